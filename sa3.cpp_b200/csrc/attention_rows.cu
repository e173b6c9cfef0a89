// attention_rows.cu -- attention with sink tokens for a few query rows: the newest tokens against a
// cache (the math and the mask of attention_sink.cu).
//
// One token a stream leaves 127 of a 128-row tile empty; what counts is to read the visible keys and
// values once, at the rate of memory, and to have enough loads in flight.  The query rows of all heads
// that share a key / value head form one 16-row operand of mma.sync m16n8k16, so a shared head's cache
// is read once for its group.  Work is split along the keys twice: the warps of a CTA take the 32-key
// steps that the window and the sinks cover in turn, and the CTAs of a cluster (1 to 16) take turns
// before that, so that a batch of one still reaches most SMs.  Every warp keeps its own running
// maximum, sum and output (f32, registers) and a ring of three steps of K and V (8 KB each, cp.async),
// of which two are in flight while one is worked on; warps are joined through shared memory and CTAs through their cluster's, in rank order, so
// there is no workspace and the result does not depend on timing.
#include <algorithm>

#include "attention_sink.h"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

constexpr int kRowsWarps = 4, kRowsStages = 3, kStepBytes = 8192;   // a step: K 32 x 128 B | V 32 x 128 B
constexpr int kRowsSmem = kRowsWarps * kRowsStages * kStepBytes;
constexpr int kPartFloats = 16 * 64 + 32;                            // O | m | l of 16 rows

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool BF>
__device__ __forceinline__ uint32_t pair_of(float lo, float hi) {
  if (BF) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  return pack_f16x2(lo, hi);
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// shared memory of CTA `rank` of the cluster, at this CTA's address p
__device__ __forceinline__ uint32_t peer(const float* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_peer(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// grid (cluster CTAs, B Hkv, 16-row tiles); row r of a tile: query i = r / group of head hk group + r % group
template <bool BF>
__global__ void __launch_bounds__(32 * kRowsWarps, 2) sink_rows_kernel(const __grid_constant__ SinkArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x, nrank = gridDim.x;
  const int b = blockIdx.y / a.Hkv, hk = blockIdx.y % a.Hkv;
  const SinkSeq s = sink_seq(a, b);
  const int row0 = blockIdx.z * 16, rows = min(16, s.qn * a.group - row0);
  // 32-key steps that some row of the tile sees: sink steps [0, ns), window steps from w0
  const int plo = s.pos0 + row0 / a.group, phi = s.pos0 + (row0 + max(rows, 1) - 1) / a.group;
  int ns = 0, w0 = 0, n = 0;
  const int hi = min(s.kn, phi + a.right + 1);
  if (rows > 0 && hi > 0) {
    ns = (min(a.sinks, hi) + 31) >> 5;
    w0 = max(max(0, plo - a.left) >> 5, ns);
    n = ns + max(0, ((hi + 31) >> 5) - w0);
  }
  const int first = rank * kRowsWarps + warp, stride = nrank * kRowsWarps;
  const uint32_t ring = smem_u32(smem) + warp * kRowsStages * kStepBytes;
  const uint16_t* kp = static_cast<const uint16_t*>(a.k.p) + (long)b * a.k.sb + (long)hk * a.k.sh;
  const uint16_t* vp = static_cast<const uint16_t*>(a.v.p) + (long)b * a.v.sb + (long)hk * a.v.sh;
  auto step_key = [&](int j) { return (j < ns ? j : w0 + (j - ns)) * 32; };
  // keys that no row of the tile sees come in as zeros, whatever they hold: 0 x NaN would spoil a product
  const int lo = plo - a.left;
  auto load = [&](int c) {       // this warp's step c into ring slot c % kRowsStages
    const int j = first + c * stride;
    if (j < n) {
      const int k0 = step_key(j);
      const uint32_t dst = ring + (c % kRowsStages) * kStepBytes;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3), ch = lane & 7, key = k0 + r;
        const uint32_t off = r * 128 + ((ch ^ (r & 7)) << 4);
        const bool in = key < hi && (key >= lo || key < a.sinks);
        const long kr = in ? key : 0;
        cp16(dst + off, kp + kr * a.k.ld + 8 * ch, in);
        cp16(dst + 4096 + off, vp + kr * a.v.ld + 8 * ch, in);
      }
    }
    cp_commit();                 // (empty groups keep the count)
  };
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[8][4];
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[d][i] = 0.f;
  const int mine = first < n ? (n - first + stride - 1) / stride : 0;
  for (int c = 0; c < kRowsStages - 1; ++c) load(c);
  // this thread's rows g and g + 8
  int p[2];
  uint32_t q[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) q[k][i] = 0u;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = row0 + g + 8 * u, i = r / a.group, h = hk * a.group + r % a.group;
    p[u] = s.pos0 + i;
    if (g + 8 * u < rows) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q.p) + (long)b * a.q.sb +
                                                             (long)h * a.q.sh + (long)i * a.q.ld);
#pragma unroll
      for (int k = 0; k < 4; ++k) {        // dims 16 k + 2 t (, + 1) and 16 k + 8 + 2 t
        q[k][u] = src[8 * k + t];
        q[k][2 + u] = src[8 * k + 4 + t];
      }
    }
  }
  for (int c = 0; c < mine; ++c) {
    cp_wait<kRowsStages - 2>();
    __syncwarp();
    load(c + kRowsStages - 1);   // (the slot of step c - 1, which the whole warp has read)
    const uint32_t base = ring + (c % kRowsStages) * kStepBytes;
    const int k0 = step_key(first + c * stride);
    float sc[4][4];              // four groups of 8 keys
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[kg][i] = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {     // dims 32 half ..: matrices of 8 dims each
        uint32_t f[4];
        const int r = 8 * kg + (lane & 7), ch = 4 * half + (lane >> 3);
        ldm4(f, base + r * 128 + ((ch ^ (r & 7)) << 4));
        mma<BF>(sc[kg], q[2 * half], f[0], f[1]);
        mma<BF>(sc[kg], q[2 * half + 1], f[2], f[3]);
      }
    }
    const bool all = k0 + 32 <= s.kn && k0 + 31 <= plo + a.right && (k0 + 31 < a.sinks || k0 >= phi - a.left);
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int kg = 0; kg < 4; ++kg)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!all && !sink_sees(a, s, p[i >> 1], k0 + 8 * kg + 2 * t + (i & 1))) sc[kg][i] = -INFINITY;
        mx[i >> 1] = fmaxf(mx[i >> 1], sc[kg][i]);
      }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
      mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2)) * a.sl2;
      const float mn = fmaxf(m[u], mx[u]), al = mn == -INFINITY ? 1.f : exp2_of(m[u] - mn);
      m[u] = mn;
      l[u] *= al;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        o[d][2 * u] *= al;
        o[d][2 * u + 1] *= al;
      }
    }
    uint32_t pa[2][4];
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mb = m[i >> 1] == -INFINITY ? 0.f : m[i >> 1];
        e[i] = exp2_of(fmaf(sc[kg][i], a.sl2, -mb));
        l[i >> 1] += e[i];
      }
      pa[kg >> 1][2 * (kg & 1)] = pair_of<BF>(e[0], e[1]);
      pa[kg >> 1][2 * (kg & 1) + 1] = pair_of<BF>(e[2], e[3]);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int d = 0; d < 4; ++d) {              // 16 dims: two n tiles
        uint32_t f[4];
        const int r = 16 * kk + (lane & 15), ch = 2 * d + (lane >> 4);
        ldm4t(f, base + 4096 + r * 128 + ((ch ^ (r & 7)) << 4));
        mma<BF>(o[2 * d], pa[kk], f[0], f[1]);
        mma<BF>(o[2 * d + 1], pa[kk], f[2], f[3]);
      }
  }
  cp_wait<0>();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
  }
  // join the warps, then the cluster's CTAs: part = [16][64] O | [16] m | [16] l
  float* part = reinterpret_cast<float*>(smem);      // [kRowsWarps + 1][kPartFloats], the last the CTA's
  __syncthreads();
  {
    float* w = part + warp * kPartFloats;
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[(g + 8 * (i >> 1)) * 64 + 8 * d + 2 * t + (i & 1)] = o[d][i];
    if (t == 0) {
      w[1024 + g] = m[0];
      w[1024 + g + 8] = m[1];
      w[1040 + g] = l[0];
      w[1040 + g + 8] = l[1];
    }
  }
  __syncthreads();
  const int r = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * 8;     // a row's 8 columns
  float M = -INFINITY, L = 0.f, v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, part[w * kPartFloats + 1024 + r]);
  for (int w = 0; w < kRowsWarps; ++w) {
    const float* x = part + w * kPartFloats;
    const float f = M == -INFINITY ? 1.f : exp2_of(x[1024 + r] - M);
    L = fmaf(f, x[1040 + r], L);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf(f, x[r * 64 + d0 + e], v[e]);
  }
  if (nrank > 1) {
    float* own = part + kRowsWarps * kPartFloats;
#pragma unroll
    for (int e = 0; e < 8; ++e) own[r * 64 + d0 + e] = v[e];
    if (d0 == 0) {
      own[1024 + r] = M;
      own[1040 + r] = L;
    }
    cluster_barrier();
    if (rank == 0) {
      M = -INFINITY;
      L = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
      for (int c0 = 0; c0 < nrank; c0 += 8) {      // eight peers' values are requested before the first is used
        float mc[8], lc[8], top = M;
        float4 x0[8], x1[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          mc[c] = -INFINITY;
          if (c0 + c >= nrank) continue;
          const uint32_t base = peer(own, c0 + c);
          mc[c] = ld_peer(base + 4 * (1024 + r));
          lc[c] = ld_peer(base + 4 * (1040 + r));
          x0[c] = ld_peer4(base + 4 * (r * 64 + d0));
          x1[c] = ld_peer4(base + 4 * (r * 64 + d0 + 4));
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) top = fmaxf(top, mc[c]);
        const float f0 = top == -INFINITY ? 1.f : exp2_of(M - top);
        M = top;
        L *= f0;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= f0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c0 + c >= nrank) continue;
          const float f = M == -INFINITY ? 1.f : exp2_of(mc[c] - M);
          const float x[8] = {x0[c].x, x0[c].y, x0[c].z, x0[c].w, x1[c].x, x1[c].y, x1[c].z, x1[c].w};
          L = fmaf(f, lc[c], L);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = fmaf(f, x[e], v[e]);
        }
      }
    }
    cluster_barrier();       // (no CTA leaves while its shared memory is read)
  }
  if (rank == 0 && r < rows) {
    const int i = (row0 + r) / a.group, h = hk * a.group + (row0 + r) % a.group;
    const bool empty = M == -INFINITY && L == L;     // no visible key (a NaN score stays a NaN)
    const float inv = 1.f / L;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = empty ? 0u : pair_of<BF>(v[2 * e] * inv, v[2 * e + 1] * inv);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o.p) + (long)b * a.o.sb + (long)h * a.o.sh + (long)i * a.o.ld + d0) =
        make_uint4(w[0], w[1], w[2], w[3]);
    if (d0 == 0 && a.lse) a.lse[((long)b * a.H + h) * a.Sq + i] = empty ? -INFINITY : M + log2f(L);
  }
}

template <bool BF>
int launch(Ctx* c, const SinkArgs& a, std::string& err) {
  auto kern = sink_rows_kernel<BF>;
  if (smem_attr(reinterpret_cast<const void*>(kern), kRowsSmem, c->device, "attention_sink smem attribute", err)) return 1;
  const int tiles = (a.Sq * a.group + 15) / 16;
  // CTAs per tile: a power of two up to 16, as long as all stay resident, two per SM (more than that
  // run in two waves: 8 x 24 heads, 1088 keys, 17.5 us with two CTAs, 12.2 with one; 1 x 24 heads,
  // 40000 keys, 57 us with 16, 46 with 8).  Up to 4 pay when every warp keeps two of its 32-key steps
  // (1 x 24 heads, 576 keys: 6.6 us with one, 6.1 with four), more when it keeps five (4 x 8 heads, 2051
  // keys: 8.1 us with four, 9.0 with eight; 1 x 8 heads, 65536 keys: 92 us with four, 49 with eight).
  const long span = std::min<long>(a.Sk, (long)a.sinks + std::min<long>((long)a.left + a.right + std::min(a.Sq, 16), a.Sk));
  int nrank = 1;
  while (nrank < 16 && (long)a.B * a.Hkv * tiles * nrank <= (long)c->sm_count &&
         span > (long)nrank * kRowsWarps * (nrank < 4 ? 64 : 160))
    nrank *= 2;
  if (nrank > 8 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return check_launch("attention_sink cluster attribute", err);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)nrank; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = use_pdl(c) ? 1 : 0;
  cfg.gridDim = dim3((unsigned)nrank, (unsigned)(a.B * a.Hkv), (unsigned)tiles);
  cfg.blockDim = dim3(32 * kRowsWarps);
  cfg.dynamicSmemBytes = kRowsSmem;
  cfg.stream = c->stream;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  ProfScope prof_(c, "attn_sink.rows");
  if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) return check_launch("attention with sinks, few rows", err);
  return check_launch("attention with sinks, few rows", err);
}

}  // namespace

// Up to 16 query rows (a group's tile of a 128-row kernel would be nearly empty), and more while all
// 16-row tiles are resident at once, two per SM: the 128-row kernel does not split a row's keys, so
// few of its tiles take the time of the longest window (us here / there: 1 x 24 heads, 192 rows,
// 4000 keys 34 / 47; 8 key heads of a group of 4, 32 rows, 8192 keys 21 / 90; 1 x 24 heads, 192 rows
// in a window of 128 keys 6.1 / 8.3).  Beyond that a tile reads the keys for 16 rows where the other
// reads them for 128 (8 x 24 heads, 32 rows, 1088 keys: 22 / 20; 64 rows 34 / 20).
bool sink_rows_applies(const Ctx* c, const SinkArgs& a) {
  return a.Sq <= 16 || (long)a.B * a.Hkv * (((long)a.Sq * a.group + 15) / 16) <= 2 * (long)c->sm_count;
}

int sink_rows_forward(Ctx* c, const SinkArgs& a, bool bf16, std::string& err) {
  return bf16 ? launch<true>(c, a, err) : launch<false>(c, a, err);
}

}  // namespace sa3k
