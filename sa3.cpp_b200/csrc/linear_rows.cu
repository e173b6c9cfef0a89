// linear_rows.cu -- the frozen linear with bias, activation and residual for a few rows (single
// tokens, one sample's conditioning): every weight is read once, straight from its stored form.
//
// With S rows a 128-row GEMM tile would be nearly empty and its 6144 / 256 = 24 output tiles would
// leave most SMs idle; the floor is the time to read W (codes and scales: 1.125 bytes a weight for
// Q8_0, 0.75 for Q4_K, 2 for F16).  So the weight is the M operand of mma.sync m16n8k16 (16 output
// features x 16 of k) and the rows of x are its N operand, 8 at a time; f16 holds the codes exactly,
// each 32-wide block's product is scaled in f32, and sums are f32.  (Tensor cores only to keep the
// arithmetic out of the way: at 8 rows they are 2% busy.)
//
// A CTA owns 16 output features; its warps take the 32-wide blocks of k in turn, so that neighbours
// read neighbouring 32-byte sectors of a row, and add their sums through shared memory in warp order.
// Within a block thread t of four holds k = 8 t .. 8 t + 7 of its row: one 8-byte load of Q8_0 codes
// (16 for f16, 4 for Q4_K) and one 16-byte load of x, with the products' k order permuted to match.
#include "activation.cuh"
#include "linear.h"
#include "ops_api.h"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

struct RowsArgs {
  const void* codes;      // [out][in] of the form
  const float* scales;    // [in/32][out] f32 (Q8_0) or float2 (Q4_K)
  const void* x;          // [S][in]
  const float* bias;
  const void* residual;   // [S][out] or null
  void* z;                // [S][out] or null
  void* y;                // [S][out]
  int in, out, S, act;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight weights of one row, as the halves of four pairs.
template <int FORM>
struct Codes;
template <>
struct Codes<kTypeQ8_0> {
  uint2 c;
  __device__ __forceinline__ void load(const void* p, long row, int in, int k) {
    c = __ldg(reinterpret_cast<const uint2*>(static_cast<const int8_t*>(p) + row * in + k));
  }
  __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
    // 0x64uu is 1024 + uu: with the sign bit flipped, code + 128
    const uint32_t u[2] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = hsub2(__byte_perm(u[i >> 1], 0x64646464u, (i & 1) ? 0x4342 : 0x4140), 0x64806480u);
  }
};
template <>
struct Codes<kTypeQ4_K> {
  uint32_t c;
  __device__ __forceinline__ void load(const void* p, long row, int in, int k) {
    c = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p) + (row * in + k) / 2));
  }
  __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = c >> (8 * i);
      h[i] = hsub2((b & 0xfu) | ((b & 0xf0u) << 12) | 0x64006400u, 0x64006400u);
    }
  }
};
template <>
struct Codes<kTypeF16> {
  uint4 c;
  __device__ __forceinline__ void load(const void* p, long row, int in, int k) {
    c = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + row * in + k));
  }
  __device__ __forceinline__ void pairs(uint32_t (&h)[4]) const {
    h[0] = c.x; h[1] = c.y; h[2] = c.z; h[3] = c.w;
  }
};

__device__ __forceinline__ uint4 load_x(const __half* x) { return __ldg(reinterpret_cast<const uint4*>(x)); }
__device__ __forceinline__ uint4 load_x(const float* x) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(x)), b = __ldg(reinterpret_cast<const float4*>(x + 4));
  return make_uint4(pack_f16x2(a.x, a.y), pack_f16x2(a.z, a.w), pack_f16x2(b.x, b.y), pack_f16x2(b.z, b.w));
}

// NT: groups of 8 rows of x.  blockDim.x / 32 warps share the blocks of k.
template <int FORM, class T, int NT>
__global__ void __launch_bounds__(256) linear_rows_kernel(const RowsArgs a) {
  extern __shared__ float red[];      // [warps][16 features][8 NT rows]
  pdl_prologue();
  constexpr int N = 8 * NT, U = 4;    // U blocks of k in flight per warp
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int f0 = blockIdx.x * 16, nb = a.in / 32;
  const long ra = min(f0 + g, a.out - 1), rb = min(f0 + g + 8, a.out - 1);
  const T* x = static_cast<const T*>(a.x);
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  for (int b0 = warp; b0 < nb; b0 += nw * U) {
    Codes<FORM> ca[U], cb[U];
    float2 sa[U], sb[U];
    uint4 xv[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + u * nw;
      if (b >= nb) continue;
      ca[u].load(a.codes, ra, a.in, 32 * b + 8 * t);
      cb[u].load(a.codes, rb, a.in, 32 * b + 8 * t);
      if (FORM == kTypeQ8_0) {
        sa[u].x = __ldg(a.scales + (long)b * a.out + ra);
        sb[u].x = __ldg(a.scales + (long)b * a.out + rb);
      } else if (FORM == kTypeQ4_K) {
        sa[u] = __ldg(reinterpret_cast<const float2*>(a.scales) + (long)b * a.out + ra);
        sb[u] = __ldg(reinterpret_cast<const float2*>(a.scales) + (long)b * a.out + rb);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = 8 * n + g;
        xv[u][n] = r < a.S ? load_x(x + (long)r * a.in + 32 * b + 8 * t) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b0 + u * nw >= nb) continue;
      uint32_t ha[4], hb[4];
      ca[u].pairs(ha);
      cb[u].pairs(hb);
      const uint32_t m0[4] = {ha[0], hb[0], ha[1], hb[1]}, m1[4] = {ha[2], hb[2], ha[3], hb[3]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 v = xv[u][n];
        if (FORM == kTypeF16) {
          mma16816(acc[n], m0, v.x, v.y);
          mma16816(acc[n], m1, v.z, v.w);
        } else {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(d, m0, v.x, v.y);
          mma16816(d, m1, v.z, v.w);
          acc[n][0] = fmaf(sa[u].x, d[0], acc[n][0]);
          acc[n][1] = fmaf(sa[u].x, d[1], acc[n][1]);
          acc[n][2] = fmaf(sb[u].x, d[2], acc[n][2]);
          acc[n][3] = fmaf(sb[u].x, d[3], acc[n][3]);
          if (FORM == kTypeQ4_K) {      // value = d sc q - dmin m: the block's sum of x, by a row of ones
            const uint32_t one[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
            float e[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(e, one, v.x, v.y);
            mma16816(e, one, v.z, v.w);
            acc[n][0] = fmaf(-sa[u].y, e[0], acc[n][0]);
            acc[n][1] = fmaf(-sa[u].y, e[1], acc[n][1]);
            acc[n][2] = fmaf(-sb[u].y, e[2], acc[n][2]);
            acc[n][3] = fmaf(-sb[u].y, e[3], acc[n][3]);
          }
        }
      }
    }
  }
  // element (feature, row): thread holds features g, g + 8 and rows 8 n + 2 t, + 1
  float* mine = red + warp * 16 * N;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[(8 * n + 2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[n][i];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * N; e += blockDim.x) {
    const int r = e >> 4, f = f0 + (e & 15);
    if (r >= a.S || f >= a.out) continue;
    float v = 0.f;
    for (int w = 0; w < nw; ++w) v += red[w * 16 * N + e];
    if (a.bias) v += a.bias[f];
    const long i = (long)r * a.out + f;
    if (a.z) static_cast<T*>(a.z)[i] = from_f32<T>(v);
    v = act_value(a.act, v);
    if (a.residual) v += to_f32(static_cast<const T*>(a.residual)[i]);
    static_cast<T*>(a.y)[i] = from_f32<T>(v);
  }
}

template <int FORM, class T>
int launch_rows(Ctx* c, const RowsArgs& a, std::string& err) {
  const int nt = a.S <= 8 ? 1 : a.S <= 16 ? 2 : 4;
  const int tiles = (a.out + 15) / 16;
  // warps per tile: enough for about eight warps on every SM, as long as each has some blocks of k
  int nw = 1;
  while (nw < 8 && (long)tiles * nw < 8 * (long)c->sm_count && a.in / 32 >= 4 * nw) nw *= 2;
  const size_t smem = (size_t)nw * 16 * 8 * nt * sizeof(float);
  ProfScope prof_(c, "linear.rows");
  const dim3 grid((unsigned)tiles), block(32 * nw);
  if (nt == 1) launch_pdl(c, linear_rows_kernel<FORM, T, 1>, grid, block, smem, a);
  else if (nt == 2) launch_pdl(c, linear_rows_kernel<FORM, T, 2>, grid, block, smem, a);
  else launch_pdl(c, linear_rows_kernel<FORM, T, 4>, grid, block, smem, a);
  return check_launch("linear of a few rows", err);
}

}  // namespace

bool linear_rows_applies(int64_t S) { return S <= 32; }

int linear_rows(Ctx* c, const Weight* w, const float* bias, int act, int type, const void* x, int64_t S,
                const void* residual, void* z, void* y, std::string& err) {
  RowsArgs a;
  const int form = w->type == kTypeQ8_0 || w->type == kTypeQ4_K ? w->type : kTypeF16;
  a.codes = form == kTypeF16 ? static_cast<const void*>(w->f16) : static_cast<const void*>(w->codes);
  a.scales = w->scales;
  a.x = x; a.bias = bias; a.residual = residual; a.z = z; a.y = y;
  a.in = (int)w->in; a.out = (int)w->out; a.S = (int)S; a.act = act;
  if (type == kTypeF16)
    return form == kTypeQ8_0 ? launch_rows<kTypeQ8_0, __half>(c, a, err)
                             : form == kTypeQ4_K ? launch_rows<kTypeQ4_K, __half>(c, a, err)
                                                 : launch_rows<kTypeF16, __half>(c, a, err);
  return form == kTypeQ8_0 ? launch_rows<kTypeQ8_0, float>(c, a, err)
                           : form == kTypeQ4_K ? launch_rows<kTypeQ4_K, float>(c, a, err)
                                               : launch_rows<kTypeF16, float>(c, a, err);
}

}  // namespace sa3k
