// layernorm.cu -- layer normalisation over the rows of a matrix, forward and backward.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps),  y = (x - mu) r gamma + beta
//   backward  xh = (x - mu) r, g = dy gamma:
//             dx = r (g - mean(g) - xh mean(g xh)),  dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// Both are bound by memory: each value of x (and dy) is read once and held in registers while its
// row's sums are formed, and each result is written once.  The variance is taken around the mean
// of the held values, not from a sum of squares, and what the f32 mean m is off by, the mean e of the
// x - m, is taken out of it and of every x - m: a large common offset costs the forward no digits (rows
// of 1e4 + N(0, 1): y was off by 1e-3 without e).  The backward takes mean and rstd as they are kept, in
// f32.  All arithmetic is f32 whatever the types; a result is rounded once, when it is stored.
//
// A row belongs to TPR threads: a part of a warp for short rows, else a whole block.  The backward
// keeps every thread's columns' sums of dy xh and dy in registers over all the rows that its block
// walks, and writes one partial row per block; a second kernel adds the partials in block order,
// so the parameter gradients do not depend on timing.
#include <cmath>
#include <type_traits>

#include "../../include/sa3k.h"
#include "ops_api.h"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

// out[i] (+)= sum over b of part[b][which][i], `planes` of them per b: a block takes 8 columns (a 32-byte
// sector) in 64 slices of the partial rows, which are then added in order.
__global__ void __launch_bounds__(512) fold_partials_kernel(const float* part, int nblocks, int planes, int cols, float* out0,
                                                            float* out1, int acc0, int acc1) {
  __shared__ float s[8][65];
  pdl_prologue();
  const int e = threadIdx.x & 7, w = threadIdx.x >> 3, i = blockIdx.x * 8 + e;
  float* out = blockIdx.y == 0 ? out0 : out1;
  if (!out) return;
  const float* p = part + (long)blockIdx.y * cols + i;
  float v = 0.f;
  if (i < cols) {
#pragma unroll 4
    for (int b = w; b < nblocks; b += 64) v += p[(long)b * planes * cols];
  }
  s[e][w] = v;
  __syncthreads();
  const int c = threadIdx.x >> 5;       // warps 0 .. 7: a column each
  if (c >= 8) return;
  v = warp_sum(s[c][threadIdx.x & 31] + s[c][32 + (threadIdx.x & 31)]);
  const int o = blockIdx.x * 8 + c;
  if ((threadIdx.x & 31) == 0 && o < cols) out[o] = (blockIdx.y == 0 ? acc0 : acc1) ? out[o] + v : v;
}

}  // namespace

int k_fold_partials(Ctx* c, const float* part, int nblocks, int planes, int cols, float* out0, float* out1, int acc0,
                    int acc1, std::string& err) {
  ProfScope prof_(c, "fold_partials");
  launch_pdl(c, fold_partials_kernel, dim3((unsigned)((cols + 7) / 8), (unsigned)planes), dim3(512), 0, part, nblocks, planes,
             cols, out0, out1, acc0, acc1);
  return check_launch("fold partials", err);
}

namespace {

struct LnArgs {
  long rows;
  int cols;
  const void* x; long x_ld;
  const void* dy; long dy_ld;     // backward
  void* out; long out_ld;         // forward y, backward dx
  const float* gamma;
  const float* beta;
  float* mean; float* rstd;       // forward: written when not null; backward: read
  float eps;
  float* part;                    // backward: [gridDim.x][2][cols] partial dgamma | dbeta
};

// Sums over the TPR threads of a row; every thread gets them.  `red`: 2 x 32 pairs, alternated by the
// caller (`ph`) so that one barrier per reduction is enough.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float a, int tpr, float2 (*red)[32], int ph) {
  if (BLOCK) {
    a = warp_sum(a);
    const int nw = blockDim.x >> 5;
    if (nw > 1) {
      if ((threadIdx.x & 31) == 0) red[ph][threadIdx.x >> 5].x = a;
      __syncthreads();
      a = warp_sum((threadIdx.x & 31) < nw ? red[ph][threadIdx.x & 31].x : 0.f);
    }
  } else {
    for (int o = tpr >> 1; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  return a;
}

// Two sums at once.  In a block each half of a warp keeps one of them from the first exchange on: 5 + 6
// shuffles instead of 20.
template <bool BLOCK>
__device__ __forceinline__ float2 row_sum2(float a, float b, int tpr, float2 (*red)[32], int ph) {
  if (BLOCK) {
    const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const bool hi = lane & 16;
    float v = (hi ? b : a) + __shfl_xor_sync(0xffffffffu, hi ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (nw > 1) {
      if ((lane & 15) == 0) (hi ? red[ph][threadIdx.x >> 5].y : red[ph][threadIdx.x >> 5].x) = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int w = lane & 15, k = 0; k < 2; ++k, w += 16)
        if (w < nw) v += hi ? red[ph][w].y : red[ph][w].x;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
  }
  for (int o = tpr >> 1; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_float2(a, b);
}

// Chunk c of a thread's columns: 8 consecutive ones from (c TPR + t) 8 (VEC, 16-byte accesses), or
// the 8 columns t + (8 c + e) TPR (rows whose width or alignment allows no vector access).
template <bool VEC>
__device__ __forceinline__ int col_of(int c, int e, int t, int tpr) {
  return VEC ? (c * tpr + t) * 8 + e : t + (8 * c + e) * tpr;
}

template <bool VEC, class T>
__device__ __forceinline__ void load_chunk(const T* p, int c, int t, int tpr, int cols, float (&v)[8]) {
  if (VEC) {
    const int i = col_of<true>(c, 0, t, tpr);
    if (i < cols) {
      load8(p + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = col_of<false>(c, e, t, tpr);
      v[e] = i < cols ? to_f32(p[i]) : 0.f;
    }
  }
}

template <bool VEC, class T>
__device__ __forceinline__ void store_chunk(T* p, int c, int t, int tpr, int cols, const float (&v)[8]) {
  if (VEC) {
    const int i = col_of<true>(c, 0, t, tpr);
    if (i < cols) store8(p + i, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = col_of<false>(c, e, t, tpr);
      if (i < cols) p[i] = from_f32<T>(v[e]);
    }
  }
}

// rstd of a row from the sums of d^2 and d, d = x - m; off = mean(d), what the mean m is off by
__device__ __forceinline__ float ln_rstd(float2 s, const LnArgs& a, float& off) {
  const float inv = 1.f / (float)a.cols;
  off = s.y * inv;
  const float var = fmaf(-off, off, s.x * inv);
  return 1.0f / sqrtf((var < 0.f ? 0.f : var) + a.eps);     // (a NaN stays one)
}

// Forward with the row in registers: NV chunks of 8 columns per thread.  With one vector
// chunk a block is held to 32 registers a thread (no spills; the scalar form would), so that an SM holds
// its full 2048 threads: what bounds the kernel is how many rows are between their loads and their stores
// (4352 x 1536 f32 to f16 12.0 us against 12.6 without, 16384 rows 36.7 against 38.7; gamma and beta
// loaded ahead of the sums cost registers: 13.7).  With the mean's correction 11.9 and 37.1.
template <class TX, class TY, bool BLOCK, int NV, bool VEC>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256, BLOCK && NV == 1 && VEC ? 2 : 1) ln_fwd_kernel(const LnArgs a, int tpr) {
  __shared__ float2 red[2][32];
  pdl_prologue();
  const int t = BLOCK ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = BLOCK ? 1 : blockDim.x / tpr;
  const long r = (long)blockIdx.x * per + (BLOCK ? 0 : threadIdx.x / tpr);
  const bool ok = r < a.rows;
  const TX* x = static_cast<const TX*>(a.x) + (ok ? r : 0) * a.x_ld;
  float v[NV][8];
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c) load_chunk<VEC>(x, c, t, tpr, a.cols, v[c]);
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[c][e];
  const float mu = row_sum<BLOCK>(s, tpr, red, 0) / (float)a.cols;
  float q = 0.f, sd = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] -= mu;
      if (col_of<VEC>(c, e, t, tpr) < a.cols) {
        sd += v[c][e];
        q = fmaf(v[c][e], v[c][e], q);
      }
    }
  float off;
  const float rs = ln_rstd(row_sum2<BLOCK>(q, sd, tpr, red, 1), a, off);
  if (!ok) return;
  if (t == 0) {
    if (a.mean) a.mean[r] = isfinite(off) ? mu + off : mu;     // (a row with an infinity has that mean)
    if (a.rstd) a.rstd[r] = rs;
  }
  TY* y = static_cast<TY*>(a.out) + r * a.out_ld;
  const float nor = -off * rs;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if constexpr (VEC && std::is_same<TY, float>::value) {     // four values at a time: fewer registers
      const int i = col_of<true>(c, 0, t, tpr);
      if (i >= a.cols) continue;
#pragma unroll
      for (int h = 0; h < 8; h += 4) {
        const float4 one = make_float4(1.f, 1.f, 1.f, 1.f), zero = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 gm = a.gamma ? *reinterpret_cast<const float4*>(a.gamma + i + h) : one;
        const float4 bt = a.beta ? *reinterpret_cast<const float4*>(a.beta + i + h) : zero;
        *reinterpret_cast<float4*>(y + i + h) =
            make_float4(fmaf(fmaf(v[c][h], rs, nor), gm.x, bt.x), fmaf(fmaf(v[c][h + 1], rs, nor), gm.y, bt.y),
                        fmaf(fmaf(v[c][h + 2], rs, nor), gm.z, bt.z), fmaf(fmaf(v[c][h + 3], rs, nor), gm.w, bt.w));
      }
      continue;
    }
    float gm[8], bt[8], o[8];
    if (a.gamma) load_chunk<VEC>(a.gamma, c, t, tpr, a.cols, gm);
    if (a.beta) load_chunk<VEC>(a.beta, c, t, tpr, a.cols, bt);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      o[e] = fmaf(fmaf(v[c][e], rs, nor), a.gamma ? gm[e] : 1.f, a.beta ? bt[e] : 0.f);
    store_chunk<VEC>(y, c, t, tpr, a.cols, o);
  }
}

// Forward of rows too long for the registers of a block: three passes over the row (the later two
// from L2), element by element.
template <class TX, class TY>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const LnArgs a) {
  __shared__ float2 red[2][32];
  pdl_prologue();
  const long r = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + r * a.x_ld;
  float s = 0.f;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) s += to_f32(x[i]);
  const float mu = row_sum<true>(s, 0, red, 0) / (float)a.cols;
  float q = 0.f, sd = 0.f;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float d = to_f32(x[i]) - mu;
    sd += d;
    q = fmaf(d, d, q);
  }
  float off;
  const float rs = ln_rstd(row_sum2<true>(q, sd, 0, red, 1), a, off);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[r] = isfinite(off) ? mu + off : mu;     // (a row with an infinity has that mean)
    if (a.rstd) a.rstd[r] = rs;
  }
  TY* y = static_cast<TY*>(a.out) + r * a.out_ld;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x)
    y[i] = from_f32<TY>(fmaf((to_f32(x[i]) - mu - off) * rs, a.gamma ? a.gamma[i] : 1.f, a.beta ? a.beta[i] : 0.f));
}

// Backward with the row in registers; the block's threads walk rows with stride gridDim.x (x rows
// per block).  PARAMS: the parameter gradients' sums are kept and written as partials.
template <class TX, class TY, bool BLOCK, int NV, bool VEC, bool PARAMS>
__global__ void __launch_bounds__(1024) ln_bwd_kernel(const LnArgs a, int tpr) {
  __shared__ float2 red[2][32];
  extern __shared__ float fold[];   // sub-warp rows: [2][cols] sums of the block
  pdl_prologue();
  const int t = BLOCK ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = BLOCK ? 1 : blockDim.x / tpr;
  const long r0 = (long)blockIdx.x * per + (BLOCK ? 0 : threadIdx.x / tpr), step = (long)gridDim.x * per;
  float gm[NV][8], sg[NV][8], sb[NV][8];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (a.gamma) load_chunk<VEC>(a.gamma, c, t, tpr, a.cols, gm[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!a.gamma) gm[c][e] = 1.f;
      sg[c][e] = sb[c][e] = 0.f;
    }
  }
  const float inv = 1.f / (float)a.cols;
  const long base = (long)blockIdx.x * per;
  int ph = 0;
  for (long rb = base; rb < a.rows; rb += step, ph ^= 1) {   // the same count for every thread of the block
    const long r = rb + (r0 - base);
    const bool ok = r < a.rows;
    const long rr = ok ? r : a.rows - 1;
    const TX* x = static_cast<const TX*>(a.x) + rr * a.x_ld;
    const TY* dy = static_cast<const TY*>(a.dy) + rr * a.dy_ld;
    float xv[NV][8], dv[NV][8];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      load_chunk<VEC>(x, c, t, tpr, a.cols, xv[c]);
      load_chunk<VEC>(dy, c, t, tpr, a.cols, dv[c]);
    }
    const float mu = a.mean[rr], rs = a.rstd[rr];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xv[c][e] = (xv[c][e] - mu) * rs;       // xh (columns past the row have dy = 0)
        if (PARAMS && ok) {
          sg[c][e] = fmaf(dv[c][e], xv[c][e], sg[c][e]);
          sb[c][e] += dv[c][e];
        }
        dv[c][e] *= gm[c][e];
        if (col_of<VEC>(c, e, t, tpr) < a.cols) {
          s1 += dv[c][e];
          s2 = fmaf(dv[c][e], xv[c][e], s2);
        }
      }
    const float2 s = row_sum2<BLOCK>(s1, s2, tpr, red, ph);
    const float m1 = s.x * inv, m2 = s.y * inv;
    if (a.out && ok) {
      TX* dx = static_cast<TX*>(a.out) + r * a.out_ld;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = rs * (dv[c][e] - m1 - xv[c][e] * m2);
        store_chunk<VEC>(dx, c, t, tpr, a.cols, o);
      }
    }
  }
  if (!PARAMS) return;
  float* part = a.part + (long)blockIdx.x * 2 * a.cols;
  if (BLOCK) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      store_chunk<VEC>(part, c, t, tpr, a.cols, sg[c]);
      store_chunk<VEC>(part + a.cols, c, t, tpr, a.cols, sb[c]);
    }
  } else {
    // the block's rows one after another: a fixed order
    for (int i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) fold[i] = 0.f;
    for (int k = 0; k < per; ++k) {
      __syncthreads();
      if (threadIdx.x / tpr != k) continue;
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = col_of<VEC>(c, e, t, tpr);
          if (i < a.cols) {
            fold[i] += sg[c][e];
            fold[a.cols + i] += sb[c][e];
          }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) part[i] = fold[i];
  }
}

// Backward of rows of 257 to 8192 columns with vector access.  The block's next rows of x and dy come
// into a ring in shared memory by bulk copies, pairs of rows ahead, so that memory stays busy through
// the reductions; and two rows are reduced together: their four sums take 6 shuffles a warp (each step
// sends away the half that the lane does not keep) and one barrier, where row by row it was 40 and two.
// Packed f32 pairs halve the instructions, which bounded the kernel (270 a warp and row, 2.4 a clock).
// A thread takes about 85 registers without spills (they went to L2, the ring having taken L1: 44 us
// for 16383 x 1536 with the fold instead of 37), so the blocks per SM follow from the threads of a row; rows of more
// than 5120 columns have 64 registers a thread and read the slot again instead of holding its values.
constexpr int kLnMaxSlots = 8;
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// (a0, b0, a1, b1) summed over the block; `red` is alternated by the caller
__device__ __forceinline__ float4 block_sum4(float a0, float b0, float a1, float b1, float4* red) {
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const bool hi = lane & 16, sel = lane & 8;
  float a = (hi ? a1 : a0) + __shfl_xor_sync(0xffffffffu, hi ? a0 : a1, 16);
  float b = (hi ? b1 : b0) + __shfl_xor_sync(0xffffffffu, hi ? b0 : b1, 16);
  float v = (sel ? b : a) + __shfl_xor_sync(0xffffffffu, sel ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((lane & 7) == 0) reinterpret_cast<float*>(red + (threadIdx.x >> 5))[lane >> 3] = v;
  __syncthreads();
  float4 s = red[0];
#pragma unroll 2
  for (int w = 1; w < nw; ++w) {
    const float4 x = red[w];
    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
  }
  return s;
}

template <class TX, class TY, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) ln_bwd_ring_kernel(const LnArgs a, int slots, int* err) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float4 red[2][32];
  __shared__ __align__(8) uint64_t full[kLnMaxSlots];
  const int t = threadIdx.x, i0 = 8 * t;
  const uint32_t xb = (uint32_t)a.cols * sizeof(TX), yb = (uint32_t)a.cols * sizeof(TY), row_bytes = xb + yb;
  if (t == 0) {
    for (int k = 0; k < slots; ++k) mbar_init(&full[k], 1);
    fence_barrier_init();
  }
  __syncthreads();
  pdl_prologue();
  const long first = blockIdx.x, step = gridDim.x;          // a pair: rows r and r + step
  auto fetch = [&](long r, int slot) {                      // (thread 0)
    const int n = r + step < a.rows ? 2 : 1;
    mbar_arrive_expect_tx(&full[slot], n * row_bytes);
    for (int k = 0; k < n; ++k) {
      uint8_t* dst = ring + (size_t)(2 * slot + k) * row_bytes;
      bulk_load(dst, static_cast<const TX*>(a.x) + (r + k * step) * a.x_ld, xb, &full[slot]);
      bulk_load(dst + xb, static_cast<const TY*>(a.dy) + (r + k * step) * a.dy_ld, yb, &full[slot]);
    }
  };
  if (t == 0)
    for (int k = 0; k < slots; ++k)
      if (first + 2 * k * step < a.rows) fetch(first + 2 * k * step, k);
  const bool in = i0 < a.cols;
  uint64_t gm[4], sg[4], sb[4];            // pairs of f32 (two lanes of work per instruction)
#pragma unroll
  for (int e = 0; e < 4; ++e) gm[e] = f2(1.f, 1.f), sg[e] = sb[e] = f2(0.f, 0.f);
  if (a.gamma && in) {
    float v[8];
    load8(a.gamma + i0, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) gm[e] = f2(v[2 * e], v[2 * e + 1]);
  }
  const float inv = 1.f / (float)a.cols;
  bool ok = true;
  int slot = 0, ph = 0;
  uint32_t phase = 0;
  float mu[2] = {0.f, 0.f}, rs[2] = {0.f, 0.f};
  auto stats = [&](long r, float (&m)[2], float (&q)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (r + k * step < a.rows) {
        m[k] = a.mean[r + k * step];
        q[k] = a.rstd[r + k * step];
      }
  };
  float mu_next[2] = {0.f, 0.f}, rs_next[2] = {0.f, 0.f};
  stats(first, mu_next, rs_next);
  for (long r = first; r < a.rows; r += 2 * step, ph ^= 1) {
    const bool two = r + step < a.rows;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mu[k] = mu_next[k];
      rs[k] = rs_next[k];
    }
    stats(r + 2 * step, mu_next, rs_next);
    if (ok) ok = mbar_wait(&full[slot], phase, err, kErrTimeoutFull);
    const uint8_t* src = ring + (size_t)(2 * slot) * row_bytes;
    float s1[2] = {0.f, 0.f}, s2[2] = {0.f, 0.f};
    constexpr bool HOLD = MAXT < 1024;
    uint64_t xh[2][4], g[2][4];
    auto row_of = [&](int k) {       // xh and g of row k from the slot
      float xv[8], dv[8];
      load8(reinterpret_cast<const TX*>(src + k * row_bytes) + i0, xv);
      load8(reinterpret_cast<const TY*>(src + k * row_bytes + xb) + i0, dv);
      const uint64_t nmu = f2(-mu[k], -mu[k]), rs2 = f2(rs[k], rs[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        xh[k][e] = fmul2(fadd2(f2(xv[2 * e], xv[2 * e + 1]), nmu), rs2);
        g[k][e] = f2(dv[2 * e], dv[2 * e + 1]);       // (dy; times gamma below)
      }
    };
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!in || (k && !two)) continue;
      row_of(k);
      uint64_t p1 = f2(0.f, 0.f), p2 = p1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sg[e] = ffma2(g[k][e], xh[k][e], sg[e]);
        sb[e] = fadd2(sb[e], g[k][e]);
        g[k][e] = fmul2(g[k][e], gm[e]);
        p1 = fadd2(p1, g[k][e]);
        p2 = ffma2(g[k][e], xh[k][e], p2);
      }
      float u, v;
      f2split(p1, u, v);
      s1[k] = u + v;
      f2split(p2, u, v);
      s2[k] = u + v;
    }
    const float4 sum = block_sum4(s1[0], s2[0], s1[1], s2[1], red[ph]);
    // (every thread has read the slot before the sum's barrier, unless it reads it again)
    if (HOLD && t == 0 && ok && r + 2 * slots * step < a.rows) fetch(r + 2 * slots * step, slot);
    if (a.out && in && ok) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k && !two) continue;
        if (!HOLD) {
          row_of(k);
#pragma unroll
          for (int e = 0; e < 4; ++e) g[k][e] = fmul2(g[k][e], gm[e]);
        }
        const float m1 = (k ? sum.z : sum.x) * inv, m2 = (k ? sum.w : sum.y) * inv, c = -m1 * rs[k];
        const uint64_t nm2 = f2(-m2, -m2), rs2 = f2(rs[k], rs[k]), c2 = f2(c, c);
        float o[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) f2split(ffma2(ffma2(xh[k][e], nm2, g[k][e]), rs2, c2), o[2 * e], o[2 * e + 1]);
        store8(static_cast<TX*>(a.out) + (r + k * step) * a.out_ld + i0, o);
      }
    }
    if (!HOLD) {
      __syncthreads();
      if (t == 0 && ok && r + 2 * slots * step < a.rows) fetch(r + 2 * slots * step, slot);
    }
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if (!in || !a.part) return;
  float* part = a.part + (long)blockIdx.x * 2 * a.cols;
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) f2split(sg[e], v[2 * e], v[2 * e + 1]);
  store8(part + i0, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) f2split(sb[e], v[2 * e], v[2 * e + 1]);
  store8(part + a.cols + i0, v);
}

// Backward of rows too long for the registers: dx in two passes over the row.
template <class TX, class TY>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(const LnArgs a) {
  __shared__ float2 red[2][32];
  pdl_prologue();
  const long r = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + r * a.x_ld;
  const TY* dy = static_cast<const TY*>(a.dy) + r * a.dy_ld;
  const float mu = a.mean[r], rs = a.rstd[r];
  float s1 = 0.f, s2 = 0.f;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float g = to_f32(dy[i]) * (a.gamma ? a.gamma[i] : 1.f);
    s1 += g;
    s2 = fmaf(g, (to_f32(x[i]) - mu) * rs, s2);
  }
  const float2 s = row_sum2<true>(s1, s2, 0, red, 0);
  const float m1 = s.x / (float)a.cols, m2 = s.y / (float)a.cols;
  TX* dx = static_cast<TX*>(a.out) + r * a.out_ld;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float g = to_f32(dy[i]) * (a.gamma ? a.gamma[i] : 1.f);
    dx[i] = from_f32<TX>(rs * (g - m1 - (to_f32(x[i]) - mu) * rs * m2));
  }
}

// Parameter gradients of long rows: block (column group, row slice), one thread per column.
template <class TX, class TY>
__global__ void __launch_bounds__(256) ln_param_long_kernel(const LnArgs a) {
  pdl_prologue();
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= a.cols) return;
  float sg = 0.f, sb = 0.f;
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float d = to_f32(static_cast<const TY*>(a.dy)[r * a.dy_ld + i]);
    sg = fmaf(d, (to_f32(static_cast<const TX*>(a.x)[r * a.x_ld + i]) - a.mean[r]) * a.rstd[r], sg);
    sb += d;
  }
  float* part = a.part + (long)blockIdx.x * 2 * a.cols;
  part[i] = sg;
  part[a.cols + i] = sb;
}

constexpr int kLnMaxRegCols = 32768;   // 1024 threads x 32 values

// Threads per row and chunks per thread.  Rows of up to 256 columns take a part of a warp (the
// smallest power of two that holds them at 8 columns a thread); longer ones a whole block of at
// most 1024 threads, at 8, 16 or 32 columns a thread.  In the forward rows of up to 1024 columns stay
// with one warp, at up to 32 columns a thread: no barrier, and all of a row's loads in flight (32768 x
// 1000 f32 -> f16: 46 us with blocks, 42 with warps; 4352 x 1536: 12.0 with blocks, 15.2 with warps).
struct LnShape {
  bool block;
  int tpr, threads, nv;
};
LnShape ln_shape(int cols, bool forward) {
  LnShape s;
  if (cols <= (forward ? 1024 : 256)) {
    s.block = false;
    s.tpr = 1;
    while (s.tpr * 8 < cols && s.tpr < 32) s.tpr *= 2;
    s.threads = 256;
    s.nv = (cols + 255) / 256;
    return s;
  }
  s.block = true;
  s.nv = cols <= 8192 ? 1 : cols <= 16384 ? 2 : 4;
  s.threads = ((cols + 8 * s.nv - 1) / (8 * s.nv) + 31) / 32 * 32;
  s.tpr = s.threads;
  return s;
}

template <class TX, class TY, bool BLOCK, int NV>
int fwd_launch(Ctx* c, const LnArgs& a, const LnShape& s, bool vec, std::string& err) {
  const long per = BLOCK ? 1 : s.threads / s.tpr;
  const dim3 grid((unsigned)((a.rows + per - 1) / per));
  ProfScope prof_(c, "layernorm.fwd");
  if (vec) launch_pdl(c, ln_fwd_kernel<TX, TY, BLOCK, NV, true>, grid, dim3(s.threads), 0, a, s.tpr);
  else launch_pdl(c, ln_fwd_kernel<TX, TY, BLOCK, NV, false>, grid, dim3(s.threads), 0, a, s.tpr);
  return check_launch("layernorm forward", err);
}

template <class TX, class TY>
int fwd_typed(Ctx* c, const LnArgs& a, bool vec, std::string& err) {
  if (a.cols > kLnMaxRegCols) {
    ProfScope prof_(c, "layernorm.fwd");
    launch_pdl(c, ln_fwd_long_kernel<TX, TY>, dim3((unsigned)a.rows), dim3(1024), 0, a);
    return check_launch("layernorm forward", err);
  }
  const LnShape s = ln_shape(a.cols, true);
  if (!s.block) {
    switch (s.nv) {
      case 1: return fwd_launch<TX, TY, false, 1>(c, a, s, vec, err);
      case 2: return fwd_launch<TX, TY, false, 2>(c, a, s, vec, err);
      case 3: return fwd_launch<TX, TY, false, 3>(c, a, s, vec, err);
      default: return fwd_launch<TX, TY, false, 4>(c, a, s, vec, err);
    }
  }
  if (s.nv == 1) return fwd_launch<TX, TY, true, 1>(c, a, s, vec, err);
  if (s.nv == 2) return fwd_launch<TX, TY, true, 2>(c, a, s, vec, err);
  return fwd_launch<TX, TY, true, 4>(c, a, s, vec, err);
}

// Blocks of the backward: enough to fill the SMs at the registers it takes, no more than rows.
int bwd_blocks(Ctx* c, const LnArgs& a, const LnShape& s) {
  const long per = s.block ? 1 : s.threads / s.tpr;
  const long need = (a.rows + per - 1) / per;
  const long fit = (long)c->sm_count * std::max(1, 1024 / s.threads);
  return (int)std::max(1L, std::min(need, fit));
}

// The ring kernel's launch for a row's threads: blocks per SM, and pairs of rows in their share of 200
// KB (the longest f32 rows, 64 KB of x and dy, have one).
struct RingShape {
  int threads, per_sm, slots, blocks;
};
RingShape ring_shape(Ctx* c, const LnArgs& a, size_t row_bytes) {
  RingShape r;
  r.threads = ((a.cols + 7) / 8 + 31) / 32 * 32;
  r.per_sm = r.threads <= 96 ? 8 : r.threads <= 192 ? 4 : r.threads <= 320 ? 2 : 1;
  r.slots = (int)std::max<size_t>(1, std::min<size_t>(kLnMaxSlots, (size_t)200 * 1024 / r.per_sm / (2 * row_bytes)));
  r.blocks = (int)std::min<long>((long)c->sm_count * r.per_sm, a.rows);
  return r;
}

template <class TX, class TY>
int ring_launch(Ctx* c, const LnArgs& a, const RingShape& r, std::string& err) {
  const size_t smem = (size_t)r.slots * 2 * a.cols * (sizeof(TX) + sizeof(TY));
  auto kern = r.threads <= 96    ? ln_bwd_ring_kernel<TX, TY, 96, 8>
              : r.threads <= 192 ? ln_bwd_ring_kernel<TX, TY, 192, 4>
              : r.threads <= 320 ? ln_bwd_ring_kernel<TX, TY, 320, 2>
              : r.threads <= 640 ? ln_bwd_ring_kernel<TX, TY, 640, 1>
                                 : ln_bwd_ring_kernel<TX, TY, 1024, 1>;
  if (smem_attr(reinterpret_cast<const void*>(kern), 200 * 1024, c->device, "layernorm smem attribute", err)) return 1;
  ProfScope prof_(c, "layernorm.bwd");
  launch_pdl(c, kern, dim3(r.blocks), dim3(r.threads), smem, a, r.slots, c->d_err);
  return check_launch("layernorm backward", err);
}

template <class TX, class TY, bool BLOCK, int NV, bool VEC>
int bwd_launch(Ctx* c, const LnArgs& a, const LnShape& s, int blocks, std::string& err) {
  const size_t smem = BLOCK ? 0 : (size_t)2 * a.cols * sizeof(float);
  ProfScope prof_(c, "layernorm.bwd");
  if (a.part) launch_pdl(c, ln_bwd_kernel<TX, TY, BLOCK, NV, VEC, true>, dim3(blocks), dim3(s.threads), smem, a, s.tpr);
  else launch_pdl(c, ln_bwd_kernel<TX, TY, BLOCK, NV, VEC, false>, dim3(blocks), dim3(s.threads), 0, a, s.tpr);
  return check_launch("layernorm backward", err);
}

template <class TX, class TY>
int bwd_typed(Ctx* c, LnArgs a, bool vec, float* dgamma, float* dbeta, int accumulate, std::string& err) {
  const bool params = dgamma || dbeta;
  const bool lng = a.cols > kLnMaxRegCols;
  LnShape s{};
  RingShape ring{};
  bool use_ring = false;
  int blocks;
  if (lng) {
    blocks = (int)std::min<long>(a.rows, 64);
  } else {
    s = ln_shape(a.cols, false);
    use_ring = vec && s.block && s.nv == 1;
    if (use_ring) {
      ring = ring_shape(c, a, (size_t)a.cols * (sizeof(TX) + sizeof(TY)));
      blocks = ring.blocks;
    } else {
      blocks = bwd_blocks(c, a, s);
    }
  }
  if (params) {
    a.part = static_cast<float*>(scratch_get(c, kSlotLnPart, (size_t)blocks * 2 * a.cols * sizeof(float), err));
    if (!a.part) return 1;
  }
  int rc = 0;
  if (lng) {
    ProfScope prof_(c, "layernorm.bwd");
    if (a.out) launch_pdl(c, ln_bwd_long_kernel<TX, TY>, dim3((unsigned)a.rows), dim3(1024), 0, a);
    if (params)
      launch_pdl(c, ln_param_long_kernel<TX, TY>, dim3(blocks, (unsigned)((a.cols + 255) / 256)), dim3(256), 0, a);
    rc = check_launch("layernorm backward", err);
  } else if (!s.block) {
    rc = vec ? bwd_launch<TX, TY, false, 1, true>(c, a, s, blocks, err) : bwd_launch<TX, TY, false, 1, false>(c, a, s, blocks, err);
  } else if (use_ring) {
    rc = ring_launch<TX, TY>(c, a, ring, err);
  } else if (s.nv == 1) {
    rc = bwd_launch<TX, TY, true, 1, false>(c, a, s, blocks, err);
  } else if (s.nv == 2) {
    rc = vec ? bwd_launch<TX, TY, true, 2, true>(c, a, s, blocks, err) : bwd_launch<TX, TY, true, 2, false>(c, a, s, blocks, err);
  } else {
    rc = vec ? bwd_launch<TX, TY, true, 4, true>(c, a, s, blocks, err) : bwd_launch<TX, TY, true, 4, false>(c, a, s, blocks, err);
  }
  if (rc || !params) return rc;
  return k_fold_partials(c, a.part, blocks, 2, a.cols, dgamma, dbeta, accumulate, accumulate, err);
}

// type-erased dispatch over the nine (x, y) type pairs
template <class F>
int with_type(int type, F&& f, const char* what, std::string& err) {
  switch (type) {
    case kTypeF32: return f(float{});
    case kTypeF16: return f(__half{});
    case kTypeBF16: return f(__nv_bfloat16{});
    default: err = std::string(what) + ": the type must be F32, F16 or BF16"; return 1;
  }
}

size_t type_size(int type) { return type == kTypeF32 ? 4 : 2; }

int check_matrix(const char* what, const void* p, int type, int64_t rows, int64_t cols, int64_t ld, std::string& err) {
  if (type != kTypeF32 && type != kTypeF16 && type != kTypeBF16) {
    err = std::string("layernorm: the type of ") + what + " must be F32, F16 or BF16";
    return 1;
  }
  if (rows > 0 && !p) { err = std::string("layernorm: ") + what + " is NULL"; return 1; }
  if (reinterpret_cast<uintptr_t>(p) % type_size(type)) { err = std::string("layernorm: ") + what + " is not aligned to its type"; return 1; }
  if (rows > 1 && ld < cols) { err = std::string("layernorm: the row stride of ") + what + " is smaller than a row"; return 1; }
  return 0;
}

int check_shape(int64_t rows, int64_t cols, std::string& err) {
  if (rows < 0 || cols < 1 || cols > (1 << 20) || rows > 0x7fffffff) {
    err = "layernorm: need 0 <= rows < 2^31 and 1 <= cols <= 2^20";
    return 1;
  }
  return 0;
}

bool vec_ok(const void* p, int type, int64_t rows, int64_t ld) {
  return aligned16(p) && (rows < 2 || (ld * (int64_t)type_size(type)) % 16 == 0);
}

}  // namespace
}  // namespace sa3k

using namespace sa3k;

extern "C" {

int sa3k_layernorm_fwd(sa3k_ctx* ctx, int64_t rows, int64_t cols, int x_type, const void* x, int64_t x_ld,
                       const float* gamma, const float* beta, float eps, int y_type, void* y, int64_t y_ld,
                       float* mean, float* rstd, char* err, int err_len) {
  return api_call(ctx, err, err_len, [&](Ctx* c, std::string& e) {
    if (check_shape(rows, cols, e) || check_matrix("x", x, x_type, rows, cols, x_ld, e) ||
        check_matrix("y", y, y_type, rows, cols, y_ld, e))
      return 1;
    if (!(eps >= 0.f)) { e = "layernorm: eps must not be negative"; return 1; }
    if (rows == 0) return 0;
    LnArgs a{};
    a.rows = rows; a.cols = (int)cols;
    a.x = x; a.x_ld = x_ld; a.out = y; a.out_ld = y_ld;
    a.gamma = gamma; a.beta = beta; a.mean = mean; a.rstd = rstd; a.eps = eps;
    const bool vec = cols % 8 == 0 && vec_ok(x, x_type, rows, x_ld) && vec_ok(y, y_type, rows, y_ld) &&
                     aligned16(gamma) && aligned16(beta);
    return with_type(x_type, [&](auto tx) {
      return with_type(y_type, [&](auto ty) { return fwd_typed<decltype(tx), decltype(ty)>(c, a, vec, e); }, "y", e);
    }, "x", e);
  });
}

int sa3k_layernorm_bwd(sa3k_ctx* ctx, int64_t rows, int64_t cols, int x_type, const void* x, int64_t x_ld,
                       const float* gamma, const float* mean, const float* rstd, int y_type, const void* dy,
                       int64_t dy_ld, void* dx, int64_t dx_ld, float* dgamma, float* dbeta, int accumulate, char* err,
                       int err_len) {
  return api_call(ctx, err, err_len, [&](Ctx* c, std::string& e) {
    if (check_shape(rows, cols, e) || check_matrix("x", x, x_type, rows, cols, x_ld, e) ||
        check_matrix("dy", dy, y_type, rows, cols, dy_ld, e) ||
        (dx && check_matrix("dx", dx, x_type, rows, cols, dx_ld, e)))
      return 1;
    if (rows > 0 && (!mean || !rstd)) { e = "layernorm: the backward needs the forward's mean and rstd"; return 1; }
    if (rows == 0) {
      for (float* g : {dgamma, dbeta})
        if (g && !accumulate && cudaMemsetAsync(g, 0, (size_t)cols * 4, c->stream) != cudaSuccess)
          return check_launch("layernorm memset", e);
      return 0;
    }
    if (!dx && !dgamma && !dbeta) return 0;
    LnArgs a{};
    a.rows = rows; a.cols = (int)cols;
    a.x = x; a.x_ld = x_ld; a.dy = dy; a.dy_ld = dy_ld; a.out = dx; a.out_ld = dx_ld;
    a.gamma = gamma; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    const bool vec = cols % 8 == 0 && vec_ok(x, x_type, rows, x_ld) && vec_ok(dy, y_type, rows, dy_ld) &&
                     (!dx || vec_ok(dx, x_type, rows, dx_ld)) && aligned16(gamma);
    return with_type(x_type, [&](auto tx) {
      return with_type(y_type, [&](auto ty) {
        return bwd_typed<decltype(tx), decltype(ty)>(c, a, vec, dgamma, dbeta, accumulate, e);
      }, "dy", e);
    }, "x", e);
  });
}

}  // extern "C"
