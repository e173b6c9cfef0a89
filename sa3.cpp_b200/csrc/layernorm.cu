// layernorm.cu -- layer normalisation over the rows of a matrix, forward and backward.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps),  y = (x - mu) r gamma + beta
//   backward  xh = (x - mu) r, g = dy gamma:
//             dx = r (g - mean(g) - xh mean(g xh)),  dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// Both are bound by memory: each value of x (and dy) is read once and held in registers while its
// row's sums are formed, and each result is written once.  The variance is taken around the mean
// of the held values, not from a sum of squares, so a large common offset costs no digits.  All
// arithmetic is f32 whatever the types; a result is rounded once, when it is stored.
//
// A row belongs to TPR threads: a part of a warp for short rows, else a whole block.  The backward
// keeps every thread's columns' sums of dy xh and dy in registers over all the rows that its block
// walks, and writes one partial row per block; a second kernel adds the partials in block order,
// so the parameter gradients do not depend on timing.
#include <cmath>

#include "../../include/sa3k.h"
#include "ops_api.h"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

// out[i] (+)= sum over blocks of part[block][which][i]: 32 columns x 32 slices of the blocks per
// thread block, the slices added in order.
__global__ void __launch_bounds__(1024) fold_partials_kernel(const float* part, int nblocks, int cols, float* out0,
                                                             float* out1, int acc0, int acc1) {
  __shared__ float s[32][33];
  pdl_prologue();
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float* out = blockIdx.y == 0 ? out0 : out1;
  if (!out) return;
  const float* p = part + (long)blockIdx.y * cols + i;
  float v = 0.f;
  if (i < cols)
    for (int b = w; b < nblocks; b += 32) v += p[(long)b * 2 * cols];
  s[w][threadIdx.x & 31] = v;
  __syncthreads();
  // warp w takes column w of the 32: its lanes hold the 32 slices
  v = warp_sum(s[threadIdx.x & 31][w]);
  const int o = blockIdx.x * 32 + w;
  if ((threadIdx.x & 31) == 0 && o < cols) out[o] = (blockIdx.y == 0 ? acc0 : acc1) ? out[o] + v : v;
}

}  // namespace

int k_fold_partials(Ctx* c, const float* part, int nblocks, int cols, float* out0, float* out1, int acc0, int acc1,
                    std::string& err) {
  ProfScope prof_(c, "fold_partials");
  launch_pdl(c, fold_partials_kernel, dim3((unsigned)((cols + 31) / 32), 2), dim3(1024), 0, part, nblocks, cols, out0, out1,
             acc0, acc1);
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

// Sum of two values over the TPR threads of a row; every thread gets it.  `red`: 2 x 32 pairs,
// alternated by the caller (`ph`) so that one barrier per reduction is enough.
template <bool BLOCK>
__device__ __forceinline__ float2 row_sum(float a, float b, int tpr, float2 (*red)[32], int ph) {
  if (BLOCK) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    const int nw = blockDim.x >> 5;
    if (nw > 1) {
      if ((threadIdx.x & 31) == 0) red[ph][threadIdx.x >> 5] = make_float2(a, b);
      __syncthreads();
      const float2 t = (threadIdx.x & 31) < nw ? red[ph][threadIdx.x & 31] : make_float2(0.f, 0.f);
      a = t.x;
      b = t.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
    }
  } else {
    for (int o = tpr >> 1; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
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

// Forward with the row in registers: NV chunks of 8 columns per thread.
template <class TX, class TY, bool BLOCK, int NV, bool VEC>
__global__ void __launch_bounds__(1024) ln_fwd_kernel(const LnArgs a, int tpr) {
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
  const float mu = row_sum<BLOCK>(s, 0.f, tpr, red, 0).x / (float)a.cols;
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = v[c][e] - mu;
      if (col_of<VEC>(c, e, t, tpr) < a.cols) q = fmaf(d, d, q);
    }
  const float rs = 1.0f / sqrtf(row_sum<BLOCK>(q, 0.f, tpr, red, 1).x / (float)a.cols + a.eps);
  if (!ok) return;
  if (t == 0) {
    if (a.mean) a.mean[r] = mu;
    if (a.rstd) a.rstd[r] = rs;
  }
  TY* y = static_cast<TY*>(a.out) + r * a.out_ld;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    float gm[8], bt[8], o[8];
    if (a.gamma) load_chunk<VEC>(a.gamma, c, t, tpr, a.cols, gm);
    if (a.beta) load_chunk<VEC>(a.beta, c, t, tpr, a.cols, bt);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      o[e] = fmaf((v[c][e] - mu) * rs, a.gamma ? gm[e] : 1.f, a.beta ? bt[e] : 0.f);
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
  const float mu = row_sum<true>(s, 0.f, 0, red, 0).x / (float)a.cols;
  float q = 0.f;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
    const float d = to_f32(x[i]) - mu;
    q = fmaf(d, d, q);
  }
  const float rs = 1.0f / sqrtf(row_sum<true>(q, 0.f, 0, red, 1).x / (float)a.cols + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[r] = mu;
    if (a.rstd) a.rstd[r] = rs;
  }
  TY* y = static_cast<TY*>(a.out) + r * a.out_ld;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x)
    y[i] = from_f32<TY>(fmaf((to_f32(x[i]) - mu) * rs, a.gamma ? a.gamma[i] : 1.f, a.beta ? a.beta[i] : 0.f));
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
    const float2 s = row_sum<BLOCK>(s1, s2, tpr, red, ph);
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
  const float2 s = row_sum<true>(s1, s2, 0, red, 0);
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
// most 1024 threads, at 8, 16 or 32 columns a thread.
struct LnShape {
  bool block;
  int tpr, threads, nv;
};
LnShape ln_shape(int cols) {
  LnShape s;
  if (cols <= 256) {
    s.block = false;
    s.tpr = 1;
    while (s.tpr * 8 < cols) s.tpr *= 2;
    s.threads = 256;
    s.nv = 1;
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
  const LnShape s = ln_shape(a.cols);
  if (!s.block) return fwd_launch<TX, TY, false, 1>(c, a, s, vec, err);
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
  int blocks;
  if (lng) {
    blocks = (int)std::min<long>(a.rows, 64);
  } else {
    s = ln_shape(a.cols);
    blocks = bwd_blocks(c, a, s);
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
  } else if (s.nv == 1) {
    rc = vec ? bwd_launch<TX, TY, true, 1, true>(c, a, s, blocks, err) : bwd_launch<TX, TY, true, 1, false>(c, a, s, blocks, err);
  } else if (s.nv == 2) {
    rc = vec ? bwd_launch<TX, TY, true, 2, true>(c, a, s, blocks, err) : bwd_launch<TX, TY, true, 2, false>(c, a, s, blocks, err);
  } else {
    rc = vec ? bwd_launch<TX, TY, true, 4, true>(c, a, s, blocks, err) : bwd_launch<TX, TY, true, 4, false>(c, a, s, blocks, err);
  }
  if (rc || !params) return rc;
  return k_fold_partials(c, a.part, blocks, a.cols, dgamma, dbeta, accumulate, accumulate, err);
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
  if (rows < 0 || cols < 1 || cols > (1 << 24) || rows > 0x7fffffff) {
    err = "layernorm: need 0 <= rows < 2^31 and 1 <= cols <= 2^24";
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
