// linear_act.cu -- the adapted frozen linear with an activation and a residual.
//
//   z = g (x W^T + s (x A^T) B^T) + bias,   y = act(z) + residual
//   backward: dz = dy act'(z);  dbias = colsum(dz);  dx and the adapter gradients as in linear.cu
//             for the upstream gradient dz (the residual's gradient is dy itself)
#include <cmath>

#include "../../include/sa3k.h"
#include "activation.cuh"
#include "linear.h"
#include "lora_kernels.h"
#include "ops_api.h"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

// y = act(zf) + residual, z = zf rounded
template <class T>
__global__ void __launch_bounds__(256) act_residual_kernel(const float* zf, long n, int act, const T* residual, T* z, T* y) {
  pdl_prologue();
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const float v = zf[i];
    if (z) z[i] = from_f32<T>(v);
    y[i] = from_f32<T>(act_value(act, v) + (residual ? to_f32(residual[i]) : 0.f));
  }
}

// Output of a split-K product: partial sums added in split order, column scale, bias, activation and
// residual; W columns per thread.  A pass of its own over all SMs: the last CTA of each tile adding its
// own splits took most of the time (33 x 6144 x 1536: 32 us, with this pass 19).
template <class T, int W>
__global__ void __launch_bounds__(128) act_splits_kernel(const float* __restrict__ partial, int splits, long n, int N,
                                                         const float* __restrict__ scale, const float* __restrict__ bias, int act,
                                                         const T* residual, T* __restrict__ z, T* y) {   // (y may be the residual)
  pdl_prologue();
  const long i = ((long)blockIdx.x * 128 + threadIdx.x) * W;
  if (i >= n) return;
  float v[W];
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    if constexpr (W == 4) {
      const float4 p = *reinterpret_cast<const float4*>(partial + (long)s * n + i);
      v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
    } else {
      v[0] += partial[(long)s * n + i];
    }
  }
  const int col = (int)(i % N);
#pragma unroll
  for (int e = 0; e < W; ++e) {
    if (scale) v[e] *= scale[col + e];
    if (bias) v[e] += bias[col + e];
    if (z) z[i + e] = from_f32<T>(v[e]);
    v[e] = act_value(act, v[e]);
    if (residual) v[e] += to_f32(residual[i + e]);
    y[i + e] = from_f32<T>(v[e]);
  }
}

template <class T>
int act_splits(Ctx* c, const GemmDesc& d, const float* partial, int splits, T* y, std::string& err) {
  const long n = (long)d.M * d.N;
  const T* res = static_cast<const T*>(d.epi->residual);
  T* z = static_cast<T*>(d.epi->z);
  ProfScope prof_(c, "linear_act.splits");
  if (d.N % 4 == 0)
    launch_pdl(c, act_splits_kernel<T, 4>, dim3((unsigned)((n / 4 + 127) / 128)), dim3(128), 0, partial, splits, n, d.N, d.col_scale,
               d.col_bias, d.epi->act, res, z, y);
  else
    launch_pdl(c, act_splits_kernel<T, 1>, dim3((unsigned)((n + 127) / 128)), dim3(128), 0, partial, splits, n, d.N, d.col_scale,
               d.col_bias, d.epi->act, res, z, y);
  return check_launch("linear_act splits", err);
}

// dz = f16(g dy act'(z)), and with part the partial column sums over the block's kActRows rows:
// part[blockIdx.y][0] of dy act'(z) (the bias gradient), with DORA [1] of dy act'(z) (z - bias) / g (dora's dg).
// One pass: dy and z are read and dz is written once, in 16-byte accesses of 8 columns a thread (VEC)
// or one column a thread (widths and bases that allow none).  Bound by memory: 2047 x 6144 f16 moves
// 75 MB.
constexpr int kActRows = 16;
template <class T, int ACT, bool VEC, bool DORA>
__global__ void __launch_bounds__(128) act_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ z, const float* __restrict__ bias,
                                                      const float* __restrict__ g, long S,
                                                      long out, __half* __restrict__ dz, long dz_ld, float* __restrict__ part) {
  pdl_prologue();
  constexpr int W = VEC ? 8 : 1;
  const long o = ((long)blockIdx.x * 128 + threadIdx.x) * W;
  if (o >= out) return;
  const long t0 = (long)blockIdx.y * kActRows, t1 = min(S, t0 + kActRows);
  float go[W], bo[W], inv[W], sb[W], sg[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    if (DORA) {
      go[e] = g[o + e];
      bo[e] = bias ? bias[o + e] : 0.f;
      inv[e] = 1.f / go[e];
    }
    sb[e] = sg[e] = 0.f;
  }
  constexpr int U = 2;        // rows whose loads are in flight together
  for (long t = t0; t < t1; t += U) {
    float d[U][8], v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= t1) continue;
      if constexpr (VEC) {
        load8(dy + (t + u) * out + o, d[u]);
        if (z) load8(z + (t + u) * out + o, v[u]);
      } else {
        d[u][0] = to_f32(dy[(t + u) * out + o]);
        if (z) v[u][0] = to_f32(z[(t + u) * out + o]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= t1) continue;
      float q[8];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (!z) v[u][e] = 0.f;
        const float x = d[u][e] * act_slope(ACT, v[u][e]);
        q[e] = DORA ? x * go[e] : x;
        sb[e] += x;
        if (DORA) sg[e] = fmaf(x, (v[u][e] - bo[e]) * inv[e], sg[e]);
      }
      if constexpr (VEC) store8(dz + (t + u) * dz_ld + o, q);
      else dz[(t + u) * dz_ld + o] = __float2half_rn(q[0]);
    }
  }
  if (!part) return;
  float* p = part + (long)blockIdx.y * (DORA ? 2 : 1) * out + o;
#pragma unroll
  for (int e = 0; e < W; ++e) {
    p[e] = sb[e];
    if (DORA) p[out + e] = sg[e];
  }
}

int64_t pad64(int64_t v) { return (v + 63) / 64 * 64; }
size_t al(size_t b) { return (b + 255) & ~(size_t)255; }

int check_args(const Ctx* c, const Weight* w, const sa3k_adapter* ad, const float* bias, int act, int type, int64_t S,
               std::string& err) {
  if (w->device != c->device) { err = "linear_act: the weight is on another device than the context"; return 1; }
  if (act < kActNone || act > kActGeluTanh) { err = "linear_act: unknown activation"; return 1; }
  if (type != kTypeF32 && type != kTypeF16) { err = "linear_act: the type must be F32 or F16"; return 1; }
  if (S < 0 || S > (1 << 20) - 16) { err = "linear_act: S must be from 0 to 2^20 - 16"; return 1; }
  if (!aligned16(bias)) { err = "linear_act: bias must start on 16 bytes"; return 1; }
  if (!ad) return 0;
  if (ad->rank < 1 || ad->rank > 16 || !ad->A || !ad->B) { err = "adapter rank must be 1..16 with A and B"; return 1; }
  if (!aligned16(ad->A) || !aligned16(ad->B) || !aligned16(ad->magnitude) || !aligned16(ad->base_norm_sq)) {
    err = "linear_act: the adapter's arrays must start on 16 bytes";
    return 1;
  }
  if (ad->magnitude && !ad->base_norm_sq) { err = "dora adapter needs base_norm_sq"; return 1; }
  return 0;
}

// x, y, ...: given, and on 16 bytes where the kernels read it in vectors (`vec`), else on its own type
int check_rows(const char* what, const void* p, int type, bool vec, std::string& err) {
  if (!p) { err = std::string("linear_act: ") + what + " is NULL"; return 1; }
  if (reinterpret_cast<uintptr_t>(p) % (vec ? 16 : type == kTypeF32 ? 4 : 2)) {
    err = std::string("linear_act: ") + what + (vec ? " must start on 16 bytes" : " is not aligned to its type");
    return 1;
  }
  return 0;
}

// x as the f16 operand (converted into scratch when it is f32)
int operand(Ctx* c, int type, const void* x, int64_t n, const __half*& x_h, std::string& err) {
  if (type == kTypeF16) {
    x_h = static_cast<const __half*>(x);
    return 0;
  }
  __half* p = static_cast<__half*>(scratch_get(c, kSlotActX, (size_t)n * sizeof(__half), err));
  if (!p || k_cvt_f16(c, static_cast<const float*>(x), n, p, err)) return 1;
  x_h = p;
  return 0;
}

// the adapter's derived operands and u^T, in one scratch buffer
int prepare_adapter(Ctx* c, const Weight* w, const sa3k_adapter* ad, const __half* x_h, int64_t S, AdapterPrep& prep,
                    __half*& ut, std::string& err) {
  prep.rank = ad->rank; prep.in = w->in; prep.out = w->out; prep.s = ad->scale;
  prep.A = ad->A; prep.B = ad->B; prep.m = ad->magnitude; prep.bns = ad->base_norm_sq;
  const size_t pb = al(adapter_prep_bytes(w->in, w->out, ad->magnitude != nullptr));
  char* mem = static_cast<char*>(scratch_get(c, kSlotActAdapter, pb + (size_t)(16 * pad64(S)) * sizeof(__half), err));
  if (!mem) return 1;
  adapter_bind(prep, mem);
  ut = reinterpret_cast<__half*>(mem + pb);
  return adapter_prepare(c, w, prep, err);
}

template <class T>
int act_residual(Ctx* c, const float* zf, int64_t n, int act, const void* residual, void* z, void* y, std::string& err) {
  ProfScope prof_(c, "linear_act.epilogue");
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, (int64_t)c->sm_count * 8);
  launch_pdl(c, act_residual_kernel<T>, dim3(grid), dim3(256), 0, zf, (long)n, act, static_cast<const T*>(residual),
             static_cast<T*>(z), static_cast<T*>(y));
  return check_launch("linear_act epilogue", err);
}

int linear_act_forward(Ctx* c, const Weight* w, const sa3k_adapter* ad, const float* bias, int act, int type,
                       const void* x, int64_t S, const void* residual, void* z, void* y, std::string& err) {
  if (!ad && linear_rows_applies(S)) return linear_rows(c, w, bias, act, type, x, S, residual, z, y, err);
  const __half* x_h;
  if (operand(c, type, x, S * w->in, x_h, err)) return 1;
  AdapterPrep prep;
  __half* ut = nullptr;
  if (ad && prepare_adapter(c, w, ad, x_h, S, prep, ut, err)) return 1;
  LinearFwd f;
  f.w = w; f.ad = ad ? &prep : nullptr; f.bias = bias; f.x_h = x_h; f.M = S;
  f.ut = ut; f.ut_ld = pad64(S);
  if (!dequantizes_inside(c, *w)) {     // activation and residual in the GEMM's epilogue
    ActEpi e;
    e.act = act; e.residual = residual; e.z = z;
    f.epi = &e;
    if (type == kTypeF16) f.y_h = static_cast<__half*>(y);
    else f.y = static_cast<float*>(y);
    return linear_forward(c, f, err);
  }
  // a base that is dequantized inside the GEMM: the f32 product, then one pass
  float* zf = static_cast<float*>(scratch_get(c, kSlotActZ, (size_t)(S * w->out) * sizeof(float), err));
  if (!zf) return 1;
  f.y = zf;
  if (linear_forward(c, f, err)) return 1;
  return type == kTypeF16 ? act_residual<__half>(c, zf, S * w->out, act, residual, z, y, err)
                          : act_residual<float>(c, zf, S * w->out, act, residual, z, y, err);
}

template <class T, int ACT>
int act_bwd_as(Ctx* c, const T* dy, const T* z, const float* bias, const float* g, int64_t S, int64_t out, __half* dz,
               int64_t dz_ld, float* part, std::string& err) {
  const bool vec = out % 8 == 0 && aligned16(dy) && aligned16(z);
  const int64_t per = vec ? 1024 : 128;
  const dim3 grid((unsigned)((out + per - 1) / per), (unsigned)((S + kActRows - 1) / kActRows));
  ProfScope prof_(c, "linear_act.dz");
  auto kern = g ? (vec ? act_bwd_kernel<T, ACT, true, true> : act_bwd_kernel<T, ACT, false, true>)
                : (vec ? act_bwd_kernel<T, ACT, true, false> : act_bwd_kernel<T, ACT, false, false>);
  launch_pdl(c, kern, grid, dim3(128), 0, dy, z, bias, g, (long)S, (long)out, dz, (long)dz_ld, part);
  return check_launch("linear_act dz", err);
}

template <class T>
int act_bwd(Ctx* c, const void* dyv, const void* zv, const float* bias, const float* g, int act, int64_t S, int64_t out,
            __half* dz, int64_t dz_ld, float* part, std::string& err) {
  const T* dy = static_cast<const T*>(dyv);
  const T* z = static_cast<const T*>(zv);
  switch (act) {
    case kActSilu: return act_bwd_as<T, kActSilu>(c, dy, z, bias, g, S, out, dz, dz_ld, part, err);
    case kActGelu: return act_bwd_as<T, kActGelu>(c, dy, z, bias, g, S, out, dz, dz_ld, part, err);
    case kActGeluTanh: return act_bwd_as<T, kActGeluTanh>(c, dy, z, bias, g, S, out, dz, dz_ld, part, err);
    default: return act_bwd_as<T, kActNone>(c, dy, z, bias, g, S, out, dz, dz_ld, part, err);
  }
}

int linear_act_backward(Ctx* c, const Weight* w, const sa3k_adapter* ad, const float* bias, int act, int type,
                        const void* x, int64_t S, const void* z, const void* dy, void* dx, float* dbias, float* dA,
                        float* dB, float* dm, int accumulate, std::string& err) {
  const int64_t in = w->in, out = w->out;
  const bool dora = ad && ad->magnitude;
  const __half* x_h = nullptr;
  AdapterPrep prep;
  __half* ut = nullptr;
  if (ad) {
    if (operand(c, type, x, S * in, x_h, err)) return 1;
    if (prepare_adapter(c, w, ad, x_h, S, prep, ut, err) || lora_u(c, x_h, S, in, prep, ut, pad64(S), err)) return 1;
  }
  const int64_t dz_ld = (out + 7) / 8 * 8;   // (TMA reads rows that start on 16 bytes)
  // scratch: dz | dut | dg | cb | c3 | partial sums
  const int chunks = (int)((S + kActRows - 1) / kActRows), planes = dora ? 2 : 1;
  const bool sums = dbias || dora;
  const size_t b_dz = al((size_t)(S * dz_ld) * 2), b_dut = ad ? al((size_t)(16 * pad64(S)) * 2) : 0,
               b_dg = dora ? al((size_t)out * 4) : 0, b_cb = dora ? al((size_t)(16 * out) * 2) : 0, b_c3 = dora ? al(1024) : 0,
               b_part = sums ? al((size_t)chunks * planes * out * 4) : 0;
  char* mem = static_cast<char*>(scratch_get(c, kSlotActPart, b_dz + b_dut + b_dg + b_cb + b_c3 + b_part, err));
  if (!mem) return 1;
  LinearBwd b;
  b.w = w; b.ad = ad ? &prep : nullptr; b.bias = bias; b.x_h = x_h; b.M = S; b.ut = ut; b.ut_ld = pad64(S);
  b.dz = reinterpret_cast<__half*>(mem);
  b.dut = reinterpret_cast<__half*>(mem + b_dz);
  b.dg = reinterpret_cast<float*>(mem + b_dz + b_dut);
  b.cb = reinterpret_cast<__half*>(mem + b_dz + b_dut + b_dg);
  b.c3 = reinterpret_cast<float*>(mem + b_dz + b_dut + b_dg + b_cb);
  float* part = sums ? reinterpret_cast<float*>(mem + b_dz + b_dut + b_dg + b_cb + b_c3) : nullptr;
  const float* g = dora ? prep.g : nullptr;
  if (type == kTypeF16 ? act_bwd<__half>(c, dy, z, bias, g, act, S, out, b.dz, dz_ld, part, err)
                       : act_bwd<float>(c, dy, z, bias, g, act, S, out, b.dz, dz_ld, part, err))
    return 1;
  if (sums && k_fold_partials(c, part, chunks, planes, (int)out, dbias, dora ? b.dg : nullptr, accumulate, 0, err)) return 1;
  b.dz_ready = true;
  b.dz_ld = dz_ld;
  if (type == kTypeF16) b.dx_h = static_cast<__half*>(dx);
  else b.dx = static_cast<float*>(dx);
  b.dA = dA; b.dB = dB; b.dm = dm; b.grad_accumulate = accumulate;
  return linear_backward(c, b, err);
}

}  // namespace

int k_act_splits(Ctx* c, const GemmDesc& d, const float* partial, int splits, std::string& err) {
  return d.out_h ? act_splits<__half>(c, d, partial, splits, d.out_h, err) : act_splits<float>(c, d, partial, splits, d.out, err);
}

}  // namespace sa3k

using namespace sa3k;

extern "C" {

int sa3k_linear_act_fwd(sa3k_ctx* ctx, const sa3k_weight* w, const sa3k_adapter* ad, const float* bias, int act, int type,
                        const void* x, int64_t S, const void* residual, void* z, void* y, char* err, int err_len) {
  return api_call(ctx, err, err_len, [&](Ctx* c, std::string& e) {
    if (!w) { e = "linear_act: the weight is NULL"; return 1; }
    if (check_args(c, &w->w, ad, bias, act, type, S, e)) return 1;
    if (S == 0) return 0;
    if (check_rows("x", x, type, true, e) || check_rows("y", y, type, false, e) ||
        (residual && check_rows("residual", residual, type, false, e)) || (z && check_rows("z", z, type, false, e)))
      return 1;
    return linear_act_forward(c, &w->w, ad, bias, act, type, x, S, residual, z, y, e);
  });
}

int sa3k_linear_act_bwd(sa3k_ctx* ctx, const sa3k_weight* w, const sa3k_adapter* ad, const float* bias, int act, int type,
                        const void* x, int64_t S, const void* z, const void* dy, void* dx, float* dbias, float* dA,
                        float* dB, float* dm, int accumulate, char* err, int err_len) {
  return api_call(ctx, err, err_len, [&](Ctx* c, std::string& e) {
    if (!w) { e = "linear_act: the weight is NULL"; return 1; }
    const bool dora = ad && ad->magnitude;
    if (check_args(c, &w->w, ad, bias, act, type, S, e)) return 1;
    if (ad && (!dA || !dB || (dora && !dm))) { e = "linear_act: an adapter needs dA and dB, and dm for dora"; return 1; }
    // (rows of B^T and of dora's factors are operands of TMA: 16-byte steps of halves)
    if (ad && w->w.out % 8) { e = "linear_act: the backward of an adapter needs an output width that is a multiple of 8"; return 1; }
    if (S > 0) {
      if (check_rows("dy", dy, type, false, e) || (ad && check_rows("x", x, type, true, e)) ||
          (z && check_rows("z", z, type, false, e)) || (dx && check_rows("dx", dx, type, true, e)))
        return 1;
      if (!z && (act != kActNone || dora)) { e = "linear_act: the backward needs the forward's z"; return 1; }
    }
    if (S == 0) {
      if (accumulate) return 0;
      const size_t n[4] = {(size_t)w->w.out, ad ? (size_t)(ad->rank * w->w.in) : 0, ad ? (size_t)(ad->rank * w->w.out) : 0,
                           dora ? (size_t)w->w.out : 0};
      float* p[4] = {dbias, dA, dB, dm};
      for (int i = 0; i < 4; ++i)
        if (p[i] && n[i] && cudaMemsetAsync(p[i], 0, n[i] * 4, c->stream) != cudaSuccess) return check_launch("linear_act memset", e);
      return 0;
    }
    return linear_act_backward(c, &w->w, ad, bias, act, type, x, S, z, dy, dx, dbias, dA, dB, dm, accumulate, e);
  });
}

}  // extern "C"
