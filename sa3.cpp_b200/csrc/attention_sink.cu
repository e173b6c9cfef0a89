// attention_sink.cu -- attention over a sliding window with sink tokens, head_dim 64.
//
// Query row i of a batch entry stands at position p = i (+ kv_len - q_len with align_end) and sees
// key j < kv_len when j <= p + right and (j < sinks or j >= p - left): the window, plus the first
// `sinks` tokens that stay visible after the window has moved on.
//   o = sum_j P_j v_j,  P_j = exp2(scale log2(e) q k_j - lse),  lse = log2 sum_j exp2(...)
//   backward: dV = P^T dO,  dS = P o (dO V^T - D),  D = rowsum(dO o O),
//             dQ = scale dS K,  dK = scale dS^T Q (summed over the query heads of a shared head)
// Rows that see nothing get o = 0 and lse = -inf, and take no part in the gradients.
#include "attention_sink.h"

#include <climits>
#include <cmath>

#include "../../include/sa3k.h"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

template <class T>
__device__ __forceinline__ const T* row_ptr(const SinkTensor& t, int b, int h, int r) {
  return static_cast<const T*>(t.p) + (long)b * t.sb + (long)h * t.sh + (long)r * t.ld;
}
template <class T>
__device__ __forceinline__ T* row_out(const SinkTensor& t, int b, int h, int r) {
  return static_cast<T*>(t.p) + (long)b * t.sb + (long)h * t.sh + (long)r * t.ld;
}

template <class T>
__device__ __forceinline__ float dot64(const float* x, const T* y) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < 64; c += 8) {
    float v[8];
    load8(y + c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x[c + e], v[e], s);
  }
  return s;
}

// A warp per query row: lanes take 32 keys at a time for the scores, then two columns each of o.
template <class T>
__global__ void __launch_bounds__(128) sink_fwd_rows_kernel(const SinkArgs a) {
  __shared__ float sq[4][64];
  pdl_prologue();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long row = (long)blockIdx.x * 4 + w;
  if (row >= (long)a.B * a.H * a.Sq) return;
  const int i = (int)(row % a.Sq), h = (int)(row / a.Sq % a.H), b = (int)(row / a.Sq / a.H);
  const SinkSeq s = sink_seq(a, b);
  if (i >= s.qn) return;
  const T* q = row_ptr<T>(a.q, b, h, i);
  sq[w][lane] = to_f32(q[lane]);
  sq[w][lane + 32] = to_f32(q[lane + 32]);
  __syncwarp();
  const int p = s.pos0 + i, hk = h / a.group;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  const int hi = min(s.kn, p + a.right + 1);
  for (int j0 = 0; j0 < hi; j0 += 32) {
    if (j0 >= a.sinks && j0 + 31 < p - a.left) continue;
    const int j = j0 + lane;
    const bool see = sink_sees(a, s, p, j);
    const float x = see ? dot64(sq[w], row_ptr<T>(a.k, b, hk, j)) * a.sl2 : -INFINITY;
    float mx = x;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx == -INFINITY) continue;
    const float mn = fmaxf(m, mx), al = exp2f(m - mn), pr = see ? exp2f(x - mn) : 0.f;
    m = mn;
    l = l * al + warp_sum(pr);
    o0 *= al;
    o1 *= al;
    for (int t = 0; t < 32; ++t) {
      const float pt = __shfl_sync(0xffffffffu, pr, t);
      const bool st = __shfl_sync(0xffffffffu, (int)see, t);
      if (!st) continue;
      const T* v = row_ptr<T>(a.v, b, hk, j0 + t);
      o0 = fmaf(pt, to_f32(v[2 * lane]), o0);
      o1 = fmaf(pt, to_f32(v[2 * lane + 1]), o1);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* o = row_out<T>(a.o, b, h, i);
  o[2 * lane] = from_f32<T>(o0 * inv);
  o[2 * lane + 1] = from_f32<T>(o1 * inv);
  if (lane == 0 && a.lse) a.lse[row] = l > 0.f ? m + log2f(l) : -INFINITY;
}

// A warp per query row: D, then dq.
template <class T>
__global__ void __launch_bounds__(128) sink_dq_rows_kernel(const SinkArgs a) {
  __shared__ float sq[4][64], sd[4][64];
  pdl_prologue();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long row = (long)blockIdx.x * 4 + w;
  if (row >= (long)a.B * a.H * a.Sq) return;
  const int i = (int)(row % a.Sq), h = (int)(row / a.Sq % a.H), b = (int)(row / a.Sq / a.H);
  const SinkSeq s = sink_seq(a, b);
  if (i >= s.qn) return;
  const T* q = row_ptr<T>(a.q, b, h, i);
  const T* d = row_ptr<T>(a.dO, b, h, i);
  const T* ov = row_ptr<T>(a.o, b, h, i);
  float D = 0.f;
  for (int c = lane; c < 64; c += 32) {
    sq[w][c] = to_f32(q[c]);
    sd[w][c] = to_f32(d[c]);
    D = fmaf(sd[w][c], to_f32(ov[c]), D);
  }
  D = warp_sum(D);
  __syncwarp();
  if (lane == 0) a.D[row] = D;
  const int p = s.pos0 + i, hk = h / a.group;
  const float lse = a.lse[row];
  float g0 = 0.f, g1 = 0.f;
  const int hi = lse == -INFINITY ? 0 : min(s.kn, p + a.right + 1);
  for (int j0 = 0; j0 < hi; j0 += 32) {
    if (j0 >= a.sinks && j0 + 31 < p - a.left) continue;
    const int j = j0 + lane;
    const bool see = sink_sees(a, s, p, j);
    float ds = 0.f;
    if (see) {
      const float pr = exp2f(dot64(sq[w], row_ptr<T>(a.k, b, hk, j)) * a.sl2 - lse);
      ds = pr * (dot64(sd[w], row_ptr<T>(a.v, b, hk, j)) - D);
    }
    for (int t = 0; t < 32; ++t) {
      const float dt = __shfl_sync(0xffffffffu, ds, t);
      if (!__shfl_sync(0xffffffffu, (int)see, t)) continue;
      const T* k = row_ptr<T>(a.k, b, hk, j0 + t);
      g0 = fmaf(dt, to_f32(k[2 * lane]), g0);
      g1 = fmaf(dt, to_f32(k[2 * lane + 1]), g1);
    }
  }
  T* dq = row_out<T>(a.dq, b, h, i);
  dq[2 * lane] = from_f32<T>(g0 * a.scale);
  dq[2 * lane + 1] = from_f32<T>(g1 * a.scale);
}

// A warp per key row: dk and dv over every query row and query head that sees it.
template <class T>
__global__ void __launch_bounds__(128) sink_dkdv_rows_kernel(const SinkArgs a) {
  __shared__ float sk[4][64], sv[4][64];
  pdl_prologue();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long row = (long)blockIdx.x * 4 + w;
  if (row >= (long)a.B * a.Hkv * a.Sk) return;
  const int j = (int)(row % a.Sk), hk = (int)(row / a.Sk % a.Hkv), b = (int)(row / a.Sk / a.Hkv);
  const SinkSeq s = sink_seq(a, b);
  if (j >= s.kn) return;
  const T* k = row_ptr<T>(a.k, b, hk, j);
  const T* v = row_ptr<T>(a.v, b, hk, j);
  for (int c = lane; c < 64; c += 32) {
    sk[w][c] = to_f32(k[c]);
    sv[w][c] = to_f32(v[c]);
  }
  __syncwarp();
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  // positions p with p + right >= j, and p - left <= j unless j is a sink
  const int lo = max(0, j - a.right - s.pos0);
  const int hi = j < a.sinks ? s.qn : (int)min((long)s.qn, (long)j + a.left - s.pos0 + 1);
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h)
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const long r = ((long)b * a.H + h) * a.Sq + i;
      bool see = i < hi && sink_sees(a, s, s.pos0 + i, j);
      float pr = 0.f, ds = 0.f;
      if (see) {
        const float lse = a.lse[r];
        pr = exp2f(dot64(sk[w], row_ptr<T>(a.q, b, h, i)) * a.sl2 - lse);
        ds = pr * (dot64(sv[w], row_ptr<T>(a.dO, b, h, i)) - a.D[r]);
      }
      for (int t = 0; t < 32; ++t) {
        const float pt = __shfl_sync(0xffffffffu, pr, t), dt = __shfl_sync(0xffffffffu, ds, t);
        if (!__shfl_sync(0xffffffffu, (int)see, t)) continue;
        const T* q = row_ptr<T>(a.q, b, h, i0 + t);
        const T* d = row_ptr<T>(a.dO, b, h, i0 + t);
        k0 = fmaf(dt, to_f32(q[2 * lane]), k0);
        k1 = fmaf(dt, to_f32(q[2 * lane + 1]), k1);
        v0 = fmaf(pt, to_f32(d[2 * lane]), v0);
        v1 = fmaf(pt, to_f32(d[2 * lane + 1]), v1);
      }
    }
  T* dk = row_out<T>(a.dk, b, hk, j);
  T* dv = row_out<T>(a.dv, b, hk, j);
  dk[2 * lane] = from_f32<T>(k0 * a.scale);
  dk[2 * lane + 1] = from_f32<T>(k1 * a.scale);
  dv[2 * lane] = from_f32<T>(v0);
  dv[2 * lane + 1] = from_f32<T>(v1);
}

template <class T>
int forward(Ctx* c, const SinkArgs& a, std::string& err) {
  const long rows = (long)a.B * a.H * a.Sq;
  ProfScope prof_(c, "attn_sink.fwd");
  launch_pdl(c, sink_fwd_rows_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, a);
  return check_launch("attention with sinks, forward", err);
}

template <class T>
int backward(Ctx* c, const SinkArgs& a, std::string& err) {
  const long rows = (long)a.B * a.H * a.Sq, keys = (long)a.B * a.Hkv * a.Sk;
  if (rows > 0) {
    ProfScope prof_(c, "attn_sink.dq");
    launch_pdl(c, sink_dq_rows_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, a);
    if (check_launch("attention with sinks, dq", err)) return 1;
  }
  if (!a.dk.p || keys == 0) return 0;
  ProfScope prof_(c, "attn_sink.dkdv");
  launch_pdl(c, sink_dkdv_rows_kernel<T>, dim3((unsigned)((keys + 3) / 4)), dim3(128), 0, a);
  return check_launch("attention with sinks, dk / dv", err);
}

// --------------------------------------------------------------------------- argument checks
constexpr int kFar = 1 << 29;    // "no bound": positions stay far below it

int check_tensor(const char* what, const sa3k_tensor4* t, int B, int H, int S, bool out, SinkTensor& d, std::string& err) {
  if (!t || !t->data) { err = std::string("attention_sink: ") + what + " is NULL"; return 1; }
  d.p = t->data;
  // (the stride of a dimension with one entry is never used)
  d.sb = B > 1 ? t->batch_stride : 64;
  d.sh = H > 1 ? t->head_stride : 64;
  d.ld = S > 1 ? t->row_stride : 64;
  if (!aligned16(d.p) || d.sb % 8 || d.sh % 8 || d.ld % 8) {
    err = std::string("attention_sink: ") + what + " must start on 16 bytes, with strides that are multiples of 8 elements";
    return 1;
  }
  if (d.sb < 0 || d.sh < 0 || d.ld < 0 || d.sb >= (1l << 38) || d.sh >= (1l << 38) || d.ld >= (1l << 38)) {
    err = std::string("attention_sink: the strides of ") + what + " must be from 0 to 2^38";
    return 1;
  }
  // rows of 64 values must not overlap where they are written: every stride holds a row, and the
  // dimensions nest (sorted by stride, each holds the extent of those below it)
  if (out) {
    long st[3] = {d.sb, d.sh, d.ld}, n[3] = {B, H, S};
    long below = 64;
    bool used[3] = {false, false, false};
    for (int k = 0; k < 3; ++k) {
      int best = -1;
      for (int i = 0; i < 3; ++i)
        if (!used[i] && (best < 0 || n[i] < 2 || (n[best] > 1 && st[i] < st[best]))) best = i;
      used[best] = true;
      if (n[best] < 2) continue;
      if (st[best] < below) { err = std::string("attention_sink: rows of ") + what + " overlap"; return 1; }
      below = st[best] * (n[best] - 1) + below;
    }
  }
  return 0;
}

int set_args(Ctx* c, const sa3k_sink_attn* p, SinkArgs& a, std::string& err) {
  if (!p) { err = "attention_sink: the description is NULL"; return 1; }
  if (p->type != kTypeF16 && p->type != kTypeBF16) { err = "attention_sink: the type must be F16 or BF16"; return 1; }
  if (p->head_dim != 64) { err = "attention_sink: head_dim must be 64"; return 1; }
  if (p->B < 0 || p->Sq < 0 || p->Sk < 0 || p->H < 1 || p->H_kv < 1 || p->H % p->H_kv) {
    err = "attention_sink: need B, Sq, Sk >= 0 and H a positive multiple of H_kv";
    return 1;
  }
  if (p->Sq >= kFar / 2 || p->Sk >= kFar / 2) { err = "attention_sink: Sq and Sk must be below 2^28"; return 1; }
  if ((int64_t)p->B * p->H > 65535) { err = "attention_sink: B * H must be at most 65535"; return 1; }
  if (!(p->scale > 0.f) || !std::isfinite(p->scale)) { err = "attention_sink: scale must be positive"; return 1; }
  if (p->sinks < 0) { err = "attention_sink: sinks must not be negative"; return 1; }
  a.B = p->B; a.H = p->H; a.Hkv = p->H_kv; a.group = p->H / p->H_kv;
  a.Sq = p->Sq; a.Sk = p->Sk;
  a.scale = p->scale;
  a.sl2 = p->scale * 1.4426950408889634f;
  a.left = p->left < 0 || p->left > kFar ? kFar : (int)p->left;
  a.right = p->right < 0 || p->right > kFar ? kFar : (int)p->right;
  a.sinks = (int)std::min<int64_t>(p->sinks, p->Sk);
  a.align_end = p->align_end ? 1 : 0;
  a.q_len = p->q_len;
  a.kv_len = p->kv_len;
  a.err = c->d_err;
  return 0;
}

}  // namespace
}  // namespace sa3k

using namespace sa3k;

extern "C" {

int sa3k_attention_sink_fwd(sa3k_ctx* ctx, const sa3k_sink_attn* p, const sa3k_tensor4* q, const sa3k_tensor4* k,
                            const sa3k_tensor4* v, const sa3k_tensor4* o, float* lse, char* err, int err_len) {
  return api_call(ctx, err, err_len, [&](Ctx* c, std::string& e) {
    SinkArgs a{};
    if (set_args(c, p, a, e)) return 1;
    if (a.B == 0 || a.Sq == 0) return 0;
    if (check_tensor("q", q, a.B, a.H, a.Sq, false, a.q, e) || check_tensor("o", o, a.B, a.H, a.Sq, true, a.o, e)) return 1;
    if (a.Sk > 0 && (check_tensor("k", k, a.B, a.Hkv, a.Sk, false, a.k, e) ||
                     check_tensor("v", v, a.B, a.Hkv, a.Sk, false, a.v, e)))
      return 1;
    a.lse = lse;
    return p->type == kTypeF16 ? forward<__half>(c, a, e) : forward<__nv_bfloat16>(c, a, e);
  });
}

int sa3k_attention_sink_bwd(sa3k_ctx* ctx, const sa3k_sink_attn* p, const sa3k_tensor4* q, const sa3k_tensor4* k,
                            const sa3k_tensor4* v, const sa3k_tensor4* o, const sa3k_tensor4* dO, const float* lse,
                            const sa3k_tensor4* dq, const sa3k_tensor4* dk, const sa3k_tensor4* dv, char* err,
                            int err_len) {
  return api_call(ctx, err, err_len, [&](Ctx* c, std::string& e) {
    SinkArgs a{};
    if (set_args(c, p, a, e)) return 1;
    if ((dk != nullptr) != (dv != nullptr)) { e = "attention_sink: give both dk and dv, or neither"; return 1; }
    if (a.B == 0) return 0;
    if (a.Sq > 0) {
      if (check_tensor("q", q, a.B, a.H, a.Sq, false, a.q, e) || check_tensor("o", o, a.B, a.H, a.Sq, false, a.o, e) ||
          check_tensor("dO", dO, a.B, a.H, a.Sq, false, a.dO, e) || check_tensor("dq", dq, a.B, a.H, a.Sq, true, a.dq, e))
        return 1;
      if (!lse) { e = "attention_sink: the backward needs the forward's lse"; return 1; }
    }
    if (a.Sk > 0) {
      if (check_tensor("k", k, a.B, a.Hkv, a.Sk, false, a.k, e) || check_tensor("v", v, a.B, a.Hkv, a.Sk, false, a.v, e))
        return 1;
      if (dk && (check_tensor("dk", dk, a.B, a.Hkv, a.Sk, true, a.dk, e) ||
                 check_tensor("dv", dv, a.B, a.Hkv, a.Sk, true, a.dv, e)))
        return 1;
    }
    a.lse = const_cast<float*>(lse);
    a.D = static_cast<float*>(scratch_get(c, kSlotSinkD, (size_t)std::max<long>(1, (long)a.B * a.H * a.Sq) * sizeof(float), e));
    if (!a.D) return 1;
    return p->type == kTypeF16 ? backward<__half>(c, a, e) : backward<__nv_bfloat16>(c, a, e);
  });
}

}  // extern "C"
