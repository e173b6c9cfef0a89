// attention_sink.h -- arguments of the windowed attention with sink tokens (attention_sink.cu).
#pragma once

#include "ops_api.h"

namespace sa3k {

// One strided [batch][head][row][64] tensor, strides in elements.
struct SinkTensor {
  void* p = nullptr;
  long sb = 0, sh = 0, ld = 0;
};

struct SinkArgs {
  int B, H, Hkv, group;            // group = H / Hkv query heads share a key / value head
  int Sq, Sk;
  float scale, sl2;                // sl2 = scale * log2(e)
  int left, right;                 // INT_MAX / 2 where unbounded
  int sinks;
  int align_end;
  const int* q_len;                // [B] or null
  const int* kv_len;               // [B] or null
  SinkTensor q, k, v, o, dO, dq, dk, dv;
  float* lse;                      // [B][H][Sq], log2 units
  float* D;                        // backward scratch [B][H][Sq]: rowsum(dO o O)
  int* next_item;                  // backward scratch: the dk / dv pass's work counter, zeroed by the dq pass
  int* err;
};

// What one batch entry looks like: its lengths, and the position of query row 0.
struct SinkSeq {
  int qn, kn, pos0;
};
__device__ __forceinline__ SinkSeq sink_seq(const SinkArgs& a, int b) {
  SinkSeq s;
  s.qn = a.q_len ? min(max(a.q_len[b], 0), a.Sq) : a.Sq;
  s.kn = a.kv_len ? min(max(a.kv_len[b], 0), a.Sk) : a.Sk;
  s.pos0 = a.align_end ? s.kn - s.qn : 0;
  return s;
}

// Key j is seen from position p: not past p + right, and within `left` behind p or a sink.
__device__ __forceinline__ bool sink_sees(const SinkArgs& a, const SinkSeq& s, int p, int j) {
  return j < s.kn && j <= p + a.right && (j < a.sinks || j >= p - a.left);
}

// the forward for a few query rows per key / value head (attention_rows.cu)
bool sink_rows_applies(const Ctx* c, const SinkArgs& a);
int sink_rows_forward(Ctx* c, const SinkArgs& a, bool bf16, std::string& err);

}  // namespace sa3k
