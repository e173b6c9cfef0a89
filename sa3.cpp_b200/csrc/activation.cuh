// activation.cuh -- the activations of the fused linear and their slopes, in f32.
//
//   silu       z s(z),  s(u) = 1 / (1 + exp(-u))
//   gelu       z Phi(z) = 0.5 z (1 + erf(z / sqrt 2))
//   gelu_tanh  0.5 z (1 + tanh(u)),  u = sqrt(2 / pi) (z + 0.044715 z^3);  0.5 (1 + tanh u) = s(2 u)
// The exponential and the division are the fast f32 forms (a few units in the last place), far
// below the rounding of a 16-bit result.
#pragma once

namespace sa3k {

enum : int { kActNone = 0, kActSilu = 1, kActGelu = 2, kActGeluTanh = 3 };

__device__ __forceinline__ float act_sigmoid(float u) { return __fdividef(1.f, 1.f + __expf(-u)); }

__device__ __forceinline__ float act_tanh_arg(float z) {   // 2 u of the tanh form
  constexpr float c2 = 1.5957691216057308f;                // 2 sqrt(2 / pi)
  return c2 * z * fmaf(0.044715f * z, z, 1.f);
}

__device__ __forceinline__ float act_value(int act, float z) {
  if (act == kActSilu) return z * act_sigmoid(z);
  if (act == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == kActGeluTanh) return z * act_sigmoid(act_tanh_arg(z));
  return z;
}

__device__ __forceinline__ float act_slope(int act, float z) {
  if (act == kActSilu) {
    const float s = act_sigmoid(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (act == kActGelu)
    return fmaf(z * 0.3989422804014327f, __expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
  if (act == kActGeluTanh) {
    const float s = act_sigmoid(act_tanh_arg(z));
    return fmaf(z * s * (1.f - s), 1.5957691216057308f * fmaf(3.f * 0.044715f * z, z, 1.f), s);
  }
  return 1.f;
}

}  // namespace sa3k
