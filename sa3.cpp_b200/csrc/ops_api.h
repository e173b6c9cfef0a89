// ops_api.h -- what the transformer-block operators (layernorm.cu, attention_sink.cu, linear_act.cu)
// share: element types, entry-point guards.
#pragma once

#include <cuda_bf16.h>

#include <cstring>
#include <exception>

#include "sa3k_internal.h"

namespace sa3k {

enum : int { kTypeBF16 = 30 };   // ggml's id

// The context's device is current while this lives; the caller's device is put back after it.
struct DeviceScope {
  int prev = -1, dev;
  explicit DeviceScope(int d) : dev(d) {
    if (cudaGetDevice(&prev) == cudaSuccess && prev != dev) cudaSetDevice(dev);
  }
  ~DeviceScope() {
    if (prev >= 0 && prev != dev) cudaSetDevice(prev);
  }
};

inline int api_error(char* err, int len, const char* msg) {
  if (err && len > 0) {
    std::strncpy(err, msg, (size_t)len - 1);
    err[len - 1] = 0;
  }
  return 1;
}

// Body of an entry point: fn(std::string& err) returns 0 or fills err; nothing it throws leaves.
template <class F>
int api_call(sa3k_ctx* ctx, char* err, int len, F&& fn) {
  if (!ctx) return api_error(err, len, "ctx is NULL");
  try {
    DeviceScope scope(ctx->c.device);
    std::string e;
    if (fn(&ctx->c, e) == 0) return 0;
    return api_error(err, len, e.c_str());
  } catch (const std::exception& x) {
    return api_error(err, len, x.what());
  } catch (...) {
    return api_error(err, len, "unknown error");
  }
}

// out0[i] (+)= sum over b of part[b][0][i] and, of two planes, out1[i] (+)= sum over b of part[b][1][i]
// (either may be null), summed in a fixed order (layernorm.cu)
int k_fold_partials(Ctx* c, const float* part, int nblocks, int planes, int cols, float* out0, float* out1, int acc0,
                    int acc1, std::string& err);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 8 consecutive values from / to 16-byte aligned memory
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  uint4 a;
  __half2* h = reinterpret_cast<__half2*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = a;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 a;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = a;
}

}  // namespace sa3k
