// attn_prims.cuh -- device helpers shared by the tcgen05 attention kernels (attention_tc.cu,
// attention_sink.cu): 4-D TMA tiles, tensor-memory stores, 64-wide operand descriptors, waits.
#pragma once

#include "sa3k_common.cuh"

namespace sa3k {

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// max of 64 values held as raw f32 bits (four independent chains of three-input max)
__device__ __forceinline__ float rowmax64(const uint32_t (&v)[64]) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 64; c += 8)
#pragma unroll
    for (int u = 0; u < 4; ++u) m[u] = max3(m[u], __uint_as_float(v[c + 2 * u]), __uint_as_float(v[c + 2 * u + 1]));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// K-major [rows][64] f16 tile (128-byte rows, 128B swizzle): descriptor of the tile, and the
// descriptor at k-step kk (16 wide = 32 bytes further: +2 in the start-address field)
__device__ __forceinline__ uint64_t kdesc0(uint32_t base) { return make_sdesc(base, 16, 1024); }
__device__ __forceinline__ uint64_t kstep(uint64_t d0, int kk) { return d0 + (uint64_t)(2 * kk); }
// the same tile read MN-major (its rows are the reduction index): 16 rows = 2048 bytes per k-step
__device__ __forceinline__ uint64_t mndesc0(uint32_t base) { return make_sdesc(base, 8192, 1024); }
__device__ __forceinline__ uint64_t mnstep(uint64_t d0, int kk) { return d0 + (uint64_t)(128 * kk); }

struct Waiter {
  volatile int* abort_flag;
  int* err;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity, int code) const {
    const uint32_t a = smem_u32(bar);
    if (mbar_try_wait(a, parity)) return true;     // fast path: already complete
    if (*abort_flag) return false;
    const unsigned long long t0 = globaltimer();
    for (uint32_t i = 1;; ++i) {
      if (mbar_try_wait(a, parity)) return true;
      if ((i & 63u) == 0) {
        if (*abort_flag) return false;
        if (globaltimer() - t0 > kWaitLimitNs) {
          record_error(err, code);
          *abort_flag = 1;
          return false;
        }
      }
    }
  }
};

// Four k-steps of one product, issued warp-wide by one elected lane: the operands advance inside, so an
// MMA costs the warp a few instructions (issued one by one, with softmax warps on the same scheduler,
// the issue was slower than the tensor core).  D = A B for acc 0, D += A B otherwise; AS, BS: steps of
// the descriptors per k-step.
template <int AS, int BS>
__device__ __forceinline__ void umma4_ss_w(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.s64 a1, %1, %5;\n\tadd.s64 b1, %2, %6;\n\t"
      "add.s64 a2, a1, %5;\n\tadd.s64 b2, b1, %6;\n\t"
      "add.s64 a3, a2, %5;\n\tadd.s64 b3, b2, %6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "n"(AS), "n"(BS)
      : "memory");
}

// The same with A in tensor memory (packed 16-bit pairs): k-steps at a, a + 8, a + HALF, a + HALF + 8.
template <int HALF, int BS>
__device__ __forceinline__ void umma4_ts_w(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.s32 a1, %1, 8;\n\tadd.s64 b1, %2, %6;\n\t"
      "add.s32 a2, %1, %5;\n\tadd.s64 b2, b1, %6;\n\t"
      "add.s32 a3, a2, 8;\n\tadd.s64 b3, b2, %6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "n"(HALF), "n"(BS)
      : "memory");
}

// A value that is the same in every lane, for the compiler to know it too (uniform registers).
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

}  // namespace sa3k
