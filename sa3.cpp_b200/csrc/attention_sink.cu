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

#include <algorithm>
#include <climits>
#include <cmath>

#include "../../include/sa3k.h"
#include "attn_prims.cuh"
#include "sa3k_common.cuh"

namespace sa3k {
namespace {

// ---------------------------------------------------------------------------- tensor-core tiles
// The kernels below share one shape: tiles of 64 rows x 64 values (8 KB, 128-byte swizzle) stream
// in by TMA, S = Q K^T and its like are formed in tensor memory, threads own one TMEM lane (tile
// row) each, and P / dS go back to tensor memory as packed 16-bit pairs to be the next product's A
// operand.  Several CTAs share an SM and its tensor memory (three of the forward, two of dq; dk / dv has
// one with three sets of buffers), so one CTA's softmax and the start and end of its work run under the
// others' products.  The first tile of a window, the last of a sequence and the tiles at its edges are
// masked; tiles that no row of the CTA sees are never loaded, so the work follows the window and not
// the sequence.
constexpr int kSoftWarps = 8, kSinkThreads = 32 * (kSoftWarps + 2);
constexpr int kTile = 8192;                 // 64 rows x 64 values x 2 bytes

struct SeqMap {       // a tensor map whose (head, row, batch) dimensions are sorted by stride
  CUtensorMap m;
  int h, s, b;        // coordinate (1 .. 3) of each dimension
  int hmul, bmul;     // 0 where the tensor is broadcast over that dimension
};

__device__ __forceinline__ void load_tile(void* dst, const SeqMap& t, uint64_t* bar, int b, int h, int row) {
  const int hc = h * t.hmul, bc = b * t.bmul;
  auto pick = [&](int k) { return t.h == k ? hc : t.s == k ? row : bc; };
  tma_load_4d(dst, &t.m, bar, 0, pick(1), pick(2), pick(3));
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  return pack_f16x2(lo, hi);
}

template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// kind::f16 instruction descriptor: M = 128, N = 64, A K-major, both operands f16 or both bf16
template <bool BF>
__host__ __device__ constexpr uint32_t sink_idesc(int b_mn) {
  return make_idesc_f16(128, 64, 0, b_mn) | (BF ? (1u << 7) | (1u << 10) : 0u);
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// The 64-key tiles that rows at positions [plo, phi] see: the sink tiles [0, ns), then the window's
// [w0, w0 + n - ns).
struct KeyTiles {
  int ns, w0, n;
  __device__ __forceinline__ int tile(int j) const { return j < ns ? j : w0 + (j - ns); }
};
__device__ __forceinline__ KeyTiles key_tiles(const SinkArgs& a, const SinkSeq& s, int plo, int phi) {
  KeyTiles k{0, 0, 0};
  const int hi = min(s.kn, phi + a.right + 1);
  if (hi <= 0 || phi < plo) return k;
  k.ns = uniform((min(a.sinks, hi) + 63) >> 6);
  k.w0 = uniform(max(max(0, plo - a.left) >> 6, k.ns));
  k.n = uniform(k.ns + max(0, ((hi + 63) >> 6) - k.w0));
  return k;
}

// Every row at positions [plo, phi] sees every key of [k0, k0 + 64).
__device__ __forceinline__ bool tile_all_seen(const SinkArgs& a, const SinkSeq& s, int plo, int phi, int k0) {
  return k0 + 64 <= s.kn && k0 + 63 <= plo + a.right && (k0 + 63 < a.sinks || k0 >= phi - a.left);
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; }

// bit c: position p sees key k0 + c
__device__ __forceinline__ uint64_t seen_mask(const SinkArgs& a, const SinkSeq& s, int p, int k0) {
  return low_bits(min(s.kn, p + a.right + 1) - k0) & (low_bits(a.sinks - k0) | ~low_bits(p - a.left - k0));
}

// Rows [from, 64) of a 64-row tile in shared memory become zeros (t of n threads).  What a buffer
// holds behind a sequence's end may be NaN, and 0 x NaN would spoil a product.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int t, int n) {
  for (int i = from * 8 + t; i < 512; i += n) reinterpret_cast<uint4*>(tile)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// A warp's 32 rows of 8 NC values (NC chunks of 16 bytes per lane, its lane's row) to global memory
// by way of shared memory, so that a store instruction writes whole 128- or 64-byte rows instead of
// 16 bytes of 32 rows (measured on the forward's 128-row tiles: 6000 cycles a CTA against 1500).
// `buf`: 32 rows x PITCH bytes of this warp's own; `out`: row 0's first value; rows at or past n stay.
template <int NC, int PITCH = 128>
__device__ __forceinline__ void store_rows(uint8_t* buf, const uint4 (&w)[NC], uint16_t* out, long ld, int n, int lane) {
  // (chunks are swizzled within a row: by the row in rows of 128 bytes, by half of it in rows of 64)
  auto at = [](int r, int q) { return r * PITCH + ((PITCH == 128 ? q ^ (r & 7) : q ^ ((r >> 1) & 3)) << 4); };
#pragma unroll
  for (int q = 0; q < NC; ++q) *reinterpret_cast<uint4*>(buf + at(lane, q)) = w[q];
  __syncwarp();
  constexpr int PER = 32 / NC;       // rows per store
#pragma unroll
  for (int k = 0; k < 32 / PER; ++k) {
    const int r = k * PER + lane / NC, q = lane % NC;
    const uint4 v = *reinterpret_cast<const uint4*>(buf + at(r, q));
    if (r < n) *reinterpret_cast<uint4*>(out + (long)r * ld + 8 * q) = v;
  }
}

// =================================================================================== forward
// CTA: 128 query rows of one (batch entry, head): four softmax warps (a thread per row), and one warp
// that issues loads and products.  Three CTAs share an SM.
// TMEM: S [0, 64), O [64, 128).  smem: Q 16 KB | P 16 KB | 2 x K 8 KB | 2 x V 8 KB | barriers.
// The threads copy S to registers and give its columns back at once, and P goes through shared
// memory, so S of the next tile is formed under this tile's exponentials, and P V under the next
// one's: a tile's chain is the softmax alone (with P over S's columns the products' latency was 40%
// of it).  What then bounds the kernel is the exponentials (16 a clock per SM, 512 clocks a tile) and
// the f32 work around them.  All of them take the MUFU unit: a polynomial for every fourth pair, with the
// clamp and the scaling that keep NaN and give masked scores 0, was slower (36.0 us against 35.6, 100.7 against 98.2).
// Measured per call: 35.6 us for 2 x 24 heads, 2048 rows in a band of 256 with 64 sinks (379
// TFLOP/s), 98.2 us for 24 heads, 8192 causal rows in a window of 1024 (493 TFLOP/s).
constexpr int kFwdThreads = 160;
constexpr int kFwdSmem = 32768 + 4 * kTile + 128 + 1024;

template <bool BF>
__global__ void __launch_bounds__(kFwdThreads, 3)
    sink_fwd_kernel(const __grid_constant__ SeqMap mq, const __grid_constant__ SeqMap mk, const __grid_constant__ SeqMap mv,
                    const __grid_constant__ SinkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sP = smem + 16384;
  uint8_t* sK = smem + 32768;             // [2]
  uint8_t* sV = sK + 2 * kTile;           // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * kTile);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;            // [2]
  uint64_t* v_full = bars + 3;            // [2]
  uint64_t* s_full = bars + 5;            // S of a tile is there
  uint64_t* s_read = bars + 6;            // it is in the threads' registers
  uint64_t* p_full = bars + 7;            // P is in shared memory (and the tile before's P V is done)
  uint64_t* pv_done = bars + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 9);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 128) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 4);
    mbar_init(p_full, 4);
    mbar_init(pv_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&mq.m);
    tma_prefetch_desc(&mk.m);
    tma_prefetch_desc(&mv.m);
  }
  if (warp == 4) {
    __syncwarp();
    tmem_alloc(tmem_slot, 128);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  pdl_trigger();   // (tensor memory is taken: see pdl_trigger)
  const uint32_t tbase = (uint32_t)uniform((int)*tmem_slot);
  pdl_wait();

  const int bh = blockIdx.y, b = bh / a.H, h = bh % a.H, r0 = blockIdx.x * 128;
  const SinkSeq s = sink_seq(a, b);
  const int rows = min(128, s.qn - r0), plo = s.pos0 + r0, phi = plo + rows - 1;
  const KeyTiles kt = rows > 0 ? key_tiles(a, s, plo, phi) : KeyTiles{0, 0, 0};
  const WaiterW<> waitw{abort_flag, a.err};

  if (warp == 4) {
    constexpr uint32_t id_s = sink_idesc<BF>(0), id_o = sink_idesc<BF>(1);
    constexpr uint64_t kSlot = kTile >> 4;
    const uint64_t qd = kdesc0(smem_u32(sQ)), pd = kdesc0(smem_u32(sP)), kd = kdesc0(smem_u32(sK)), vd = mndesc0(smem_u32(sV));
    const int hk = h / a.group;
    auto load = [&](uint8_t* dst, const SeqMap& m, uint64_t* bar, int c) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, kTile);
        load_tile(dst + (c & 1) * kTile, m, bar, b, hk, kt.tile(c) * 64);
      }
      __syncwarp();
    };
    auto scores = [&](int c) {       // S = Q K^T of tile c
      if (!waitw(&k_full[c & 1], (uint32_t)((c >> 1) & 1), kErrTimeoutFull)) return false;
      tc_fence_after();
      const uint64_t k = kd + (c & 1) * kSlot;
      umma4_ss_w<2, 2>(tbase, qd, k, id_s, 0u);
      umma_commit_w(s_full);
      return true;
    };
    bool ok = kt.n > 0;
    if (ok) {
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, 2 * kTile);
        load_tile(sQ, mq, q_full, b, h, r0);
        load_tile(sQ + kTile, mq, q_full, b, h, r0 + 64);
      }
      for (int c = 0; c < min(2, kt.n); ++c) {
        load(sK, mk, &k_full[c], c);
        load(sV, mv, &v_full[c], c);
      }
      ok = waitw(q_full, 0, kErrTimeoutFull) && scores(0);
    }
    for (int c = 0; c < kt.n && ok; ++c) {
      if (!waitw(s_read, (uint32_t)(c & 1), kErrTimeoutOther)) break;
      if (c + 1 < kt.n && !scores(c + 1)) break;
      if (c + 2 < kt.n) load(sK, mk, &k_full[c & 1], c + 2);                       // (S(c) has read its K)
      if (!waitw(p_full, (uint32_t)(c & 1), kErrTimeoutReady)) break;
      if (!waitw(&v_full[c & 1], (uint32_t)((c >> 1) & 1), kErrTimeoutFull)) break;
      tc_fence_after();
      const uint64_t v = vd + (c & 1) * kSlot;
      umma4_ss_w<2, 128>(tbase + 64, pd, v, id_o, c > 0 ? 1u : 0u);
      umma_commit_w(pv_done);
      if (c > 0 && c + 1 < kt.n) load(sV, mv, &v_full[(c + 1) & 1], c + 1);       // (P V(c - 1) had read its V at p_full)
    }
  } else if (rows > 0) {
    const int row = 32 * warp + lane, i = r0 + row, p = plo + row;
    const uint32_t tS = tbase + ((uint32_t)(32 * warp) << 16), tO = tS + 64;
    uint8_t* prow = sP + row * 128;
    // tiles that every row sees whole: sink tiles below fs, window tiles of [f0, f1)
    const int top = min(plo + a.right + 1, s.kn);
    const int fs = max(0, min(a.sinks, top)) >> 6, f0 = (max(0, phi - a.left) + 63) >> 6, f1 = max(f0, top >> 6);
    const uint64_t sc2 = f2(a.sl2, a.sl2);
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int c = 0; c < kt.n; ++c) {
      const int t = kt.tile(c);
      if (!waitw(s_full, (uint32_t)(c & 1), kErrTimeoutAccum)) { ok = false; break; }
      tc_fence_after();
      uint32_t v[64];
      tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
      tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      if (!(t < fs || (t >= f0 && t < f1))) {
        const uint64_t mask = seen_mask(a, s, p, t * 64);
        const uint32_t ml = (uint32_t)mask, mh = (uint32_t)(mask >> 32);
        if (__any_sync(0xffffffffu, ml != 0xffffffffu)) {      // (32 rows' edge often lies in one half)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((ml >> e) & 1u)) v[e] = 0xff800000u;
        }
        if (__any_sync(0xffffffffu, mh != 0xffffffffu)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((mh >> e) & 1u)) v[32 + e] = 0xff800000u;
        }
      }
      const float mx = rowmax64(v) * a.sl2;
      // the exponent's base stays unless the row's maximum grew by more than 2^8: P then stays below
      // 2^8, and O is rescaled rarely
      const bool grow = mx > m_used + 8.f;
      bool waited = c == 0;
      if (__any_sync(0xffffffffu, grow)) {
        float alpha = 1.f;
        if (grow) {
          alpha = m_used == -INFINITY ? 0.f : ex2(m_used - mx);
          m_used = mx;
        }
        l *= alpha;
        if (c > 0) {
          if (!waitw(pv_done, (uint32_t)((c - 1) & 1), kErrTimeoutAccum)) { ok = false; break; }
          waited = true;
          tc_fence_after();
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            uint32_t o[16];
            tmem_ld16(tO + 16 * q, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(tO + 16 * q, o);
          }
          tmem_st_wait();
        }
      }
      const float mb = m_used == -INFINITY ? 0.f : m_used;
      const uint64_t nb2 = f2(-mb, -mb);
      uint64_t ls[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        float x0, x1;
        f2split(ffma2(f2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), sc2, nb2), x0, x1);
        const float p0 = ex2(x0), p1 = ex2(x1);
        ls[e & 1] = fadd2(ls[e & 1], f2(p0, p1));
        v[e] = pack2<BF>(p0, p1);
      }
      float l0, l1, l2, l3;
      f2split(ls[0], l0, l1);
      f2split(ls[1], l2, l3);
      l += (l0 + l1) + (l2 + l3);
      // P's buffer is free once the tile before's P V is done
      if (!waited && !waitw(pv_done, (uint32_t)((c - 1) & 1), kErrTimeoutAccum)) { ok = false; break; }
#pragma unroll
      for (int q = 0; q < 8; ++q)
        *reinterpret_cast<uint4*>(prow + ((q ^ (row & 7)) << 4)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      if (t * 64 + 64 > s.kn && s.kn < a.Sk) {   // values behind the sequence's end (its last tile)
        if (!waitw(&v_full[c & 1], (uint32_t)((c >> 1) & 1), kErrTimeoutFull)) { ok = false; break; }
        zero_rows(sV + (c & 1) * kTile, max(0, s.kn - t * 64), row, 128);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    const bool have = ok && kt.n > 0 && waitw(pv_done, (uint32_t)((kt.n - 1) & 1), kErrTimeoutAccum);
    tc_fence_after();
    const bool empty = m_used == -INFINITY && l == l;   // no visible key (a NaN score stays a NaN)
    const float inv = 1.f / l;
    uint16_t* out = static_cast<uint16_t*>(a.o.p) + (long)b * a.o.sb + (long)h * a.o.sh + (long)(r0 + 32 * warp) * a.o.ld;
    if (have) {
      uint32_t o[64];
      tmem_ld32(tO, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
      tmem_ld32(tO + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
      tmem_ld_wait();
      uint4 w[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = empty ? 0u : pack2<BF>(__uint_as_float(o[8 * q + 2 * e]) * inv, __uint_as_float(o[8 * q + 2 * e + 1]) * inv);
        w[q] = make_uint4(x[0], x[1], x[2], x[3]);
      }
      store_rows<8>(sQ + 4096 * warp, w, out, a.o.ld, rows - 32 * warp, lane);   // (the products have read Q)
    } else if (ok && row < rows) {      // no row sees a key
#pragma unroll
      for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(out + (long)lane * a.o.ld + 8 * q) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (ok && a.lse && row < rows) a.lse[(long)bh * a.Sq + i] = empty ? -INFINITY : m_used + log2f(l);
  }
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tbase, 128);
  }
}

// ======================================================================================== dq
// CTA: 128 query rows of one (batch entry, head); both warpgroups hold all of them and take 32 of
// a tile's 64 keys each.  The threads copy S and dP to registers and give their columns back at
// once, so the next tile's products run under this tile's exponentials; dS has columns of its own.
// Measured: 49 us for 4 x 24 heads, 1088 rows in a band of 256 with 64 sinks, 60 us for 3 x 24 heads of
// 2047 ragged rows in a window of 512 (two persistent CTAs per SM over all tiles took 52 and 69).
// TMEM: S [0, 64), dP [64, 128), dQ [128, 192), dS in two buffers of 32 columns at 192 and 224.
constexpr int kDqStages = 3;
constexpr int kDqSmem = 49152 + kDqStages * 2 * kTile + 256 + 1024;

template <bool BF>
__global__ void __launch_bounds__(kSinkThreads, 2)
    sink_dq_kernel(const __grid_constant__ SeqMap mq, const __grid_constant__ SeqMap mdo, const __grid_constant__ SeqMap mo,
                   const __grid_constant__ SeqMap mk, const __grid_constant__ SeqMap mv, const __grid_constant__ SinkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                   // Q 16 KB | dO 16 KB | O 16 KB
  uint8_t* sKV = smem + 49152;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + kDqStages * 2 * kTile);
  uint64_t* q_full = bars;
  uint64_t* kv_full = q_full + 1;
  uint64_t* kv_empty = kv_full + kDqStages;
  uint64_t* s_full = kv_empty + kDqStages;
  uint64_t* s_read = s_full + 1;
  uint64_t* ds_full = s_read + 1;       // [2] per dS buffer: with one barrier, the next tile's phase could
  uint64_t* ds_free = ds_full + 2;      // [2]   end before the issuing warp has seen this one's
  uint64_t* acc_full = ds_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == kSoftWarps && lane == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kDqStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, kSoftWarps);
    mbar_init(&ds_full[0], kSoftWarps);
    mbar_init(&ds_full[1], kSoftWarps);
    mbar_init(&ds_free[0], 1);
    mbar_init(&ds_free[1], 1);
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&mq.m);
    tma_prefetch_desc(&mdo.m);
    tma_prefetch_desc(&mo.m);
    tma_prefetch_desc(&mk.m);
    tma_prefetch_desc(&mv.m);
  }
  if (warp == kSoftWarps + 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  pdl_trigger();   // (tensor memory is taken: see pdl_trigger)
  const uint32_t tbase = (uint32_t)uniform((int)*tmem_slot);
  pdl_wait();

  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.next_item = 0;     // for the dk / dv pass
  const int bh = blockIdx.y, b = bh / a.H, h = bh % a.H, r0 = blockIdx.x * 128;
  const SinkSeq s = sink_seq(a, b);
  const int rows = min(128, s.qn - r0), plo = s.pos0 + r0, phi = plo + rows - 1;
  const KeyTiles kt = rows > 0 ? key_tiles(a, s, plo, phi) : KeyTiles{0, 0, 0};
  const Waiter wait{abort_flag, a.err};
  const WaiterW<> waitw{abort_flag, a.err};

  if (warp == kSoftWarps) {
    if (lane == 0 && rows > 0) {
      mbar_arrive_expect_tx(q_full, 6 * kTile);
      for (int g = 0; g < 2; ++g) {
        load_tile(sQ + kTile * g, mq, q_full, b, h, r0 + 64 * g);
        load_tile(sQ + 2 * kTile + kTile * g, mdo, q_full, b, h, r0 + 64 * g);
        load_tile(sQ + 4 * kTile + kTile * g, mo, q_full, b, h, r0 + 64 * g);
      }
      for (int j = 0; j < kt.n; ++j) {
        const int st = j % kDqStages;
        if (j >= kDqStages && !wait(&kv_empty[st], (uint32_t)((j / kDqStages) & 1) ^ 1u, kErrTimeoutEmpty)) break;
        uint8_t* p = sKV + st * 2 * kTile;
        mbar_arrive_expect_tx(&kv_full[st], 2 * kTile);
        load_tile(p, mk, &kv_full[st], b, h / a.group, kt.tile(j) * 64);
        load_tile(p + kTile, mv, &kv_full[st], b, h / a.group, kt.tile(j) * 64);
      }
    }
  } else if (warp == kSoftWarps + 1) {
    constexpr uint32_t id_s = sink_idesc<BF>(0), id_g = sink_idesc<BF>(1);
    const uint64_t qd = kdesc0(smem_u32(sQ)), dd = kdesc0(smem_u32(sQ + 2 * kTile));
    bool ok = kt.n > 0 && waitw(q_full, 0, kErrTimeoutFull);
    auto grad = [&](int j) {     // dQ += dS K of tile j
      if (!waitw(&ds_full[j & 1], (uint32_t)((j >> 1) & 1), kErrTimeoutReady)) return false;
      tc_fence_after();
      const uint64_t kmn = mndesc0(smem_u32(sKV + (j % kDqStages) * 2 * kTile));
      umma4_ts_w<16, 128>(tbase + 128, tbase + 192 + 32 * (j & 1), kmn, id_g, j > 0 ? 1u : 0u);
      umma_commit_w(&ds_free[j & 1]);
      umma_commit_w(&kv_empty[j % kDqStages]);
      return true;
    };
    for (int j = 0; j < kt.n && ok; ++j) {
      const int st = j % kDqStages;
      if (!waitw(&kv_full[st], (uint32_t)((j / kDqStages) & 1), kErrTimeoutFull)) { ok = false; break; }
      if (j > 0 && !waitw(s_read, (uint32_t)((j - 1) & 1), kErrTimeoutOther)) { ok = false; break; }
      tc_fence_after();
      const uint64_t kd = kdesc0(smem_u32(sKV + st * 2 * kTile)), vd = kdesc0(smem_u32(sKV + st * 2 * kTile + kTile));
      umma4_ss_w<2, 2>(tbase, qd, kd, id_s, 0u);
      umma4_ss_w<2, 2>(tbase + 64, dd, vd, id_s, 0u);
      umma_commit_w(s_full);
      if (j > 0) ok = grad(j - 1);
    }
    if (ok) ok = grad(kt.n - 1);
    if (ok) umma_commit_w(acc_full);
  } else if (rows > 0) {
    const int g = warp >> 2, quarter = warp & 3, row = 32 * quarter + lane, i = r0 + row, p = plo + row;
    const uint32_t lane_off = (uint32_t)(32 * quarter) << 16;
    const uint32_t tS = tbase + lane_off + 32 * g, tP = tS + 64;
    const bool mine = row < rows;
    float lse = INFINITY, D = 0.f;
    if (mine) {
      lse = a.lse[(long)bh * a.Sq + i];
      if (lse == -INFINITY) lse = INFINITY;      // a row that sees nothing: P = 0
    }
    bool ok = waitw(q_full, 0, kErrTimeoutFull);
    if (ok) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int off = row * 128 + ((q ^ (row & 7)) << 4);
        const uint4 x = *reinterpret_cast<const uint4*>(sQ + 2 * kTile + off), y = *reinterpret_cast<const uint4*>(sQ + 4 * kTile + off);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 u = unpack2<BF>(xs[e]), w = unpack2<BF>(ys[e]);
          D = fmaf(u.x, w.x, D);
          D = fmaf(u.y, w.y, D);
        }
      }
      if (g == 0 && mine) a.D[(long)bh * a.Sq + i] = D;
    }
    const uint64_t sc2 = f2(a.sl2, a.sl2), nl2 = f2(-lse, -lse), nd2 = f2(-D, -D);
    for (int j = 0; j < kt.n && ok; ++j) {
      const int t = kt.tile(j);
      if (!waitw(s_full, (uint32_t)(j & 1), kErrTimeoutAccum)) { ok = false; break; }
      tc_fence_after();
      uint32_t sv[32], pv[32];
      tmem_ld32(tS, sv);
      tmem_ld32(tP, pv);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      uint32_t mask = 0xffffffffu;
      const bool edge = !tile_all_seen(a, s, plo, phi, t * 64);
      if (edge) mask = (uint32_t)(seen_mask(a, s, p, t * 64) >> (32 * g));
      uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x0, x1, d0, d1;
        f2split(ffma2(f2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, nl2), x0, x1);
        const float p0 = ex2(x0), p1 = ex2(x1);
        f2split(fmul2(f2(p0, p1), fadd2(f2(__uint_as_float(pv[2 * e]), __uint_as_float(pv[2 * e + 1])), nd2)), d0, d1);
        if (edge) {
          if (!((mask >> (2 * e)) & 1u)) d0 = 0.f;
          if (!((mask >> (2 * e + 1)) & 1u)) d1 = 0.f;
        }
        pk[e] = pack2<BF>(d0, d1);
      }
      if (j >= 2 && !waitw(&ds_free[j & 1], (uint32_t)(((j >> 1) - 1) & 1), kErrTimeoutOther)) { ok = false; break; }
      tc_fence_after();
      tmem_st16(tbase + lane_off + 192 + 32 * (j & 1) + 16 * g, pk);
      if (t * 64 + 64 > s.kn && s.kn < a.Sk) {   // keys behind the sequence's end
        const int st = j % kDqStages;
        if (!waitw(&kv_full[st], (uint32_t)((j / kDqStages) & 1), kErrTimeoutFull)) { ok = false; break; }
        zero_rows(sKV + st * 2 * kTile, max(0, s.kn - t * 64), (int)threadIdx.x, 32 * kSoftWarps);
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[j & 1]);
    }
    const bool have = ok && kt.n > 0 && waitw(acc_full, 0, kErrTimeoutAccum);
    tc_fence_after();
    uint32_t o[32];
    if (have) {
      tmem_ld32(tbase + lane_off + 128 + 32 * g, o);
      tmem_ld_wait();
    }
    uint16_t* out = static_cast<uint16_t*>(a.dq.p) + (long)b * a.dq.sb + (long)h * a.dq.sh + (long)(r0 + 32 * quarter) * a.dq.ld + 32 * g;
    if (have) {
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = pack2<BF>(__uint_as_float(o[8 * q + 2 * e]) * a.scale, __uint_as_float(o[8 * q + 2 * e + 1]) * a.scale);
        w[q] = make_uint4(x[0], x[1], x[2], x[3]);
      }
      // (the products have read Q and dO: 32 KB for the 8 warps' rows)
      store_rows<4>(sQ + 4096 * warp, w, out, a.dq.ld, rows - 32 * quarter, lane);
    } else if (ok && mine) {      // no row sees a key
#pragma unroll
      for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(out + (long)lane * a.dq.ld + 8 * q) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __syncthreads();
  if (warp == kSoftWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tbase, 256);
  }
}

// ==================================================================================== dk, dv
// Persistent, one CTA per SM: an item is 128 keys of one (batch entry, key / value head); the 64-row
// query tiles that see them, of every query head of the group, stream past, and the tiles of one item
// after the other form one stream of steps.  16 softmax warps in two sets take alternate steps (in a
// set a thread owns a key row and 32 of the step's 64 query columns), and there are three buffers for
// S^T and dP^T, so a set finds its next scores ready: with one CTA of 8 warps and one buffer twice per
// SM every step waited for four products in series (1450 clocks a step and SM, then 700; 4 x 24 heads,
// 1088 rows in a band of 256 with 64 sinks: 80 us then, 66 since scores and gradients have an issuing
// warp each).
// Items are handed out by a counter, heaviest first (those with sinks are seen by every later query).
// TMEM: buffer u < 3 at 128 u: S^T [0, 64), dP^T [64, 128) (P^T, dS^T of columns 32 g .. overwrite the
// first 16 columns of their own halves); dV at 384, dK at 448.
// smem: 2 x (K 16 KB, V 16 KB) | 6 x (Q 8 KB, dO 8 KB) | 16 x 2 KB output rows | 16 x lse, D | items | barriers
constexpr int kDkvSets = 2, kDkvStages = 6, kDkvItems = 4;
constexpr int kDkvWarps = 8 * kDkvSets, kDkvThreads = 32 * (kDkvWarps + 3);
constexpr int kDkvSmem = 65536 + kDkvStages * 2 * kTile + kDkvWarps * (2048 + 256) + 256 + 512 + 1024;

struct DkvItem {      // n > 0 steps: query tiles [qt0, qt1) of each of the group's heads; n < 0: no more items
  int b, hk, k0, keys, qt0, qt1, n, pos0, qn, kn;
};

template <bool BF>
__global__ void __launch_bounds__(kDkvThreads, 1)
    sink_dkdv_kernel(const __grid_constant__ SeqMap mk, const __grid_constant__ SeqMap mv, const __grid_constant__ SeqMap mq,
                     const __grid_constant__ SeqMap mdo, const __grid_constant__ SinkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sKV = smem;                                  // [2] K | V
  uint8_t* sQd = smem + 65536;                          // [kDkvStages] Q | dO
  uint8_t* sOut = sQd + kDkvStages * 2 * kTile;         // [warps][32 rows x 64 bytes]
  float* s_ld = reinterpret_cast<float*>(sOut + kDkvWarps * 2048);          // [warps][16 column pairs][lse 2 | D 2]
  DkvItem* items = reinterpret_cast<DkvItem*>(s_ld + 64 * kDkvWarps);       // [kDkvItems]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(items) + 256);
  uint64_t* kv_full = bars;                             // [2]
  uint64_t* kv_empty = kv_full + 2;                     // [2] the item's last scores are done
  uint64_t* q_full = kv_empty + 2;
  uint64_t* q_empty = q_full + kDkvStages;              // dV and dK of the slot's tile are done
  // scores of a step are there: [6], a barrier per buffer and set.  With one per buffer a set would look at
  // every second phase only, and could not tell the next phase but one from the last it saw
  uint64_t* s_full = q_empty + kDkvStages;
  uint64_t* ds_full = s_full + 3 * kDkvSets;            // [3]
  uint64_t* g_done = ds_full + 3;                       // [3] dV and dK of the buffer's step are done
  uint64_t* acc_full = g_done + 3;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* item_full = acc_empty + 1;                  // [kDkvItems]
  uint64_t* item_empty = item_full + kDkvItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(item_empty + kDkvItems);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == kDkvWarps && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < kDkvStages; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 3 * kDkvSets; ++i) mbar_init(&s_full[i], 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&ds_full[i], 8);
      mbar_init(&g_done[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, kDkvWarps);
    for (int i = 0; i < kDkvItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kDkvWarps + 2);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&mk.m);
    tma_prefetch_desc(&mv.m);
    tma_prefetch_desc(&mq.m);
    tma_prefetch_desc(&mdo.m);
  }
  if (warp == kDkvWarps + 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  pdl_trigger();   // (tensor memory is taken: see pdl_trigger)
  const uint32_t tbase = (uint32_t)uniform((int)*tmem_slot);
  pdl_wait();
  const Waiter wait{abort_flag, a.err};
  const WaiterW<> waitw{abort_flag, a.err};

  if (warp == kDkvWarps) {
    const int nbh = a.B * a.Hkv, ktiles = (a.Sk + 127) / 128, nitems = nbh * ktiles;
    int ni = 0, t = 0, L = blockIdx.x;      // items handed on, steps, the item's number
    bool ok = true;
    while (ok) {
      DkvItem it;
      it.n = -1;
      if (L < nitems) {
        const int bh = L % nbh;
        it.b = bh / a.Hkv;
        it.hk = bh % a.Hkv;
        it.k0 = L / nbh * 128;
        const SinkSeq s = sink_seq(a, it.b);
        it.pos0 = s.pos0;
        it.qn = s.qn;
        it.kn = s.kn;
        it.keys = min(128, s.kn - it.k0);
        const int lo = max(0, it.k0 - a.right - s.pos0);
        const int hi = it.k0 < a.sinks ? s.qn : min(s.qn, it.k0 + it.keys + a.left - s.pos0);
        it.qt0 = lo >> 6;
        it.qt1 = lo < hi ? (hi + 63) >> 6 : it.qt0;
        it.n = it.keys > 0 ? (it.qt1 - it.qt0) * a.group : 0;
        for (int i = lane; it.n == 0 && i < it.keys * 8; i += 32) {     // keys that no query sees
          const long r = it.k0 + (i >> 3);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const SinkTensor& out = u ? a.dk : a.dv;
            uint16_t* p = static_cast<uint16_t*>(out.p) + (long)it.b * out.sb + (long)it.hk * out.sh + r * out.ld + 8 * (i & 7);
            *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
      if (it.n != 0 && lane == 0) {
        const int slot = ni % kDkvItems, kb = ni & 1;
        ok = ni < kDkvItems || wait(&item_empty[slot], (uint32_t)((ni / kDkvItems - 1) & 1), kErrTimeoutEmpty);
        if (ok) {
          items[slot] = it;
          mbar_arrive(&item_full[slot]);
          if (it.n > 0) ok = ni < 2 || wait(&kv_empty[kb], (uint32_t)((ni / 2 - 1) & 1), kErrTimeoutEmpty);
        }
        if (ok && it.n > 0) {
          uint8_t* kv = sKV + 32768 * kb;
          mbar_arrive_expect_tx(&kv_full[kb], 4 * kTile);
          for (int g = 0; g < 2; ++g) {
            load_tile(kv + kTile * g, mk, &kv_full[kb], it.b, it.hk, it.k0 + 64 * g);
            load_tile(kv + 2 * kTile + kTile * g, mv, &kv_full[kb], it.b, it.hk, it.k0 + 64 * g);
          }
          for (int h = it.hk * a.group; h < (it.hk + 1) * a.group && ok; ++h)
            for (int q = it.qt0; q < it.qt1; ++q, ++t) {
              const int st = t % kDkvStages;
              if (t >= kDkvStages && !wait(&q_empty[st], (uint32_t)((t / kDkvStages - 1) & 1), kErrTimeoutEmpty)) { ok = false; break; }
              uint8_t* p = sQd + st * 2 * kTile;
              mbar_arrive_expect_tx(&q_full[st], 2 * kTile);
              load_tile(p, mq, &q_full[st], it.b, h, q * 64);
              load_tile(p + kTile, mdo, &q_full[st], it.b, h, q * 64);
            }
        }
      }
      if (it.n < 0) break;
      if (it.n > 0) ++ni;
      if (lane == 0) L = (int)gridDim.x + atomicAdd(a.next_item, 1);
      L = __shfl_sync(0xffffffffu, L, 0);
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
  } else if (warp >= kDkvWarps + 1) {
    // Two warps issue the products, one the scores (up to three steps ahead), one the gradients: the
    // waits and the issue of all 16 products of a step in one warp took 1700 clocks, more than the softmax.
    const bool grads = warp == kDkvWarps + 2;
    int st = 0, u = 0, f = 0;                // ring slot, buffer and barrier of the step, with the parity of their use
    uint32_t st_ph = 0, u_ph = 0;
    auto step = [&]() {
      if (++st == kDkvStages) { st = 0; st_ph ^= 1u; }
      if (++u == 3) { u = 0; u_ph ^= 1u; }
      if (++f == 3 * kDkvSets) f = 0;
    };
    bool ok = true;
    int t = 0;
    for (int item = 0; ok; ++item) {
      const int slot = item % kDkvItems;
      if (!waitw(&item_full[slot], (uint32_t)((item / kDkvItems) & 1), kErrTimeoutOther)) break;
      const int n = uniform(items[slot].n);
      if (n < 0) break;
      if (!grads) {              // S^T = K Q^T and dP^T = V dO^T
        constexpr uint32_t id_s = sink_idesc<BF>(0);
        const int kb = item & 1;
        const uint32_t ka = smem_u32(sKV) + 32768 * kb;
        const uint64_t kd = kdesc0(ka), vd = kdesc0(ka + 2 * kTile);
        ok = waitw(&kv_full[kb], (uint32_t)((item >> 1) & 1), kErrTimeoutFull);
        for (int j = 0; j < n && ok; ++j, ++t) {
          if (t >= 3 && !(ok = waitw(&g_done[u], u_ph ^ 1u, kErrTimeoutOther))) break;
          if (!(ok = waitw(&q_full[st], st_ph, kErrTimeoutFull))) break;
          tc_fence_after();
          const uint32_t qa = smem_u32(sQd) + st * 2 * kTile, tS = tbase + 128 * u;
          umma4_ss_w<2, 2>(tS, kd, kdesc0(qa), id_s, 0u);
          umma4_ss_w<2, 2>(tS + 64, vd, kdesc0(qa + kTile), id_s, 0u);
          umma_commit_w(&s_full[f]);
          step();
        }
        if (ok) umma_commit_w(&kv_empty[kb]);
      } else {
        constexpr uint32_t id_g = sink_idesc<BF>(1);
        for (int j = 0; j < n && ok; ++j) {
          if (!(ok = waitw(&ds_full[u], u_ph, kErrTimeoutReady))) break;
          if (j == 0 && item > 0 && !(ok = waitw(acc_empty, (uint32_t)((item - 1) & 1), kErrTimeoutOther))) break;
          tc_fence_after();
          const uint32_t qa = smem_u32(sQd) + st * 2 * kTile, tS = tbase + 128 * u, acc = j > 0 ? 1u : 0u;
          umma4_ts_w<32, 128>(tbase + 384, tS, mndesc0(qa + kTile), id_g, acc);         // dV += P^T dO
          umma4_ts_w<32, 128>(tbase + 448, tS + 64, mndesc0(qa), id_g, acc);            // dK += dS^T Q
          umma_commit_w(&g_done[u]);
          umma_commit_w(&q_empty[st]);
          step();
        }
        if (ok) umma_commit_w(acc_full);
      }
      if (lane == 0) mbar_arrive(&item_empty[slot]);
    }
  } else {
    const int set = warp >> 3, g = (warp >> 2) & 1, wg = warp >> 2, quarter = warp & 3, row = 32 * quarter + lane;
    const uint32_t lane_off = (uint32_t)(32 * quarter) << 16;
    const uint64_t sc2 = f2(a.sl2, a.sl2);
    uint8_t* stg = sOut + warp * 2048;
    float* ldb = s_ld + 64 * warp;
    bool ok = true;
    int t0 = 0;                                 // the item's first step
    for (int item = 0; ok; ++item) {
      if (!waitw(&item_full[item % kDkvItems], (uint32_t)((item / kDkvItems) & 1), kErrTimeoutOther)) break;
      const DkvItem& it = items[item % kDkvItems];
      if (it.n < 0) break;
      const int k0 = it.k0, kj = k0 + row, qn = it.qn, pos0 = it.pos0, n = it.n, qt0 = it.qt0, qt1 = it.qt1;
      // rows of the item and their window: query tiles at positions [e0, e1) see every key of the item
      const bool whole = k0 + 128 <= it.kn, inside = kj < it.kn;
      const int e0 = k0 + 127 - a.right, e1 = k0 + 127 < a.sinks ? INT_MAX : k0 + a.left - 62;
      // lane c holds the lse and the D of the group's column c, fetched one of the set's steps ahead
      auto fetch = [&](int h, int q) {
        const int i = q * 64 + 32 * g + lane;
        float2 v = make_float2(INFINITY, 0.f);
        if (i < qn) {
          const long r = ((long)it.b * a.H + h) * a.Sq + i;
          v = make_float2(a.lse[r], a.D[r]);        // (not looked at before its step: the loads stay in flight)
        }
        return v;
      };
      int j = (t0 & 1) == set ? 0 : 1;          // the set's first step of the item
      int h = it.hk * a.group, q = qt0 + j;
      auto wrap = [&]() {
        while (q >= qt1) {
          q -= qt1 - qt0;
          ++h;
        }
      };
      wrap();
      float2 next = j < n ? fetch(h, q) : make_float2(0.f, 0.f);
      for (; j < n && ok; j += 2) {
        const int t = t0 + j, u = t % 3, q0 = q * 64, pq = pos0 + q0;
        __syncwarp();                            // the step before's values have been read
        ldb[4 * (lane >> 1) + (lane & 1)] = next.x == -INFINITY ? INFINITY : next.x;      // a row that sees nothing: P = 0
        ldb[4 * (lane >> 1) + 2 + (lane & 1)] = next.y;
        q += 2;
        wrap();
        if (j + 2 < n) next = fetch(h, q);
        __syncwarp();
        constexpr int F = 3 * kDkvSets;
        if (!waitw(&s_full[t % F], (uint32_t)((t / F) & 1), kErrTimeoutAccum)) { ok = false; break; }
        tc_fence_after();
        // queries of the tile that see key kj: position from kj - right to kj + left (any, for a sink)
        const bool edge = !whole || q0 + 64 > qn || pq < e0 || pq >= e1;
        uint32_t mask = 0xffffffffu;
        if (edge) {
          uint64_t m = low_bits(qn - q0) & ~low_bits(kj - a.right - pq);
          if (kj >= a.sinks) m &= low_bits(kj + a.left - pq + 1);
          mask = inside ? (uint32_t)(m >> (32 * g)) : 0u;
        }
        const bool some = edge && __any_sync(0xffffffffu, mask != 0xffffffffu);
        const float4* ld4 = reinterpret_cast<const float4*>(ldb);
        const uint32_t tS = tbase + 128 * u + lane_off + 32 * g, tP = tS + 64;
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t sv[16], pv[16], pk[8], dk[8];
          tmem_ld16(tS + 16 * hf, sv);
          tmem_ld16(tP + 16 * hf, pv);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 w4 = ld4[8 * hf + e];     // lse and D of two queries, one broadcast read
            float x0, x1, d0, d1;
            f2split(ffma2(f2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sc2, f2(-w4.x, -w4.y)), x0, x1);
            float p0 = ex2(x0), p1 = ex2(x1);
            f2split(fmul2(f2(p0, p1), fadd2(f2(__uint_as_float(pv[2 * e]), __uint_as_float(pv[2 * e + 1])), f2(-w4.z, -w4.w))),
                    d0, d1);
            if (some) {
              const uint32_t mm = mask >> (16 * hf);
              if (!((mm >> (2 * e)) & 1u)) p0 = d0 = 0.f;
              if (!((mm >> (2 * e + 1)) & 1u)) p1 = d1 = 0.f;
            }
            pk[e] = pack2<BF>(p0, p1);
            dk[e] = pack2<BF>(d0, d1);
          }
          tmem_st8(tS + 8 * hf, pk);      // (over the columns that this thread has read)
          tmem_st8(tP + 8 * hf, dk);
        }
        if (q0 + 64 > qn && qn < a.Sq) {   // query rows behind the sequence's end
          const int st = t % kDkvStages;
          if (!waitw(&q_full[st], (uint32_t)((t / kDkvStages) & 1), kErrTimeoutFull)) { ok = false; break; }
          zero_rows(sQd + st * 2 * kTile, qn - q0, (int)threadIdx.x & 255, 256);
          zero_rows(sQd + st * 2 * kTile + kTile, qn - q0, (int)threadIdx.x & 255, 256);
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[u]);
      }
      // the item's results: warpgroups 0, 1 take dV's columns 32 wg .., 2, 3 dK's
      if (!ok || !waitw(acc_full, (uint32_t)(item & 1), kErrTimeoutAccum)) break;
      t0 += n;
      tc_fence_after();
      uint32_t o[32];
      tmem_ld32(tbase + 384 + 32 * wg + lane_off, o);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
      const SinkTensor& out = wg < 2 ? a.dv : a.dk;
      const float mul = wg < 2 ? 1.f : a.scale;
      uint4 w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = pack2<BF>(__uint_as_float(o[8 * c + 2 * e]) * mul, __uint_as_float(o[8 * c + 2 * e + 1]) * mul);
        w[c] = make_uint4(x[0], x[1], x[2], x[3]);
      }
      store_rows<4, 64>(stg, w,
                        static_cast<uint16_t*>(out.p) + (long)it.b * out.sb + (long)it.hk * out.sh +
                            (long)(it.k0 + 32 * quarter) * out.ld + 32 * (wg & 1),
                        out.ld, it.keys - 32 * quarter, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[item % kDkvItems]);
    }
  }
  __syncthreads();
  if (warp == kDkvWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// Tensor map of 64-row tiles over a strided tensor; its head, row and batch dimensions go in by
// growing stride.
int make_seq_map(SeqMap* t, bool bf, const SinkTensor& x, int B, int H, int S, std::string& err) {
  PFN_encodeTiled enc = encode_tiled_fn(err);
  if (!enc) return 1;
  struct Dim { long stride, n; int which; } d[3] = {{x.sh, H, 0}, {x.ld, S, 1}, {x.sb, B, 2}};
  t->hmul = t->bmul = 1;
  if (d[0].n < 2 || x.sh == 0) { d[0].n = 1; t->hmul = 0; }
  if (d[2].n < 2 || x.sb == 0) { d[2].n = 1; t->bmul = 0; }
  std::stable_sort(d, d + 3, [](const Dim& p, const Dim& q) {
    if ((p.n > 1) != (q.n > 1)) return p.n > 1;
    return p.stride < q.stride;
  });
  cuuint64_t dims[4] = {64, 1, 1, 1}, strides[3];
  cuuint32_t box[4] = {64, 1, 1, 1}, estr[4] = {1, 1, 1, 1};
  long below = 64;
  for (int k = 0; k < 3; ++k) {
    const long st = d[k].n > 1 ? d[k].stride : below;    // (a dimension of one entry: any valid stride)
    dims[k + 1] = (cuuint64_t)d[k].n;
    strides[k] = (cuuint64_t)st * 2;
    (d[k].which == 0 ? t->h : d[k].which == 1 ? t->s : t->b) = k + 1;
    if (d[k].which == 1) box[k + 1] = 64;
    below = st * d[k].n;
  }
  const CUresult r = enc(&t->m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, x.p, dims, strides,
                         box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    err = "attention_sink: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")";
    return 1;
  }
  return 0;
}

template <bool BF>
int forward(Ctx* c, const SinkArgs& a, std::string& err) {
  if (sink_rows_applies(c, a)) return sink_rows_forward(c, a, BF, err);
  // (a stand-in key tensor for a forward without keys: its map is never loaded from)
  const bool nokeys = a.Sk == 0;
  SeqMap mq, mk, mv;
  if (make_seq_map(&mq, BF, a.q, a.B, a.H, a.Sq, err) ||
      make_seq_map(&mk, BF, nokeys ? a.q : a.k, a.B, nokeys ? a.H : a.Hkv, nokeys ? a.Sq : a.Sk, err) ||
      make_seq_map(&mv, BF, nokeys ? a.q : a.v, a.B, nokeys ? a.H : a.Hkv, nokeys ? a.Sq : a.Sk, err))
    return 1;
  auto kern = sink_fwd_kernel<BF>;
  if (smem_attr(reinterpret_cast<const void*>(kern), kFwdSmem, c->device, "attention_sink smem attribute", err)) return 1;
  ProfScope prof_(c, "attn_sink.fwd");
  launch_pdl(c, kern, dim3((unsigned)((a.Sq + 127) / 128), (unsigned)(a.B * a.H)), dim3(kFwdThreads), (size_t)kFwdSmem, mq, mk,
             mv, a);
  return check_launch("attention with sinks, forward", err);
}

template <bool BF>
int backward(Ctx* c, const SinkArgs& a, std::string& err) {
  const bool noq = a.Sq == 0, nokeys = a.Sk == 0;
  if (noq && nokeys) return 0;
  SeqMap mq, mdo, mo, mk, mv;
  const SinkTensor &to = noq ? a.k : a.o;
  const SinkTensor &tq = noq ? a.k : a.q, &td = noq ? a.k : a.dO, &tk = nokeys ? a.q : a.k, &tv = nokeys ? a.q : a.v;
  const int hq = noq ? a.Hkv : a.H, sq = noq ? a.Sk : a.Sq, hk = nokeys ? a.H : a.Hkv, sk = nokeys ? a.Sq : a.Sk;
  if (make_seq_map(&mq, BF, tq, a.B, hq, sq, err) || make_seq_map(&mdo, BF, td, a.B, hq, sq, err) ||
      make_seq_map(&mo, BF, to, a.B, hq, sq, err) ||
      make_seq_map(&mk, BF, tk, a.B, hk, sk, err) || make_seq_map(&mv, BF, tv, a.B, hk, sk, err))
    return 1;
  if (!noq) {
    auto kern = sink_dq_kernel<BF>;
    if (smem_attr(reinterpret_cast<const void*>(kern), kDqSmem, c->device, "attention_sink smem attribute", err)) return 1;
    ProfScope prof_(c, "attn_sink.dq");
    launch_pdl(c, kern, dim3((unsigned)((a.Sq + 127) / 128), (unsigned)(a.B * a.H)), dim3(kSinkThreads), (size_t)kDqSmem, mq,
               mdo, mo, mk, mv, a);
    if (check_launch("attention with sinks, dq", err)) return 1;
  }
  if (!a.dk.p || nokeys) return 0;
  auto kern = sink_dkdv_kernel<BF>;
  if (smem_attr(reinterpret_cast<const void*>(kern), kDkvSmem, c->device, "attention_sink smem attribute", err)) return 1;
  if (noq && cudaMemsetAsync(a.next_item, 0, sizeof(int), c->stream) != cudaSuccess) return check_launch("attention_sink memset", err);
  const long items = (long)a.B * a.Hkv * ((a.Sk + 127) / 128);
  ProfScope prof_(c, "attn_sink.dkdv");
  launch_pdl(c, kern, dim3((unsigned)std::min<long>(items, (long)c->sm_count)), dim3(kDkvThreads), (size_t)kDkvSmem, mk, mv, mq,
             mdo, a);
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
  // the dimensions have to nest: by growing stride, each holds the extent of those below it (an input
  // may be broadcast over heads or batch with stride 0)
  long st[3] = {d.sh, d.ld, d.sb}, n[3] = {H, S, B};
  long below = 64;
  bool used[3] = {false, false, false};
  for (int k = 0; k < 3; ++k) {
    int best = -1;
    for (int i = 0; i < 3; ++i)
      if (!used[i] && n[i] > 1 && (best < 0 || st[i] < st[best])) best = i;
    if (best < 0) break;
    used[best] = true;
    if (!out && best != 1 && st[best] == 0) continue;
    if (st[best] < below) { err = std::string("attention_sink: rows of ") + what + " overlap"; return 1; }
    below = st[best] * (n[best] - 1) + below;
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
  if ((int64_t)p->B * p->H * ((p->Sk + 127) / 128) >= (1ll << 31)) {
    err = "attention_sink: too many key tiles for one launch";
    return 1;
  }
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
    return p->type == kTypeF16 ? forward<false>(c, a, e) : forward<true>(c, a, e);
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
    // scratch: the item counter | D
    char* mem = static_cast<char*>(scratch_get(c, kSlotSinkD, 256 + (size_t)a.B * a.H * a.Sq * sizeof(float), e));
    if (!mem) return 1;
    a.next_item = reinterpret_cast<int*>(mem);
    a.D = reinterpret_cast<float*>(mem + 256);
    return p->type == kTypeF16 ? backward<false>(c, a, e) : backward<true>(c, a, e);
  });
}

}  // extern "C"
