// FlashAttention backward for sm_100a.  With c = sm_scale and the forward's
// saved O and LSE,
//   P_mn  = exp(c q_m.k_n - lse_m)          (0 where masked)
//   delta_m = sum_d dO_md O_md,  dP = dO V^T,  dS = P * (dP - delta)
//   dQ = c dS K,   dK = c sum_g dS^T Q,   dV = sum_g P^T dO
// (sum_g over the query heads that share a key/value head).  P is recomputed
// from Q, K and LSE instead of being stored.
//
// fa_bwd_stats_kernel (memory-bound) reads O and dO once and
// leaves -lse*log2(e) and -delta per query row.  fa_bwd_kernel then runs two
// kinds of work items, both one 128-row stationary tile against a stream of tiles:
//   * dK/dV items: K and V tiles stationary, every
//     (query head of the group, query tile) streamed.  The products are taken
//     transposed, S^T = K Q^T and dP^T = V dO^T, so that P^T and dS^T come out
//     with keys in the TMEM lanes and are, converted in place, the A operands
//     (from TMEM) of dV += P^T dO and dK += dS^T Q: neither goes through
//     shared memory.
//   * dQ items: Q and dO tiles stationary, K and V tiles streamed,
//     S = Q K^T, dP = dO V^T, dQ += dS K.
// S and dP are formed twice (7 products instead of 5; at head dims past 128
// three times, 9 products, see BwdCfg), and in return every
// output element is summed in one accumulator in a fixed order: no fp32 dQ
// traffic through L2, no atomics, the same bits from call to call, and shared
// heads need no second reduction.
//
// A CTA stays on its SM and takes item after item (a tile, or a slice of one
// when there are few).  Warps 0 and 3 load (TMA; one operand each), warps 1
// and 2 issue tcgen05.mma, warps 4-11 are two softmax warpgroups: each covers
// the 128 lanes and one half of the streamed tile's columns.  Per streamed
// tile i
//   warp 1 issues  [dV(i)] S(i+1)      once P(i) is stored (dQ: S(i) read)
//   warp 2 issues  dK(i)/dQ(i) dP(i+1) once dS(i) is stored
// Each pair shares one TMEM buffer (P overwrites S, dS overwrites dP), whose
// products its warp keeps in order; the two pairs touch different buffers, and
// their bursts take turns, so that neither's products queue behind a second
// burst of the other's.  One issuing warp for all four left the tensor core
// idle for the few hundred cycles that a warp's first wait after a burst of
// products takes (twice per tile, of some 3300 cycles then); with two, the
// other's products run meanwhile.  While the softmax warps turn S(i+1)
// into P the tensor core runs dK(i) and dP(i+1), and while they turn dP into
// dS it runs dV(i) and S(i+1).  P overwrites its own half of S, dS its own
// half of dP, so no warp writes columns another still has to read.
//
// What bounds it (times: ten calls back to back, the best of several such
// groups; in a long run the power limit lowers the clock).  B1 H16 S4096 D128
// (bf16, all pairs) takes 353 us, 973 TF/s of the five products that the
// formula needs and 1362 of the seven that run, against 1633 of a plain GEMM in
// a run as short; over two seconds 398 us, 1209 against the GEMM's 1360.  The
// tensor pipe is active 69 % of the time: a tile of a dK/dV item is 2048
// tensor-core cycles against some 2400 of the softmax warps' chain (S's wait,
// 64 exponentials a lane, P's store, dP's wait, dS's store).
// Causal 4 x 32 heads of S 1024 (173 us, 497 TF/s; 132 us of this kernel and 18
// of the statistics at the full clock) works through 62 such tiles per SM, 58 %
// of this kernel's cycles; the rest lies around its 14 items: the accumulators'
// read-out and stores, which nothing overlaps, were 15 % of the time (the
// stores alone 3 %), what starts and ends the pipeline was not taken apart.
// At head dim 64 the same exponentials stand against half the products: 32
// heads S 4096 516 us, 666 TF/s (645 us on a GPU already at its power limit).
// At 256, 2 x 16 heads S 4096 causal 1176 us, 585 TF/s: products of 64 streamed
// rows read each stationary operand from shared memory for half the work, some
// 2250 cycles of its bandwidth against 1536 of the tensor core's; a second
// half-tile slot for dO in place of its single one changed nothing.
//
// P and dS are handed on in halves (kHalves): B1 H16 S4096 353 us against 365
// in one piece.  16 softmax warps (32 columns each) and exponentials by
// polynomial on the FMA pipe were slower or no faster.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "fa_internal.h"
#include "ptx.cuh"

namespace fab {

template <typename T>
struct BwdElem;
template <>
struct BwdElem<__nv_bfloat16> {
  static constexpr uint32_t kFmt = kFmtBF16;
  static constexpr bool kScaled = false;  // fp32's exponent range: dS never underflows where dO does not
  static constexpr float kPExp = 0.f;
  __device__ static uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ static float2 unpack2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
template <>
struct BwdElem<__half> {
  static constexpr uint32_t kFmt = kFmtF16;
  // dS = P * (dP - delta) is rounded to fp16 as an operand, and P is about
  // 1/keys: with the small dO of real training it would fall below fp16's
  // normal range although dQ and dK do not.  dS is therefore formed times a
  // power of two that brings the bound 2 |dO_m| |V_n| (Euclidean norms, the
  // largest of the row or of the item's rows, and of the sequence's keys) to
  // [2^14, 2^15); the epilogue divides it out.  (With the largest element of dO
  // brought to [1, 2) instead, 8092 keys and rows of different size took the
  // error against 64 bits to 1.6 times the rounding's; now 1.4.)  What that
  // leaves: dS is subnormal below 2^-29 of the bound and 0 below 2^-39, so dk
  // of a key whose every probability is that small has an absolute precision.
  static constexpr bool kScaled = true;
  // P itself is an operand of dV: as P * 2^12 it keeps its precision down to
  // 2^-26, and its largest value, 1, stays far below fp16's 65504.
  static constexpr float kPExp = 12.f;
  __device__ static uint32_t pack2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ static float2 unpack2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};

// Tile shapes by padded head dim.  Streamed tiles have 128 rows up to head
// dim 128; at 256 shared memory holds the two stationary tiles (128 KB) and
// three 64-row ones.  dK and dV together exceed TMEM at 256, so there a dK/dV
// item forms S and dP over the whole head dim but 128 columns of each output,
// and two items cover a key tile: with dQ's, S and dP are formed three times,
// nine products instead of the formula's five.  Head dims 129 to 255 run as 256
// (2 x 16 heads S 2048 causal: D 160, 192 and 256 all 345 us), 65 to 127 as 128
// (D 72, 80, 96 and 128: 124 to 134 us).
//
// The two streamed operands have a ring each.  The first (Q, or K) is read by
// S(i) and again by dK(i) or dQ(i), a whole tile's time later, and its next
// load has only until S two tiles on to land; the second (dO, or V) is done
// with half a tile after it is first read.  So the first ring is the longer.
template <int kDP_>
struct BwdCfg {
  static constexpr int kDP = kDP_;
  static constexpr int kBS = kDP == 256 ? 64 : 128;  // streamed rows
  static constexpr int kRing0 = kDP == 256 ? 2 : kDP == 128 ? 3 : 4;
  static constexpr int kRing1 = kDP == 256 ? 1 : kDP == 128 ? 2 : 3;
  static constexpr int kAtoms = kDP / 64;  // 128-byte column atoms
  static constexpr int kAAtomBytes = 128 * 128;
  static constexpr int kABytes = kAAtomBytes * kAtoms;
  static constexpr int kBAtomBytes = kBS * 128;
  static constexpr int kBBytes = kBAtomBytes * kAtoms;
  static constexpr int kStatBytes = 2 * kBS * 4;  // statistics of a streamed query tile, two buffers
  static constexpr int kOutDkv = kDP == 256 ? 128 : kDP;  // output columns of one dK/dV item
  static constexpr int kDSplit = kDP / kOutDkv;
  // full/empty per slot; statistics full/empty x 2; stationary full/empty x 2;
  // S, P x 2, dP, dS x 2; issue order x 2; accumulators final x 2 and read; ragged tile x 2; next item
  // full/empty x 2; its request; teardown x 2.
  static constexpr int kNumBars = 2 * (kRing0 + kRing1) + 4 + 4 + 6 + 3 + 2 + 4 + 3 + 2;
  static constexpr int kTailBytes = 304;  // TMEM address, two abort flags with a word each, two items, the scheduler's response
  static constexpr int kSmemBytes =
      2 * kABytes + (kRing0 + kRing1) * kBBytes + 2 * kStatBytes + kNumBars * 8 + kTailBytes;
  // P and dS are handed to the tensor core in two halves where a warp works
  // through two 32-column chunks.
  static constexpr bool kHalves = kBS == 128;
  static constexpr int kThreads = 384;
  // Launched with 168 registers a thread; the load/MMA warpgroup hands some
  // to the two softmax warpgroups, which hold a 64-column row of P across
  // the wait for dP.
  static constexpr int kLaunchRegs = 168, kLoadRegs = 72, kSoftmaxRegs = 216;
  static_assert(128 * kLoadRegs + 256 * kSoftmaxRegs <= kThreads * kLaunchRegs, "register split");
  static constexpr int kTmemS = 0, kTmemP = kBS, kTmemAcc = 2 * kBS;
  static_assert(2 * kBS + kDP <= 512 && 2 * kBS + 2 * kOutDkv <= 512, "TMEM budget");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// Rows of a (batch entry, query head) in the statistics buffer, in tiles of
// kBS rows.  Packed batches give sequence b the tiles from cu_q[b] / kBS + b
// on: ceil(len / kBS) tiles always fit before the next sequence's.
__device__ __forceinline__ int64_t bwd_stat_tile0(const FaBwdParams& p, int b, int h, int q_row0, int bs) {
  return p.cu_q != nullptr ? static_cast<int64_t>(h) * p.stat_tiles + q_row0 / bs + b
                           : (static_cast<int64_t>(b) * p.Hq + h) * p.stat_tiles;
}

// The same for keys' tiles of kBS rows, in which V's norms are taken (fp16).
__device__ __forceinline__ int64_t bwd_key_tile0(const FaBwdParams& p, int b, int h, int k_row0, int bs) {
  return p.cu_k != nullptr ? static_cast<int64_t>(h) * p.key_tiles + k_row0 / bs + b
                           : (static_cast<int64_t>(b) * p.Hkv + h) * p.key_tiles;
}

// The exponent of dS's scale where dO's and V's norms are the roots of g2, v2.
__device__ __forceinline__ float bwd_scale_exp(float g2, float v2) {
  const float b = 0.5f * (log2f(g2) + log2f(v2));
  return g2 > 0.f && g2 < INFINITY && v2 > 0.f && v2 < INFINITY ? fminf(13.f - floorf(b), 60.f) : 0.f;
}

// First row and length of batch entry b.  Packed offsets are clamped to the
// tensor and to the declared longest length, so that no offset makes the
// kernels touch memory outside it.
__device__ __forceinline__ void bwd_seq(const int* cu, int b, int total, int longest, int& row0, int& len) {
  if (cu == nullptr) {
    row0 = 0;
    len = longest;
    return;
  }
  row0 = min(max(cu[b], 0), total);
  len = min(min(max(cu[b + 1], row0), total) - row0, longest);
}

// Rows of a packed tensor that belong to no sequence (before cu[0], after
// cu[B]) get zero gradients, from CTAs along x.  which: 0 dq, 1 dk, 2 dv.
template <typename T>
__device__ __forceinline__ void bwd_zero_rest(const FaBwdParams& p, int which) {
  const bool is_q = which == 0;
  const int* cu = is_q ? p.cu_q : p.cu_k;
  const int total = is_q ? p.total_q : p.total_k, heads = is_q ? p.Hq : p.Hkv;
  const int head = min(max(cu[0], 0), total);
  const int tail = max(min(max(cu[p.B], 0), total), head);
  T* out = reinterpret_cast<T*>(is_q ? p.dq : which == 1 ? p.dk : p.dv);
  const int64_t ss = is_q ? p.dq_ss : which == 1 ? p.dk_ss : p.dv_ss;
  const int64_t sh = is_q ? p.dq_sh : which == 1 ? p.dk_sh : p.dv_sh;
  const int rest = head + total - tail;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < static_cast<int64_t>(rest) * heads * p.D; i += gridDim.x * int64_t(blockDim.x)) {
    const int d = static_cast<int>(i % p.D);
    const int h = static_cast<int>(i / p.D % heads);
    int row = static_cast<int>(i / p.D / heads);
    if (row >= head) row += tail - head;
    out[row * ss + h * sh + d] = static_cast<T>(0.f);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) fa_bwd_zero_rest_kernel(const FaBwdParams p) {
  bwd_zero_rest<T>(p, blockIdx.y);
}

// Per query row: -lse * log2(e), plus kPExp, (-inf for rows that saw no key and for the
// padding rows of the last tile, so that P is 0 there) and -delta, as
// [tile][2][kBS]; for fp16 also the row's squared norm of dO and the tile's
// largest, and from further CTAs those of V's rows, the tiles' largest
// only.  One CTA per kBS-row tile; kLanes lanes share a row, eight
// columns each, so a warp reads whole 128-byte lines.  Measured: 4 x 32 heads,
// S 1024, 67 MB, 15 us (18 with 256 threads, 22 with 1024); 2 x 16 heads, S
// 8192, 134 MB, 25.5 us, 5.3 TB/s.
constexpr int kStatThreads = 512;
template <typename T, int kBS, int kLanes>
__global__ void __launch_bounds__(kStatThreads, 2) fa_bwd_stats_kernel(const FaBwdParams p) {
  // The main kernel may be set up meanwhile; it waits before it reads.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Rows of CTAs, in y and past its 65535 in z: query heads, for fp16
  // key/value heads, and three more for packed batches.
  int bh = blockIdx.z * gridDim.y + blockIdx.y;
  const int q_heads = p.B * p.Hq, all_heads = q_heads + (BwdElem<T>::kScaled ? p.B * p.Hkv : 0);
  if (bh >= all_heads) {
    if (p.cu_q != nullptr && bh < all_heads + 3) bwd_zero_rest<T>(p, bh - all_heads);
    return;
  }
  const bool keys = BwdElem<T>::kScaled && bh >= q_heads;
  if (keys) bh -= q_heads;
  const int heads = keys ? p.Hkv : p.Hq;
  const int b = bh / heads, h = bh % heads;
  int q0, M;
  if (keys)
    bwd_seq(p.cu_k, b, p.total_k, p.N, q0, M);
  else
    bwd_seq(p.cu_q, b, p.total_q, p.M, q0, M);
  const int m0 = blockIdx.x * kBS;
  if (m0 >= M) return;
  // For keys both operands are V.
  const int64_t o_ss = keys ? p.v_ss : p.o_ss, g_ss = keys ? p.v_ss : p.g_ss;
  const T* v = reinterpret_cast<const T*>(p.v) + (p.cu_k ? q0 * p.v_ss : b * p.v_sb) + h * p.v_sh;
  const T* o = keys ? v : reinterpret_cast<const T*>(p.o) + (p.cu_q ? q0 * p.o_ss : b * p.o_sb) + h * p.o_sh;
  const T* g = keys ? v : reinterpret_cast<const T*>(p.dout) + (p.cu_q ? q0 * p.g_ss : b * p.g_sb) + h * p.g_sh;
  const float* lse = p.lse + (p.cu_q ? q0 * p.l_ss : b * p.l_sb) + h * p.l_sh;
  const int64_t tile = (keys ? bwd_key_tile0(p, b, h, q0, kBS) : bwd_stat_tile0(p, b, h, q0, kBS)) + blockIdx.x;
  float* st = p.stats + tile * (2 * kBS);
  constexpr int kRows = kStatThreads / kLanes;  // rows of one pass over the CTA
  const int sub = threadIdx.x % kLanes, r0 = threadIdx.x / kLanes;
  const int col = sub * 8;
  float amax = 0.f;
  // All of a thread's loads are under way before the first is used: the
  // kernel's time is one trip to memory where there are few rows.
  constexpr int kSteps = kBS / kRows;
  uint4 ow[kSteps], gw[kSteps];
  float l[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int m = m0 + r0 + i * kRows;
    ow[i] = gw[i] = make_uint4(0, 0, 0, 0);
    l[i] = -INFINITY;
    if (m < M) {
      const T* orow = o + m * o_ss + col;
      const T* grow = g + m * g_ss + col;
      if (col + 8 <= p.D) {
        ow[i] = *reinterpret_cast<const uint4*>(orow);
        gw[i] = *reinterpret_cast<const uint4*>(grow);
      } else if (col < p.D) {
        alignas(16) T part[2][8] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < p.D) part[0][e] = orow[e], part[1][e] = grow[e];
        ow[i] = *reinterpret_cast<const uint4*>(part[0]);
        gw[i] = *reinterpret_cast<const uint4*>(part[1]);
      }
      if (sub == 0 && !keys) l[i] = lse[m * p.l_ss];
    }
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int r = r0 + i * kRows;
    float dot = 0.f, norm = 0.f;
    const uint32_t* ov = reinterpret_cast<const uint32_t*>(&ow[i]);
    const uint32_t* gv = reinterpret_cast<const uint32_t*>(&gw[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 of = BwdElem<T>::unpack2(ov[e]), gf = BwdElem<T>::unpack2(gv[e]);
      dot = fmaf(of.x, gf.x, dot);
      dot = fmaf(of.y, gf.y, dot);
      if constexpr (BwdElem<T>::kScaled) norm = fmaf(gf.x, gf.x, fmaf(gf.y, gf.y, norm));
    }
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, off);
      if constexpr (BwdElem<T>::kScaled) norm += __shfl_xor_sync(0xffffffffu, norm, off);
    }
    if (sub == 0) {
      if (!keys) {
        const bool none = l[i] == -INFINITY;
        st[r] = none ? -INFINITY : fmaf(-l[i], 1.4426950408889634f, BwdElem<T>::kPExp);
        st[kBS + r] = none ? 0.f : -dot;
      }
      if constexpr (BwdElem<T>::kScaled) {
        if (!keys) p.row_norm[tile * kBS + r] = norm;
        if (norm < INFINITY) amax = fmaxf(amax, norm);
      }
    }
  }
  if constexpr (BwdElem<T>::kScaled) {
    __shared__ float red[kStatThreads / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kStatThreads / 32; ++w) amax = fmaxf(amax, red[w]);
      (keys ? p.key_max : p.tile_max)[tile] = amax;
    }
  }
}

// A 32-column chunk of a warp's 32 output rows: lane r brings row r's values,
// packed.  Four lanes exchange their 16-byte pieces (a 4 x 4 transpose in two
// steps) and store 64 consecutive bytes of one row at a time, 8 lines per
// instruction instead of 32.  An SM writes some 30 bytes a cycle whichever way
// (measured; 32-byte stores of whole sectors without the exchange were 3 %
// slower at 4 x 32 heads, S 1024, causal).  `row` is the warp's first row at
// the chunk's first column, `stride` in bytes; `rows` and `cols` say how much
// of the chunk exists.  16-byte aligned rows.
template <typename T>
__device__ __forceinline__ void bwd_store_chunk(int64_t row, int64_t stride, int rows, int cols, const uint32_t (&w)[16]) {
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1, high = lane & 2;
  uint32_t t[16], u[16];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? w[h + e] : w[h + 4 + e], 1);
      t[h + e] = odd ? other : w[h + e];
      t[h + 4 + e] = odd ? w[h + 4 + e] : other;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, high ? t[e] : t[8 + e], 2);
    u[e] = high ? other : t[e];
    u[8 + e] = high ? t[8 + e] : other;
  }
  // u holds piece lane % 4 of the four rows of this group of lanes.
  const int col = (lane & 3) * 8;
  T* dst = reinterpret_cast<T*>(row + (lane & ~3) * stride) + col;
  rows -= lane & ~3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < rows) {
      if (col + 8 <= cols) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < cols)
            reinterpret_cast<uint16_t*>(dst)[e] =
                static_cast<uint16_t>((e & 1) ? u[4 * i + e / 2] >> 16 : u[4 * i + e / 2] & 0xFFFFu);
      }
    }
    dst = reinterpret_cast<T*>(reinterpret_cast<int64_t>(dst) + stride);
  }
}

// Warp-collective bounded wait for a phase, in few instructions: these kernels
// hold some sixty waits, and with the general one (ptx.cuh) inlined at each
// they outgrew the instruction cache.  Each try suspends for a microsecond at
// most; after kWaitTries, or once another warp of the CTA has given up, the
// warp leaves its code in the abort flag and unwinds.  The word after the flag,
// read with it, is the number of tries not to make: 0 but in tests.
constexpr int kWaitTries = 4000000;
__device__ __forceinline__ bool bwd_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int code) {
  // Usually complete already: one test, no loop.
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n, a, m;\n\t"
      "mov.u32 n, %4;\n\t"
      "WAIT:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
      "@p bra DONE;\n\t"
      "ld.volatile.shared.v2.u32 {a, m}, [%3];\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.le.u32 q, n, m;\n\t"
      "setp.ne.or.u32 q, a, 0, q;\n\t"
      "@!q bra WAIT;\n\t"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(smem_u32(const_cast<const int*>(abort))), "n"(kWaitTries)
      : "memory");
  if (__all_sync(0xffffffffu, ok != 0)) return true;
  *abort = code;
  return false;
}

// A work item: one stationary tile (and, at head dim 256, one half of the
// output columns) against a slice of its streamed tiles.
struct BwdItem {
  int kind;                // kItemDkv, kItemDq, or kItemEnd: no more
  int b, h, tile;          // batch entry, head (of the stationary tile), 128-row tile
  int dcol0;               // first output column
  int q_row0, k_row0;      // the sequence's first rows in a packed tensor
  int M, N;                // its lengths
  int row0;                // first stationary row within the sequence
  int first, per_head;     // streamed tiles [first, first + per_head) of each head
  int begin, nt;           // this slice: streamed tiles begin .. begin + nt of all heads'
  int begin_head, begin_tile;  // begin / per_head, begin % per_head
  int slice, slices;
  int two;                 // P and dS as two 16-bit parts each
  // The tile's first row in dK or dQ [0] and in dV [1], the bytes between
  // rows, and the slice's sums where there are several slices.
  int64_t out[2], stride[2], part;
};
enum BwdItemKind : int { kItemEnd, kItemDkv, kItemDq };

// Streamed tiles of a stationary tile are cut into slices when there are too
// few stationary tiles to fill the GPU; slice s of `slices` takes an even
// share, and with more than one each leaves fp32 sums that
// fa_bwd_join_kernel adds in slice order.
__device__ __forceinline__ void bwd_slices(int total, int slice_len, int max_slices, int& slices, int& share) {
  slices = min(max_slices, max(1, (total + slice_len - 1) / slice_len));
  share = (total + slices - 1) / slices;
}

// P and dS are rounded to 16 bits as operands.  Over many rows that adds as
// much error to a gradient as its own rounding does (together 1.4 times), but
// where few rows or keys are summed a handful of values decides, and whole
// gradients were up to 1.8 times as far off as by their rounding alone.  Short
// sequences, and all sequences of a call with few query rows (over its heads),
// take each value as two 16-bit parts with a product for each.  Measured: 4
// heads of 300 tokens, one of 1024 and 4 of 500 by 700 (D 256) take the same
// time within 2 %; 8 heads of 1 query and 32768 keys 156 instead of 129 us.
constexpr int kTwoPartLength = 128, kTwoPartRows = 2048;

// False: nothing to do (a tile or slice that this sequence does not have).
template <int kDP, bool kDkv>
__device__ __forceinline__ bool bwd_item(const FaBwdParams& p, int index, BwdItem& w) {
  using C = BwdCfg<kDP>;
  constexpr int kDSplit = kDkv ? C::kDSplit : 1;
  const int tiles = kDkv ? p.k_tiles : p.q_tiles;
  const int heads = kDkv ? p.Hkv : p.Hq;
  const int max_slices = kDkv ? p.dkv_slices : p.dq_slices;
  w.slice = index % max_slices;
  index /= max_slices;
  w.dcol0 = kDSplit > 1 ? index % kDSplit * C::kOutDkv : 0;
  index /= kDSplit;
  // The tile is the fast index, so that CTAs at work together share a head's
  // operands in L2; longest (causal) first.
  w.tile = kDkv ? index % tiles : tiles - 1 - index % tiles;
  w.b = index / tiles / heads;
  w.h = index / tiles % heads;
  bwd_seq(p.cu_q, w.b, p.total_q, p.M, w.q_row0, w.M);
  bwd_seq(p.cu_k, w.b, p.total_k, p.N, w.k_row0, w.N);
  w.row0 = w.tile * 128;
  if (w.row0 >= (kDkv ? w.N : w.M)) return false;
  int last;
  if constexpr (kDkv) {
    w.first = p.causal ? w.row0 / C::kBS : 0;  // query m sees key n iff m >= n
    last = (w.M + C::kBS - 1) / C::kBS;
  } else {
    w.first = 0;
    last = ((p.causal ? min(w.N, w.row0 + 128) : w.N) + C::kBS - 1) / C::kBS;
  }
  w.per_head = max(0, last - w.first);
  const int total = w.per_head * (kDkv ? p.group : 1);
  int share;
  bwd_slices(total, kDkv ? p.dkv_slice_len : p.dq_slice_len, max_slices, w.slices, share);
  if (w.slice >= w.slices) return false;
  w.begin = w.slice * share;
  w.nt = max(0, min(share, total - w.begin));
  w.two = p.few_rows || min(w.M, w.N) <= kTwoPartLength;
  w.begin_head = w.per_head > 0 ? w.begin / w.per_head : 0;
  w.begin_tile = w.begin - w.begin_head * w.per_head;
  w.kind = kDkv ? kItemDkv : kItemDq;
  return true;
}

// fp32 sums of a slice: [slot][accumulator][column][row].
template <int kDP, bool kDkv>
__device__ __forceinline__ int64_t bwd_part_slot(const FaBwdParams& p, const BwdItem& w) {
  using C = BwdCfg<kDP>;
  int64_t tile;
  if constexpr (kDkv) {
    tile = p.cu_k != nullptr ? static_cast<int64_t>(w.h) * p.part_k_tiles + w.k_row0 / 128 + w.b + w.tile
                             : (static_cast<int64_t>(w.b) * p.Hkv + w.h) * p.part_k_tiles + w.tile;
    return (tile * C::kDSplit + w.dcol0 / C::kOutDkv) * p.dkv_slices + w.slice;
  } else {
    tile = p.cu_q != nullptr ? static_cast<int64_t>(w.h) * p.part_q_tiles + w.q_row0 / 128 + w.b + w.tile
                             : (static_cast<int64_t>(w.b) * p.Hq + w.h) * p.part_q_tiles + w.tile;
    return tile * p.dq_slices + w.slice;
  }
}

// Where the item's results go.
template <typename T, int kDP, bool kDkv>
__device__ __forceinline__ void bwd_outputs(const FaBwdParams& p, BwdItem& w) {
  constexpr int64_t kSize = sizeof(T);
  auto at = [&](const void* base, int64_t sb, int64_t sh, int64_t ss, int row0) {
    return reinterpret_cast<int64_t>(base) + ((p.cu_q ? row0 * ss : w.b * sb) + w.h * sh + w.row0 * ss) * kSize;
  };
  if constexpr (kDkv) {
    w.out[0] = at(p.dk, p.dk_sb, p.dk_sh, p.dk_ss, w.k_row0);
    w.out[1] = at(p.dv, p.dv_sb, p.dv_sh, p.dv_ss, w.k_row0);
    w.stride[0] = p.dk_ss * kSize;
    w.stride[1] = p.dv_ss * kSize;
    w.part = reinterpret_cast<int64_t>(p.dkv_part + bwd_part_slot<kDP, true>(p, w) * (2 * BwdCfg<kDP>::kOutDkv * 128));
  } else {
    w.out[0] = w.out[1] = at(p.dq, p.dq_sb, p.dq_sh, p.dq_ss, w.q_row0);
    w.stride[0] = w.stride[1] = p.dq_ss * kSize;
    w.part = reinterpret_cast<int64_t>(p.dq_part + bwd_part_slot<kDP, false>(p, w) * (kDP * 128));
  }
}

// What warp (half, rows wq * 32 ...) of the tile writes: dK/dV items:
// warpgroup 0 dK, 1 dV; dQ items: each half of the columns.
template <typename T, int kDP>
struct BwdOut {
  int64_t row, stride;  // the warp's first row at its first column, bytes between rows
  int rows, left;       // rows of the warp's 32, columns from there on, that exist
  int cols;             // columns of a warp
  int acc;              // its first accumulator column
  float* part;          // this lane's column 0 of the slice's sums
  __device__ __forceinline__ BwdOut(const BwdItem& w, int half, int wq, int head_dim) {
    const bool dkv = w.kind == kItemDkv;
    cols = dkv ? BwdCfg<kDP>::kOutDkv : kDP / 2;
    const int col0 = dkv ? w.dcol0 : half * cols;
    stride = half ? w.stride[1] : w.stride[0];
    row = (half ? w.out[1] : w.out[0]) + wq * 32 * stride + col0 * static_cast<int>(sizeof(T));
    rows = (dkv ? w.N : w.M) - w.row0 - wq * 32;
    left = head_dim - col0;
    acc = half * cols;
    part = reinterpret_cast<float*>(w.part) + acc * 128 + wq * 32 + (threadIdx.x & 31);
  }
  // 32 columns from the warp's column cc on.
  __device__ __forceinline__ void store(int cc, const float (&v)[32]) const {
    if (rows <= 0 || cc >= left) return;
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = BwdElem<T>::pack2(v[2 * e], v[2 * e + 1]);
    bwd_store_chunk<T>(row + cc * static_cast<int>(sizeof(T)), stride, rows, left - cc, w);
  }
};

// Shared memory and barriers of a CTA.
template <int kDP>
struct BwdCta {
  using C = BwdCfg<kDP>;
  uint8_t *sA0, *sA1, *sB0, *sB1;
  float* sStat;
  uint64_t *full0, *empty0, *full1, *empty1, *st_full, *st_empty, *a_full, *a_empty, *s, *pr, *dp, *ds, *turn, *done, *acc_free,
      *fix, *sched_full, *sched_empty, *clc, *drained;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  BwdItem* item;  // [2]
  uint32_t clc_resp;
  __device__ __forceinline__ explicit BwdCta(uint8_t* smem) {
    sA0 = smem;
    sA1 = sA0 + C::kABytes;
    sB0 = sA1 + C::kABytes;
    sB1 = sB0 + C::kRing0 * C::kBBytes;
    sStat = reinterpret_cast<float*>(sB1 + C::kRing1 * C::kBBytes);
    full0 = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sStat) + 2 * C::kStatBytes);
    empty0 = full0 + C::kRing0;
    full1 = empty0 + C::kRing0;
    empty1 = full1 + C::kRing1;
    st_full = empty1 + C::kRing1;
    st_empty = st_full + 2;
    a_full = st_empty + 2;
    a_empty = a_full + 2;
    s = a_empty + 2;    // S(i) complete
    pr = s + 1;         // [2] P(i) half stored, stored (dK/dV); [1] S(i) read (dQ)
    dp = pr + 2;        // dP(i) complete
    ds = dp + 1;        // [2] dS(i) half stored, stored
    turn = ds + 2;      // [2] issue order of the two issuers
    done = turn + 2;    // [2] accumulator final
    acc_free = done + 2;  // accumulators read
    fix = acc_free + 1;   // [2] ragged tile landed, before its rows are cleared
    sched_full = fix + 2;
    sched_empty = sched_full + 2;
    clc = sched_empty + 2;
    drained = clc + 1;
    tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
    clc_resp = (smem_u32(tmem_slot + 6) + 15u) & ~15u;  // 16 bytes
    item = reinterpret_cast<BwdItem*>(tmem_slot + 12);
    static_assert(48 + 2 * sizeof(BwdItem) <= C::kTailBytes, "two items in the tail");
  }
};

// A position in a ring (or in a barrier's phases, with one slot).
struct BwdPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++slot == size) {
      slot = 0;
      phase ^= 1;
    }
  }
};

// The roles below run one copy of their code each, whatever the item's kind
// and whichever of their two warps they are: with a copy for every
// combination the kernel was four times the size, and items of a few tiles
// spent most of their time fetching instructions.

// --------------------------------------------------------------- producers
// Role 0 (warp 0): the first stationary and streamed operands (K and Q, or Q
// and K) and the statistics; role 1 (warp 3): the second ones (V and dO, or
// dO and V).  The whole warp runs this; lane 0 issues the copies.
struct BwdProducer {
  BwdPos ring, a, stat, fix;
  bool any = false;
  int tiles = 0, stats = 0;
};

template <int kDP>
__device__ __forceinline__ bool bwd_produce(const FaBwdParams& p, const BwdCta<kDP>& c, int role, const CUtensorMap* map_a,
                                            const CUtensorMap* map_s, const BwdItem& w, BwdProducer& n) {
  using C = BwdCfg<kDP>;
  constexpr int kBS = C::kBS;
  if (w.nt == 0) return true;
  const int lane = threadIdx.x & 31;
  const bool packed = p.cu_q != nullptr, dkv = w.kind == kItemDkv;
  const int map_b = packed ? 0 : w.b;
  uint64_t* const full = role == 0 ? c.full0 : c.full1;
  uint64_t* const empty = role == 0 ? c.empty0 : c.empty1;
  uint8_t* const ring = role == 0 ? c.sB0 : c.sB1;
  const int size = role == 0 ? C::kRing0 : C::kRing1;
  if (!bwd_wait(c.a_empty + role, n.a.phase ^ 1, c.abort_flag, kDevTimeoutEmpty)) return false;
  if (lane == 0) {
    mbar_arrive_expect_tx(c.a_full + role, C::kABytes);
#pragma unroll 1
    for (int a = 0; a < C::kAtoms; ++a)
      tma_load_4d((role ? c.sA1 : c.sA0) + a * C::kAAtomBytes, map_a, c.a_full + role, a * 64,
                  (dkv ? w.k_row0 : w.q_row0) + w.row0, w.h, map_b);
  }
  n.a.next(1);
  if (role == 0 && !n.any) {
    // The statistics kernel's output is read from here on.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    fence_proxy_async_global();
  }
  n.any = true;
  // A packed sequence's last tile runs into the next sequence's rows.  Rows of
  // the summed dimension must be zero there (0 x NaN is NaN), so such a tile
  // is cleared past the end before it is handed on.
  const int len = dkv ? w.M : w.N;  // valid streamed rows of the sequence
  const int ragged = packed && len % kBS != 0 ? len / kBS - w.first : -1;
  const int row_first = (dkv ? w.q_row0 : w.k_row0) + w.first * kBS;
  int ti = w.begin_tile;
  int head = (dkv ? w.h * p.group : w.h / p.group) + w.begin_head;
  const bool stats = dkv && role == 0;
  const float* stat = p.stats + (bwd_stat_tile0(p, w.b, head, w.q_row0, kBS) + w.first) * (2 * kBS);
  const int64_t stat_head = static_cast<int64_t>(p.stat_tiles) * (2 * kBS);
#pragma unroll 1
  for (int i = 0; i < w.nt; ++i) {
    if (!bwd_wait(empty + n.ring.slot, n.ring.phase ^ 1, c.abort_flag, kDevTimeoutEmpty)) return false;
    uint8_t* dst = ring + n.ring.slot * C::kBBytes;
    uint64_t* const landed = full + n.ring.slot;
    n.ring.next(size);
    ++n.tiles;
    const bool fix = ti == ragged;
    if (lane == 0) {
      uint64_t* bar = fix ? c.fix + role : landed;
      mbar_arrive_expect_tx(bar, C::kBBytes + p.starve_bytes);
#pragma unroll
      for (int a = 0; a < C::kAtoms; ++a)
        tma_load_4d(dst + a * C::kBAtomBytes, map_s, bar, a * 64, row_first + ti * kBS, head, map_b);
    }
    if (stats) {
      if (!bwd_wait(c.st_empty + n.stat.slot, n.stat.phase ^ 1, c.abort_flag, kDevTimeoutEmpty)) return false;
      if (lane == 0) {
        mbar_arrive_expect_tx(c.st_full + n.stat.slot, C::kStatBytes);
        bulk_load_g2s(c.sStat + n.stat.slot * (2 * kBS), stat + ti * (2 * kBS), C::kStatBytes, c.st_full + n.stat.slot);
      }
      n.stat.next(2);
      ++n.stats;
    }
    if (fix) {
      if (!bwd_wait(c.fix + role, n.fix.phase, c.abort_flag, kDevTimeoutKV)) return false;
      n.fix.next(1);
      const int rows = len % kBS, chunks = (kBS - rows) * 8;  // 16-byte pieces of one atom's rows past the end
#pragma unroll 1
      for (int a = 0; a < C::kAtoms; ++a)
#pragma unroll 1
        for (int k = lane; k < chunks; k += 32)
          *reinterpret_cast<uint4*>(dst + a * C::kBAtomBytes + rows * 128 + k * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(landed);
    }
    if (++ti == w.per_head) {
      ti = 0;
      ++head;
      stat += stat_head;
    }
  }
  return true;
}

// ------------------------------------------------------------- MMA issuers
// Role 0 (warp 1): S and dV.  Role 1 (warp 2): dP and dK or dQ.  A slot of a
// ring is free when both roles' products that read it are complete.
struct BwdIssuer {
  BwdPos s, o;      // the rings of the first and of the second product's operand
  BwdPos item, it;  // items, streamed tiles
};

template <typename T, int kDP, bool kTwo>
__device__ __forceinline__ bool bwd_issue(const BwdCta<kDP>& c, uint32_t tmem, bool leader, int role, const BwdItem& w,
                                          BwdIssuer& n) {
  using C = BwdCfg<kDP>;
  constexpr int kBS = C::kBS;
  if (w.nt == 0) return true;
  const int nt = w.nt;
  const bool dkv = w.kind == kItemDkv;
  constexpr uint32_t kFmt = BwdElem<T>::kFmt;
  constexpr uint32_t idesc_s = umma_idesc(kFmt, 128, kBS, 0, 0);
  const uint32_t idesc_o = dkv ? umma_idesc(kFmt, 128, C::kOutDkv, 0, 1) : umma_idesc(kFmt, 128, kDP, 0, 1);
  constexpr uint32_t kHi = umma_desc_hi(1024, kLayoutSw128);
  const uint32_t a_lo = umma_desc_lo(smem_u32(role == 0 ? c.sA0 : c.sA1), 16);
  // The streamed operand of the role's first product (S or dP), and, MN-major
  // from this item's first output column, that of its second.
  const uint32_t b_lo = umma_desc_lo(smem_u32(role == 0 ? c.sB0 : c.sB1), 16);
  const uint32_t bn_lo = umma_desc_lo(smem_u32(role == 0 ? c.sB1 : c.sB0) + (w.dcol0 / 64) * C::kBAtomBytes,
                                      C::kBAtomBytes);
  // This role's buffer, the barriers of its first product and of what the
  // softmax warps make of it, its rings.
  const uint32_t tBuf = tmem + (role == 0 ? C::kTmemS : C::kTmemP);
  const uint32_t tAcc = tmem + C::kTmemAcc + (role == 0 ? C::kOutDkv : 0);
  uint64_t* const ready = role == 0 ? c.s : c.dp;
  uint64_t* const stored = role == 0 ? c.pr : c.ds;
  const int size_s = role == 0 ? C::kRing0 : C::kRing1, size_o = role == 0 ? C::kRing1 : C::kRing0;
  uint64_t* const full_s = role == 0 ? c.full0 : c.full1;
  uint64_t* const empty_s = role == 0 ? c.empty0 : c.empty1;
  uint64_t* const full_o = role == 0 ? c.full1 : c.full0;
  uint64_t* const empty_o = role == 0 ? c.empty1 : c.empty0;
  const bool sum = role == 1 || dkv;  // has a second product: dV, dK or dQ
  // With one slot the tile of the next dP lands where the last one was, after
  // the burst's first half: it can only be waited for in between.
  const bool one_burst = C::kRing1 > 1 || role == 0;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    return bwd_wait(bar, parity, c.abort_flag, code);
  };
  auto commit = [&](uint64_t* bar) {
    if (leader) mma_commit(bar);
  };
  // D[128 x kOut] += A (TMEM, kBS wide) x B(slot).  Each softmax warpgroup's
  // half of A starts at its half of the fp32 columns; `part` 0 takes the first
  // half of each warpgroup's columns, 1 the rest.  `rest`: the second part of
  // values in two parts.
  auto second_product = [&](bool acc, int part, bool rest = false) {
    uint32_t vb = bn_lo + n.o.slot * (C::kBBytes >> 4) + part * ((kBS / 64 * 16 * 128) >> 4);
    uint32_t at = tBuf + part * (kBS / 8) + (rest ? kBS / 4 : 0);
    asm volatile("" : "+r"(vb), "+r"(at));
#pragma unroll
    for (int x = 0; x < kBS / 32; ++x) {
      constexpr int kHalf = kBS / 32;  // steps of a warpgroup's columns
      const int kk = x / (kHalf / 2) * kHalf + x % (kHalf / 2);
      const uint64_t bd = umma_desc_join(vb + ((kk * 16 * 128) >> 4), kHi);
      if (leader) mma_ts_f16(tAcc, at + (kk / kHalf) * (kBS / 2) + (kk % kHalf) * 8, bd, idesc_o, (acc || x > 0) ? 1u : 0u);
    }
  };

  // One pass per streamed tile, after one for the first tile's first product
  // alone, which needs no wait for the previous item's last products: it
  // overwrites a buffer that those read, in issue order.
#pragma unroll 1
  for (int i = -1; i < nt; ++i) {
    const bool more = i + 1 < nt;
    // All waits come before the burst, so that its products go out together.
    if (i < 0) {
      if (!wait(c.a_full + role, n.item.phase, kDevTimeoutQ)) return false;
    } else {
      if (sum && !wait(full_o + n.o.slot, n.o.phase, kDevTimeoutKV)) return false;
      // The first product into an accumulator waits until the previous item's
      // sums have been read.
      if (i == 0 && !wait(c.acc_free, n.item.phase ^ 1, kDevTimeoutAcc)) return false;
    }
    if (more && (one_burst || i < 0) && !wait(full_s + n.s.slot, n.s.phase, kDevTimeoutKV)) return false;
    if (i >= 0) {
      // Bursts alternate between the issuers: role 0's i-th, role 1's i-th.
      if (!wait(c.turn + (role ^ 1), n.it.phase ^ (role ^ 1), kDevTimeoutP)) return false;
      if (sum && C::kHalves) {
        if (!wait(stored, n.it.phase, kDevTimeoutP)) return false;
        tc_fence_after();
        second_product(i > 0, 0);
      }
      if (!wait(stored + 1, n.it.phase, kDevTimeoutP)) return false;
      tc_fence_after();
      if (sum) {
        if (!C::kHalves) second_product(i > 0, 0);
        second_product(true, 1);
        if (kTwo && w.two)
#pragma unroll 1
          for (int part = 0; part < 2; ++part) second_product(true, part, true);
        commit(empty_o + n.o.slot);
      }
      n.o.next(size_o);
      n.it.next(1);
      if (!more) {
        if (leader) mbar_arrive(c.turn + role);
        break;
      }
      if (!one_burst && !wait(full_s + n.s.slot, n.s.phase, kDevTimeoutKV)) return false;
    }
    tc_fence_after();
    // D[128 x kBS] = A (stationary) x B(slot)^T over the head dim.
    uint32_t qa = a_lo, kb = b_lo + n.s.slot * (C::kBBytes >> 4);
    asm volatile("" : "+r"(qa), "+r"(kb));
#pragma unroll
    for (int kk = 0; kk < kDP / 16; ++kk) {
      const int a = kk >> 2;
      const uint32_t off = (kk & 3) * 32;
      const uint64_t ad = umma_desc_join(qa + ((a * C::kAAtomBytes + off) >> 4), kHi);
      const uint64_t bd = umma_desc_join(kb + ((a * C::kBAtomBytes + off) >> 4), kHi);
      // The other issuer may go on when this burst is nearly out.
      if (kk == kDP / 32 && i >= 0 && leader) mbar_arrive(c.turn + role);
      if (leader) mma_ss_f16(tBuf, ad, bd, idesc_s, kk > 0 ? 1u : 0u);
    }
    commit(ready);
    // A slot counts two releases, one by each role, except that V tiles of dQ
    // items are read by role 1 alone, which gives both.
    commit(empty_s + n.s.slot);
    if (role == 1 && !dkv) commit(empty_s + n.s.slot);
    if (i + 2 == nt) commit(c.a_empty + role);
    n.s.next(size_s);
  }
  commit(c.done + (role ^ 1));
  n.item.next(1);
  return true;
}

// ----------------------------------------------------------------- softmax
struct BwdSoftmax {
  BwdPos it, item, stat;
};

// What packing 32 values left of them, packed in turn.
template <typename T>
__device__ __forceinline__ void bwd_rest(const float* x, const uint32_t (&pk)[16], uint32_t (&rest)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float2 f = BwdElem<T>::unpack2(pk[e]);
    rest[e] = BwdElem<T>::pack2(x[2 * e] - f.x, x[2 * e + 1] - f.y);
  }
}

// The streamed tiles of one item.
template <typename T, int kDP, bool kTwo, bool kDkv>
__device__ __forceinline__ bool bwd_tiles(const FaBwdParams& p, const BwdCta<kDP>& c, uint32_t tS, uint32_t tP, int half,
                                          int r, float row_nl, float row_nd, float cta_scale, const BwdItem& w,
                                          BwdSoftmax& n) {
  using C = BwdCfg<kDP>;
  constexpr int kBS = C::kBS, kCols = kBS / 2, kChunks = kCols / 32;  // columns of one warpgroup
  const int lane = threadIdx.x & 31;
  const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
  const int my = w.row0 + r;  // position of this lane's row in the sequence
  // Never-visible scores become -inf whatever the scale's sign.
  const uint32_t out = p.scale_log2 < 0.f ? 0x7f800000u : 0xff800000u;
  auto arrive = [&](uint64_t* bar) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  int ti = w.begin_tile;
#pragma unroll 1
  for (int i = 0; i < w.nt; ++i) {
    // Positions of this tile's columns: queries (dK/dV) or keys.
    const int pos0 = (w.first + ti) * kBS + half * kCols;
    const int lo = kDkv && p.causal ? my - pos0 : 0;
    const int hi = kDkv ? kCols : (p.causal ? min(w.N, my + 1) : w.N) - pos0;
    const bool need_mask = kDkv ? p.causal && pos0 < w.row0 + 127
                                : pos0 + kCols > w.N || (p.causal && pos0 + kCols - 1 > w.row0);
    const float* st = c.sStat + n.stat.slot * (2 * kBS) + half * kCols;
    if (kDkv && !bwd_wait(c.st_full + n.stat.slot, n.stat.phase, c.abort_flag, kDevTimeoutKV)) return false;
    if (!bwd_wait(c.s, n.it.phase, c.abort_flag, kDevTimeoutS)) return false;
    tc_fence_after();
    // Chunks of 32 columns; the next one's load is under way while one is
    // worked on.
    float pr[kCols];
    uint32_t rr[kChunks][32];
    tmem_ld32(tS, rr[0]);
#pragma unroll
    for (int cc = 0; cc < kChunks; ++cc) {
      tmem_wait_ld();
      if (cc + 1 < kChunks) tmem_ld32(tS + (cc + 1) * 32, rr[cc + 1]);
      if (!kDkv && cc + 1 == kChunks) {
        arrive(c.pr + 1);
        if (C::kHalves && lane == 0) mbar_arrive(c.pr);  // its phases go with the tiles of both kinds
      }
      // The first half of P is handed on while the second is worked out.
      if (kDkv && C::kHalves && cc == 1) {
        tmem_wait_st();
        arrive(c.pr);
      }
      if (need_mask) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (cc * 32 + e < lo || cc * 32 + e >= hi) rr[cc][e] = out;
      }
      [[maybe_unused]] uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const int x = cc * 32 + e;
        float4 nl = make_float4(row_nl, row_nl, row_nl, row_nl);
        if constexpr (kDkv) nl = *reinterpret_cast<const float4*>(st + x);
        const float2 a = __ffma2_rn(make_float2(__uint_as_float(rr[cc][e]), __uint_as_float(rr[cc][e + 1])), c2,
                                    make_float2(nl.x, nl.y));
        const float2 d = __ffma2_rn(make_float2(__uint_as_float(rr[cc][e + 2]), __uint_as_float(rr[cc][e + 3])), c2,
                                    make_float2(nl.z, nl.w));
        pr[x] = ex2_approx(a.x);
        pr[x + 1] = ex2_approx(a.y);
        pr[x + 2] = ex2_approx(d.x);
        pr[x + 3] = ex2_approx(d.y);
        if constexpr (kDkv) {
          pk[e / 2] = BwdElem<T>::pack2(pr[x], pr[x + 1]);
          pk[e / 2 + 1] = BwdElem<T>::pack2(pr[x + 2], pr[x + 3]);
        }
      }
      // P of 32 columns takes 16 of them: columns that are in registers.
      if constexpr (kDkv) {
        tmem_st16(tS + cc * 16, pk);
        if (kTwo && w.two) {
          tmem_wait_ld();  // the second parts go where the last chunks of S were
          uint32_t rest[16];
          bwd_rest<T>(pr + cc * 32, pk, rest);
          tmem_st16(tS + kCols / 2 + cc * 16, rest);
        }
      }
    }
    if constexpr (kDkv) {
      tmem_wait_st();
      arrive(c.pr + 1);
    }
    if (!bwd_wait(c.dp, n.it.phase, c.abort_flag, kDevTimeoutS)) return false;
    tc_fence_after();
    tmem_ld32(tP, rr[0]);
#pragma unroll
    for (int cc = 0; cc < kChunks; ++cc) {
      tmem_wait_ld();
      if (cc + 1 < kChunks) tmem_ld32(tP + (cc + 1) * 32, rr[cc + 1]);
      if (C::kHalves && cc == 1) {
        tmem_wait_st();
        arrive(c.ds);
      }
      uint32_t pk[16];
      float value[32];
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const int x = cc * 32 + e;
        float4 nd = make_float4(row_nd, row_nd, row_nd, row_nd);
        if constexpr (kDkv) nd = *reinterpret_cast<const float4*>(st + kBS + x);
        float2 d0 = __fadd2_rn(make_float2(__uint_as_float(rr[cc][e]), __uint_as_float(rr[cc][e + 1])),
                               make_float2(nd.x, nd.y));
        float2 d1 = __fadd2_rn(make_float2(__uint_as_float(rr[cc][e + 2]), __uint_as_float(rr[cc][e + 3])),
                               make_float2(nd.z, nd.w));
        d0 = __fmul2_rn(make_float2(pr[x], pr[x + 1]), d0);
        d1 = __fmul2_rn(make_float2(pr[x + 2], pr[x + 3]), d1);
        if constexpr (kDkv && BwdElem<T>::kScaled) {
          d0 = __fmul2_rn(d0, make_float2(cta_scale, cta_scale));
          d1 = __fmul2_rn(d1, make_float2(cta_scale, cta_scale));
        }
        pk[e / 2] = BwdElem<T>::pack2(d0.x, d0.y);
        pk[e / 2 + 1] = BwdElem<T>::pack2(d1.x, d1.y);
        value[e] = d0.x, value[e + 1] = d0.y, value[e + 2] = d1.x, value[e + 3] = d1.y;
      }
      tmem_st16(tP + cc * 16, pk);
      if (kTwo && w.two) {
        tmem_wait_ld();
        uint32_t rest[16];
        bwd_rest<T>(value, pk, rest);
        tmem_st16(tP + kCols / 2 + cc * 16, rest);
      }
    }
    tmem_wait_st();
    arrive(c.ds + 1);
    if constexpr (kDkv) {
      if (lane == 0) mbar_arrive(c.st_empty + n.stat.slot);
      n.stat.next(2);
    }
    n.it.next(1);
    if (++ti == w.per_head) ti = 0;
  }
  return true;
}

__device__ __forceinline__ float bwd_warp_max(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
  return x;
}
// The largest squared norm of the sequence's V rows.
template <int kBS>
__device__ __forceinline__ float bwd_key_norm(const FaBwdParams& p, const BwdItem& w, int h) {
  const float* at = p.key_max + bwd_key_tile0(p, w.b, h, w.k_row0, kBS);
  float big = 0.f;
  for (int x = threadIdx.x & 31; x * kBS < w.N; x += 32) big = fmaxf(big, at[x]);
  return bwd_warp_max(big);
}

template <typename T, int kDP, bool kTwo>
__device__ __forceinline__ bool bwd_softmax(const FaBwdParams& p, const BwdCta<kDP>& c, uint32_t tmem, const BwdItem& w,
                                            BwdSoftmax& n) {
  using C = BwdCfg<kDP>;
  constexpr int kBS = C::kBS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = (warp - 4) >> 2;
  const int wq = warp & 3;
  const int r = wq * 32 + lane;  // TMEM lane: stationary row
  const uint32_t mine = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  const uint32_t tS = mine + C::kTmemS + half * (kBS / 2), tP = mine + C::kTmemP + half * (kBS / 2);
  const bool dkv = w.kind == kItemDkv;
  float unscale = 1.f;  // what the epilogue takes back of dS's scale
  if (w.nt > 0) {
    if (dkv) {
      float cta_scale = 1.f;
      if constexpr (BwdElem<T>::kScaled) {
        // The largest |dO| over every row that this item sums.
        float big = 0.f;
        for (int x = lane; x < w.nt; x += 32) {
          const int j = w.begin + x;
          big = fmaxf(big, p.tile_max[bwd_stat_tile0(p, w.b, w.h * p.group + j / w.per_head, w.q_row0, kBS) + w.first +
                                      j % w.per_head]);
        }
        const float e = bwd_scale_exp(bwd_warp_max(big), bwd_key_norm<kBS>(p, w, w.h));
        cta_scale = exp2f(e - BwdElem<T>::kPExp);
        unscale = exp2f(-e);
      }
      if (!bwd_tiles<T, kDP, kTwo, true>(p, c, tS, tP, half, r, 0.f, 0.f, cta_scale, w, n)) return false;
    } else {
      float row_nl = 0.f, row_nd = 0.f;
      const int my = w.row0 + r;
      [[maybe_unused]] float v2 = 0.f;
      if constexpr (BwdElem<T>::kScaled) v2 = bwd_key_norm<kBS>(p, w, w.h / p.group);
      if (my < w.M) {
        const int64_t st_tile = bwd_stat_tile0(p, w.b, w.h, w.q_row0, kBS) + my / kBS;
        row_nl = p.stats[st_tile * (2 * kBS) + my % kBS];
        row_nd = p.stats[st_tile * (2 * kBS) + kBS + my % kBS];
        if constexpr (BwdElem<T>::kScaled) {
          const float e = bwd_scale_exp(p.row_norm[st_tile * kBS + my % kBS], v2);
          row_nl += e - BwdElem<T>::kPExp;  // P, hence dS, times 2^e
          unscale = exp2f(-e);
        }
      }
      if (!bwd_tiles<T, kDP, kTwo, false>(p, c, tS, tP, half, r, row_nl, row_nd, 1.f, w, n)) return false;
    }
    if (!bwd_wait(c.done + (dkv ? half : 0), n.item.phase, c.abort_flag, kDevTimeoutO)) return false;
    tc_fence_after();
    n.item.next(1);
  }
  const BwdOut<T, kDP> out(w, half, wq, p.D);
  const float mul = dkv && half == 1 ? exp2f(-BwdElem<T>::kPExp) : p.scale * unscale;
#pragma unroll 1
  for (int cc = 0; cc < out.cols; cc += 32) {
    float v[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = 0.f;  // where no pair is visible
    if (w.nt > 0) {
      uint32_t rr[32];
      tmem_ld32(mine + C::kTmemAcc + out.acc + cc, rr);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(rr[e]) * mul;
    }
    if (w.slices > 1) {
#pragma unroll
      for (int e = 0; e < 32; ++e) out.part[(cc + e) * 128] = v[e];
    } else {
      out.store(cc, v);
    }
  }
  if (w.nt > 0) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.acc_free);
  }
  return true;
}

// One CTA per SM works through items: its own block index, then those of
// blocks that have not started, which it takes from the hardware scheduler
// (cluster launch control).  Loads, products and softmax run ahead into the
// next item, so only the accumulators' read-out separates two items.
// kTwo: items may have P and dS in two parts (a kernel of its own: as a branch
// in the one for all calls it cost the others 2 to 5 %).
template <typename T, int kDP, bool kTwo>
__global__ void __launch_bounds__(384, 1)
    fa_bwd_kernel(const __grid_constant__ FaBwdParams p, const __grid_constant__ CUtensorMap k_a,
                  const __grid_constant__ CUtensorMap v_a, const __grid_constant__ CUtensorMap q_b,
                  const __grid_constant__ CUtensorMap g_b, const __grid_constant__ CUtensorMap q_a,
                  const __grid_constant__ CUtensorMap g_a, const __grid_constant__ CUtensorMap k_b,
                  const __grid_constant__ CUtensorMap v_b) {
  using C = BwdCfg<kDP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const BwdCta<kDP> c(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kRing0; ++s) {
      mbar_init(c.full0 + s, 1);
      mbar_init(c.empty0 + s, 2);  // both issuers
    }
    for (int s = 0; s < C::kRing1; ++s) {
      mbar_init(c.full1 + s, 1);
      mbar_init(c.empty1 + s, 2);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(c.a_full + x, 1);
      mbar_init(c.a_empty + x, 1);
      mbar_init(c.sched_full + x, 1);
      mbar_init(c.sched_empty + x, 11);  // every warp but warp 0
      mbar_init(c.pr + x, 8);  // one arrival per softmax warp
      mbar_init(c.ds + x, 8);
      mbar_init(c.turn + x, 1);
      mbar_init(c.st_full + x, 1);
      mbar_init(c.st_empty + x, 8);
      mbar_init(c.fix + x, 1);
      mbar_init(c.done + x, 1);
      mbar_init(c.drained + x, 1);
    }
    mbar_init(c.s, 1);
    mbar_init(c.dp, 1);
    mbar_init(c.acc_free, 8);
    mbar_init(c.clc, 1);
    *c.abort_flag = *reinterpret_cast<volatile int*>(&g_fab_device_error) != 0 ? -1 : 0;
    c.abort_flag[2] = 0;
    c.abort_flag[1] = c.abort_flag[3] = p.spared_tries;
    // The swizzled tiles need the base that the alignment above asks for.
    if (smem_u32(smem_raw) & 1023u) {
      record_device_error(kDevTimeoutTeardown);
      *c.abort_flag = -1;
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(c.tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *c.tmem_slot;
  const bool skip = *c.abort_flag != 0;
  // The q-th item, for every warp but warp 0, which posts them.
  auto get_item = [&](int q, BwdItem& w) {
    w.kind = kItemEnd;
    if (!bwd_wait(c.sched_full + (q & 1), (q >> 1) & 1, c.abort_flag, kDevTimeoutSched)) return;
    w = c.item[q & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(c.sched_empty + (q & 1));
  };

  // Each warpgroup re-splits its registers first, whatever it does after.
  if (warp < 4) {
    setmaxnreg_dec<C::kLoadRegs>();
    if ((warp == 0 || warp == 3) && !skip) {
      const int role = warp == 0 ? 0 : 1;
      BwdProducer n;
      BwdItem w;
      int index = static_cast<int>(blockIdx.x);
      BwdPos answer;
      // The scheduler's next block index, -1 when there is none.
      auto ask = [&]() -> int {
        if (lane == 0) {
          mbar_arrive_expect_tx(c.clc, 16);
          clc_try_cancel(c.clc_resp, c.clc);
        }
        // The answer must have landed before this CTA may leave: the second
        // abort flag stays zero till then, so only the tries bound this wait.
        const bool ok = bwd_wait(c.clc, answer.phase, c.abort_flag + 2, kDevTimeoutSched);
        answer.next(1);
        return ok ? clc_first_cta_x(c.clc_resp) : -1;
      };
#pragma unroll 1
      for (int q = 0;; ++q) {
        if (role == 0) {
          // The next item that exists: this block's, then the scheduler's.
          bool found = false;
#pragma unroll 1
          while (index >= 0 && !found) {
            found = index < p.num_dkv ? bwd_item<kDP, true>(p, index, w) : bwd_item<kDP, false>(p, index - p.num_dkv, w);
            if (!found) index = ask();
          }
          if (!found)
            w.kind = kItemEnd;
          else if (w.kind == kItemDkv)
            bwd_outputs<T, kDP, true>(p, w);
          else
            bwd_outputs<T, kDP, false>(p, w);
          // Whatever is posted, the slot's last item must have been read.
          if (q >= 2 && !bwd_wait(c.sched_empty + (q & 1), ((q - 2) >> 1) & 1, c.abort_flag, kDevTimeoutSched)) break;
          if (lane == 0) {
            c.item[q & 1] = w;
            mbar_arrive(c.sched_full + (q & 1));
          }
        } else {
          get_item(q, w);
        }
        if (w.kind == kItemEnd) break;
        const bool dkv = w.kind == kItemDkv;
        const CUtensorMap* map_a = dkv ? (role ? &v_a : &k_a) : role ? &g_a : &q_a;
        const CUtensorMap* map_s = dkv ? (role ? &g_b : &q_b) : role ? &v_b : &k_b;
        if (!bwd_produce<kDP>(p, c, role, map_a, map_s, w, n)) break;
        // All of this item's loads are under way: time to ask for the next.
        if (role == 0) index = ask();
      }
      // No copy may still be landing when a producer leaves: the last one
      // into every buffer, whether or not its tile was handed on.
      if (n.any) bwd_wait(c.a_full + role, n.a.phase ^ 1, c.abort_flag + 2, kDevTimeoutTeardown);
      uint64_t* const full = role == 0 ? c.full0 : c.full1;
      const int size = role == 0 ? C::kRing0 : C::kRing1;
      BwdPos last = n.ring;  // the oldest of the last `size` loads, if there were as many
      if (n.tiles < size) last = BwdPos();
      else last.phase ^= 1;
#pragma unroll 1
      for (int x = min(n.tiles, size); x > 0; --x) {
        bwd_wait(full + last.slot, last.phase, c.abort_flag + 2, kDevTimeoutTeardown);
        last.next(size);
      }
      BwdPos stat = n.stat;
      if (n.stats < 2) stat = BwdPos();
      else stat.phase ^= 1;
#pragma unroll 1
      for (int x = min(n.stats, 2); x > 0; --x) {
        bwd_wait(c.st_full + stat.slot, stat.phase, c.abort_flag + 2, kDevTimeoutTeardown);
        stat.next(2);
      }
    } else if (!skip) {
      const bool leader = elect_one();
      const int role = warp - 1;
      BwdIssuer n;
      BwdItem w;
#pragma unroll 1
      for (int q = 0;; ++q) {
        get_item(q, w);
        if (w.kind == kItemEnd || !bwd_issue<T, kDP, kTwo>(c, tmem, leader, role, w, n)) break;
      }
      // Drain the tensor pipe before TMEM is released.
      if (leader) mma_commit(c.drained + role);
      bwd_wait(c.drained + role, 0, c.abort_flag + 2, kDevTimeoutTeardown);
    }
  } else {
    setmaxnreg_inc<C::kSoftmaxRegs>();
    if (!skip) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the statistics
      BwdSoftmax n;
      BwdItem w;
#pragma unroll 1
      for (int q = 0;; ++q) {
        get_item(q, w);
        if (w.kind == kItemEnd || !bwd_softmax<T, kDP, kTwo>(p, c, tmem, w, n)) break;
      }
    }
  }

  // A warp that gave up left its code.
  __syncthreads();
  if (threadIdx.x == 0 && c.abort_flag[0] > 0) record_device_error(c.abort_flag[0]);
  if (threadIdx.x == 0 && c.abort_flag[2] > 0) record_device_error(c.abort_flag[2]);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the slices of every tile that has more than one, in slice order, and
// stores the result.  blockIdx.x: tile (as an item without its slice),
// blockIdx.y: 32-column chunk of a thread's columns.  28 heads over 4, S 2048:
// 8.4 us for the 64 key tiles' dK and dV.
template <typename T, int kDP, bool kDkv>
__global__ void __launch_bounds__(256) fa_bwd_join_kernel(const FaBwdParams p) {
  const int max_slices = kDkv ? p.dkv_slices : p.dq_slices;
  BwdItem w;
  if (!bwd_item<kDP, kDkv>(p, static_cast<int>(blockIdx.x) * max_slices, w) || w.slices <= 1) return;
  bwd_outputs<T, kDP, kDkv>(p, w);
  const BwdOut<T, kDP> out(w, threadIdx.x >> 7, (threadIdx.x >> 5) & 3, p.D);
  const int cc = blockIdx.y * 32;
  constexpr int64_t kSlot = (kDkv ? 2 * BwdCfg<kDP>::kOutDkv : kDP) * 128;
  const float* src = out.part + cc * 128;
  float v[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) v[e] = src[e * 128];
  for (int s = 1; s < w.slices; ++s) {
    src += kSlot;
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] += src[e * 128];
  }
  out.store(cc, v);
}

}  // namespace fab
