// FlashAttention backward for sm_100a.  With c = sm_scale and the forward's
// saved O and LSE,
//   P_mn  = exp(c q_m.k_n - lse_m)          (0 where masked)
//   delta_m = sum_d dO_md O_md,  dP = dO V^T,  dS = P * (dP - delta)
//   dQ = c dS K,   dK = c sum_g dS^T Q,   dV = sum_g P^T dO
// (sum_g over the query heads that share a key/value head).  P is recomputed
// from Q, K and LSE instead of being stored.
//
// Two launches.  fa_bwd_stats_kernel (memory-bound) reads O and dO once and
// leaves -lse*log2(e) and -delta per query row.  fa_bwd_kernel then runs two
// kinds of CTAs, both one 128-row stationary tile against a stream of tiles:
//   * dK/dV CTAs (blockIdx.x < num_dkv): K and V tiles stationary, every
//     (query head of the group, query tile) streamed.  The products are taken
//     transposed, S^T = K Q^T and dP^T = V dO^T, so that P^T and dS^T come out
//     with keys in the TMEM lanes and are, converted in place, the A operands
//     (from TMEM) of dV += P^T dO and dK += dS^T Q: neither goes through
//     shared memory.
//   * dQ CTAs: Q and dO tiles stationary, K and V tiles streamed,
//     S = Q K^T, dP = dO V^T, dQ += dS K.
// S and dP are formed twice (7 products instead of 5), and in return every
// output element is summed in one accumulator in a fixed order: no fp32 dQ
// traffic through L2, no atomics, the same bits from call to call, and shared
// heads need no second reduction.
//
// Warp 0 loads (TMA), warp 1 issues tcgen05.mma, warps 4-11 are two softmax
// warpgroups: each covers the 128 lanes and one half of the streamed tile's
// columns.  Per streamed tile i the issue order is
//   [dV(i)] S(i+1)  |  dK/dQ(i) dP(i+1)
// where the first group waits for P(i) (or, in dQ CTAs, for S(i) to have been
// read) and the second for dS(i): while the softmax warps turn S(i+1) into P
// the tensor core runs dK(i) and dP(i+1), and while they turn dP into dS it
// runs dV(i) and S(i+1).  P overwrites its own half of S, dS its own half of
// dP, so no warp writes columns another still has to read.
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
  __device__ static float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
};
template <>
struct BwdElem<__half> {
  static constexpr uint32_t kFmt = kFmtF16;
  // dS = P * (dP - delta) is rounded to fp16 as an operand, and P is about
  // 1/keys: with the small dO of real training it would fall below fp16's
  // normal range although dQ and dK do not.  dS is therefore formed times a
  // power of two that brings the largest |dO| of its row (dQ) or of the CTA's
  // rows (dK) to [1, 2); the epilogue divides it out.
  static constexpr bool kScaled = true;
  // P itself is an operand of dV: as P * 2^12 it keeps its precision down to
  // 2^-26, and its largest value, 1, stays far below fp16's 65504.
  static constexpr float kPExp = 12.f;
  __device__ static uint32_t pack2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ static float to_f(__half x) { return __half2float(x); }
};

// Tile shapes by padded head dim.  Streamed tiles have 128 rows up to head
// dim 128; at 256 shared memory holds the two stationary tiles (128 KB) and
// three 64-row ones.  dK and dV together exceed TMEM at 256, so there a dK/dV
// CTA forms S and dP over the whole head dim but 128 columns of each output,
// and two CTAs cover a key tile.
template <int kDP_>
struct BwdCfg {
  static constexpr int kDP = kDP_;
  static constexpr int kBS = kDP == 256 ? 64 : 128;                      // streamed rows
  static constexpr int kRing = kDP == 256 ? 3 : kDP == 128 ? 4 : 8;      // streamed tiles in shared memory
  static constexpr int kAtoms = kDP / 64;                                // 128-byte column atoms
  static constexpr int kAAtomBytes = 128 * 128;
  static constexpr int kABytes = kAAtomBytes * kAtoms;
  static constexpr int kBAtomBytes = kBS * 128;
  static constexpr int kBBytes = kBAtomBytes * kAtoms;
  // Statistics of the streamed query tiles: one buffer per resident one.
  static constexpr int kStatBufs = (kRing + 1) / 2;
  static constexpr int kStatBytes = 2 * kBS * 4;
  static constexpr int kOutDkv = kDP == 256 ? 128 : kDP;                 // output columns of one dK/dV CTA
  static constexpr int kDSplit = kDP / kOutDkv;
  static constexpr int kNumBars = 2 * kRing + 2 + 4 + 2;
  static constexpr int kSmemBytes = 1024 + 2 * kABytes + kRing * kBBytes + kStatBufs * kStatBytes + kNumBars * 8 + 16;
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

// Per query row: -lse * log2(e), plus kPExp, (-inf for rows that saw no key and for the
// padding rows of the last tile, so that P is 0 there) and -delta, as
// [tile][2][kBS]; for fp16 also the row's scale exponent and the tile's
// largest |dO|.  One CTA per kBS-row tile; kLanes lanes share a row, eight
// columns each, so a warp reads whole 128-byte lines.
template <typename T, int kBS, int kLanes>
__global__ void __launch_bounds__(256) fa_bwd_stats_kernel(const FaBwdParams p) {
  const int bh = blockIdx.y;
  const int b = bh / p.Hq, h = bh % p.Hq;
  int q0, M;
  bwd_seq(p.cu_q, b, p.total_q, p.M, q0, M);
  const int m0 = blockIdx.x * kBS;
  if (m0 >= M) return;
  const T* o = reinterpret_cast<const T*>(p.o) + (p.cu_q ? q0 * p.o_ss : b * p.o_sb) + h * p.o_sh;
  const T* g = reinterpret_cast<const T*>(p.dout) + (p.cu_q ? q0 * p.g_ss : b * p.g_sb) + h * p.g_sh;
  const float* lse = p.lse + (p.cu_q ? q0 * p.l_ss : b * p.l_sb) + h * p.l_sh;
  const int64_t tile = bwd_stat_tile0(p, b, h, q0, kBS) + blockIdx.x;
  float* st = p.stats + tile * (2 * kBS);
  constexpr int kRows = 256 / kLanes;  // rows of one pass over the CTA
  const int sub = threadIdx.x % kLanes, r0 = threadIdx.x / kLanes;
  const int col = sub * 8;
  float amax = 0.f;
#pragma unroll 4
  for (int r = r0; r < kBS; r += kRows) {
    const int m = m0 + r;
    float dot = 0.f, big = 0.f;
    if (m < M && col < p.D) {
      const T* orow = o + m * p.o_ss + col;
      const T* grow = g + m * p.g_ss + col;
      if (col + 8 <= p.D) {
        const uint4 ow = *reinterpret_cast<const uint4*>(orow), gw = *reinterpret_cast<const uint4*>(grow);
        const T* oe = reinterpret_cast<const T*>(&ow);
        const T* ge = reinterpret_cast<const T*>(&gw);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float gv = BwdElem<T>::to_f(ge[e]);
          dot = fmaf(BwdElem<T>::to_f(oe[e]), gv, dot);
          big = fmaxf(big, fabsf(gv));
        }
      } else {
        for (int e = 0; col + e < p.D; ++e) {
          const float gv = BwdElem<T>::to_f(grow[e]);
          dot = fmaf(BwdElem<T>::to_f(orow[e]), gv, dot);
          big = fmaxf(big, fabsf(gv));
        }
      }
    }
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, off);
      if constexpr (BwdElem<T>::kScaled) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
    }
    if (sub == 0) {
      const float l = m < M ? lse[m * p.l_ss] : -INFINITY;
      const bool none = l == -INFINITY;
      st[r] = none ? -INFINITY : fmaf(-l, 1.4426950408889634f, BwdElem<T>::kPExp);
      st[kBS + r] = none ? 0.f : -dot;
      if constexpr (BwdElem<T>::kScaled) {
        // 2^e * big in [1, 2); rows of zeros (and of infinities) keep their scale.
        const float e = big > 0.f && big < INFINITY ? -floorf(log2f(big)) : 0.f;
        p.row_exp[tile * kBS + r] = e;
        if (big < INFINITY) amax = fmaxf(amax, big);
      }
    }
  }
  if constexpr (BwdElem<T>::kScaled) {
    __shared__ float red[8];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) amax = fmaxf(amax, red[w]);
      p.tile_max[tile] = amax;
    }
  }
}

// Rows of a packed tensor that belong to no sequence (before cu[0], after
// cu[B]) get zero gradients.  blockIdx.y: dq, dk, dv.
template <typename T>
__global__ void __launch_bounds__(256) fa_bwd_zero_rest_kernel(const FaBwdParams p) {
  const bool is_q = blockIdx.y == 0;
  const int* cu = is_q ? p.cu_q : p.cu_k;
  const int total = is_q ? p.total_q : p.total_k, heads = is_q ? p.Hq : p.Hkv;
  const int head = min(max(cu[0], 0), total);
  const int tail = max(min(max(cu[p.B], 0), total), head);
  T* out = reinterpret_cast<T*>(is_q ? p.dq : blockIdx.y == 1 ? p.dk : p.dv);
  const int64_t ss = is_q ? p.dq_ss : blockIdx.y == 1 ? p.dk_ss : p.dv_ss;
  const int64_t sh = is_q ? p.dq_sh : blockIdx.y == 1 ? p.dk_sh : p.dv_sh;
  const int rest = head + total - tail;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < static_cast<int64_t>(rest) * heads * p.D; i += gridDim.x * 256ll) {
    const int d = static_cast<int>(i % p.D);
    const int h = static_cast<int>(i / p.D % heads);
    int row = static_cast<int>(i / p.D / heads);
    if (row >= head) row += tail - head;
    out[row * ss + h * sh + d] = static_cast<T>(0.f);
  }
}

// 32 fp32 values as part of an output row (16-byte aligned).
template <typename T>
__device__ __forceinline__ void bwd_store32(T* dst, const float (&v)[32], int ncols) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e] = BwdElem<T>::pack2(v[2 * e], v[2 * e + 1]);
  if (ncols >= 32) {
    uint4* d4 = reinterpret_cast<uint4*>(dst);
#pragma unroll
    for (int e = 0; e < 4; ++e) d4[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
  } else {
    uint16_t* d1 = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < ncols) d1[e] = static_cast<uint16_t>((e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu);
  }
}

// One CTA's work.  kDkv: a key tile against its query tiles, else a query
// tile against its key tiles.  a0/a1 are the maps of the stationary operands
// (K and V, or Q and dO), b0/b1 of the streamed ones (Q and dO, or K and V).
template <typename T, int kDP, bool kDkv>
__device__ __forceinline__ void fa_bwd_body(const FaBwdParams& p, const CUtensorMap* a0, const CUtensorMap* a1,
                                            const CUtensorMap* b0, const CUtensorMap* b1, int index,
                                            uint8_t* smem_raw) {
  using C = BwdCfg<kDP>;
  constexpr int kBS = C::kBS, kRing = C::kRing;
  constexpr int kOut = kDkv ? C::kOutDkv : kDP;  // columns of each accumulator
  constexpr int kDSplit = kDkv ? C::kDSplit : 1;

  // ---- work item: the tile is the fast index, longest (causal) first
  const int tiles = kDkv ? p.k_tiles : p.q_tiles;
  const int heads = kDkv ? p.Hkv : p.Hq;
  const int dcol0 = kDSplit > 1 ? index % kDSplit * kOut : 0;
  index /= kDSplit;
  const int tile = kDkv ? index % tiles : tiles - 1 - index % tiles;
  const int b = index / tiles / heads, h = index / tiles % heads;
  int q_row0, k_row0, M, N;
  bwd_seq(p.cu_q, b, p.total_q, p.M, q_row0, M);
  bwd_seq(p.cu_k, b, p.total_k, p.N, k_row0, N);
  const int map_b = p.cu_q != nullptr ? 0 : b;
  const int row0 = tile * 128;  // first stationary row within the sequence
  if (row0 >= (kDkv ? N : M)) return;
  // Streamed tiles [first, first + per_head) of each of `group` heads.
  int first = 0, last;
  if constexpr (kDkv) {
    if (p.causal) first = row0 / kBS;  // query m sees key n iff m >= n
    last = (M + kBS - 1) / kBS;
  } else {
    const int seen = p.causal ? min(N, row0 + 128) : N;
    last = (seen + kBS - 1) / kBS;
  }
  const int per_head = max(0, last - first);
  const int nt = per_head * (kDkv ? p.group : 1);
  const int h_stream0 = kDkv ? h * p.group : h / p.group;

  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  uint8_t* sA0 = smem;
  uint8_t* sA1 = sA0 + C::kABytes;
  uint8_t* sB = sA1 + C::kABytes;
  float* sStat = reinterpret_cast<float*>(sB + kRing * C::kBBytes);
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sStat) + C::kStatBufs * C::kStatBytes);
  uint64_t* bar_empty = bar_full + kRing;
  uint64_t* bar_a = bar_empty + kRing;  // [2]
  uint64_t* bar_s = bar_a + 2;          // S(i) complete
  uint64_t* bar_p = bar_s + 1;          // P(i) stored (dK/dV), S(i) read (dQ)
  uint64_t* bar_dp = bar_p + 1;         // dP(i) complete
  uint64_t* bar_ds = bar_dp + 1;        // dS(i) stored
  uint64_t* bar_done = bar_ds + 1;      // accumulators final
  uint64_t* bar_fix = bar_done + 1;     // ragged tile landed, before its rows are cleared
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_fix + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(bar_full + s, 1);
      mbar_init(bar_empty + s, 1);
    }
    mbar_init(bar_a, 1);
    mbar_init(bar_a + 1, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_p, 8);  // one arrival per softmax warp
    mbar_init(bar_dp, 1);
    mbar_init(bar_ds, 8);
    mbar_init(bar_done, 1);
    mbar_init(bar_fix, 1);
    *abort_flag = *reinterpret_cast<volatile int*>(&g_fab_device_error) != 0 ? 1 : 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const bool skip = *abort_flag != 0;

  // Each warpgroup re-splits its registers first, whatever it does after.
  if (warp < 4) {
    setmaxnreg_dec<C::kLoadRegs>();
  if (warp == 0 && !skip && nt > 0) {
    // ------------------------------------------------------------ producer
    // The whole warp runs this; lane 0 issues the copies.
    const bool packed = p.cu_q != nullptr;
    const int stat_len = kDkv ? M : N;  // valid streamed rows of the sequence
    const int row_base = kDkv ? q_row0 : k_row0;
    if (lane == 0) {
      const int a_row = (kDkv ? k_row0 : q_row0) + row0;
      mbar_arrive_expect_tx(bar_a, C::kABytes);
      for (int a = 0; a < C::kAtoms; ++a) tma_load_4d(sA0 + a * C::kAAtomBytes, a0, bar_a, a * 64, a_row, h, map_b);
      mbar_arrive_expect_tx(bar_a + 1, C::kABytes);
      for (int a = 0; a < C::kAtoms; ++a)
        tma_load_4d(sA1 + a * C::kAAtomBytes, a1, bar_a + 1, a * 64, a_row, h, map_b);
    }
    bool ok = true;
    uint32_t fixes = 0;
    int issued = 0;
    int g = 0, ti = first;  // head of the group and tile of streamed pair t / 2
    for (int t = 0; t < 2 * nt; ++t) {
      const int s = t % kRing;
      const bool second = (t & 1) != 0;
      if (!(ok = mbar_wait_warp(bar_empty + s, ((t / kRing) & 1) ^ 1, abort_flag, kDevTimeoutEmpty))) break;
      const int rows_left = stat_len - ti * kBS;
      // A packed sequence's last tile runs into the next sequence's rows.
      // Rows of the summed dimension must be zero there (0 x NaN is NaN), so
      // such a tile is cleared past the end before it is handed on.  V tiles
      // of dQ CTAs are exempt: they only feed dP columns that are masked.
      const bool fix = packed && rows_left < kBS && (kDkv || !second);
      uint64_t* bar = fix ? bar_fix : bar_full + s;
      if (lane == 0) {
        // A query tile brings its rows' statistics along (same barrier; its
        // buffer is free when its slot is: both were last used for dK).
        const bool stat = kDkv && !second;
        mbar_arrive_expect_tx(bar, C::kBBytes + (stat ? C::kStatBytes : 0));
        if (stat)
          bulk_load_g2s(sStat + (t / 2) % C::kStatBufs * (2 * kBS),
                        p.stats + (bwd_stat_tile0(p, b, h_stream0 + g, q_row0, kBS) + ti) * (2 * kBS), C::kStatBytes, bar);
        uint8_t* dst = sB + s * C::kBBytes;
        const CUtensorMap* map = second ? b1 : b0;
        for (int a = 0; a < C::kAtoms; ++a)
          tma_load_4d(dst + a * C::kBAtomBytes, map, bar, a * 64, row_base + ti * kBS, h_stream0 + g, map_b);
      }
      issued = t + 1;
      if (fix) {
        if (!(ok = mbar_wait_warp(bar_fix, fixes & 1, abort_flag, kDevTimeoutKV))) break;
        ++fixes;
        uint8_t* dst = sB + s * C::kBBytes;
        const int chunks = (kBS - rows_left) * 8;  // 16-byte pieces of one atom's rows past the end
        for (int a = 0; a < C::kAtoms; ++a)
          for (int c = lane; c < chunks; c += 32)
            *reinterpret_cast<uint4*>(dst + a * C::kBAtomBytes + rows_left * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_full + s);
      }
      if (second && ++ti == last) {
        ti = first;
        ++g;
      }
    }
    // No copy may still be landing when the CTA leaves.
    volatile int no_abort = 0;
    if (lane == 0) {
      mbar_wait(bar_a, 0, &no_abort, kDevTimeoutTeardown);
      mbar_wait(bar_a + 1, 0, &no_abort, kDevTimeoutTeardown);
      for (int x = max(0, issued - kRing); x < issued; ++x)
        mbar_wait(bar_full + (x % kRing), (x / kRing) & 1, &no_abort, kDevTimeoutTeardown);
    }
    __syncwarp();
  } else if (warp == 1 && !skip && nt > 0) {
    // ---------------------------------------------------------- MMA issuer
    const bool leader = elect_one();
    constexpr uint32_t kFmt = BwdElem<T>::kFmt;
    constexpr uint32_t idesc_s = umma_idesc(kFmt, 128, kBS, 0, 0);
    constexpr uint32_t idesc_o = umma_idesc(kFmt, 128, kOut, 0, 1);
    constexpr uint32_t kHi = umma_desc_hi(1024, kLayoutSw128);
    const uint32_t a0_lo = umma_desc_lo(smem_u32(sA0), 16);
    const uint32_t a1_lo = umma_desc_lo(smem_u32(sA1), 16);
    const uint32_t b_lo = umma_desc_lo(smem_u32(sB), 16);
    // The same tiles as MN-major operands, from this CTA's first output column.
    const uint32_t bn_lo = umma_desc_lo(smem_u32(sB) + (dcol0 / 64) * C::kBAtomBytes, C::kBAtomBytes);
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
      return mbar_wait_warp(bar, parity, abort_flag, code);
    };
    // D[128 x kBS] = A (stationary) x B(slot)^T over the head dim.
    auto issue_s = [&](uint32_t d, uint32_t alo, int s) {
      uint32_t qa = alo, kb = b_lo + s * (C::kBBytes >> 4);
      asm volatile("" : "+r"(qa), "+r"(kb));
#pragma unroll
      for (int kk = 0; kk < kDP / 16; ++kk) {
        const int a = kk >> 2;
        const uint32_t off = (kk & 3) * 32;
        const uint64_t ad = umma_desc_join(qa + ((a * C::kAAtomBytes + off) >> 4), kHi);
        const uint64_t bd = umma_desc_join(kb + ((a * C::kBAtomBytes + off) >> 4), kHi);
        if (leader) mma_ss_f16(d, ad, bd, idesc_s, kk > 0 ? 1u : 0u);
      }
    };
    // D[128 x kOut] += A (TMEM, kBS wide) x B(slot).  Each softmax warpgroup's
    // half of A starts at its half of the fp32 columns.
    auto issue_o = [&](uint32_t d, uint32_t a, int s, bool acc) {
      uint32_t vb = bn_lo + s * (C::kBBytes >> 4);
      asm volatile("" : "+r"(vb));
#pragma unroll
      for (int kk = 0; kk < kBS / 16; ++kk) {
        constexpr int kHalf = kBS / 32;
        const uint32_t at = a + (kk / kHalf) * (kBS / 2) + (kk % kHalf) * 8;
        const uint64_t bd = umma_desc_join(vb + ((kk * 16 * 128) >> 4), kHi);
        if (leader) mma_ts_f16(d, at, bd, idesc_o, (acc || kk > 0) ? 1u : 0u);
      }
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) mma_commit(bar);
    };
    const uint32_t tS = tmem + C::kTmemS, tP = tmem + C::kTmemP;
    const uint32_t tAcc0 = tmem + C::kTmemAcc, tAcc1 = tAcc0 + kOut;
    auto slot = [](int t) { return t % kRing; };
    auto par = [](int t) { return static_cast<uint32_t>((t / kRing) & 1); };

    bool ok = wait(bar_a, 0, kDevTimeoutQ) && wait(bar_full + slot(0), par(0), kDevTimeoutKV);
    if (ok) {
      tc_fence_after();
      issue_s(tS, a0_lo, slot(0));
      commit(bar_s);
      ok = wait(bar_a + 1, 0, kDevTimeoutQ) && wait(bar_full + slot(1), par(1), kDevTimeoutKV);
    }
    if (ok) {
      tc_fence_after();
      issue_s(tP, a1_lo, slot(1));
      commit(bar_dp);
      if constexpr (!kDkv) commit(bar_empty + slot(1));
    }
    for (int i = 0; ok && i < nt; ++i) {
      const int t0 = 2 * i, t1 = 2 * i + 1;
      if (!(ok = wait(bar_p, i & 1, kDevTimeoutP))) break;
      tc_fence_after();
      if constexpr (kDkv) {
        issue_o(tAcc1, tS, slot(t1), i > 0);
        commit(bar_empty + slot(t1));
      }
      if (i + 1 < nt) {
        if (!(ok = wait(bar_full + slot(t0 + 2), par(t0 + 2), kDevTimeoutKV))) break;
        tc_fence_after();
        issue_s(tS, a0_lo, slot(t0 + 2));
        commit(bar_s);
      }
      if (!(ok = wait(bar_ds, i & 1, kDevTimeoutP))) break;
      tc_fence_after();
      issue_o(tAcc0, tP, slot(t0), i > 0);
      commit(bar_empty + slot(t0));
      if (i + 1 < nt) {
        if (!(ok = wait(bar_full + slot(t1 + 2), par(t1 + 2), kDevTimeoutKV))) break;
        tc_fence_after();
        issue_s(tP, a1_lo, slot(t1 + 2));
        commit(bar_dp);
        if constexpr (!kDkv) commit(bar_empty + slot(t1 + 2));
      }
    }
    // Drain the tensor pipe; the softmax warps read the accumulators after this.
    commit(bar_done);
    volatile int no_abort = 0;
    mbar_wait_warp(bar_done, 0, &no_abort, kDevTimeoutTeardown);
  }
  } else {
    setmaxnreg_inc<C::kSoftmaxRegs>();
  if (!skip) {
    // ------------------------------------------------------------- softmax
    const int half = (warp - 4) >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;  // TMEM lane: stationary row
    const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
    constexpr int kCols = kBS / 2;  // columns of one warpgroup
    const uint32_t tS = tmem + lane_base + C::kTmemS + half * kCols;
    const uint32_t tP = tmem + lane_base + C::kTmemP + half * kCols;
    const int my = row0 + r;  // position of this lane's row in the sequence
    const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
    float row_nl = 0.f, row_nd = 0.f, unscale = 1.f, cta_scale = 1.f;
    if constexpr (!kDkv) {
      if (nt > 0 && my < M) {
        const int64_t st_tile = bwd_stat_tile0(p, b, h, q_row0, kBS) + my / kBS;
        row_nl = p.stats[st_tile * (2 * kBS) + my % kBS];
        row_nd = p.stats[st_tile * (2 * kBS) + kBS + my % kBS];
        if constexpr (BwdElem<T>::kScaled) {
          const float e = p.row_exp[st_tile * kBS + my % kBS];
          row_nl += e - BwdElem<T>::kPExp;  // P, hence dS, times 2^e
          unscale = exp2f(-e);
        }
      }
    } else if constexpr (BwdElem<T>::kScaled) {
      // Largest |dO| over every row this CTA sums.
      float big = 0.f;
      for (int x = lane; x < nt; x += 32)
        big = fmaxf(big, p.tile_max[bwd_stat_tile0(p, b, h_stream0 + x / per_head, q_row0, kBS) + first + x % per_head]);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
      const float e = big > 0.f ? floorf(log2f(big)) : 0.f;
      cta_scale = exp2f(-e - BwdElem<T>::kPExp);
      unscale = exp2f(e);
    }
    // One streamed tile.  `masked`: some pair of this warpgroup's columns is
    // not visible; `pos0` is the position of its first column.
    auto step = [&](auto masked, int i, int pos0) -> bool {
      constexpr bool kMasked = decltype(masked)::value;
      [[maybe_unused]] const float* st = sStat + i % C::kStatBufs * (2 * kBS) + half * kCols;
      // Visible columns [lo, hi) of this lane.
      const int lo = kMasked && kDkv ? my - pos0 : 0;
      const int hi = kMasked && !kDkv ? (p.causal ? min(N, my + 1) : N) - pos0 : kCols;
      if constexpr (kDkv) {
        // The statistics land with the query tile; S(i) implies it, but only
        // this wait orders the copy before this thread's reads.
        if (!mbar_wait_warp(bar_full + (2 * i) % kRing, ((2 * i) / kRing) & 1, abort_flag, kDevTimeoutKV)) return false;
      }
      if (!mbar_wait_warp(bar_s, i & 1, abort_flag, kDevTimeoutS)) return false;
      tc_fence_after();
      float pr[kCols];
      {
        uint32_t rr[kCols / 32][32];
#pragma unroll
        for (int cc = 0; cc < kCols / 32; ++cc) tmem_ld32(tS + cc * 32, rr[cc]);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < kCols; ++x) pr[x] = __uint_as_float(rr[x / 32][x % 32]);
      }
      if constexpr (!kDkv) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p);
      }
#pragma unroll
      for (int cc = 0; cc < kCols / 32; ++cc) {
        [[maybe_unused]] uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const int x = cc * 32 + e;
          float4 nl = make_float4(row_nl, row_nl, row_nl, row_nl);
          if constexpr (kDkv) nl = *reinterpret_cast<const float4*>(st + x);
          const float2 a = __ffma2_rn(make_float2(pr[x], pr[x + 1]), c2, make_float2(nl.x, nl.y));
          const float2 d = __ffma2_rn(make_float2(pr[x + 2], pr[x + 3]), c2, make_float2(nl.z, nl.w));
          pr[x] = ex2_approx(a.x);
          pr[x + 1] = ex2_approx(a.y);
          pr[x + 2] = ex2_approx(d.x);
          pr[x + 3] = ex2_approx(d.y);
          if constexpr (kMasked) {
#pragma unroll
            for (int y = x; y < x + 4; ++y)
              if (y < lo || y >= hi) pr[y] = 0.f;
          }
          if constexpr (kDkv) {
            pk[e / 2] = BwdElem<T>::pack2(pr[x], pr[x + 1]);
            pk[e / 2 + 1] = BwdElem<T>::pack2(pr[x + 2], pr[x + 3]);
          }
        }
        if constexpr (kDkv) tmem_st16(tS + cc * 16, pk);
      }
      if constexpr (kDkv) {
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p);
      }
      if (!mbar_wait_warp(bar_dp, i & 1, abort_flag, kDevTimeoutS)) return false;
      tc_fence_after();
      uint32_t rr[kCols / 32][32];
#pragma unroll
      for (int cc = 0; cc < kCols / 32; ++cc) tmem_ld32(tP + cc * 32, rr[cc]);
      tmem_wait_ld();
#pragma unroll
      for (int cc = 0; cc < kCols / 32; ++cc) {
        [[maybe_unused]] uint32_t pk[16];
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
          if constexpr (kMasked) {
            // P is 0 there, but dP may be infinite or NaN.
            if (x < lo || x >= hi) d0.x = 0.f;
            if (x + 1 < lo || x + 1 >= hi) d0.y = 0.f;
            if (x + 2 < lo || x + 2 >= hi) d1.x = 0.f;
            if (x + 3 < lo || x + 3 >= hi) d1.y = 0.f;
          }
          pk[e / 2] = BwdElem<T>::pack2(d0.x, d0.y);
          pk[e / 2 + 1] = BwdElem<T>::pack2(d1.x, d1.y);
        }
        tmem_st16(tP + cc * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_ds);
      return true;
    };
    bool ok = true;
    int ti = first;
    for (int i = 0; ok && i < nt; ++i) {
      // Streamed rows of this tile: query positions (dK/dV) or key positions.
      const int pos0 = ti * kBS + half * kCols;
      bool need_mask;
      if constexpr (kDkv)
        need_mask = p.causal && pos0 < row0 + 127;
      else
        need_mask = pos0 + kCols > N || (p.causal && pos0 + kCols - 1 > row0);
      ok = need_mask ? step(std::true_type{}, i, pos0) : step(std::false_type{}, i, pos0);
      if (++ti == last) ti = first;
    }

    // ------------------------------------------------------------ epilogue
    // dK/dV: warpgroup 0 writes dK (acc 0), warpgroup 1 dV (acc 1); dQ: each
    // warpgroup half of the columns.
    if (nt > 0 && ok) ok = mbar_wait_warp(bar_done, 0, abort_flag, kDevTimeoutO);
    tc_fence_after();
    const bool row_ok = my < (kDkv ? N : M);
    T* out;
    float mul;
    int col0, ncol;
    uint32_t t_acc;
    if constexpr (kDkv) {
      const bool is_v = half == 1;
      out = reinterpret_cast<T*>(is_v ? p.dv : p.dk);
      const int64_t ss = is_v ? p.dv_ss : p.dk_ss, sh = is_v ? p.dv_sh : p.dk_sh, sb = is_v ? p.dv_sb : p.dk_sb;
      out += (p.cu_k ? k_row0 * ss : b * sb) + h * sh + my * ss;
      mul = is_v ? exp2f(-BwdElem<T>::kPExp) : p.scale * unscale;
      col0 = dcol0;
      ncol = kOut;
      t_acc = tmem + lane_base + C::kTmemAcc + (is_v ? kOut : 0);
    } else {
      out = reinterpret_cast<T*>(p.dq) + (p.cu_q ? q_row0 * p.dq_ss : b * p.dq_sb) + h * p.dq_sh + my * p.dq_ss;
      mul = p.scale * unscale;
      col0 = half * (kOut / 2);
      ncol = kOut / 2;
      t_acc = tmem + lane_base + C::kTmemAcc + col0;
    }
    if (ok) {
#pragma unroll 1
      for (int cc = 0; cc < ncol / 32; ++cc) {
        float v[32];
        if (nt > 0) {
          uint32_t rr[32];
          tmem_ld32(t_acc + cc * 32, rr);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(rr[e]) * mul;
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;  // no pair is visible
        }
        const int left = p.D - col0 - cc * 32;
        if (row_ok && left > 0) bwd_store32<T>(out + col0 + cc * 32, v, left);
      }
    }
  }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int kDP>
__global__ void __launch_bounds__(384, 1)
    fa_bwd_kernel(const __grid_constant__ FaBwdParams p, const __grid_constant__ CUtensorMap k_a,
                  const __grid_constant__ CUtensorMap v_a, const __grid_constant__ CUtensorMap q_b,
                  const __grid_constant__ CUtensorMap g_b, const __grid_constant__ CUtensorMap q_a,
                  const __grid_constant__ CUtensorMap g_a, const __grid_constant__ CUtensorMap k_b,
                  const __grid_constant__ CUtensorMap v_b) {
  extern __shared__ uint8_t smem_raw[];
  const int x = static_cast<int>(blockIdx.x);
  if (x < p.num_dkv)
    fa_bwd_body<T, kDP, true>(p, &k_a, &v_a, &q_b, &g_b, x, smem_raw);
  else
    fa_bwd_body<T, kDP, false>(p, &q_a, &g_a, &k_b, &v_b, x - p.num_dkv, smem_raw);
}

}  // namespace fab
