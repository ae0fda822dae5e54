// The attention backward's translation unit of libfa_b200.so: its kernels,
// their launch and the C entry points.  Compiled apart from capi.cu so that
// the forward kernels' register allocation does not depend on it; like every
// unit it has its own copy of the device status word.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "fa_b200.h"
#include "fa_internal.h"
#include "fa_bwd_kernel.cuh"

namespace fab {

int fa_bwd_take_device_error(int* code) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_fab_device_error, sizeof(int)) != cudaSuccess) return kErrCuda;
  if (v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_fab_device_error, &zero, sizeof(int)) != cudaSuccess) return kErrCuda;
  }
  *code = v;
  return kOk;
}

// Read by every later launch.
static std::atomic<int> g_spared_tries{0}, g_starve_bytes{0};
void fa_bwd_set_wait_limit(uint64_t ns) {
  g_spared_tries = ns == 0 || ns / 1000 >= kWaitTries ? 0 : kWaitTries - std::max(static_cast<int>(ns / 1000), 1);
}
void fa_bwd_starve_loads(bool starve) { g_starve_bytes = starve ? 16 : 0; }

namespace {

int padded_head_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
int stat_rows(int D) { return D <= 128 ? 128 : 64; }  // BwdCfg::kBS

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// A slice no shorter than this is worth its own read-out (see choose_slices).
constexpr int64_t kMinSliceTiles = 6;
constexpr int kSms = 148;  // plans depend on sizes only, so that results do not depend on the device at hand

// What a call launches and how its workspace is laid out (byte offsets).
struct BwdPlan {
  int bs;  // rows of a streamed tile
  int q_tiles, k_tiles;
  int64_t stat_tiles;
  int dkv_slice_len, dkv_slices, dq_slice_len, dq_slices;
  int64_t part_k_tiles, part_q_tiles;
  int64_t key_tiles;
  int64_t dkv_tiles, dq_tiles;  // stationary tiles of all heads, a half-head's each where a tile takes two items
  size_t row_norm, tile_max, key_max, dkv_part, dq_part, bytes;
};

// Streamed tiles a tile works through, summed over the tiles of one head (of
// the longest sequence).
int64_t streamed_tiles(int64_t tiles, int64_t other_rows, int bs, bool causal, bool dkv) {
  const int64_t all = ceil_div(other_rows, bs);
  if (!causal) return tiles * all;
  int64_t sum = 0;
  for (int64_t t = 0; t < tiles; ++t) {
    const int64_t n = dkv ? all - t * 128 / bs : ceil_div(std::min(other_rows, (t + 1) * 128), bs);
    sum += n > 0 ? n : 0;
  }
  return sum;
}

// Slices of the longest tile's `longest` streamed tiles when an SM's share of
// the whole work is `share` of them: a tile half as long again as 5/4 of the
// share would finish last, alone.  A slice costs a round of fp32 sums and the
// join kernel.  Measured on B200, sliced and unsliced: 28 heads over 4, S 2048
// causal 114 against 183 us; 4 over 1, S 4096, D 256 causal 200 against 359;
// 8 heads, 1 query, 32768 keys 124 against 364; one head, S 1024 causal, 41
// against 59.  Slices of half the share cost 8 to 50 % more than these, of
// 3/2 of it up to 14 % (one head, S 8192, causal); a minimum of 4 tiles 20 %
// more at one head, S 1024.
void choose_slices(int64_t longest, double share, int* len, int* slices) {
  const int64_t want = std::max<int64_t>(kMinSliceTiles, static_cast<int64_t>(share * 1.25 + 0.5));
  *len = static_cast<int>(std::min<int64_t>(longest < 1 ? 1 : longest, want));
  *slices = 1;
  if (longest * 2 >= want * 3) *slices = static_cast<int>(std::min<int64_t>(ceil_div(longest, want), 1 << 15));
  if (*slices == 1) *len = 0x7fffffff;
}

BwdPlan make_plan(const fab_attention_bwd_params* p) {
  BwdPlan w{};
  const bool packed = p->cu_seqlens_q != nullptr;
  const int bs = w.bs = stat_rows(p->head_dim);
  const int dsplit = p->head_dim > 128 ? 2 : 1;
  const int group = p->heads_q / p->heads_kv;
  const int64_t M = packed ? std::min(p->seqlen_q, p->total_q) : p->seqlen_q;
  const int64_t N = packed ? std::min(p->seqlen_k, p->total_k) : p->seqlen_k;
  w.q_tiles = static_cast<int>(ceil_div(M, 128));
  w.k_tiles = static_cast<int>(ceil_div(N, 128));
  // Tiles of one head in the numbering of the statistics and partial sums.
  w.stat_tiles = packed ? p->total_q / bs + int64_t(p->batch) + 1 : ceil_div(M, bs);
  w.part_q_tiles = packed ? p->total_q / 128 + int64_t(p->batch) + 1 : w.q_tiles;
  w.part_k_tiles = packed ? p->total_k / 128 + int64_t(p->batch) + 1 : w.k_tiles;
  const int64_t per_q = int64_t(p->heads_q) * (packed ? 1 : p->batch), per_kv = int64_t(p->heads_kv) * (packed ? 1 : p->batch);
  // The work in products of 128 x bs x 128: a streamed tile costs a dK/dV item
  // four (S, dP, dV, dK) and a dQ item three.  A packed batch's lengths are
  // not known here; its tiles are taken to be as long as the longest.
  const bool causal = p->causal != 0;
  double dkv = 0, dq = 0;
  if (w.k_tiles > 0) dkv = double(streamed_tiles(w.k_tiles, M, bs, causal, true)) / w.k_tiles * group * dsplit * per_kv * w.part_k_tiles;
  if (w.q_tiles > 0) dq = double(streamed_tiles(w.q_tiles, N, bs, causal, false)) / w.q_tiles * per_q * w.part_q_tiles;
  const double share = (4 * dkv + 3 * dq) / kSms;
  // (Where there is no tile, a long sum of nothing is not cut: no item would
  // write its slices, and there is nothing to join.)
  choose_slices(w.k_tiles > 0 ? ceil_div(M, bs) * group : 0, share / 4, &w.dkv_slice_len, &w.dkv_slices);
  choose_slices(w.q_tiles > 0 ? ceil_div(N, bs) : 0, share / 3, &w.dq_slice_len, &w.dq_slices);
  const int64_t tiles = w.stat_tiles * per_q;
  size_t at = round256(size_t(tiles) * 2 * bs * sizeof(float));
  w.row_norm = at;
  if (p->dtype == kDtypeF16) at += round256(size_t(tiles) * bs * sizeof(float));
  w.tile_max = at;
  if (p->dtype == kDtypeF16) at += round256(size_t(tiles) * sizeof(float));
  w.key_max = at;
  w.key_tiles = packed ? p->total_k / bs + int64_t(p->batch) + 1 : ceil_div(N, bs);
  if (p->dtype == kDtypeF16) at += round256(size_t(w.key_tiles) * per_kv * sizeof(float));
  w.dkv_tiles = int64_t(p->batch) * p->heads_kv * w.k_tiles * dsplit;
  w.dq_tiles = int64_t(p->batch) * p->heads_q * w.q_tiles;
  const int dp = padded_head_dim(p->head_dim);
  w.dkv_part = at;
  if (w.dkv_slices > 1) at += size_t(w.part_k_tiles) * per_kv * w.dkv_slices * 2 * dp * 128 * sizeof(float);
  w.dq_part = at;
  if (w.dq_slices > 1) at += size_t(w.part_q_tiles) * per_q * w.dq_slices * dp * 128 * sizeof(float);
  w.bytes = at;
  return w;
}

// Can the items, the heads of both kinds and the tiles of one head be numbered
// in 31 bits?
bool numbered(const fab_attention_bwd_params* p, const BwdPlan& w) {
  constexpr double kMost = 0x7fffffff;
  return double(w.dkv_tiles) * w.dkv_slices + double(w.dq_tiles) * w.dq_slices <= kMost &&
         double(p->batch) * (double(p->heads_q) + p->heads_kv) + 65538 <= kMost && w.stat_tiles <= kMost &&
         w.key_tiles <= kMost && w.part_q_tiles <= kMost && w.part_k_tiles <= kMost;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Outer strides in whole 16-byte units; a dim of one element has none.
bool strides16(int64_t s_b, int64_t batch, int64_t s_h, int64_t heads, int64_t s_s, int64_t rows) {
  return (batch <= 1 || s_b % 8 == 0) && (heads <= 1 || s_h % 8 == 0) && (rows <= 1 || s_s % 8 == 0);
}

// Everything the host can check.  *empty: no gradient has an element.
int validate(const fab_attention_bwd_params* p, bool* empty) {
  *empty = false;
  if (p == nullptr) return kErrInvalidArg;
  if (p->dtype != kDtypeF16 && p->dtype != kDtypeBF16) return p->dtype == kDtypeF32 ? kErrUnsupported : kErrInvalidArg;
  if (p->batch < 0 || p->heads_q < 0 || p->heads_kv < 0 || p->seqlen_q < 0 || p->seqlen_k < 0 || p->head_dim <= 0)
    return kErrInvalidArg;
  if (p->head_dim > 256) return kErrUnsupported;
  if (!std::isfinite(p->sm_scale)) return kErrInvalidArg;
  const bool packed = p->cu_seqlens_q != nullptr;
  if (packed != (p->cu_seqlens_k != nullptr)) return kErrInvalidArg;
  if (packed && ((reinterpret_cast<uintptr_t>(p->cu_seqlens_q) & 3u) || (reinterpret_cast<uintptr_t>(p->cu_seqlens_k) & 3u)))
    return kErrInvalidArg;
  if (packed && (p->total_q < 0 || p->total_k < 0)) return kErrInvalidArg;
  if (p->batch == 0) {
    *empty = true;
    return kOk;
  }
  if (p->heads_kv == 0 ? p->heads_q != 0 : p->heads_q % p->heads_kv != 0) return kErrInvalidArg;
  if (int64_t(p->batch) * p->heads_q > 0x7fffffff) return kErrUnsupported;
  const int64_t q_rows = packed ? p->total_q : p->seqlen_q, k_rows = packed ? p->total_k : p->seqlen_k;
  const int64_t nb = packed ? 1 : p->batch;
  const bool has_q = q_rows > 0 && p->heads_q > 0, has_k = k_rows > 0 && p->heads_kv > 0;
  if (!has_q && !has_k) {
    *empty = true;
    return kOk;
  }
  if (p->heads_q == 0) return kErrInvalidArg;  // key/value heads without a query head
  if (has_q) {
    if (!p->q || !p->o || !p->dout || !p->lse || !p->dq) return kErrInvalidArg;
    if (!aligned16(p->q) || !aligned16(p->o) || !aligned16(p->dout) || !aligned16(p->dq) ||
        (reinterpret_cast<uintptr_t>(p->lse) & 3u))
      return kErrInvalidArg;
    if (!strides16(p->q_stride_b, nb, p->q_stride_h, p->heads_q, p->q_stride_s, q_rows) || !strides16(p->o_stride_b, nb, p->o_stride_h, p->heads_q, p->o_stride_s, q_rows) ||
        !strides16(p->dout_stride_b, nb, p->dout_stride_h, p->heads_q, p->dout_stride_s, q_rows) ||
        !strides16(p->dq_stride_b, nb, p->dq_stride_h, p->heads_q, p->dq_stride_s, q_rows))
      return kErrInvalidArg;
  }
  if (has_k) {
    if (!p->k || !p->v || !p->dk || !p->dv) return kErrInvalidArg;
    if (!aligned16(p->k) || !aligned16(p->v) || !aligned16(p->dk) || !aligned16(p->dv)) return kErrInvalidArg;
    if (!strides16(p->k_stride_b, nb, p->k_stride_h, p->heads_kv, p->k_stride_s, k_rows) || !strides16(p->v_stride_b, nb, p->v_stride_h, p->heads_kv, p->v_stride_s, k_rows) ||
        !strides16(p->dk_stride_b, nb, p->dk_stride_h, p->heads_kv, p->dk_stride_s, k_rows) || !strides16(p->dv_stride_b, nb, p->dv_stride_h, p->heads_kv, p->dv_stride_s, k_rows))
      return kErrInvalidArg;
  }
  return kOk;
}

template <typename T, int kBS>
void launch_stats(const FaBwdParams& kp, cudaStream_t stream) {
  constexpr bool kKeys = BwdElem<T>::kScaled;
  const int64_t rows = int64_t(kp.B) * (kp.Hq + (kKeys ? kp.Hkv : 0)) + (kp.cu_q != nullptr ? 3 : 0);
  const int64_t y = std::min<int64_t>(rows, 65535);
  const dim3 grid(static_cast<unsigned>(ceil_div(kKeys ? std::max(kp.M, kp.N) : kp.M, kBS)), static_cast<unsigned>(y),
                  static_cast<unsigned>(ceil_div(rows, y)));
  // Lanes per row: eight columns each.
  if constexpr (kBS == 64) {
    fa_bwd_stats_kernel<T, 64, 32><<<grid, kStatThreads, 0, stream>>>(kp);
  } else {
    if (kp.D <= 64)
      fa_bwd_stats_kernel<T, 128, 8><<<grid, kStatThreads, 0, stream>>>(kp);
    else
      fa_bwd_stats_kernel<T, 128, 16><<<grid, kStatThreads, 0, stream>>>(kp);
  }
}

template <typename T, int kDP, bool kTwo>
int launch(const fab_attention_bwd_params* p, const BwdPlan& w, FaBwdParams& kp, cudaStream_t stream) {
  using C = BwdCfg<kDP>;
  auto kern = fa_bwd_kernel<T, kDP, kTwo>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), C::kSmemBytes);
  if (rc) return rc;
  // The kernel's register split was sized for this launch allocation; a build
  // compiled to another one is refused.
  static const int regs = [&] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, reinterpret_cast<const void*>(kern)) == cudaSuccess ? a.numRegs : -1;
  }();
  if (regs != C::kLaunchRegs) return regs < 0 ? kErrLaunch : kErrUnsupported;
  const bool packed = kp.cu_q != nullptr;
  const int64_t q_rows = packed ? kp.total_q : kp.M, k_rows = packed ? kp.total_k : kp.N;
  const CUtensorMapDataType dt =
      p->dtype == kDtypeBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int mb = packed ? 1 : kp.B;
  // Each operand as a stationary (128 rows) and as a streamed (kBS rows) tile.
  CUtensorMap qa, ga, ka, va, qb, gb, kb, vb;
  auto map = [&](CUtensorMap* m, const void* base, int64_t rows, int heads, int64_t ss, int64_t sh, int64_t sb, int box) {
    return make_bhsd_map(m, base, dt, 2, kp.D, static_cast<int>(rows), heads, mb, ss, sh, packed ? 0 : sb, 64, box,
                         CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (q_rows > 0 && k_rows > 0) {
    if ((rc = map(&qa, p->q, q_rows, kp.Hq, p->q_stride_s, p->q_stride_h, p->q_stride_b, 128))) return rc;
    if ((rc = map(&ga, p->dout, q_rows, kp.Hq, p->dout_stride_s, p->dout_stride_h, p->dout_stride_b, 128))) return rc;
    if ((rc = map(&ka, p->k, k_rows, kp.Hkv, p->k_stride_s, p->k_stride_h, p->k_stride_b, 128))) return rc;
    if ((rc = map(&va, p->v, k_rows, kp.Hkv, p->v_stride_s, p->v_stride_h, p->v_stride_b, 128))) return rc;
    if constexpr (C::kBS == 128) {
      qb = qa, gb = ga, kb = ka, vb = va;
    } else {
      if ((rc = map(&qb, p->q, q_rows, kp.Hq, p->q_stride_s, p->q_stride_h, p->q_stride_b, C::kBS))) return rc;
      if ((rc = map(&gb, p->dout, q_rows, kp.Hq, p->dout_stride_s, p->dout_stride_h, p->dout_stride_b, C::kBS))) return rc;
      if ((rc = map(&kb, p->k, k_rows, kp.Hkv, p->k_stride_s, p->k_stride_h, p->k_stride_b, C::kBS))) return rc;
      if ((rc = map(&vb, p->v, k_rows, kp.Hkv, p->v_stride_s, p->v_stride_h, p->v_stride_b, C::kBS))) return rc;
    }
  } else {
    // Nothing attends to anything: the items write zeros and read no map.
    qa = ga = ka = va = qb = gb = kb = vb = CUtensorMap{};
  }
  const int64_t dkv = w.dkv_tiles * kp.dkv_slices, grid = dkv + w.dq_tiles * kp.dq_slices;
  kp.num_dkv = static_cast<int>(dkv);
  const bool stats = q_rows > 0 && k_rows > 0 && kp.M > 0;
  if (stats)
    launch_stats<T, C::kBS>(kp, stream);
  else if (packed)
    fa_bwd_zero_rest_kernel<T><<<dim3(8, 3), 256, 0, stream>>>(kp);
  if (grid > 0) {
    // Set up while the statistics kernel still runs.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = stats ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kern, kp, ka, va, qb, gb, qa, ga, kb, vb) != cudaSuccess) {
      cudaGetLastError();
      return kErrLaunch;
    }
    if (kp.dkv_slices > 1)
      fa_bwd_join_kernel<T, kDP, true>
          <<<dim3(static_cast<unsigned>(w.dkv_tiles), C::kOutDkv / 32), 256, 0, stream>>>(kp);
    if (kp.dq_slices > 1)
      fa_bwd_join_kernel<T, kDP, false>
          <<<dim3(static_cast<unsigned>(w.dq_tiles), kDP / 64), 256, 0, stream>>>(kp);
  }
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

template <typename T, int kDP>
int launch_parts(const fab_attention_bwd_params* p, const BwdPlan& w, FaBwdParams& kp, cudaStream_t stream) {
  const bool two = kp.few_rows || kp.cu_q != nullptr || std::min(kp.M, kp.N) <= kTwoPartLength;
  return two ? launch<T, kDP, true>(p, w, kp, stream) : launch<T, kDP, false>(p, w, kp, stream);
}

template <typename T>
int launch_dim(const fab_attention_bwd_params* p, const BwdPlan& w, FaBwdParams& kp, cudaStream_t stream) {
  switch (padded_head_dim(kp.D)) {
    case 64:
      return launch_parts<T, 64>(p, w, kp, stream);
    case 128:
      return launch_parts<T, 128>(p, w, kp, stream);
    default:
      return launch_parts<T, 256>(p, w, kp, stream);
  }
}

}  // namespace
}  // namespace fab

using namespace fab;

extern "C" {

int fab_attention_bwd_workspace(const fab_attention_bwd_params* p, size_t* bytes) {
  if (bytes == nullptr) return kErrInvalidArg;
  *bytes = 0;
  bool empty = false;
  const int rc = validate(p, &empty);
  if (rc || empty) return rc;
  const BwdPlan w = make_plan(p);
  if (!numbered(p, w)) return kErrUnsupported;
  *bytes = w.bytes;
  return kOk;
}

int fab_attention_bwd(const fab_attention_bwd_params* p, void* stream) {
  bool empty = false;
  const int rc = validate(p, &empty);
  if (rc || empty) return rc;
  const BwdPlan w = make_plan(p);
  if (!numbered(p, w)) return kErrUnsupported;
  if (w.bytes > 0 && (p->workspace == nullptr || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) != 0 ||
                      p->workspace_bytes < w.bytes))
    return kErrWorkspace;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  FaBwdParams kp{};
  kp.o = p->o;
  kp.dout = p->dout;
  kp.lse = p->lse;
  kp.dq = p->dq;
  kp.dk = p->dk;
  kp.dv = p->dv;
  kp.o_sb = p->o_stride_b;
  kp.o_sh = p->o_stride_h;
  kp.o_ss = p->o_stride_s;
  kp.g_sb = p->dout_stride_b;
  kp.g_sh = p->dout_stride_h;
  kp.g_ss = p->dout_stride_s;
  kp.l_sb = p->lse_stride_b;
  kp.l_sh = p->lse_stride_h;
  kp.l_ss = p->lse_stride_s;
  kp.dq_sb = p->dq_stride_b;
  kp.dq_sh = p->dq_stride_h;
  kp.dq_ss = p->dq_stride_s;
  kp.dk_sb = p->dk_stride_b;
  kp.dk_sh = p->dk_stride_h;
  kp.dk_ss = p->dk_stride_s;
  kp.dv_sb = p->dv_stride_b;
  kp.dv_sh = p->dv_stride_h;
  kp.dv_ss = p->dv_stride_s;
  kp.stats = reinterpret_cast<float*>(ws);
  kp.row_norm = reinterpret_cast<float*>(ws + w.row_norm);
  kp.tile_max = reinterpret_cast<float*>(ws + w.tile_max);
  kp.key_max = reinterpret_cast<float*>(ws + w.key_max);
  kp.key_tiles = static_cast<int>(w.key_tiles);
  kp.v = p->v;
  kp.v_sb = p->v_stride_b;
  kp.v_sh = p->v_stride_h;
  kp.v_ss = p->v_stride_s;
  kp.stat_tiles = static_cast<int>(w.stat_tiles);
  kp.B = p->batch;
  kp.Hq = p->heads_q;
  kp.Hkv = p->heads_kv;
  kp.M = p->seqlen_q;
  kp.N = p->seqlen_k;
  kp.D = p->head_dim;
  kp.group = p->heads_q / p->heads_kv;
  kp.scale = p->sm_scale;
  // A scale of zero keeps its zero in dq and dk; inside the exponential a
  // vanishing one does the same and keeps masked scores masked.
  kp.scale_log2 = (p->sm_scale == 0.f ? 1e-30f : p->sm_scale) * 1.4426950408889634f;
  kp.causal = p->causal ? 1 : 0;
  kp.few_rows = int64_t(p->heads_q) * (p->cu_seqlens_q != nullptr ? p->total_q : int64_t(p->batch) * p->seqlen_q) <= kTwoPartRows;
  kp.cu_q = p->cu_seqlens_q;
  kp.cu_k = p->cu_seqlens_k;
  kp.total_q = p->total_q;
  kp.total_k = p->total_k;
  if (kp.cu_q != nullptr) {
    kp.M = kp.M < kp.total_q ? kp.M : kp.total_q;
    kp.N = kp.N < kp.total_k ? kp.N : kp.total_k;
  }
  kp.spared_tries = g_spared_tries;
  kp.starve_bytes = g_starve_bytes;
  kp.q_tiles = w.q_tiles;
  kp.k_tiles = w.k_tiles;
  kp.dkv_slice_len = w.dkv_slice_len;
  kp.dkv_slices = w.dkv_slices;
  kp.dq_slice_len = w.dq_slice_len;
  kp.dq_slices = w.dq_slices;
  kp.part_k_tiles = static_cast<int>(w.part_k_tiles);
  kp.part_q_tiles = static_cast<int>(w.part_q_tiles);
  kp.dkv_part = reinterpret_cast<float*>(ws + w.dkv_part);
  kp.dq_part = reinterpret_cast<float*>(ws + w.dq_part);
  auto st = static_cast<cudaStream_t>(stream);
  return p->dtype == kDtypeBF16 ? launch_dim<__nv_bfloat16>(p, w, kp, st) : launch_dim<__half>(p, w, kp, st);
}

}  // extern "C"
