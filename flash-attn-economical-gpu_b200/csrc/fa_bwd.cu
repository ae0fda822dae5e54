// The attention backward's translation unit of libfa_b200.so: its kernels,
// their launch and the C entry points.  Compiled apart from capi.cu so that
// the forward kernels' register allocation does not depend on it; like every
// unit it has its own copy of the device status word.
#include <cudaTypedefs.h>

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

namespace {

int padded_head_dim(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
int stat_rows(int D) { return D <= 128 ? 128 : 64; }  // BwdCfg::kBS

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t round256(size_t x) { return (x + 255) / 256 * 256; }

struct BwdWorkspace {
  int64_t tiles_per_head;
  size_t row_exp, tile_max, bytes;  // byte offsets behind the statistics
};

BwdWorkspace workspace_plan(const fab_attention_bwd_params* p) {
  BwdWorkspace w{};
  const int bs = stat_rows(p->head_dim);
  int64_t tiles;
  if (p->cu_seqlens_q != nullptr) {
    w.tiles_per_head = p->total_q / bs + int64_t(p->batch) + 1;
    tiles = w.tiles_per_head * p->heads_q;
  } else {
    w.tiles_per_head = ceil_div(p->seqlen_q, bs);
    tiles = w.tiles_per_head * p->heads_q * p->batch;
  }
  w.row_exp = round256(size_t(tiles) * 2 * bs * sizeof(float));
  w.tile_max = w.bytes = w.row_exp;
  if (p->dtype == kDtypeF16) {
    w.tile_max = w.row_exp + round256(size_t(tiles) * bs * sizeof(float));
    w.bytes = w.tile_max + round256(size_t(tiles) * sizeof(float));
  }
  return w;
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
  const dim3 grid(static_cast<unsigned>(ceil_div(kp.M, kBS)), static_cast<unsigned>(kp.B * kp.Hq));
  // Lanes per row: eight columns each.
  if constexpr (kBS == 64) {
    fa_bwd_stats_kernel<T, 64, 32><<<grid, 256, 0, stream>>>(kp);
  } else {
    if (kp.D <= 64)
      fa_bwd_stats_kernel<T, 128, 8><<<grid, 256, 0, stream>>>(kp);
    else
      fa_bwd_stats_kernel<T, 128, 16><<<grid, 256, 0, stream>>>(kp);
  }
}

template <typename T, int kDP>
int launch(const fab_attention_bwd_params* p, FaBwdParams& kp, cudaStream_t stream) {
  using C = BwdCfg<kDP>;
  auto kern = fa_bwd_kernel<T, kDP>;
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
    if (static_cast<int64_t>(kp.B) * kp.Hq > 65535) return kErrUnsupported;
    if (kp.M > 0) launch_stats<T, C::kBS>(kp, stream);
  } else {
    // Nothing attends to anything: the CTAs write zeros and read no map.
    qa = ga = ka = va = qb = gb = kb = vb = CUtensorMap{};
  }
  if (packed) fa_bwd_zero_rest_kernel<T><<<dim3(8, 3), 256, 0, stream>>>(kp);
  const int64_t dkv = static_cast<int64_t>(kp.B) * kp.Hkv * kp.k_tiles * C::kDSplit;
  const int64_t grid = dkv + static_cast<int64_t>(kp.B) * kp.Hq * kp.q_tiles;
  if (grid > 0x7fffffffLL) return kErrUnsupported;
  kp.num_dkv = static_cast<int>(dkv);
  if (grid > 0)
    kern<<<static_cast<unsigned>(grid), C::kThreads, C::kSmemBytes, stream>>>(kp, ka, va, qb, gb, qa, ga, kb, vb);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

template <typename T>
int launch_dim(const fab_attention_bwd_params* p, FaBwdParams& kp, cudaStream_t stream) {
  switch (padded_head_dim(kp.D)) {
    case 64:
      return launch<T, 64>(p, kp, stream);
    case 128:
      return launch<T, 128>(p, kp, stream);
    default:
      return launch<T, 256>(p, kp, stream);
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
  *bytes = workspace_plan(p).bytes;
  return kOk;
}

int fab_attention_bwd(const fab_attention_bwd_params* p, void* stream) {
  bool empty = false;
  const int rc = validate(p, &empty);
  if (rc || empty) return rc;
  const BwdWorkspace w = workspace_plan(p);
  if (w.bytes > 0 && (p->workspace == nullptr || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) != 0 ||
                      p->workspace_bytes < w.bytes))
    return kErrWorkspace;
  if (w.tiles_per_head > 0x7fffffffLL) return kErrUnsupported;
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
  kp.row_exp = reinterpret_cast<float*>(ws + w.row_exp);
  kp.tile_max = reinterpret_cast<float*>(ws + w.tile_max);
  kp.stat_tiles = static_cast<int>(w.tiles_per_head);
  kp.B = p->batch;
  kp.Hq = p->heads_q;
  kp.Hkv = p->heads_kv;
  kp.M = p->seqlen_q;
  kp.N = p->seqlen_k;
  kp.D = p->head_dim;
  kp.group = p->heads_q / p->heads_kv;
  kp.scale = p->sm_scale;
  kp.scale_log2 = p->sm_scale * 1.4426950408889634f;
  kp.causal = p->causal ? 1 : 0;
  kp.cu_q = p->cu_seqlens_q;
  kp.cu_k = p->cu_seqlens_k;
  kp.total_q = p->total_q;
  kp.total_k = p->total_k;
  if (kp.cu_q != nullptr) {
    kp.M = kp.M < kp.total_q ? kp.M : kp.total_q;
    kp.N = kp.N < kp.total_k ? kp.N : kp.total_k;
  }
  kp.q_tiles = static_cast<int>(ceil_div(kp.M, 128));
  kp.k_tiles = static_cast<int>(ceil_div(kp.N, 128));
  auto st = static_cast<cudaStream_t>(stream);
  return p->dtype == kDtypeBF16 ? launch_dim<__nv_bfloat16>(p, kp, st) : launch_dim<__half>(p, kp, st);
}

}  // extern "C"
