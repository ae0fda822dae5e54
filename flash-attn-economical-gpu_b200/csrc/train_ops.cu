// Translation unit of the training operators around the attention: layer
// norm and multi-axis rotary embedding (train_ops.cuh), with their C entry
// points.  The unit has its own copy of the device status word.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "fa_b200.h"
#include "fa_internal.h"
#include "train_ops.cuh"

namespace fab {

int train_ops_take_device_error(int* code) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_fab_device_error, sizeof(int)) != cudaSuccess) return kErrCuda;
  if (v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_fab_device_error, &zero, sizeof(int)) != cudaSuccess) return kErrCuda;
  }
  *code = v;
  return kOk;
}

int train_ops_set_wait_limit(uint64_t ns) {
  return cudaMemcpyToSymbol(g_fab_wait_limit_ns, &ns, sizeof(ns)) == cudaSuccess ? kOk : kErrCuda;
}

// Read by every later launch.
static std::atomic<int> g_starve_row{-1};
void train_ops_starve_row_sums(int row) { g_starve_row = row; }

namespace {

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int elt_bytes(int dtype) { return dtype == kDtypeF32 ? 4 : 2; }

// CTAs of the layer norm backward kernels, which are also the lines of partial
// dw/db sums: as many as stay resident (an SM holds 2048 16-byte vectors of
// the rows being worked on: two stages of x, dy and dres, or three of x and a
// residual, take 192 KB of shared memory), by sizes alone, so that the order of the sums does not
// depend on the device.
constexpr int kSms = 148;
constexpr int kResidentVectors = 2048;
// The most lines of any path.
int64_t max_lines(int64_t rows, int cols) {
  const int64_t per_cta = std::max<int64_t>(ceil_div(cols, 8), 64);
  return std::min<int64_t>(rows, kSms * std::max<int64_t>(2, 2048 / per_cta));
}

int launched() { return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch; }

// Threads of a CTA whose every thread holds nv vectors of v columns.
int row_threads(int cols, int v, int nv) { return static_cast<int>(ceil_div(ceil_div(cols, v * nv), 32) * 32); }

template <typename T, typename W, int V, int NV, int kMaxThreads>
int run_fwd(const LayerNormParams& p, cudaStream_t st) {
  layernorm_fwd_kernel<T, W, V, NV, kMaxThreads><<<static_cast<unsigned>(p.rows), row_threads(p.cols, V, NV), 0, st>>>(p);
  return launched();
}

// Clusters of `ctas` CTAs that are resident together: all that the SMs have
// room for, but the GPU's processing clusters are not a multiple of four CTAs
// each.  (Measured: of the clusters of 4 and 8 that fill every SM some had to
// wait for a second round; 4096 x 16384 fp32 backward 246 against 174 us.)
int64_t resident(int64_t per_sm, int ctas) { return kSms * per_sm * (ctas > 2 ? 7 : 8) / (8 * ctas); }

// How rows of `places` places (columns, and in front of them those of a cut
// 16-byte piece) are shared out, `per_cta` at most to a CTA: the CTAs of a row
// (a cluster where there are several), and each one's places.
struct Spread {
  int ctas, span;
};
Spread spread_row(int places, int per_cta, int unit) {
  int ctas = 1;
  while (int64_t(ctas) * per_cta < places) ctas *= 2;
  return {ctas, static_cast<int>(ceil_div(ceil_div(places, ctas), unit) * unit)};
}

// Rows whose 16-byte pieces do not start where the rows do: workable all the
// same where a row starts at the same place of a piece in every tensor.  Each
// worker then takes every 8th row or a multiple of that, which start alike.
enum class Rows { kEven, kOdd, kAny };
struct RowTensor {
  const void* p;  // or null
  int64_t ld;
};
template <int N>
Rows rows_kind(const RowTensor (&t)[N], int cols, int v, bool even_weights) {
  bool even = even_weights && cols % v == 0, alike = true;
  for (const RowTensor& x : t) {
    if (x.p == nullptr) continue;
    even = even && aligned(x.p, 16) && x.ld % v == 0;
    alike = alike && (reinterpret_cast<uintptr_t>(x.p) - reinterpret_cast<uintptr_t>(t[0].p)) % 16 == 0 &&
            (x.ld - t[0].ld) % v == 0 && x.ld >= 0;
  }
  return even ? Rows::kEven : alike ? Rows::kOdd : Rows::kAny;
}
int64_t like_workers(int64_t workers, int64_t rows, bool odd) {
  return !odd || workers >= rows || workers < 8 ? std::min(workers, rows) : workers / 8 * 8;
}

// `workers` rows at a time, each on `ctas` CTAs.
template <typename P>
int launch_rows(void (*kern)(P), const P& p, int64_t workers, int ctas, int threads, size_t smem, cudaStream_t st) {
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), 200 * 1024)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(workers * ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess) return kOk;
  cudaGetLastError();
  return kErrLaunch;
}

// Rows stream through resident CTAs where each gets at least this many (kFewRows
// otherwise: nothing was launched).  Measured, streamed against a CTA for every
// row: 8192 x 3584 bf16 with a residual 47.8 against 57.3 us, 1200 x 3584 15.9
// against 16.4, 148 x 3584 10.2 against 8.2; 32768 x 256 20.5 against 25.8.
constexpr int64_t kStreamRows = 2;
constexpr int kFewRows = -1;

template <typename T, typename W, int NV, int kMaxThreads, int kMinCtas, bool kWide, bool kOdd>
int run_fwd_stream(LayerNormParams p, cudaStream_t st) {
  constexpr int kStages = 3, V = 16 / sizeof(T);
  const int places = p.cols + (kOdd ? V - 1 : 0);
  const Spread row = spread_row(places, kWide ? 1024 * V : places, 32 * V);
  p.span = row.span;
  const int threads = row_threads(kWide ? row.span : places, V, NV);
  const int64_t most = resident(std::max(1, kResidentVectors / (threads * NV)), row.ctas);
  if (!kOdd && p.rows < kStreamRows * most) return kFewRows;
  const int64_t workers = like_workers(most, p.rows, kOdd);
  return launch_rows(layernorm_fwd_stream_kernel<T, W, NV, kMaxThreads, kMinCtas, kStages, kWide, kOdd>, p, workers, row.ctas,
                     threads, size_t(kStages) * NV * 2 * threads * 16, st);
}

// Rows of any length and place.
int long_threads(int cols) { return static_cast<int>(std::min<int64_t>(1024, ceil_div(cols, 32) * 32)); }

template <typename T, typename W>
int fwd(const LayerNormParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const RowTensor rows[] = {{p.x, p.ld_x}, {p.y, p.ld_y}, {p.residual, p.ld_res}, {p.residual ? p.x_out : nullptr, p.ld_xo}};
  const Rows kind = rows_kind(rows, p.cols, V, aligned(p.w, 16) && aligned(p.bias, 16));
  if (kind == Rows::kOdd && p.cols + V - 1 <= 1024 * V) return run_fwd_stream<T, W, 4, 256, 2, false, true>(p, st);
  if (kind == Rows::kOdd && p.cols + V - 1 <= kMaxCluster * 1024 * V) return run_fwd_stream<T, W, 4, 256, 2, true, true>(p, st);
  if (kind == Rows::kEven) {
    // Up to 64 vectors a warp is a CTA: at 32768 x 256 20.5 us against 24.2
    // with the wider form.
    int rc = kFewRows;
    if (p.cols <= 64 * V)
      rc = run_fwd_stream<T, W, 2, 32, 12, false, false>(p, st);
    else if (p.cols <= 1024 * V)
      rc = run_fwd_stream<T, W, 4, 256, 2, false, false>(p, st);
    else if (p.cols <= kMaxCluster * 1024 * V)
      rc = run_fwd_stream<T, W, 4, 256, 2, true, false>(p, st);
    if (rc != kFewRows) return rc;
    // One vector per thread up to 512 threads, the quickest for one row's
    // latency (148 x 3584 8.2 us against 10.2 with two); two up to there,
    // then four (148 x 8192 10.2 us with two, 16.3 with four).
    if (p.cols <= 512 * V) return run_fwd<T, W, V, 1, 512>(p, st);
    if (p.cols <= 1024 * V) return run_fwd<T, W, V, 2, 512>(p, st);
    if (p.cols <= 4096 * V) return run_fwd<T, W, V, 4, 1024>(p, st);
  }
  layernorm_fwd_long_kernel<T, W><<<static_cast<unsigned>(p.rows), long_threads(p.cols), 0, st>>>(p);
  return launched();
}

// A launch that is set up while the previous kernel of the stream runs; the
// kernel itself waits before it reads that one's results.
template <typename... Args, typename... Given>
int launch_after(void (*kernel)(Args...), unsigned grid, unsigned block, cudaStream_t st, Given... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return kOk;
  cudaGetLastError();
  return kErrLaunch;
}

template <typename T, typename W, int NV, int kMaxThreads, int kMinCtas, bool kWarpRow, bool kWide, bool kOdd>
int run_bwd(LayerNormBwdParams p, int* lines, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int places = p.cols + (kOdd ? V - 1 : 0);
  const Spread row = spread_row(places, kWide ? 1024 * V : places, 32 * V);
  p.span = row.span;
  const int threads = kWarpRow ? kMaxThreads : row_threads(kWide ? row.span : places, V, NV);
  // Rows on their way at once per worker, this one included.
  constexpr int kStages = 2;
  size_t smem = size_t(kStages) * NV * 3 * threads * 16;
  const int vectors = threads * NV;  // of one row, or of all the warps' rows
  const int64_t rows = kWarpRow ? ceil_div(p.rows, threads / 32) : p.rows;  // one after another, if by one CTA
  // Every CTA leaves a line of sums, as many bytes as two fp32 rows, which the
  // finish kernel reads: with few rows in all, fewer CTAs of several rows each,
  // but one per SM.  Measured, against a row each: 4096 x 1024 bf16 (four) 19.4
  // and 25.6 us, 600 x 3584 (two; four 21.5) 19.4 and 21.1, 4096 x 256 (two;
  // four 13.3) 11.4 and 15.3.
  constexpr int kLineRows = !kWarpRow && NV == 2 ? 4 : 2;
  const int64_t most = std::min({resident(std::max(1, kResidentVectors / vectors), row.ctas), max_lines(p.rows, p.cols),
                                 std::max<int64_t>(kSms / row.ctas, ceil_div(rows, kLineRows))});
  *lines = static_cast<int>(like_workers(most, rows, kOdd && !kWarpRow));
  if (kWarpRow) smem = std::max(smem, size_t(threads / 32) * p.cols * sizeof(float));
  return launch_rows(layernorm_bwd_kernel<T, W, NV, kMaxThreads, kMinCtas, kWarpRow, kWide, kOdd, kStages>, p, *lines,
                     row.ctas, threads, smem, st);
}

template <typename T, typename W>
int bwd(const LayerNormBwdParams& p, void* dw, void* db, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const RowTensor rows[] = {{p.x, p.ld_x}, {p.dy, p.ld_dy}, {p.dx, p.ld_dx}, {p.dres, p.ld_dres}};
  const Rows kind = rows_kind(rows, p.cols, V, aligned(p.w, 16));
  const int places = p.cols + (kind == Rows::kOdd ? V - 1 : 0);
  int rc, lines = 0;
  if (kind == Rows::kAny || places > kMaxCluster * 1024 * V) {
    lines = static_cast<int>(max_lines(p.rows, p.cols));
    // The column sums first: dx may lie over dy.
    if (p.part != nullptr)
      layernorm_bwd_long_cols_kernel<T>
          <<<dim3(static_cast<unsigned>(ceil_div(p.cols, 1024)), static_cast<unsigned>(lines)), long_threads(p.cols), 0, st>>>(p);
    layernorm_bwd_long_kernel<T, W><<<static_cast<unsigned>(p.rows), long_threads(p.cols), 0, st>>>(p);
    rc = launched();
  } else if (kind == Rows::kOdd) {
    if (places <= 64 * V)
      rc = run_bwd<T, W, 2, 256, 2, true, false, true>(p, &lines, st);
    else if (places <= 1024 * V)
      rc = run_bwd<T, W, 4, 256, 2, false, false, true>(p, &lines, st);
    else
      rc = run_bwd<T, W, 4, 256, 2, false, true, true>(p, &lines, st);
  } else if (p.cols <= 64 * V) {
    // A warp for each row (32768 x 512 bf16: 37.9 us against 50.2 with a CTA).
    rc = run_bwd<T, W, 2, 256, 2, true, false, false>(p, &lines, st);
  } else if (p.cols <= 256 * V) {
    // Two vectors per thread while that leaves four warps or more for a row
    // (8192 x 2048 bf16: 39.9 us against 44.0 with four).
    rc = run_bwd<T, W, 2, 128, 4, false, false, false>(p, &lines, st);
  } else if (p.cols <= 512 * V) {
    rc = run_bwd<T, W, 4, 128, 4, false, false, false>(p, &lines, st);
  } else if (p.cols <= 1024 * V) {
    rc = run_bwd<T, W, 4, 256, 2, false, false, false>(p, &lines, st);
  } else {
    rc = run_bwd<T, W, 4, 256, 2, false, true, false>(p, &lines, st);
  }
  if (rc || p.part == nullptr) return rc;
  return launch_after(layernorm_bwd_finish_kernel<W>, static_cast<unsigned>(ceil_div(2 * int64_t(p.cols), 32)), 1024u, st,
                      static_cast<const float*>(p.part), lines, p.cols, static_cast<W*>(dw), static_cast<W*>(db));
}

// The (T, W) pairs: weights in the activations' type or fp32.
template <typename F>
int by_types(int dtype, int w_dtype, F f) {
  if (dtype == kDtypeF32 && w_dtype == kDtypeF32) return f(float{}, float{});
  if (dtype == kDtypeBF16 && w_dtype == kDtypeBF16) return f(__nv_bfloat16{}, __nv_bfloat16{});
  if (dtype == kDtypeBF16 && w_dtype == kDtypeF32) return f(__nv_bfloat16{}, float{});
  if (dtype == kDtypeF16 && w_dtype == kDtypeF16) return f(__half{}, __half{});
  if (dtype == kDtypeF16 && w_dtype == kDtypeF32) return f(__half{}, float{});
  return kErrUnsupported;
}

template <typename T, int V>
int run_rope(RopeParams& p, cudaStream_t st) {
  const int nvec = p.half / V + (p.head_dim - 2 * p.half) / V;
  p.slots = (p.heads_q + p.heads_k + kRopeHeads - 1) / kRopeHeads;
  const int64_t blocks = ceil_div(int64_t(p.tokens) * nvec * p.slots, 256);
  if (blocks > 0x7fffffffLL) return kErrUnsupported;
  rope_axes_kernel<T, V><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);
  return launched();
}

// Can every access take V values at once?  Also settles whether the tables can.
template <typename T, int V>
bool rope_in_vectors(RopeParams& p) {
  auto even = [&](const void* ptr, int64_t a, int64_t b) { return aligned(ptr, V * sizeof(T)) && a % V == 0 && b % V == 0; };
  const bool vec = p.half % V == 0 && p.head_dim % V == 0 && even(p.q, p.q_st, p.q_sh) && even(p.q_out, p.qo_st, p.qo_sh) &&
                   (p.heads_k == 0 || (even(p.k, p.k_st, p.k_sh) && even(p.k_out, p.ko_st, p.ko_sh)));
  p.vec_table = vec && aligned(p.cos, 16) && aligned(p.sin, 16);
  for (int i = 0; i < p.axes; ++i)
    if (p.ends[i] % V != 0) p.vec_table = 0;
  return vec;
}

// 16-byte accesses, else (16-bit types, say 20 pairs of a head of 80) 8-byte
// ones, else single values.  Measured: 16384 tokens, 24 heads of 80, 12 + 8
// pairs, bf16, 45 us in 8-byte pieces, 125 in single values.
template <typename T>
int rope(RopeParams& p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (rope_in_vectors<T, V>(p)) return run_rope<T, V>(p, st);
  if constexpr (V > 4)
    if (rope_in_vectors<T, 4>(p)) return run_rope<T, 4>(p, st);
  p.vec_table = 0;
  return run_rope<T, 1>(p, st);
}

}  // namespace
}  // namespace fab

using namespace fab;

extern "C" {

int fab_layernorm(const void* x, const void* residual, const void* w, const void* bias, void* y, void* x_out,
                  float* mean, float* rstd, int64_t rows, int cols, int64_t ld_x, int64_t ld_res, int64_t ld_y,
                  int64_t ld_xo, float eps, int dtype, int w_dtype, void* stream) {
  if (rows < 0 || cols <= 0 || rows > 0x7fffffffLL) return kErrInvalidArg;
  if (!(eps >= 0.f) || !std::isfinite(eps)) return kErrInvalidArg;
  if (rows == 0) return kOk;
  if (!x || !w || !y || (residual != nullptr && x_out == nullptr) || (mean == nullptr) != (rstd == nullptr))
    return kErrInvalidArg;
  const uintptr_t e = elt_bytes(dtype), we = elt_bytes(w_dtype);
  if (!aligned(x, e) || !aligned(residual, e) || !aligned(y, e) || !aligned(x_out, e) || !aligned(w, we) ||
      !aligned(bias, we) || !aligned(mean, 4) || !aligned(rstd, 4))
    return kErrInvalidArg;
  LayerNormParams p{x, residual, w, bias, y, x_out, mean, rstd, ld_x, ld_res, ld_y, ld_xo, rows, cols, eps, 0, g_starve_row};
  auto st = static_cast<cudaStream_t>(stream);
  return by_types(dtype, w_dtype, [&](auto t, auto wt) { return fwd<decltype(t), decltype(wt)>(p, st); });
}

int fab_layernorm_bwd_workspace(int64_t rows, int cols, size_t* bytes) {
  if (bytes == nullptr || rows < 0 || cols <= 0) return kErrInvalidArg;
  *bytes = size_t(max_lines(rows, cols)) * 2 * size_t(cols) * sizeof(float);
  return kOk;
}

int fab_layernorm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd,
                      const void* dresidual, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes,
                      int64_t rows, int cols, int64_t ld_dy, int64_t ld_x, int64_t ld_dres, int64_t ld_dx, int dtype,
                      int w_dtype, void* stream) {
  if (rows < 0 || cols <= 0 || rows > 0x7fffffffLL) return kErrInvalidArg;
  const uintptr_t e = elt_bytes(dtype), we = elt_bytes(w_dtype);
  if (!aligned(dw, we) || !aligned(db, we)) return kErrInvalidArg;
  auto st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    // Sums over no rows.
    if (dw != nullptr && cudaMemsetAsync(dw, 0, size_t(cols) * we, st) != cudaSuccess) return kErrCuda;
    if (db != nullptr && cudaMemsetAsync(db, 0, size_t(cols) * we, st) != cudaSuccess) return kErrCuda;
    return kOk;
  }
  if (!dy || !x || !w || !mean || !rstd || !dx) return kErrInvalidArg;
  if (!aligned(dy, e) || !aligned(x, e) || !aligned(dresidual, e) || !aligned(dx, e) || !aligned(w, we) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return kErrInvalidArg;
  const bool sums = dw != nullptr || db != nullptr;
  if (sums && (workspace == nullptr || !aligned(workspace, 16) ||
               workspace_bytes < size_t(max_lines(rows, cols)) * 2 * size_t(cols) * sizeof(float)))
    return kErrWorkspace;
  LayerNormBwdParams p{dy, x, w, mean, rstd, dresidual, dx, sums ? static_cast<float*>(workspace) : nullptr,
                       ld_dy, ld_x, ld_dres, ld_dx, rows, cols, 0, g_starve_row};
  return by_types(dtype, w_dtype,
                  [&](auto t, auto wt) { return bwd<decltype(t), decltype(wt)>(p, dw, db, st); });
}

int fab_rope_axes(const fab_rope_axes_params* a, void* stream) {
  if (a == nullptr) return kErrInvalidArg;
  if (a->tokens < 0 || a->heads_q < 0 || a->heads_k < 0 || a->head_dim <= 0 || a->table_rows < 0) return kErrInvalidArg;
  if (a->axes < 1 || a->axes > kMaxRopeAxes) return kErrInvalidArg;
  if (a->dtype != kDtypeF16 && a->dtype != kDtypeBF16 && a->dtype != kDtypeF32) return kErrInvalidArg;
  RopeParams p{};
  int64_t half = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0) return kErrInvalidArg;
    half += a->sections[i];
    if (2 * half > a->head_dim) return kErrInvalidArg;
    p.ends[i] = static_cast<int>(half);
  }
  if (half == 0) return kErrInvalidArg;
  if (a->tokens == 0 || a->heads_q + a->heads_k == 0) return kOk;
  const uintptr_t e = elt_bytes(a->dtype);
  if (!a->positions || !aligned(a->positions, a->positions_64bit ? 8 : 4)) return kErrInvalidArg;
  if (a->table_rows > 0 && (!a->cos || !a->sin || !aligned(a->cos, 4) || !aligned(a->sin, 4))) return kErrInvalidArg;
  if (a->heads_q > 0 && (!a->q || !a->q_out || !aligned(a->q, e) || !aligned(a->q_out, e))) return kErrInvalidArg;
  if (a->heads_k > 0 && (!a->k || !a->k_out || !aligned(a->k, e) || !aligned(a->k_out, e))) return kErrInvalidArg;
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.pos = a->positions;
  p.cos = a->cos;
  p.sin = a->sin;
  p.q_st = a->q_stride_t, p.q_sh = a->q_stride_h;
  p.k_st = a->k_stride_t, p.k_sh = a->k_stride_h;
  p.qo_st = a->q_out_stride_t, p.qo_sh = a->q_out_stride_h;
  p.ko_st = a->k_out_stride_t, p.ko_sh = a->k_out_stride_h;
  p.pos_sa = a->positions_stride_axis, p.pos_st = a->positions_stride_t;
  p.tokens = a->tokens;
  p.heads_q = a->heads_q;
  p.heads_k = a->heads_k;
  p.head_dim = a->head_dim;
  p.half = static_cast<int>(half);
  p.axes = a->axes;
  p.table_rows = a->table_rows;
  p.sin_sign = a->inverse ? -1.f : 1.f;
  p.pos64 = a->positions_64bit ? 1 : 0;
  auto st = static_cast<cudaStream_t>(stream);
  if (a->dtype == kDtypeBF16) return rope<__nv_bfloat16>(p, st);
  if (a->dtype == kDtypeF16) return rope<__half>(p, st);
  return rope<float>(p, st);
}

}  // extern "C"
