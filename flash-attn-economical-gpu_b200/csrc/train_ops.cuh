// Memory-bound operators around the attention of a trained block: layer norm
// forward and backward (with the weight's and bias's gradients) and rotary
// embedding over several position axes.  All arithmetic is fp32; a value is
// rounded once, when it is stored in its tensor's type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "ptx.cuh"

namespace fab {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }

// V consecutive values in 16-byte accesses (two for eight floats).
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec {
  T e[V];
};
// Two 16-bit values of one word, converted together.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int V>
__device__ __forceinline__ void to_floats(const Vec<T, V>& v, float (&f)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 x = unpack2<T>(w[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_float<T>(v.e[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
  if constexpr (V * sizeof(T) == 16) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    to_floats<T, V>(*reinterpret_cast<const Vec<T, V>*>(&w), f);
  } else if constexpr (V * sizeof(T) == 32) {
    const uint4 w[2] = {reinterpret_cast<const uint4*>(p)[0], reinterpret_cast<const uint4*>(p)[1]};
    to_floats<T, V>(*reinterpret_cast<const Vec<T, V>*>(w), f);
  } else {
    to_floats<T, V>(*reinterpret_cast<const Vec<T, V>*>(p), f);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  Vec<T, V> v;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v.e[i] = from_float<T>(f[i]);
  }
  if constexpr (V * sizeof(T) == 16)
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
  else
    *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// The 16-byte vectors of the kernels below, worked on in pairs (two fp32
// operations per instruction).
template <typename T>
struct Pairs {
  static constexpr int kN = 8 / sizeof(T);  // pairs in 16 bytes
};
template <typename T>
__device__ __forceinline__ void to_pairs(const uint4& w, float2 (&f)[Pairs<T>::kN]) {
  if constexpr (sizeof(T) == 2) {
    f[0] = unpack2<T>(w.x), f[1] = unpack2<T>(w.y), f[2] = unpack2<T>(w.z), f[3] = unpack2<T>(w.w);
  } else {
    f[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    f[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
  }
}
template <typename T>
__device__ __forceinline__ uint4 from_pairs(const float2 (&f)[Pairs<T>::kN]) {
  if constexpr (sizeof(T) == 2)
    return make_uint4(pack2<T>(f[0].x, f[0].y), pack2<T>(f[1].x, f[1].y), pack2<T>(f[2].x, f[2].y), pack2<T>(f[3].x, f[3].y));
  else
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}
// 2 * N weights of type W (N pairs), 16-byte aligned for N * 2 * sizeof(W) >= 16.
template <typename W, int N>
__device__ __forceinline__ void load_pairs(const W* p, float2 (&f)[N]) {
  if constexpr (sizeof(W) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float4 v = *reinterpret_cast<const float4*>(p + 2 * i);
      f[i] = make_float2(v.x, v.y);
      f[i + 1] = make_float2(v.z, v.w);
    }
  } else {
    static_assert(N == 4, "16-bit weights go with 16-bit rows");
    to_pairs<W>(*reinterpret_cast<const uint4*>(p), f);
  }
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Sum over the CTA of K values at once, the result in every thread.  `red`
// holds K * 32 floats; a caller that reduces again synchronises in between.
template <int K>
__device__ __forceinline__ void warp_sum(float (&v)[K]) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
}
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
  warp_sum<K>(v);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[k * 32 + warp] = v[k];
  __syncthreads();
  if (warps <= 8) {
    // Every thread adds the few warps' sums itself, in warp order.
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = red[k * 32];
    for (int w = 1; w < warps; ++w)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += red[k * 32 + w];
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane < warps ? red[k * 32 + lane] : 0.f;
    warp_sum<K>(v);
  }
}

// block_sum for CTAs of at most eight warps that reduce once per row: `red`
// holds K * 8 floats, zero where there is no warp, and every thread adds the
// eight itself (two 16-byte reads), in warp order.
template <int K>
__device__ __forceinline__ void few_warps_sum(float (&v)[K], float* red) {
  warp_sum<K>(v);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[k * 8 + (threadIdx.x >> 5)] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const float4 a = *reinterpret_cast<const float4*>(red + k * 8), b = *reinterpret_cast<const float4*>(red + k * 8 + 4);
    v[k] = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
  }
}

// Rows wider than a CTA's share of shared memory belong to a cluster of CTAs,
// each with its columns.  A CTA's columns are counted in places: column c is
// place c + shift, where the row starts `shift` elements past a 16-byte
// boundary, so that places 0, V, 2V, ... lie on boundaries.  (V values are 16
// bytes.)
constexpr int kMaxCluster = 8;
struct RowShare {
  int rank, ctas;      // place in the cluster
  int first, places;   // first place, places of this CTA
  int lo, hi;          // this CTA's places that are columns
};
template <bool kWide>
__device__ __forceinline__ RowShare row_share(int cols, int shift, int span) {
  RowShare r{0, 1, 0, cols + shift, shift, cols + shift};
  if constexpr (kWide) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r.rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r.ctas));
    r.first = r.rank * span;
    r.places = max(0, min(span, r.hi - r.first));
    r.lo -= r.first;
    r.hi -= r.first;
  }
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}

// The sums over a row of K values at a time, in one of two buffers in turn:
// every thread has left a buffer for good when the other one's sums are
// complete.  A CTA alone: few_warps_sum.  A cluster: each warp's sum goes to
// every CTA, and its bytes complete that CTA's barrier.  (A barrier of the
// cluster, which also waits for the row's stores to global memory, took longer:
// 4096 x 12288 bf16 forward 104 us against 78.)  The kernels hold
//   float red[2][kSumFloats<kWide, K>], RowBars bars  in shared memory
// as variables of their own: through a reference the reads of a lone CTA's
// sums became generic ones, 4 % of the backward's time.
template <bool kWide, int K>
constexpr int kSumFloats = K * 8 * (kWide ? kMaxCluster : 1);
struct RowBars {
  uint64_t bar[2];
  int abort;
};
template <bool kWide, int kFloats>
__device__ __forceinline__ void init_sums(float (&red)[2][kFloats], RowBars& bars) {
  for (int i = threadIdx.x; i < 2 * kFloats; i += blockDim.x) red[i / kFloats][i % kFloats] = 0.f;
  if constexpr (kWide) {
    if (threadIdx.x == 0) {
      mbar_init(bars.bar, 1);
      mbar_init(bars.bar + 1, 1);
      mbar_fence_init();
      bars.abort = 0;
    }
    cluster_sync();
  } else {
    __syncthreads();
  }
}
// K sums over the cluster; false when a peer's never came.  `withheld`: this
// CTA sends none.
template <int K>
__device__ __forceinline__ bool cluster_sum(float (&v)[K], float* red, uint64_t* bar, uint32_t parity, RowBars& bars,
                                            const RowShare& r, bool withheld) {
  const int lane = threadIdx.x & 31;
  warp_sum<K>(v);
  if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, K * 4 * (blockDim.x >> 5) * r.ctas);
  if (lane < r.ctas && !withheld) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      asm volatile(
          "{\n\t.reg .u32 to, bar;\n\t"
          "mapa.shared::cluster.u32 to, %0, %2;\n\t"
          "mapa.shared::cluster.u32 bar, %1, %2;\n\t"
          "st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [to], %3, [bar];\n\t}" ::"r"(
              smem_u32(red + (k * kMaxCluster + r.rank) * 8 + (threadIdx.x >> 5))),
          "r"(smem_u32(bar)), "r"(lane), "r"(__float_as_uint(v[k]))
          : "memory");
  }
  __syncwarp();
  const bool ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, &bars.abort, kDevTimeoutRowSum));
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.f;
    for (int x = 0; x < 2 * r.ctas; ++x) {
      const float4 a = *reinterpret_cast<const float4*>(red + k * kMaxCluster * 8 + x * 4);
      v[k] += (a.x + a.y) + (a.z + a.w);
    }
  }
  return ok;
}

// A row whose ends lie inside 16-byte pieces (kOdd): those pieces' places that
// are no columns.
template <typename T>
struct RowEnds {
  static constexpr int V = 16 / sizeof(T);
  int lo, hi;  // columns are places [lo, hi)
  __device__ __forceinline__ bool cut(int c) const { return c < lo || c + V > hi; }
  __device__ __forceinline__ bool in(int c) const { return c >= lo && c < hi; }
  // Values at no column become 0.
  __device__ __forceinline__ void clip(int c, float2 (&f)[V / 2]) const {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      if (!in(c + 2 * e)) f[e].x = 0.f;
      if (!in(c + 2 * e + 1)) f[e].y = 0.f;
    }
  }
  __device__ __forceinline__ void copy(T* to, const T* from, int c) const {
#pragma unroll 1
    for (int e = 0; e < V; ++e)
      if (in(c + e)) to[e] = from[e];
  }
  __device__ __forceinline__ void store(T* to, const uint4& v, int c) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (in(c + e)) {
        if constexpr (sizeof(T) == 2)
          reinterpret_cast<uint16_t*>(to)[e] = static_cast<uint16_t>(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
        else
          reinterpret_cast<uint32_t*>(to)[e] = w[e];
      }
  }
  // Weights of the places from c on, 0 at no column.
  template <typename W>
  __device__ __forceinline__ void weights(const W* w, int c, float2 (&f)[V / 2]) const {
#pragma unroll
    for (int e = 0; e < V / 2; ++e)
      f[e] = make_float2(in(c + 2 * e) ? to_float<W>(w[c + 2 * e]) : 0.f, in(c + 2 * e + 1) ? to_float<W>(w[c + 2 * e + 1]) : 0.f);
  }
};
// Elements from the 16-byte boundary at or before p.
template <typename T>
__device__ __forceinline__ int past_boundary(const T* p) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u) / static_cast<int>(sizeof(T));
}

// ------------------------------------------------------------ layer norm ---
struct LayerNormParams {
  const void* x;
  const void* residual;  // or null
  const void* w;
  const void* bias;  // or null
  void* y;
  void* x_out;  // x + residual, or null
  float* mean;  // or null
  float* rstd;
  int64_t ld_x, ld_res, ld_y, ld_xo;
  int64_t rows;
  int cols;
  float eps;
  int span;  // columns of a CTA where a cluster shares a row
  int starve_row;  // test hook: the row whose sums the cluster's last CTA withholds, or -1
};

// y = (x' - mean) * rsqrt(var + eps) * w + b per row, x' = x or round(x + residual).
// One CTA per row; the row stays in registers (NV vectors of V per thread), so
// it is read once, and the variance is the mean of squared distances from the
// mean, not a difference of sums.  For calls of few rows, where one row's
// latency is the time (1 x 3584 bf16 4.3 us).
template <typename T, typename W, int V, int NV, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) layernorm_fwd_kernel(const LayerNormParams p) {
  __shared__ float red[64];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ld_x;
  const T* res = reinterpret_cast<const T*>(p.residual);
  float v[NV][V];
  float sum[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (threadIdx.x + k * blockDim.x) * V;
    if (c < p.cols) {
      load_vec<T, V>(x + c, v[k]);
      if (res != nullptr) {
        float r[V];
        load_vec<T, V>(res + row * p.ld_res + c, r);
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] += r[e];
        T* xo = reinterpret_cast<T*>(p.x_out) + row * p.ld_xo + c;
        store_vec<T, V>(xo, v[k]);
        // The norm is of the rounded sum.
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[k][e] = to_float<T>(from_float<T>(v[k][e]));
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] += v[k][e];
    }
  }
  block_sum<1>(sum, red);
  const float mean = sum[0] / static_cast<float>(p.cols);
  float sq[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (threadIdx.x + k * blockDim.x) * V;
    if (c < p.cols)
#pragma unroll
      for (int e = 0; e < V; ++e) sq[0] = fmaf(v[k][e] - mean, v[k][e] - mean, sq[0]);
  }
  block_sum<1>(sq, red + 32);
  const float rstd = rsqrtf(sq[0] / static_cast<float>(p.cols) + p.eps);
  if (threadIdx.x == 0 && p.mean != nullptr) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (threadIdx.x + k * blockDim.x) * V;
    if (c < p.cols) {
      float w[V], o[V];
      load_vec<W, V>(reinterpret_cast<const W*>(p.w) + c, w);
      if (p.bias != nullptr) {
        float b[V];
        load_vec<W, V>(reinterpret_cast<const W*>(p.bias) + c, b);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf((v[k][e] - mean) * rstd, w[e], b[e]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (v[k][e] - mean) * rstd * w[e];
      }
      store_vec<T, V>(reinterpret_cast<T*>(p.y) + row * p.ld_y + c, o);
    }
  }
}

// Asynchronous 16-byte copies into shared memory that the copying thread
// alone reads back: it waits for its own groups, no barrier is needed.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// A shared-memory read that the compiler may not merge with an earlier one.
__device__ __forceinline__ uint4 read_again(const uint4* p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(smem_u32(p))
               : "memory");
  return v;
}

// The rows of a launch, streamed: each CTA takes rows blockIdx.x, + gridDim.x,
// ... and has the next kStages - 1 of them on their way into shared memory
// while it works on one, so that the memory stays busy across a row's two
// reductions; weight and bias wait in registers for all of them (read anew for
// every row they were the larger part of what L1 had to deliver).  NV 16-byte
// vectors per thread.  kOdd: rows off the 16-byte grid, of which every CTA
// takes some that start at the same offset (gridDim.x / ctas is a multiple of
// 8, or there is one row each); the pieces at their ends are cut to the row.
// Bound by memory: 8192 x 3584 bf16 with a residual moves 235 MB in 34.5 us,
// 6.8 TB/s; 8192 x 3585 takes 71 us a call against 48 (its edges' values come
// and go one by one), a cluster's 4096 x 16384 fp32 181 us for 1.07 GB.
template <typename T, typename W, int NV, int kMaxThreads, int kMinCtas, int kStages, bool kWide, bool kOdd>
__global__ void __launch_bounds__(kMaxThreads, kMinCtas) layernorm_fwd_stream_kernel(const LayerNormParams p) {
  constexpr int N = Pairs<T>::kN, V = 2 * N;
  extern __shared__ __align__(16) uint8_t smem_copies[];
  __shared__ __align__(16) float red[2][kSumFloats<kWide, 1>];
  __shared__ RowBars bars;
  uint32_t ctas = 1;
  if constexpr (kWide) asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int64_t row0 = blockIdx.x / ctas;
  const int shift = kOdd ? past_boundary(reinterpret_cast<const T*>(p.x) + row0 * p.ld_x) : 0;
  const RowShare share = row_share<kWide>(p.cols, shift, p.span);
  const int cols = share.places, col0 = share.first - shift;
  [[maybe_unused]] const RowEnds<T> ends{share.lo, share.hi};
  const bool summed = p.residual != nullptr;
  const int threads = blockDim.x;
  const int c0 = threadIdx.x * V, step = threads * V;  // first column, columns between vectors
  init_sums<kWide>(red, bars);
  [[maybe_unused]] uint32_t parity = 0;
  [[maybe_unused]] const int starve_row = share.rank == share.ctas - 1 ? p.starve_row : -1;
  float2 w[NV][N], b[NV][N];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = c0 + k * step;
#pragma unroll
    for (int e = 0; e < N; ++e) w[k][e] = b[k][e] = both(0.f);
    if (c < cols) {
      const W* pw = reinterpret_cast<const W*>(p.w) + col0;
      const W* pb = reinterpret_cast<const W*>(p.bias) + col0;
      if constexpr (kOdd) {
        ends.weights(pw, c, w[k]);
        if (p.bias != nullptr) ends.weights(pb, c, b[k]);
      } else {
        load_pairs<W, N>(pw + c, w[k]);
        if (p.bias != nullptr) load_pairs<W, N>(pb + c, b[k]);
      }
    }
  }
  // Pointers to this thread's first column of the row being fetched and of the
  // one being worked on, moved from row to row.
  const int64_t rows_apart = gridDim.x / ctas;
  const T* fx = reinterpret_cast<const T*>(p.x) + row0 * p.ld_x + col0 + c0;
  const T* fr = reinterpret_cast<const T*>(p.residual) + row0 * p.ld_res + col0 + c0;
  T* y = reinterpret_cast<T*>(p.y) + row0 * p.ld_y + col0 + c0;
  T* xo = reinterpret_cast<T*>(p.x_out) + row0 * p.ld_xo + col0 + c0;
  const int64_t dx = rows_apart * p.ld_x, dr = rows_apart * p.ld_res, dy = rows_apart * p.ld_y, dxo = rows_apart * p.ld_xo;
  // This thread's vectors of a stage: x at [k], the residual at [NV + k].
  uint4* const mine = reinterpret_cast<uint4*>(smem_copies) + threadIdx.x;
  const int stage_size = 2 * NV * threads;
  int64_t fetch_row = row0;
  [[maybe_unused]] const bool close = p.ld_x < V || (summed && p.ld_res < V);  // rows nearer than a piece
  auto fetch = [&](uint4* to) {
    if (fetch_row < p.rows) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (c0 + k * step < cols) {
          // The first and last row's cut pieces are not all inside the tensor.
          if (kOdd && ends.cut(c0 + k * step) && (fetch_row == 0 || fetch_row + 1 == p.rows || close)) {
            ends.copy(reinterpret_cast<T*>(to + k * threads), fx + k * step, c0 + k * step);
            if (summed) ends.copy(reinterpret_cast<T*>(to + (NV + k) * threads), fr + k * step, c0 + k * step);
            continue;
          }
          copy16(to + k * threads, fx + k * step);
          if (summed) copy16(to + (NV + k) * threads, fr + k * step);
        }
    }
    copy_commit();
    fetch_row += rows_apart;
    fx += dx;
    fr += dr;
  };
  const float inv = 1.f / static_cast<float>(p.cols);
  uint4* to = mine;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s, to += stage_size) fetch(to);
  const uint4* from = mine;
  uint4* const end = mine + kStages * stage_size;
  for (int64_t row = row0; row < p.rows; row += rows_apart, y += dy, xo += dxo) {
    fetch(to);
    if ((to += stage_size) == end) to = mine;
    copy_wait<kStages - 1>();
    float2 f[NV][N];
    float2 sum2 = both(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c0 + k * step < cols) {
        to_pairs<T>(from[k * threads], f[k]);
        if (summed) {
          float2 r[N];
          to_pairs<T>(from[(NV + k) * threads], r);
#pragma unroll
          for (int e = 0; e < N; ++e) r[e] = __fadd2_rn(f[k][e], r[e]);
          const uint4 raw = from_pairs<T>(r);
          if (kOdd && ends.cut(c0 + k * step))
            ends.store(xo + k * step, raw, c0 + k * step);
          else
            *reinterpret_cast<uint4*>(xo + k * step) = raw;
          to_pairs<T>(raw, f[k]);  // the norm is of the rounded sum
        }
        if (kOdd && ends.cut(c0 + k * step)) ends.clip(c0 + k * step, f[k]);
#pragma unroll
        for (int e = 0; e < N; ++e) sum2 = __fadd2_rn(sum2, f[k][e]);
      }
    }
    if ((from += stage_size) == end) from = mine;
    float sum[1] = {sum2.x + sum2.y};
    if constexpr (kWide) {
      if (!cluster_sum<1>(sum, red[0], bars.bar, parity, bars, share, row == starve_row)) break;
    } else {
      few_warps_sum<1>(sum, red[0]);
    }
    const float mean = sum[0] * inv;
    float2 sq2 = both(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (c0 + k * step < cols) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[k][e] = __fadd2_rn(f[k][e], both(-mean));
        if (kOdd && ends.cut(c0 + k * step)) ends.clip(c0 + k * step, f[k]);
#pragma unroll
        for (int e = 0; e < N; ++e) sq2 = __ffma2_rn(f[k][e], f[k][e], sq2);
      }
    float sq[1] = {sq2.x + sq2.y};
    // Each of the two sums also frees the other's buffer.
    if constexpr (kWide) {
      if (!cluster_sum<1>(sq, red[1], bars.bar + 1, parity, bars, share, false)) break;
      parity ^= 1u;
    } else {
      few_warps_sum<1>(sq, red[1]);
    }
    const float rstd = rsqrtf(sq[0] * inv + p.eps);
    if (threadIdx.x == 0 && share.rank == 0 && p.mean != nullptr) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (c0 + k * step < cols) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[k][e] = __ffma2_rn(__fmul2_rn(f[k][e], both(rstd)), w[k][e], b[k][e]);
        if (kOdd && ends.cut(c0 + k * step))
          ends.store(y + k * step, from_pairs<T>(f[k]), c0 + k * step);
        else
          *reinterpret_cast<uint4*>(y + k * step) = from_pairs<T>(f[k]);
      }
  }
  copy_wait<0>();
  if constexpr (kWide) cluster_sync();  // the others may still write their sums here
}

// Rows too long for a cluster, or that lie at different places of a 16-byte
// piece in different tensors: the same sums over three reads of the row (the
// later ones from L2).  Rare, and 2 to 4 times the streamed kernels' time.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) layernorm_fwd_long_kernel(const LayerNormParams p) {
  __shared__ float red[64];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ld_x;
  const T* res = reinterpret_cast<const T*>(p.residual);
  T* xo = reinterpret_cast<T*>(p.x_out) + row * p.ld_xo;
  // Each thread reads back only what it wrote itself.
  const T* src = res != nullptr ? xo : x;
  float sum[1] = {0.f};
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    float v = to_float<T>(x[c]);
    if (res != nullptr) {
      const T s = from_float<T>(v + to_float<T>(res[row * p.ld_res + c]));
      xo[c] = s;
      v = to_float<T>(s);
    }
    sum[0] += v;
  }
  block_sum<1>(sum, red);
  const float mean = sum[0] / static_cast<float>(p.cols);
  float sq[1] = {0.f};
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float d = to_float<T>(src[c]) - mean;
    sq[0] = fmaf(d, d, sq[0]);
  }
  block_sum<1>(sq, red + 32);
  const float rstd = rsqrtf(sq[0] / static_cast<float>(p.cols) + p.eps);
  if (threadIdx.x == 0 && p.mean != nullptr) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  T* y = reinterpret_cast<T*>(p.y) + row * p.ld_y;
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float b = p.bias != nullptr ? to_float<W>(reinterpret_cast<const W*>(p.bias)[c]) : 0.f;
    y[c] = from_float<T>(fmaf((to_float<T>(src[c]) - mean) * rstd, to_float<W>(reinterpret_cast<const W*>(p.w)[c]), b));
  }
}

struct LayerNormBwdParams {
  const void* dy;
  const void* x;
  const void* w;
  const float* mean;
  const float* rstd;
  const void* dres;  // gradient that reaches x past the norm, or null
  void* dx;
  float* part;  // [gridDim.x][2][cols]: this CTA's sums of dy * xhat and dy; or null
  int64_t ld_dy, ld_x, ld_dres, ld_dx;
  int64_t rows;
  int cols;
  int span;  // columns of a CTA where a cluster shares a row
  int starve_row;  // test hook: the row whose sums the cluster's last CTA withholds, or -1
};

// With xhat = (x - mean) * rstd and g = dy * w:
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) + dres
//   dw = sum_rows dy * xhat,  db = sum_rows dy
// Memory-bound: dy, x (and dres) in, dx out, each once.  A row belongs to one
// warp (kWarpRow, short rows: no barrier at all) or to the whole CTA; a
// "worker" (warp or CTA) i takes rows i, i + workers, ...  A thread keeps the
// same columns for all of them, so its share of dw and db stays in registers
// and leaves once.  The next kStages - 1 rows are on their way into shared
// memory while one is worked on, which keeps the memory busy across the
// reduction that every row has in its middle; the weight waits in registers.
// Wider than 1024 vectors, a row is shared by a cluster (kWide), and rows off
// the 16-byte grid are taken in whole pieces (kOdd), as in the forward kernel.
// Measured: 8192 x 3584 bf16 with dres 235 MB in 50 us, 4.7 TB/s, two fifths of
// the issue slots: what bounds it is the latency of a row's two passes over
// shared memory with the sum in between, at the 16 warps that the sums leave
// registers for.  Three stages (one CTA less), 16 warps in one CTA, and dy and
// xhat held in registers across the sum were all slower.
template <typename T, typename W, int NV, int kMaxThreads, int kMinCtas, bool kWarpRow, bool kWide, bool kOdd, int kStages>
__global__ void __launch_bounds__(kMaxThreads, kMinCtas) layernorm_bwd_kernel(const LayerNormBwdParams p) {
  constexpr int N = Pairs<T>::kN, V = 2 * N;
  extern __shared__ __align__(16) uint8_t smem_copies[];
  __shared__ __align__(16) float red[2][kSumFloats<kWide, 2>];
  __shared__ RowBars bars;
  uint32_t ctas = 1;
  if constexpr (kWide) asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int threads = blockDim.x;
  const int lanes = kWarpRow ? 32 : threads;  // threads of a row
  const int me = kWarpRow ? threadIdx.x & 31 : threadIdx.x;
  const int64_t worker = kWarpRow ? static_cast<int64_t>(blockIdx.x) * (threads >> 5) + (threadIdx.x >> 5) : blockIdx.x / ctas;
  const int64_t workers = kWarpRow ? static_cast<int64_t>(gridDim.x) * (threads >> 5) : gridDim.x / ctas;
  const int shift = kOdd ? past_boundary(reinterpret_cast<const T*>(p.x) + worker * p.ld_x) : 0;
  const RowShare share = row_share<kWide>(p.cols, shift, p.span);
  const int cols = share.places, col0 = share.first - shift;
  [[maybe_unused]] const RowEnds<T> ends{share.lo, share.hi};
  const int c0 = me * V, step = lanes * V;  // first column, columns between vectors
  const bool summed = p.dres != nullptr;
  init_sums<kWide>(red, bars);
  [[maybe_unused]] uint32_t parity = 0;
  [[maybe_unused]] const int starve_row = share.rank == share.ctas - 1 ? p.starve_row : -1;
  float2 w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = c0 + k * step;
#pragma unroll
    for (int e = 0; e < N; ++e) w[k][e] = dw[k][e] = db[k][e] = both(0.f);
    if (c < cols) {
      if constexpr (kOdd)
        ends.weights(reinterpret_cast<const W*>(p.w) + col0, c, w[k]);
      else
        load_pairs<W, N>(reinterpret_cast<const W*>(p.w) + col0 + c, w[k]);
    }
  }
  const float inv = 1.f / static_cast<float>(p.cols);
  // This thread's first column of the row being fetched and of the one being
  // worked on.  Moved from row to row; where a cluster or cut pieces need the
  // registers, formed anew (kFresh: 4096 x 12288 bf16 110 against 128 us, but
  // one CTA's rows, 8192 x 8192, 126 against 116).
  constexpr bool kFresh = kWide || kOdd;
  const T* fx = reinterpret_cast<const T*>(p.x) + worker * p.ld_x + col0 + c0;
  const T* fg = reinterpret_cast<const T*>(p.dy) + worker * p.ld_dy + col0 + c0;
  const T* fr = reinterpret_cast<const T*>(p.dres) + worker * p.ld_dres + col0 + c0;
  T* out = reinterpret_cast<T*>(p.dx) + worker * p.ld_dx + col0 + c0;
  const int64_t ax = workers * p.ld_x, ag = workers * p.ld_dy, ar = workers * p.ld_dres, ao = workers * p.ld_dx;
  // This thread's vectors of a stage: x at [k], dy at [NV + k], dres after.
  uint4* const mine = reinterpret_cast<uint4*>(smem_copies) + threadIdx.x;
  const int stage_size = 3 * NV * threads;
  [[maybe_unused]] const bool close = p.ld_x < V || p.ld_dy < V || (summed && p.ld_dres < V);  // rows nearer than a piece
  int64_t fetch_row = worker;
  auto fetch = [&](uint4* to) {
    if (fetch_row < p.rows) {
      if constexpr (kFresh) {
        fx = reinterpret_cast<const T*>(p.x) + fetch_row * p.ld_x + col0 + c0;
        fg = reinterpret_cast<const T*>(p.dy) + fetch_row * p.ld_dy + col0 + c0;
        fr = reinterpret_cast<const T*>(p.dres) + fetch_row * p.ld_dres + col0 + c0;
      }
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (c0 + k * step < cols) {
          // The first and last row's cut pieces are not all inside the tensor.
          if (kOdd && ends.cut(c0 + k * step) && (fetch_row == 0 || fetch_row + 1 == p.rows || close)) {
            ends.copy(reinterpret_cast<T*>(to + k * threads), fx + k * step, c0 + k * step);
            ends.copy(reinterpret_cast<T*>(to + (NV + k) * threads), fg + k * step, c0 + k * step);
            if (summed) ends.copy(reinterpret_cast<T*>(to + (2 * NV + k) * threads), fr + k * step, c0 + k * step);
            continue;
          }
          copy16(to + k * threads, fx + k * step);
          copy16(to + (NV + k) * threads, fg + k * step);
          if (summed) copy16(to + (2 * NV + k) * threads, fr + k * step);
        }
    }
    copy_commit();
    fetch_row += workers;
    if constexpr (!kFresh) {
      fx += ax;
      fg += ag;
      fr += ar;
    }
  };
  uint4* to = mine;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s, to += stage_size) fetch(to);
  const uint4* from = mine;
  uint4* const end = mine + kStages * stage_size;
  int turn = 0;
  float next_mean = 0.f, next_rstd = 0.f;
  if (worker < p.rows) {
    next_mean = p.mean[worker];
    next_rstd = p.rstd[worker];
  }
  for (int64_t row = worker; row < p.rows; row += workers, turn ^= 1) {
    fetch(to);
    if ((to += stage_size) == end) to = mine;
    const float2 scale = both(next_rstd), less = both(-next_mean);
    if (row + workers < p.rows) {  // the next row's, a row ahead of their use
      next_mean = p.mean[row + workers];
      next_rstd = p.rstd[row + workers];
    }
    copy_wait<kStages - 1>();
    float2 s0 = both(0.f), s1 = both(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c0 + k * step < cols) {
        // Read again after the reduction rather than held across it: the
        // registers buy another resident CTA.
        float2 h[N], g[N];
        to_pairs<T>(from[k * threads], h);
        to_pairs<T>(from[(NV + k) * threads], g);
        if (kOdd && ends.cut(c0 + k * step)) {
          ends.clip(c0 + k * step, h);
          ends.clip(c0 + k * step, g);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          h[e] = __fmul2_rn(__fadd2_rn(h[e], less), scale);
          dw[k][e] = __ffma2_rn(g[e], h[e], dw[k][e]);
          db[k][e] = __fadd2_rn(db[k][e], g[e]);
          g[e] = __fmul2_rn(g[e], w[k][e]);
          s0 = __fadd2_rn(s0, g[e]);
          s1 = __ffma2_rn(g[e], h[e], s1);
        }
      }
    }
    float s[2] = {s0.x + s0.y, s1.x + s1.y};
    if constexpr (kWarpRow) {
      warp_sum<2>(s);
    } else if constexpr (kWide) {
      if (!cluster_sum<2>(s, red[turn], bars.bar + turn, parity, bars, share, row == starve_row)) break;
      parity ^= static_cast<uint32_t>(turn);
    } else {
      few_warps_sum<2>(s, red[turn]);  // the other buffer is free again: every thread has passed this row's barrier
    }
    const float2 na = both(-s[0] * inv), nb = both(-s[1] * inv);
    if constexpr (kFresh) out = reinterpret_cast<T*>(p.dx) + row * p.ld_dx + col0 + c0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c0 + k * step < cols) {
        float2 h[N], g[N];
        to_pairs<T>(read_again(from + k * threads), h);
        to_pairs<T>(read_again(from + (NV + k) * threads), g);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          h[e] = __fmul2_rn(__fadd2_rn(h[e], less), scale);
          g[e] = __ffma2_rn(g[e], w[k][e], __ffma2_rn(h[e], nb, na));
          g[e] = __fmul2_rn(g[e], scale);
        }
        if (summed) {
          float2 r[N];
          to_pairs<T>(from[(2 * NV + k) * threads], r);
#pragma unroll
          for (int e = 0; e < N; ++e) g[e] = __fadd2_rn(g[e], r[e]);
        }
        if (kOdd && ends.cut(c0 + k * step))
          ends.store(out + k * step, from_pairs<T>(g), c0 + k * step);
        else
          *reinterpret_cast<uint4*>(out + k * step) = from_pairs<T>(g);
      }
    }
    if ((from += stage_size) == end) from = mine;
    if constexpr (!kFresh) out += ao;
  }
  copy_wait<0>();
  if constexpr (kWide) cluster_sync();  // the others may still write their sums here
  if (p.part == nullptr) return;
  float* part = p.part + static_cast<int64_t>(kWide ? worker : blockIdx.x) * 2 * p.cols;
  if constexpr (kWarpRow) {
    // The warps' sums meet in shared memory, in warp order.
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem_copies);
    const int warps = threads >> 5;
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (c0 + k * step < cols)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float2 v = which ? db[k][e] : dw[k][e];
            const int c = c0 + k * step + 2 * e;
            float* to = sums + (threadIdx.x >> 5) * p.cols + col0 + c;
            if constexpr (kOdd) {
              if (ends.in(c)) to[0] = v.x;
              if (ends.in(c + 1)) to[1] = v.y;
            } else {
              *reinterpret_cast<float2*>(to) = v;
            }
          }
      __syncthreads();
      for (int c = threadIdx.x; c < p.cols; c += threads) {
        float v = sums[c];
        for (int x = 1; x < warps; ++x) v += sums[x * p.cols + c];
        part[which * p.cols + c] = v;
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      if (c >= cols) continue;
      float* const to = part + col0 + c;
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        if constexpr (kOdd) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int d = 2 * (e + x);
            if (ends.in(c + d)) to[d] = dw[k][e + x].x, to[p.cols + d] = db[k][e + x].x;
            if (ends.in(c + d + 1)) to[d + 1] = dw[k][e + x].y, to[p.cols + d + 1] = db[k][e + x].y;
          }
        } else {
          *reinterpret_cast<float4*>(to + 2 * e) = make_float4(dw[k][e].x, dw[k][e].y, dw[k][e + 1].x, dw[k][e + 1].y);
          *reinterpret_cast<float4*>(to + p.cols + 2 * e) = make_float4(db[k][e].x, db[k][e].y, db[k][e + 1].x, db[k][e + 1].y);
        }
      }
    }
  }
}

// Rows too long for a cluster, or of unlike places: dx only, two reads of the
// row.  The column sums are another kernel's, which reads dy and x again and
// runs before this one, whose dx may lie over dy.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) layernorm_bwd_long_kernel(const LayerNormBwdParams p) {
  __shared__ float red[64];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ld_x;
  const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.ld_dy;
  const W* w = reinterpret_cast<const W*>(p.w);
  const float mean = p.mean[row], rstd = p.rstd[row];
  float s[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float g = to_float<T>(dy[c]) * to_float<W>(w[c]);
    s[0] += g;
    s[1] = fmaf(g, (to_float<T>(x[c]) - mean) * rstd, s[1]);
  }
  block_sum<2>(s, red);
  const float a = s[0] / static_cast<float>(p.cols), b = s[1] / static_cast<float>(p.cols);
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float h = (to_float<T>(x[c]) - mean) * rstd;
    float o = rstd * (to_float<T>(dy[c]) * to_float<W>(w[c]) - fmaf(h, b, a));
    if (p.dres != nullptr) o += to_float<T>(reinterpret_cast<const T*>(p.dres)[row * p.ld_dres + c]);
    reinterpret_cast<T*>(p.dx)[row * p.ld_dx + c] = from_float<T>(o);
  }
}

// The column sums of those rows: CTA (x, y) sums rows y, y + gridDim.y, ...
// of 1024 columns into its line of `part`.
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_bwd_long_cols_kernel(const LayerNormBwdParams p) {
  const int c = blockIdx.x * 1024 + threadIdx.x;
  if (c >= p.cols) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float g = to_float<T>(reinterpret_cast<const T*>(p.dy)[row * p.ld_dy + c]);
    const float h = (to_float<T>(reinterpret_cast<const T*>(p.x)[row * p.ld_x + c]) - p.mean[row]) * p.rstd[row];
    dw = fmaf(g, h, dw);
    db += g;
  }
  float* out = p.part + static_cast<int64_t>(blockIdx.y) * 2 * p.cols;
  out[c] = dw;
  out[p.cols + c] = db;
}

// dw[c] = sum_i part[i][0][c], db[c] = sum_i part[i][1][c], in a fixed order:
// 32 columns per CTA, warp x takes lines x, x + 32, ... (its loads all under
// way together), the warps' sums are added in warp order.  592 lines of 3584
// columns, 17 MB mostly from L2: 7 us, of which setting it up under the
// backward kernel (programmatic launch) hides a part.
template <typename W>
__global__ void __launch_bounds__(1024) layernorm_bwd_finish_kernel(const float* part, int lines, int cols, W* dw, W* db) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;  // column of [dw | db]
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float s = 0.f;
  if (j < 2 * cols)
#pragma unroll 8
    for (int i = warp; i < lines; i += 32) s += part[static_cast<int64_t>(i) * 2 * cols + j];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && j < 2 * cols) {
#pragma unroll
    for (int k = 1; k < 32; ++k) s += sums[k][lane];
    W* out = j < cols ? dw : db;
    if (out != nullptr) out[j < cols ? j : j - cols] = from_float<W>(s);
  }
}

// ---------------------------------------------------------------- rotary ---
constexpr int kMaxRopeAxes = 4;
struct RopeParams {
  const void* q;
  const void* k;  // or null
  void* q_out;
  void* k_out;
  const void* pos;  // [axes][tokens], int32 or int64
  const float* cos;  // [table_rows][half]
  const float* sin;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;
  int64_t pos_sa, pos_st;
  int tokens, heads_q, heads_k, head_dim;
  int half;  // rotated pairs: (i, half + i) for i < half; later columns are copied
  int axes;
  int ends[kMaxRopeAxes];  // pair i follows the first axis a with i < ends[a]
  int table_rows;
  float sin_sign;  // -1: the inverse rotation
  int pos64;
  int vec_table;  // every V pairs of a thread follow one axis and lie 16-byte aligned in the tables
  int slots;      // threads that share a token's heads
};

__device__ __forceinline__ int rope_axis(const RopeParams& p, int i) {
  int a = 0;
#pragma unroll
  for (int k = 0; k < kMaxRopeAxes - 1; ++k) a += (k < p.axes - 1 && i >= p.ends[k]) ? 1 : 0;
  return a;
}

// Table row of (axis, token), or -1 when the position is outside the table.
__device__ __forceinline__ int rope_row(const RopeParams& p, int axis, int64_t token) {
  const int64_t at = axis * p.pos_sa + token * p.pos_st;
  const int64_t r = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[at] : reinterpret_cast<const int32_t*>(p.pos)[at];
  return r >= 0 && r < p.table_rows ? static_cast<int>(r) : -1;
}

// Thread (token, slot, vi) owns V pairs of kRopeHeads heads (slot, slot +
// slots, ...): their cosines and sines are read once for all of them, and all
// of their loads are under way before the first is used.  Memory-bound: q and
// k in and out once; the table rows stay in L1 and L2.  A position outside the
// table makes its pairs NaN; nothing is read out of bounds.  Measured: a call of
// 16384 tokens, 28 + 4 heads of 128, bf16, 268 MB, takes 53 us with a cold L2
// (5.0 TB/s), 50 among other calls; with a cold L2 two heads per thread 59, one
// 69, six 67, eight 55.  fp32, 537 MB: 90 us (6.0 TB/s), 87.
constexpr int kRopeHeads = 4;
template <typename T, int V>
__global__ void __launch_bounds__(256, 3) rope_axes_kernel(const RopeParams p) {
  const int rot = p.half / V;                            // vectors of pairs
  const int nvec = rot + (p.head_dim - 2 * p.half) / V;  // and of columns to copy
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int per_token = nvec * p.slots;
  const int64_t t = id / per_token;
  if (t >= p.tokens) return;
  const int in_token = static_cast<int>(id - t * per_token);
  const int slot = in_token / nvec, vi = in_token - slot * nvec;
  const int heads = p.heads_q + p.heads_k;
  const bool turns = vi < rot;
  const int c0 = turns ? vi * V : 2 * p.half + (vi - rot) * V;
  // Loads of every head first.
  Vec<T, V> lo[kRopeHeads], hi[kRopeHeads];
  T* out[kRopeHeads];
#pragma unroll
  for (int j = 0; j < kRopeHeads; ++j) {
    const int h = slot + j * p.slots;
    if (h >= heads) continue;
    const bool is_k = h >= p.heads_q;
    const int hh = is_k ? h - p.heads_q : h;
    const T* in = reinterpret_cast<const T*>(is_k ? p.k : p.q) + t * (is_k ? p.k_st : p.q_st) + hh * (is_k ? p.k_sh : p.q_sh) + c0;
    out[j] = reinterpret_cast<T*>(is_k ? p.k_out : p.q_out) + t * (is_k ? p.ko_st : p.qo_st) + hh * (is_k ? p.ko_sh : p.qo_sh) + c0;
    lo[j] = *reinterpret_cast<const Vec<T, V>*>(in);
    if (turns) hi[j] = *reinterpret_cast<const Vec<T, V>*>(in + p.half);
  }
  if (!turns) {
#pragma unroll
    for (int j = 0; j < kRopeHeads; ++j)
      if (slot + j * p.slots < heads) *reinterpret_cast<Vec<T, V>*>(out[j]) = lo[j];
    return;
  }
  float c[V], s[V];
  if (V >= 4 && p.vec_table) {
    const int row = rope_row(p, rope_axis(p, c0), t);
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const int64_t at = static_cast<int64_t>(row < 0 ? 0 : row) * p.half + c0 + e;
      float4 cv = make_float4(NAN, NAN, NAN, NAN), sv = cv;
      if (row >= 0) {
        cv = *reinterpret_cast<const float4*>(p.cos + at);
        sv = *reinterpret_cast<const float4*>(p.sin + at);
      }
      c[e] = cv.x, s[e] = sv.x;
      if constexpr (V >= 4) {
        c[e + 1] = cv.y, c[e + 2] = cv.z, c[e + 3] = cv.w;
        s[e + 1] = sv.y, s[e + 2] = sv.z, s[e + 3] = sv.w;
      }
    }
  } else {
    int last_axis = -1, row = -1;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int a = rope_axis(p, c0 + e);
      if (a != last_axis) {
        row = rope_row(p, a, t);
        last_axis = a;
      }
      c[e] = row < 0 ? NAN : p.cos[static_cast<int64_t>(row) * p.half + c0 + e];
      s[e] = row < 0 ? NAN : p.sin[static_cast<int64_t>(row) * p.half + c0 + e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] *= p.sin_sign;
#pragma unroll
  for (int j = 0; j < kRopeHeads; ++j) {
    if (slot + j * p.slots >= heads) continue;
    float l[V], u[V], a[V], b[V];
    to_floats<T, V>(lo[j], l);
    to_floats<T, V>(hi[j], u);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      a[e] = l[e] * c[e] - u[e] * s[e];
      b[e] = u[e] * c[e] + l[e] * s[e];
    }
    store_vec<T, V>(out[j], a);
    store_vec<T, V>(out[j] + p.half, b);
  }
}

}  // namespace fab
