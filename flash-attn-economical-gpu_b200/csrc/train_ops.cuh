// Memory-bound operators around the attention of a trained block: layer norm
// forward and backward (with the weight's and bias's gradients) and rotary
// embedding over several position axes.  All arithmetic is fp32; a value is
// rounded once, when it is stored in its tensor's type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

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
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_float<T>(v.e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.e[i] = from_float<T>(f[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// Sum over the CTA of K values at once, the result in every thread.  `red`
// holds K * 32 floats; a caller that reduces again synchronises in between.
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[k * 32 + warp] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float s = lane < warps ? red[k * 32 + lane] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    v[k] = s;
  }
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
};

// y = (x' - mean) * rsqrt(var + eps) * w + b per row, x' = x or round(x + residual).
// One CTA per row; the row stays in registers (NV vectors of V per thread), so
// it is read once, and the variance is the mean of squared distances from the
// mean, not a difference of sums.
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
        for (int e = 0; e < V; ++e) v[k][e] = to_float<T>(from_float<T>(v[k][e] + r[e]));
        store_vec<T, V>(reinterpret_cast<T*>(p.x_out) + row * p.ld_xo + c, v[k]);
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

// Rows too long for the registers of one CTA: the same sums over three reads
// of the row (the later ones from L2).
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
};

// With xhat = (x - mean) * rstd and g = dy * w:
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) + dres
//   dw = sum_rows dy * xhat,  db = sum_rows dy
// CTA i takes rows i, i + gridDim.x, ...; a thread keeps the same columns for
// all of them, so its share of dw and db stays in registers and leaves once
// per CTA.
template <typename T, typename W, int V, int NV, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) layernorm_bwd_kernel(const LayerNormBwdParams p) {
  __shared__ float red[2][64];
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int e = 0; e < V; ++e) dw[k][e] = db[k][e] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(p.cols);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ld_x;
    const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.ld_dy;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float h[NV][V], g[NV][V];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (threadIdx.x + k * blockDim.x) * V;
      if (c < p.cols) {
        load_vec<T, V>(x + c, h[k]);
        load_vec<T, V>(dy + c, g[k]);
        float w[V];
        load_vec<W, V>(reinterpret_cast<const W*>(p.w) + c, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          h[k][e] = (h[k][e] - mean) * rstd;
          dw[k][e] = fmaf(g[k][e], h[k][e], dw[k][e]);
          db[k][e] += g[k][e];
          g[k][e] *= w[e];
          s[0] += g[k][e];
          s[1] = fmaf(g[k][e], h[k][e], s[1]);
        }
      }
    }
    block_sum<2>(s, red[turn]);  // the other buffer is free again: every thread has passed this row's barrier
    const float a = s[0] * inv, b = s[1] * inv;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (threadIdx.x + k * blockDim.x) * V;
      if (c < p.cols) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = rstd * (g[k][e] - fmaf(h[k][e], b, a));
        if (p.dres != nullptr) {
          float r[V];
          load_vec<T, V>(reinterpret_cast<const T*>(p.dres) + row * p.ld_dres + c, r);
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] += r[e];
        }
        store_vec<T, V>(reinterpret_cast<T*>(p.dx) + row * p.ld_dx + c, o);
      }
    }
  }
  if (p.part != nullptr) {
    float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (threadIdx.x + k * blockDim.x) * V;
      if (c < p.cols)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          out[c + e] = dw[k][e];
          out[p.cols + c + e] = db[k][e];
        }
    }
  }
}

// Rows too long for the registers: dx only, two reads of the row.
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

// The column sums those rows leave: CTA (x, y) sums rows y, y + gridDim.y, ...
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
// 32 columns per CTA, eight warps take every eighth line, their sums are added
// in warp order.
template <typename W>
__global__ void __launch_bounds__(256) layernorm_bwd_finish_kernel(const float* __restrict__ part, int lines, int cols,
                                                                   W* dw, W* db) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;  // column of [dw | db]
  float s = 0.f;
  if (j < 2 * cols)
#pragma unroll 4
    for (int i = warp; i < lines; i += 8) s += part[static_cast<int64_t>(i) * 2 * cols + j];
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && j < 2 * cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sums[k][lane];
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

// One CTA per token (and per gridDim.y share of its heads).  Thread vi of a
// head slot owns V pairs of every head of the slot: their cosines and sines
// are read once and used for all of them.  A position outside the table makes
// its pairs NaN; nothing is read out of bounds.
template <typename T, int V>
__global__ void __launch_bounds__(256) rope_axes_kernel(const RopeParams p) {
  const int64_t t = blockIdx.x;
  const int rot = p.half / V;                         // vectors of pairs
  const int nvec = rot + (p.head_dim - 2 * p.half) / V;  // and of columns to copy
  const int slots = blockDim.x / nvec;
  const int vi = threadIdx.x % nvec;
  const int slot = threadIdx.x / nvec;
  if (slot >= slots) return;
  float c[V], s[V];
  if (vi < rot) {
    int last_axis = -1, row = -1;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int i = vi * V + e;
      const int a = rope_axis(p, i);
      if (a != last_axis) {
        row = rope_row(p, a, t);
        last_axis = a;
      }
      c[e] = row < 0 ? NAN : p.cos[static_cast<int64_t>(row) * p.half + i];
      s[e] = row < 0 ? NAN : p.sin[static_cast<int64_t>(row) * p.half + i] * p.sin_sign;
    }
  }
  for (int h = blockIdx.y * slots + slot; h < p.heads_q + p.heads_k; h += slots * gridDim.y) {
    const bool is_k = h >= p.heads_q;
    const int hh = is_k ? h - p.heads_q : h;
    const T* in = reinterpret_cast<const T*>(is_k ? p.k : p.q) + t * (is_k ? p.k_st : p.q_st) + hh * (is_k ? p.k_sh : p.q_sh);
    T* out = reinterpret_cast<T*>(is_k ? p.k_out : p.q_out) + t * (is_k ? p.ko_st : p.qo_st) + hh * (is_k ? p.ko_sh : p.qo_sh);
    if (vi < rot) {
      const int i = vi * V;
      float lo[V], hi[V], a[V], b[V];
      load_vec<T, V>(in + i, lo);
      load_vec<T, V>(in + p.half + i, hi);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        a[e] = lo[e] * c[e] - hi[e] * s[e];
        b[e] = hi[e] * c[e] + lo[e] * s[e];
      }
      store_vec<T, V>(out + i, a);
      store_vec<T, V>(out + p.half + i, b);
    } else {
      const int i = 2 * p.half + (vi - rot) * V;
      *reinterpret_cast<Vec<T, V>*>(out + i) = *reinterpret_cast<const Vec<T, V>*>(in + i);
    }
  }
}

}  // namespace fab
