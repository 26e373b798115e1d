// Layer norm: y = (x - mean) * rstd * w + b over rows of D values, mean and rstd kept in fp32 for
// the backward pass
//   dx = rstd (a - mean(a) - xhat mean(a xhat)),  a = dy w,  xhat = (x - mean) rstd
//   dw = sum_rows dy xhat,  db = sum_rows dy.
// Bound by HBM: forward one read and one write of x, backward two reads and one write. A row is
// held in the registers of one warp, or of a CTA of 128 or 512 threads, EPT values per thread, so
// x is read once and the variance is the mean of squared deviations (two passes over registers,
// no cancellation). Rows wider than 8192 values are read again from cache instead.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "hgemm.cuh"
#include "textgrad.cuh"

namespace dc {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// E consecutive values (16 bytes, or one value) as floats.
template <typename T, int E>
__device__ __forceinline__ void load_e(const T* p, float* f) {
  if (E == 1) {
    f[0] = to_f(*p);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = to_f(h[i]);
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_e(T* p, const float* f) {
  if (E == 1) {
    *p = from_f<T>(f[0]);
  } else {
    uint4 u;
    T* h = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < E; ++i) h[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}
// E values of the weight or bias, in x's type or in fp32.
template <typename T, int E>
__device__ __forceinline__ void load_w(const void* w, int64_t i, bool f32, float* f) {
  if (f32) {
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = static_cast<const float*>(w)[i + j];
  } else {
    load_e<T, E>(static_cast<const T*>(w) + i, f);
  }
}

// Sums of two values over the TPR threads of a row. A CTA holds one row when TPR > 32; `red` is
// its scratch (one slot per warp), alternating between two halves so one barrier is enough.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* red, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    float2* slot = red + turn * kWarps;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = 0.f; b = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) { a += slot[i].x; b += slot[i].y; }
  }
  return make_float2(a, b);
}

struct NormParams {
  const void* x;
  int64_t ldx;
  const void* dy;
  int64_t lddy;
  const void* w;            // null: ones
  const void* b;            // null: zeros
  void* out;                // y or dx
  int64_t ldo;
  float* mean;              // [M]; forward: null when not kept
  float* rstd;
  float* part_w;            // backward: [gridDim.x, ldp] partial column sums, or null
  float* part_b;
  int64_t ldp;
  int64_t M;
  int D;
  float eps;
  int w_f32;
};

template <int TPR> struct NormCta { static constexpr int kThreads = TPR == 32 ? 256 : TPR; };

template <typename T, int E, int EPT, int TPR>
__global__ void __launch_bounds__(NormCta<TPR>::kThreads)
norm_fwd_kernel(const NormParams p) {
  constexpr int NV = EPT / E;
  constexpr int kRows = NormCta<TPR>::kThreads / TPR;
  __shared__ float2 red[2 * (TPR / 32)];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  if (row >= p.M) return;                      // whole warps (TPR == 32) or the whole CTA
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float v[EPT];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * E;
    if (c < p.D) {
      load_e<T, E>(x + c, v + i * E);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) v[i * E + j] = 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < EPT; ++i) s += v[i];
  const float inv = 1.0f / static_cast<float>(p.D);
  const float mean = row_sum2<TPR>(s, 0.f, red, turn).x * inv;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * TPR + t) * E < p.D) {
#pragma unroll
      for (int j = 0; j < E; ++j) { const float d = v[i * E + j] - mean; s += d * d; }
    }
  }
  const float var = row_sum2<TPR>(s, 0.f, red, turn).x * inv;
  const float rstd = 1.0f / sqrtf(var + p.eps);
  if (t == 0 && p.mean != nullptr) { p.mean[row] = mean; p.rstd[row] = rstd; }
  T* y = static_cast<T*>(p.out) + row * p.ldo;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * E;
    if (c < p.D) {
      float w[E], b[E], o[E];
      if (p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, w);
      if (p.b != nullptr) load_w<T, E>(p.b, c, p.w_f32, b);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float h = (v[i * E + j] - mean) * rstd;
        o[j] = h * (p.w != nullptr ? w[j] : 1.0f) + (p.b != nullptr ? b[j] : 0.0f);
      }
      store_e<T, E>(y + c, o);
    }
  }
}

// Persistent: each CTA takes every gridDim.x-th row (group of rows), its threads keep the dw / db
// sums of their own columns in registers and write one partial row at the end.
template <typename T, int E, int EPT, int TPR>
__global__ void __launch_bounds__(NormCta<TPR>::kThreads)
norm_bwd_kernel(const NormParams p) {
  constexpr int NV = EPT / E;
  constexpr int kRows = NormCta<TPR>::kThreads / TPR;
  __shared__ float2 red[2 * (TPR / 32)];
  int turn = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float w[EPT], dw[EPT], db[EPT];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * E;
#pragma unroll
    for (int j = 0; j < E; ++j) { w[i * E + j] = c < p.D ? 1.0f : 0.f; dw[i * E + j] = 0.f; db[i * E + j] = 0.f; }
    if (c < p.D && p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, w + i * E);
  }
  const float inv = 1.0f / static_cast<float>(p.D);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub; row < p.M;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float h[EPT], d[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * E;
      if (c < p.D) {
        load_e<T, E>(x + c, h + i * E);
        load_e<T, E>(dy + c, d + i * E);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) { h[i * E + j] = mean; d[i * E + j] = 0.f; }
      }
    }
    float sa = 0.f, sh = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      h[i] = (h[i] - mean) * rstd;
      dw[i] += d[i] * h[i];
      db[i] += d[i];
      d[i] *= w[i];
      sa += d[i];
      sh += d[i] * h[i];
    }
    const float2 s = row_sum2<TPR>(sa, sh, red, turn);
    const float ma = s.x * inv, mh = s.y * inv;
    T* dx = static_cast<T*>(p.out) + row * p.ldo;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * E;
      if (c < p.D) {
        float o[E];
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = rstd * (d[i * E + j] - ma - h[i * E + j] * mh);
        store_e<T, E>(dx + c, o);
      }
    }
  }
  if (p.part_w == nullptr) return;
  if (TPR == 32) {
    // The warps of the CTA hold sums of the same columns: added in warp order.
    __shared__ float acc[TPR == 32 ? 2 * 32 * EPT : 1];
    for (int s = 0; s < kRows; ++s) {
      if (sub == s) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          const int k = i * 32 + t;
          acc[k] = s == 0 ? dw[i] : acc[k] + dw[i];
          acc[32 * EPT + k] = s == 0 ? db[i] : acc[32 * EPT + k] + db[i];
        }
      }
      __syncthreads();
    }
    if (sub != 0) return;
#pragma unroll
    for (int i = 0; i < EPT; ++i) { dw[i] = acc[i * 32 + t]; db[i] = acc[32 * EPT + i * 32 + t]; }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * E;
    if (c < p.D) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        p.part_w[blockIdx.x * p.ldp + c + j] = dw[i * E + j];
        p.part_b[blockIdx.x * p.ldp + c + j] = db[i * E + j];
      }
    }
  }
}

// Rows of any width: one CTA of 512 threads per row, values read again for each pass.
constexpr int kNormWide = 512;

template <typename T>
__global__ void __launch_bounds__(kNormWide)
norm_fwd_wide_kernel(const NormParams p) {
  __shared__ float2 red[2 * (kNormWide / 32)];
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const float inv = 1.0f / static_cast<float>(p.D);
  float s = 0.f;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) s += to_f(x[c]);
  const float mean = row_sum2<kNormWide>(s, 0.f, red, turn).x * inv;
  s = 0.f;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) { const float d = to_f(x[c]) - mean; s += d * d; }
  const float rstd = 1.0f / sqrtf(row_sum2<kNormWide>(s, 0.f, red, turn).x * inv + p.eps);
  if (threadIdx.x == 0 && p.mean != nullptr) { p.mean[row] = mean; p.rstd[row] = rstd; }
  T* y = static_cast<T*>(p.out) + row * p.ldo;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) {
    float w = 1.f, b = 0.f;
    if (p.w != nullptr) load_w<T, 1>(p.w, c, p.w_f32, &w);
    if (p.b != nullptr) load_w<T, 1>(p.b, c, p.w_f32, &b);
    y[c] = from_f<T>((to_f(x[c]) - mean) * rstd * w + b);
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormWide)
norm_dx_wide_kernel(const NormParams p) {
  __shared__ float2 red[2 * (kNormWide / 32)];
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
  const float mean = p.mean[row], rstd = p.rstd[row];
  const float inv = 1.0f / static_cast<float>(p.D);
  float sa = 0.f, sh = 0.f;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) {
    float w = 1.f;
    if (p.w != nullptr) load_w<T, 1>(p.w, c, p.w_f32, &w);
    const float a = to_f(dy[c]) * w;
    sa += a;
    sh += a * ((to_f(x[c]) - mean) * rstd);
  }
  const float2 s = row_sum2<kNormWide>(sa, sh, red, turn);
  T* dx = static_cast<T*>(p.out) + row * p.ldo;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) {
    float w = 1.f;
    if (p.w != nullptr) load_w<T, 1>(p.w, c, p.w_f32, &w);
    const float a = to_f(dy[c]) * w;
    dx[c] = from_f<T>(rstd * (a - s.x * inv - (to_f(x[c]) - mean) * rstd * (s.y * inv)));
  }
}

// Partial dw / db of a row block: one thread per column.
template <typename T>
__global__ void __launch_bounds__(256)
norm_dw_wide_kernel(const NormParams p, int rows_per_block) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.D) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t r1 = min(p.M, r0 + rows_per_block);
  float sw = 0.f, sb = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float d = to_f(static_cast<const T*>(p.dy)[r * p.lddy + c]);
    const float h = (to_f(static_cast<const T*>(p.x)[r * p.ldx + c]) - p.mean[r]) * p.rstd[r];
    sw += d * h;
    sb += d;
  }
  p.part_w[blockIdx.y * p.ldp + c] = sw;
  p.part_b[blockIdx.y * p.ldp + c] = sb;
}

}  // namespace dc
