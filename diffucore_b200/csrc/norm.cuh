// Layer norm: y = (x - mean) * rstd * w + b over rows of D values, mean and rstd kept in fp32 for
// the backward pass
//   dx = rstd (a - mean(a) - xhat mean(a xhat)),  a = dy w,  xhat = (x - mean) rstd
//   dw = sum_rows dy xhat,  db = sum_rows dy.
// Bound by HBM: forward one read and one write of x, backward two reads and one write. Every value is
// read once and held in registers while its row's sums are formed; the variance is the mean of
// squared deviations from the mean (no cancellation). Only rows beyond the widest register layout
// are read again from cache.
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

template <typename T, bool VEC> struct NormUnit { using type = T; };
template <typename T> struct NormUnit<T, true> { using type = uint4; };

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
  int stages, slot;         // ring kernel: stages, bytes per row and tensor
};

template <int TPR> struct NormCta { static constexpr int kThreads = TPR == 32 ? 256 : TPR; };

// Forward, rows in registers: TPR threads per row, NU units each. A unit is 16 bytes (VEC) or one
// value, kept packed until it is used, so a warp holds a row of 4096 16-bit values in 64 registers
// per lane: 16 loads in flight per lane and no barrier at all.
template <typename T, bool VEC, int NU, int TPR>
__global__ void __launch_bounds__(NormCta<TPR>::kThreads)
norm_fwd_kernel(const NormParams p) {
  constexpr int E = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int kRows = NormCta<TPR>::kThreads / TPR;
  using Unit = typename NormUnit<T, VEC>::type;
  __shared__ float2 red[2 * (TPR / 32)];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  if (row >= p.M) return;                      // whole warps (TPR == 32) or the whole CTA
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  Unit v[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int c = (i * TPR + t) * E;
    v[i] = Unit{};                             // zero bits: zeros in every type
    if (c < p.D) v[i] = *reinterpret_cast<const Unit*>(x + c);
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const T* h = reinterpret_cast<const T*>(&v[i]);
#pragma unroll
    for (int j = 0; j < E; ++j) s += to_f(h[j]);
  }
  const float inv = 1.0f / static_cast<float>(p.D);
  const float mean = row_sum2<TPR>(s, 0.f, red, turn).x * inv;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if ((i * TPR + t) * E < p.D) {
      const T* h = reinterpret_cast<const T*>(&v[i]);
#pragma unroll
      for (int j = 0; j < E; ++j) { const float d = to_f(h[j]) - mean; s += d * d; }
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum2<TPR>(s, 0.f, red, turn).x * inv + p.eps);
  if (t == 0 && p.mean != nullptr) { p.mean[row] = mean; p.rstd[row] = rstd; }
  T* y = static_cast<T*>(p.out) + row * p.ldo;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int c = (i * TPR + t) * E;
    if (c < p.D) {
      const T* h = reinterpret_cast<const T*>(&v[i]);
      float w[E], b[E], o[E];
      if (p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, w);
      if (p.b != nullptr) load_w<T, E>(p.b, c, p.w_f32, b);
#pragma unroll
      for (int j = 0; j < E; ++j)
        o[j] = (to_f(h[j]) - mean) * rstd * (p.w != nullptr ? w[j] : 1.0f) + (p.b != nullptr ? b[j] : 0.0f);
      store_e<T, E>(y + c, o);
    }
  }
}

// Rows streamed through a ring of shared-memory stages by bulk copies: the backward pass, and the
// forward pass of rows that no 16-byte access fits. Persistent CTAs of 256 threads (512 for rows
// above 4096 values) take kRows rows at a time; each thread keeps its columns of w (and of the dw /
// db sums) in registers for all its rows. The registers that those sums take leave too little room
// to hide HBM's latency with loads in flight; the ring keeps several rows per CTA on their way
// whatever the occupancy.
//
// A bulk copy starts and ends on 16-byte boundaries. Where rows do not, the copy takes the aligned
// window around the row; the bytes before and after it belong to the neighbouring rows, and the
// first and the last row, which lack one, are read in place instead.
constexpr int kRingMax = 8;

template <int TPR> struct RingCta { static constexpr int kThreads = TPR > 256 ? TPR : 256; };

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <typename T, int E, int TPR, bool BWD>
__global__ void __launch_bounds__(RingCta<TPR>::kThreads, TPR > 256 ? 1 : 2)
norm_ring_kernel(const NormParams p) {
  constexpr int EPT = 16;
  constexpr int NV = EPT / E;
  constexpr int kRows = RingCta<TPR>::kThreads / TPR;
  constexpr int kTensors = BWD ? 2 : 1;
  extern __shared__ __align__(16) uint8_t ring[];      // [stage][row][x, dy][slot]
  __shared__ __align__(8) uint64_t full[kRingMax];
  __shared__ float2 red[2 * (RingCta<TPR>::kThreads / 32)];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int64_t blocks = (p.M + kRows - 1) / kRows;
  const uint8_t* src[2] = {static_cast<const uint8_t*>(p.x), static_cast<const uint8_t*>(p.dy)};
  const int64_t pitch[2] = {p.ldx * static_cast<int64_t>(sizeof(T)), p.lddy * static_cast<int64_t>(sizeof(T))};
  const int row_bytes = p.D * static_cast<int>(sizeof(T));
  const bool edges = E == 1;                            // rows 0 and M - 1 are read in place
  auto slot = [&](int stage, int r, int which) { return ring + ((stage * kRows + r) * kTensors + which) * p.slot; };

  // Thread 0: the copies of the rows of one block.
  auto issue = [&](int stage, int64_t block) {
    uint32_t total = 0;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      for (int r = 0; r < kRows; ++r) {
        const int64_t row = block * kRows + r;
        if (row >= p.M || (edges && (row == 0 || row == p.M - 1))) continue;
#pragma unroll
        for (int k = 0; k < kTensors; ++k) {
          const uintptr_t a = reinterpret_cast<uintptr_t>(src[k] + row * pitch[k]);
          const uintptr_t lo = a & ~uintptr_t(15), hi = (a + row_bytes + 15) & ~uintptr_t(15);
          if (pass == 0) total += static_cast<uint32_t>(hi - lo);
          else bulk_load(slot(stage, r, k), reinterpret_cast<const void*>(lo), static_cast<uint32_t>(hi - lo), &full[stage]);
        }
      }
      if (pass == 0) {
        if (total > 0) mbar_arrive_expect_tx(&full[stage], total);
        else mbar_arrive(&full[stage]);
      }
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
    for (int s = 0; s < p.stages; ++s) {
      const int64_t block = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
      if (block < blocks) issue(s, block);
    }
  }
  float w[EPT], sw[EPT], sb[EPT];                       // forward: sb is b
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * E;
#pragma unroll
    for (int j = 0; j < E; ++j) { w[i * E + j] = c < p.D ? 1.0f : 0.f; sw[i * E + j] = 0.f; sb[i * E + j] = 0.f; }
    if (c < p.D && p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, w + i * E);
    if (!BWD && c < p.D && p.b != nullptr) load_w<T, E>(p.b, c, p.w_f32, sb + i * E);
  }
  __syncthreads();
  const float inv = 1.0f / static_cast<float>(p.D);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  // Sums over a row's threads; every thread of the CTA takes part, and when it returns every thread
  // has read its values of the stage.
  auto row_sums = [&](float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    float2* sl = red + turn * (RingCta<TPR>::kThreads / 32);
    turn ^= 1;
    if (TPR > 32 && (threadIdx.x & 31) == 0) sl[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    if (TPR > 32) {
      a = 0.f; b = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) { const float2 f = sl[sub * (TPR / 32) + i]; a += f.x; b += f.y; }
    }
    return make_float2(a, b);
  };

  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int64_t row = block * kRows + sub;
    const bool live = row < p.M;
    float mean = 0.f, rstd = 0.f;
    if (BWD && live) { mean = p.mean[row]; rstd = p.rstd[row]; }
    mbar_wait(&full[stage], phase, nullptr);
    __syncwarp();
    const T* px = nullptr;
    const T* pd = nullptr;
    if (live) {
      const uint8_t* a[2];
#pragma unroll
      for (int k = 0; k < kTensors; ++k) {
        const uint8_t* g = src[k] + row * pitch[k];
        a[k] = edges && (row == 0 || row == p.M - 1) ? g : slot(stage, sub, k) + (reinterpret_cast<uintptr_t>(g) & 15);
      }
      px = reinterpret_cast<const T*>(a[0]);
      if (BWD) pd = reinterpret_cast<const T*>(a[1]);
    }
    float h[EPT], d[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * E;
      if (live && c < p.D) {
        load_e<T, E>(px + c, h + i * E);
        if (BWD) load_e<T, E>(pd + c, d + i * E);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) { h[i * E + j] = mean; d[i * E + j] = 0.f; }
      }
    }
    float2 s;
    if (BWD) {
      float sa = 0.f, sh = 0.f;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        h[i] = (h[i] - mean) * rstd;
        sw[i] += d[i] * h[i];
        sb[i] += d[i];
        d[i] = __fmul_rn(d[i], w[i]);       // the same value in the sum and in dx: a one-value row gives 0
        sa += d[i];
        sh += d[i] * h[i];
      }
      s = row_sums(sa, sh);
    } else {
      float sa = 0.f;
#pragma unroll
      for (int i = 0; i < EPT; ++i) sa += h[i];          // 0 past the row
      s = row_sums(sa, 0.f);
    }
    if (threadIdx.x == 0) {
      const int64_t next = block + static_cast<int64_t>(p.stages) * gridDim.x;
      if (next < blocks) issue(stage, next);
    }
    if (++stage == p.stages) { stage = 0; phase ^= 1; }
    if (!BWD) {
      mean = s.x * inv;
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((i * TPR + t) * E < p.D) {
#pragma unroll
          for (int j = 0; j < E; ++j) { h[i * E + j] -= mean; sq += h[i * E + j] * h[i * E + j]; }
        }
      rstd = 1.0f / sqrtf(row_sums(sq, 0.f).x * inv + p.eps);
      if (live && t == 0 && p.mean != nullptr) { p.mean[row] = mean; p.rstd[row] = rstd; }
    }
    if (live) {
      T* out = static_cast<T*>(p.out) + row * p.ldo;
      const float ma = s.x * inv, mh = s.y * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * E;
        if (c < p.D) {
          float o[E];
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const int k = i * E + j;
            o[j] = BWD ? rstd * (d[k] - ma - h[k] * mh) : h[k] * rstd * w[k] + sb[k];
          }
          store_e<T, E>(out + c, o);
        }
      }
    }
  }
  if (!BWD || p.part_w == nullptr) return;
  if (kRows > 1) {
    // The CTA's row groups hold sums of the same columns: added in the order of the groups.
    float* acc = reinterpret_cast<float*>(ring);         // no copy is under way any more
    __syncthreads();
    for (int g = 0; g < kRows; ++g) {
      if (sub == g) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          const int k = i * TPR + t;
          acc[k] = g == 0 ? sw[i] : acc[k] + sw[i];
          acc[TPR * EPT + k] = g == 0 ? sb[i] : acc[TPR * EPT + k] + sb[i];
        }
      }
      __syncthreads();
    }
    if (sub != 0) return;
#pragma unroll
    for (int i = 0; i < EPT; ++i) { sw[i] = acc[i * TPR + t]; sb[i] = acc[TPR * EPT + i * TPR + t]; }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * E;
    if (c < p.D) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        p.part_w[blockIdx.x * p.ldp + c + j] = sw[i * E + j];
        p.part_b[blockIdx.x * p.ldp + c + j] = sb[i * E + j];
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
    const float a = __fmul_rn(to_f(dy[c]), w);
    sa += a;
    sh += a * ((to_f(x[c]) - mean) * rstd);
  }
  const float2 s = row_sum2<kNormWide>(sa, sh, red, turn);
  T* dx = static_cast<T*>(p.out) + row * p.ldo;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) {
    float w = 1.f;
    if (p.w != nullptr) load_w<T, 1>(p.w, c, p.w_f32, &w);
    const float a = __fmul_rn(to_f(dy[c]), w);
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
