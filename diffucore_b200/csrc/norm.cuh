// Layer norm: y = (x - mean) * rstd * w + b over rows of D values, mean and rstd kept in fp32 for
// the backward pass
//   dx = rstd (a - mean(a) - xhat mean(a xhat)),  a = dy w,  xhat = (x - mean) rstd
//   dw = sum_rows dy xhat,  db = sum_rows dy.
// Bound by HBM: forward one read and one write of x, backward two reads and one write. Every value is
// read once and held in registers while its row's sums are formed; the variance is the mean of
// squared deviations from the mean (no cancellation). Only rows beyond the widest register layout
// are read again from cache. rstd is rsqrtf's, good to 2 units in the last place of fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>
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
  if constexpr (E == 1) {
    *p = from_f<T>(f[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    constexpr int bf16 = std::is_same<T, __nv_bfloat16>::value;
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_h2(f[0], f[1], bf16), pack_h2(f[2], f[3], bf16),
                                              pack_h2(f[4], f[5], bf16), pack_h2(f[6], f[7], bf16));
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

// A 16-byte unit of x's type as pairs of floats, and back.
template <typename T>
__device__ __forceinline__ void unit_pairs(const uint4& u, Pair (&f)[8 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(T) == 4) {
    f[0] = pair(__uint_as_float(w[0]), __uint_as_float(w[1]));
    f[1] = pair(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[i] = pair(v.x, v.y);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pairs_unit(const Pair (&f)[8 / sizeof(T)]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
    const float2 a = split(f[0]), b = split(f[1]);
    w[0] = __float_as_uint(a.x); w[1] = __float_as_uint(a.y); w[2] = __float_as_uint(b.x); w[3] = __float_as_uint(b.y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = split(f[i]);
      w[i] = pack_h2(v.x, v.y, std::is_same<T, __nv_bfloat16>::value);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
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
  float* part_w;            // backward: [parts, ldp] partial column sums, or null
  float* part_b;
  int64_t ldp;
  int parts;                // partial rows
  int64_t M;
  int D;
  float eps;
  int w_f32;
  int stages, slot;         // ring kernel: stages, bytes per row and tensor
};

template <int TPR> struct NormCta { static constexpr int kThreads = TPR == 32 ? 256 : TPR; };

// Forward of few rows, in registers: TPR threads per row, NU units each, all loaded at once. A unit is
// 16 bytes (VEC) or one value, kept packed until it is used. Rows of 32 threads need no barrier, wider
// ones two; bound by latency (one row of 4096 6 us a call, most of it the host's).
template <typename T, bool VEC, int NU, int TPR>
__global__ void __launch_bounds__(NormCta<TPR>::kThreads)
norm_fwd_kernel(const NormParams p) {
  constexpr int E = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int kRows = NormCta<TPR>::kThreads / TPR;
  using Unit = typename NormUnit<T, VEC>::type;
  __shared__ float2 red[2 * (TPR / 32)];
  pdl_enter();
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
  const float rstd = rsqrtf(row_sum2<TPR>(s, 0.f, red, turn).x * inv + p.eps);
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
// forward pass of many rows. Persistent CTAs of 128 threads (more for wide rows) take kRows rows at
// a time, TPR threads and EPT values per thread for each; warp 0 also issues the copies,
// into the stage that the previous step emptied (a warp of its own for them would cost the others a
// quarter of their registers). A thread keeps its columns of w (and of the dw / db sums) in registers for all its rows.
// Those registers leave too little occupancy to hide HBM's latency with loads in flight; the ring keeps
// several rows per CTA on their way whatever the occupancy.
//
// A bulk copy starts and ends on 16-byte boundaries. Where rows do not (E == 1), the copy takes the
// aligned window around the row; the bytes before and after it belong to the neighbouring rows, and
// the first and the last row, which lack one, are read in place instead.
constexpr int kRingMax = 8;

template <typename T, int TPR, int EPT, bool BWD> struct RingCta {
  static constexpr int kThreads = TPR > 128 ? TPR : 128;
  // With 32 values' dw / db sums in registers, w can be read from shared memory so that 384 threads fit
  // an SM instead of 256. Measured with and without: 30000 x 2048 bf16 81 / 89 us, 32768 x 4096 fp32
  // 260 / 275, but 32768 x 4096 bf16 177 / 163.
  static constexpr bool kSharedW = BWD && EPT == 32 && (sizeof(T) == 4 || TPR < 128);
  static constexpr int kWBytes = kSharedW ? TPR * EPT * 4 : 0;
  static constexpr int kSmThreads =                       // resident per SM
      EPT > 16 ? (!BWD ? 512 : kSharedW || EPT == 24 ? 384 : 256) : (BWD ? 512 : 768);
  static constexpr int kPerSm = kSmThreads > kThreads ? kSmThreads / kThreads : 1;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <typename T, int E, int EPT, int TPR, bool BWD>
__global__ void __launch_bounds__(RingCta<T, TPR, EPT, BWD>::kThreads, RingCta<T, TPR, EPT, BWD>::kPerSm)
norm_ring_kernel(const NormParams p) {
  constexpr int NV = EPT / E;
  constexpr int kThreads = RingCta<T, TPR, EPT, BWD>::kThreads;
  constexpr int kWarps = kThreads / 32;
  constexpr int kRows = kThreads / TPR;
  constexpr int kTensors = BWD ? 2 : 1;
  using Cta = RingCta<T, TPR, EPT, BWD>;
  extern __shared__ __align__(16) uint8_t ring_smem[]; // w pairs, then [stage][row][x, dy][slot]
  uint8_t* const ring = ring_smem + Cta::kWBytes;
  __shared__ __align__(8) uint64_t full[kRingMax];
  __shared__ __align__(8) uint64_t empty[kRingMax];
  __shared__ float2 red[2 * kWarps];
  const int warp = warp_id(), lane = lane_id();
  const int64_t blocks = (p.M + kRows - 1) / kRows;
  const uint8_t* src[2] = {static_cast<const uint8_t*>(p.x), static_cast<const uint8_t*>(p.dy)};
  const int64_t pitch[2] = {p.ldx * static_cast<int64_t>(sizeof(T)), p.lddy * static_cast<int64_t>(sizeof(T))};
  const int row_bytes = p.D * static_cast<int>(sizeof(T));
  auto in_place = [&](int64_t row) { return E == 1 && (row == 0 || row == p.M - 1); };
  auto slot = [&](int stage, int r, int which) { return ring + ((stage * kRows + r) * kTensors + which) * p.slot; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], kWarps); }
    fence_barrier_init();
  }
  pdl_enter();
  __syncthreads();

  // Warp 0: the copies of a block's rows into a stage, lane r row r.
  auto issue = [&](int stage, int64_t block) {
    const int64_t row = block * kRows + lane;
    const bool copies = lane < kRows && row < p.M && !in_place(row);
    uintptr_t lo[kTensors];
    uint32_t n[kTensors], total = 0;
#pragma unroll
    for (int k = 0; k < kTensors; ++k) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src[k] + row * pitch[k]);
      lo[k] = at & ~uintptr_t(15);
      n[k] = static_cast<uint32_t>(((at + row_bytes + 15) & ~uintptr_t(15)) - lo[k]);
      if (copies) total += n[k];
    }
    if constexpr (kRows > 1) {
#pragma unroll
      for (int o = 1; o < kRows; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);    // rows are in the first lanes
    }
    if (lane == 0) {
      if (total > 0) mbar_arrive_expect_tx(&full[stage], total);
      else mbar_arrive(&full[stage]);
    }
    __syncwarp();
    if (copies) {
#pragma unroll
      for (int k = 0; k < kTensors; ++k) bulk_load(slot(stage, lane, k), reinterpret_cast<const void*>(lo[k]), n[k], &full[stage]);
    }
    __syncwarp();
  };
  if (warp == 0) {
    for (int s = 0; s < p.stages; ++s) {
      const int64_t block = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
      if (block < blocks) issue(s, block);
    }
  }

  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  constexpr int kPairs = EPT / 2;
  // forward: sb is b; kSharedW: w is at ws[i * TPR + t], two pairs each
  Pair w[Cta::kSharedW ? 1 : kPairs], sw[kPairs], sb[kPairs];
  ulonglong2* const ws = reinterpret_cast<ulonglong2*>(ring_smem);
  {
    float wf[EPT], bf[EPT];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * E;
#pragma unroll
      for (int j = 0; j < E; ++j) { wf[i * E + j] = c < p.D ? 1.0f : 0.f; bf[i * E + j] = 0.f; }
      if (c < p.D && p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, wf + i * E);
      if (!BWD && c < p.D && p.b != nullptr) load_w<T, E>(p.b, c, p.w_f32, bf + i * E);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      if (!Cta::kSharedW) w[Cta::kSharedW ? 0 : i] = pair(wf[2 * i], wf[2 * i + 1]);
      else if (sub == 0 && i % 2 == 0)
        ws[i / 2 * TPR + t] = make_ulonglong2(pair(wf[2 * i], wf[2 * i + 1]).v, pair(wf[2 * i + 2], wf[2 * i + 3]).v);
      sb[i] = pair(bf[2 * i], bf[2 * i + 1]);
      sw[i] = pair(0.f, 0.f);
    }
    if (Cta::kSharedW) __syncthreads();
  }
  const float inv = 1.0f / static_cast<float>(p.D);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  // Sums over a row's threads, two halves of `red` in turn so that one barrier per sum is enough.
  auto row_sums = [&](float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      if (BWD) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (TPR > 32) {
      constexpr int kParts = TPR / 32;
      float2* sl = red + turn * kWarps;
      turn ^= 1;
      if (lane == 0) sl[warp] = v;
      named_barrier_sync(1 + sub, TPR);
      v = sl[sub * kParts + lane % kParts];
#pragma unroll
      for (int o = kParts / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        if (BWD) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      }
    }
    return v;
  };
  float mean = 0.f, rstd = 0.f;                         // backward: of the next row, loaded a row ahead
  auto load_stats = [&](int64_t block) {
    const int64_t row = block * kRows + sub;
    mean = row < p.M ? p.mean[row] : 0.f;
    rstd = row < p.M ? p.rstd[row] : 0.f;
  };
  if (BWD && blockIdx.x < blocks) load_stats(blockIdx.x);

  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int64_t row = block * kRows + sub;
    const bool live = kRows == 1 || row < p.M;
    float mu = mean, rs = rstd;
    if (BWD && block + gridDim.x < blocks) load_stats(block + gridDim.x);
    mbar_wait(&full[stage], phase, nullptr);
    __syncwarp();
    // Values past the row read as the mean: their deviation is 0 backward, and they add 0 forward.
    Pair h[kPairs], d[BWD ? kPairs : 1];
    {
      float hf[EPT], df[EPT];
      const uint8_t* gx = src[0] + row * pitch[0];
      const uint8_t* gd = src[1] + row * pitch[1];
      auto take = [&](const T* x, const T* y) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + t) * E;
          if (live && c < p.D) {
            load_e<T, E>(x + c, hf + i * E);
            if (BWD) load_e<T, E>(y + c, df + i * E);
          } else {
#pragma unroll
            for (int j = 0; j < E; ++j) { hf[i * E + j] = mu; df[i * E + j] = 0.f; }
          }
        }
      };
      if (live && in_place(row)) {
        take(reinterpret_cast<const T*>(gx), reinterpret_cast<const T*>(gd));
      } else {
        const uint8_t* sx = slot(stage, sub, 0);
        const uint8_t* sd = slot(stage, sub, kTensors - 1);
        if (E == 1) {                                    // where the row starts in its window
          sx += reinterpret_cast<uintptr_t>(gx) & 15;
          sd += reinterpret_cast<uintptr_t>(gd) & 15;
        }
        take(reinterpret_cast<const T*>(sx), reinterpret_cast<const T*>(sd));
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        h[i] = pair(hf[2 * i], hf[2 * i + 1]);
        if (BWD) d[i] = pair(df[2 * i], df[2 * i + 1]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);          // this warp's values are in registers
    // Refill the stage of the step before: the other warps are past it or nearly so.
    if (warp == 0 && block != blockIdx.x) {
      const int prev = stage == 0 ? p.stages - 1 : stage - 1;
      const int64_t next = block + static_cast<int64_t>(p.stages - 1) * gridDim.x;
      if (next < blocks) {
        const bool ok = mbar_wait(&empty[prev], stage == 0 ? phase ^ 1 : phase, nullptr);
        if (__all_sync(0xffffffffu, ok)) issue(prev, next);
      }
    }
    if (++stage == p.stages) { stage = 0; phase ^= 1; }
    float2 s = make_float2(0.f, 0.f);
    if (BWD) {
      const Pair nm = pair(-mu, -mu), rr = pair(rs, rs);
      Pair sa = pair(0.f, 0.f), sh = sa;
#pragma unroll
      for (int i = 0; i < kPairs; i += 2) {
        ulonglong2 w2 = make_ulonglong2(0, 0);
        if (Cta::kSharedW) w2 = ws[i / 2 * TPR + t];
#pragma unroll
        for (int j = i; j < i + 2; ++j) {
          const Pair wj = Cta::kSharedW ? Pair{j == i ? w2.x : w2.y} : w[Cta::kSharedW ? 0 : j];
          h[j] = (h[j] + nm) * rr;
          sw[j] = fma(d[j], h[j], sw[j]);
          sb[j] = sb[j] + d[j];
          d[j] = d[j] * wj;
          sa = sa + d[j];
          sh = fma(d[j], h[j], sh);
        }
      }
      const float2 fa = split(sa), fh = split(sh);
      s = row_sums(make_float2(fa.x + fa.y, fh.x + fh.y));
    } else {
      Pair sa = pair(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) sa = sa + h[i];
      float2 f = split(sa);
      mu = row_sums(make_float2(f.x + f.y, 0.f)).x * inv;
      const Pair nm = pair(-mu, -mu);
      sa = pair(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        h[i] = h[i] + nm;
        // the pair's two values are E-neighbours or, one value per unit, TPR columns apart
        const int c0 = E == 1 ? 2 * i * TPR + t : (2 * i / E * TPR + t) * E, c1 = E == 1 ? c0 + TPR : c0;
        if (c1 < p.D) {
          sa = fma(h[i], h[i], sa);
        } else if (E == 1 && c0 < p.D) {
          const Pair one = pair(split(h[i]).x, 0.f);
          sa = fma(one, one, sa);
        }
      }
      f = split(sa);
      rs = rsqrtf(row_sums(make_float2(f.x + f.y, 0.f)).x * inv + p.eps);
      if (live && t == 0 && p.mean != nullptr) { p.mean[row] = mu; p.rstd[row] = rs; }
    }
    if (live) {
      T* out = static_cast<T*>(p.out) + row * p.ldo;
      const Pair rr = pair(rs, rs), nma = pair(-s.x * inv, -s.x * inv), nmh = pair(-s.y * inv, -s.y * inv);
      float o[EPT];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 f = split(BWD ? (fma(h[i], nmh, d[BWD ? i : 0]) + nma) * rr : fma(h[i] * rr, w[Cta::kSharedW ? 0 : i], sb[i]));
        o[2 * i] = f.x;
        o[2 * i + 1] = f.y;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * E;
        if (c < p.D) store_e<T, E>(out + c, o + i * E);
      }
    }
  }
  if constexpr (BWD) {
    if (p.part_w == nullptr) return;
    float fw[EPT], fb[EPT];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 x = split(sw[i]), y = split(sb[i]);
      fw[2 * i] = x.x; fw[2 * i + 1] = x.y;
      fb[2 * i] = y.x; fb[2 * i + 1] = y.y;
    }
    if (kRows > 1) {
      // The CTA's row groups hold sums of the same columns: added in the order of the groups.
      float* acc = reinterpret_cast<float*>(ring);         // no copy is under way any more
      for (int g = 0; g < kRows; ++g) {
        __syncthreads();
        if (sub == g) {
#pragma unroll
          for (int i = 0; i < EPT; ++i) {
            const int k = i * TPR + t;
            acc[k] = g == 0 ? fw[i] : acc[k] + fw[i];
            acc[TPR * EPT + k] = g == 0 ? fb[i] : acc[TPR * EPT + k] + fb[i];
          }
        }
      }
      __syncthreads();
      if (sub != 0) return;
#pragma unroll
      for (int i = 0; i < EPT; ++i) { fw[i] = acc[i * TPR + t]; fb[i] = acc[TPR * EPT + i * TPR + t]; }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * E;
      if (c < p.D) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          p.part_w[blockIdx.x * p.ldp + c + j] = fw[i * E + j];
          p.part_b[blockIdx.x * p.ldp + c + j] = fb[i * E + j];
        }
      }
    }
  }
}

// Narrow rows, forward and backward: TPR threads (4 to 32) per row, two 16-byte units each, so that
// a warp has up to eight rows under way and a sum over a row is two to five shuffles. Persistent CTAs;
// w and b (or w and the dw / db sums) stay in registers, the next row's units are loaded a row
// ahead. bf16, 48 Mi values: 64 wide 36.8 us forward (5470 GB/s) and 58.0 backward (5200), 234 and 409 by
// a warp per row through the ring; 512 wide 36.3 and 57.8, 44.0 and 66.0.
constexpr int kNarrowThreads = 256;
constexpr int kNarrowUnits = 2;

// CTAs per SM: at four the forward kernel's 64 registers spill (393216 x 128 48 us, 36 with three).
template <bool BWD> struct NormNarrow { static constexpr int kPerSm = BWD ? 2 : 3; };

template <typename T, int TPR, bool BWD>
__global__ void __launch_bounds__(kNarrowThreads, NormNarrow<BWD>::kPerSm)
norm_narrow_kernel(const NormParams p) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  constexpr int kUnitPairs = E / 2, kPairs = kNarrowUnits * kUnitPairs;
  constexpr int kRows = kNarrowThreads / TPR, kWarps = kNarrowThreads / 32;
  __shared__ float2 red[BWD ? kWarps : 1][TPR * kPairs];
  pdl_enter();
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  Pair w[kPairs], sw[kPairs], sb[kPairs];                  // forward: sb is b
#pragma unroll
  for (int i = 0; i < kNarrowUnits; ++i) {
    const int c = (i * TPR + t) * E;
    float wf[E], bf[E];
#pragma unroll
    for (int j = 0; j < E; ++j) { wf[j] = 1.0f; bf[j] = 0.f; }
    if (c < p.D && p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, wf);
    if (!BWD && c < p.D && p.b != nullptr) load_w<T, E>(p.b, c, p.w_f32, bf);
#pragma unroll
    for (int j = 0; j < kUnitPairs; ++j) {
      w[i * kUnitPairs + j] = pair(wf[2 * j], wf[2 * j + 1]);
      sb[i * kUnitPairs + j] = pair(bf[2 * j], bf[2 * j + 1]);
      sw[i * kUnitPairs + j] = pair(0.f, 0.f);
    }
  }
  const float inv = 1.0f / static_cast<float>(p.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  uint4 nx[kNarrowUnits], nd[kNarrowUnits];
  float nmu = 0.f, nrs = 0.f;
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < kNarrowUnits; ++i) {
      const int c = (i * TPR + t) * E;
      nx[i] = nd[i] = make_uint4(0, 0, 0, 0);
      if (row < p.M && c < p.D) {
        nx[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + row * p.ldx + c);
        if (BWD) nd[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dy) + row * p.lddy + c);
      }
    }
    if (BWD) {
      nmu = row < p.M ? p.mean[row] : 0.f;
      nrs = row < p.M ? p.rstd[row] : 0.f;
    }
  };
  auto row_sum = [&](Pair a) {                             // both values' sums over the row's threads
    float2 f = split(a);
    if (!BWD) f.x += f.y;
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) {
      f.x += __shfl_xor_sync(0xffffffffu, f.x, o);
      if (BWD) f.y += __shfl_xor_sync(0xffffffffu, f.y, o);
    }
    return f;
  };
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  fetch(first + sub);
  for (int64_t base = first; base < p.M; base += step) {
    const int64_t row = base + sub;
    Pair h[kPairs], d[kPairs];
#pragma unroll
    for (int i = 0; i < kNarrowUnits; ++i) {
      Pair f[kUnitPairs], g[kUnitPairs];
      unit_pairs<T>(nx[i], f);
      if (BWD) unit_pairs<T>(nd[i], g);
#pragma unroll
      for (int j = 0; j < kUnitPairs; ++j) {
        h[i * kUnitPairs + j] = f[j];
        d[i * kUnitPairs + j] = BWD ? g[j] : f[j];
      }
    }
    float mu = nmu, rs = nrs;
    if (base + step < p.M) fetch(row + step);
    Pair nma = pair(0.f, 0.f), nmh = nma;
    if constexpr (BWD) {
      const Pair nm = pair(-mu, -mu), rr = pair(rs, rs);
      Pair sa = pair(0.f, 0.f), sh = sa;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        h[i] = (h[i] + nm) * rr;
        sw[i] = fma(d[i], h[i], sw[i]);
        sb[i] = sb[i] + d[i];
        d[i] = d[i] * w[i];
        sa = sa + d[i];
        sh = fma(d[i], h[i], sh);
      }
      const float2 a = split(sa), b = split(sh);
      const float2 s = row_sum(pair(a.x + a.y, b.x + b.y));
      nma = pair(-s.x * inv, -s.x * inv);
      nmh = pair(-s.y * inv, -s.y * inv);
    } else {
      Pair s = pair(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) s = s + h[i];
      mu = row_sum(s).x * inv;
      const Pair nm = pair(-mu, -mu);
      s = pair(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kNarrowUnits; ++i) {
#pragma unroll
        for (int j = i * kUnitPairs; j < (i + 1) * kUnitPairs; ++j) {
          h[j] = h[j] + nm;
          if ((i * TPR + t) * E < p.D) s = fma(h[j], h[j], s);
        }
      }
      rs = rsqrtf(row_sum(s).x * inv + p.eps);
      if (t == 0 && row < p.M && p.mean != nullptr) { p.mean[row] = mu; p.rstd[row] = rs; }
    }
    if (row < p.M) {
      T* out = static_cast<T*>(p.out) + row * p.ldo;
      const Pair rr = pair(rs, rs);
#pragma unroll
      for (int i = 0; i < kNarrowUnits; ++i) {
        const int c = (i * TPR + t) * E;
        float o[E];
#pragma unroll
        for (int j = 0; j < kUnitPairs; ++j) {
          const int k = i * kUnitPairs + j;
          const float2 f = split(BWD ? (fma(h[k], nmh, d[k]) + nma) * rr : fma(h[k] * rr, w[k], sb[k]));
          o[2 * j] = f.x;
          o[2 * j + 1] = f.y;
        }
        if (c < p.D) store_e<T, E>(out + c, o);
      }
    }
  }
  if constexpr (BWD) {
    if (p.part_w == nullptr) return;
    // The rows' sums, added over the warp's row groups and then over the warps, always in that order.
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        float2 f = split(which == 0 ? sw[i] : sb[i]);
#pragma unroll
        for (int o = 16; o >= TPR; o >>= 1) {
          f.x += __shfl_xor_sync(0xffffffffu, f.x, o);
          f.y += __shfl_xor_sync(0xffffffffu, f.y, o);
        }
        if (lane_id() < TPR) red[warp_id()][i / kUnitPairs * TPR * kUnitPairs + t * kUnitPairs + i % kUnitPairs] = f;
      }
      __syncthreads();
      float* part = (which == 0 ? p.part_w : p.part_b) + blockIdx.x * p.ldp;
      for (int c = threadIdx.x; c < p.D; c += kNarrowThreads) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) a += reinterpret_cast<const float*>(red[k])[c];
        part[c] = a;
      }
      __syncthreads();
    }
  }
}

// The affine vector of 16-byte units of a row in shared memory: units in x's type, or, for fp32
// vectors beside 16-bit rows (W32), E / 4 planes of four floats per unit, so that a warp's loads are
// consecutive. A null vector reads as `fill`.
template <typename T, bool W32>
struct AffineStage {
  static constexpr int E = 16 / static_cast<int>(sizeof(T));
  static constexpr int kPlanes = W32 ? E / 4 : 1;

  __device__ static void store(uint4* dst, const void* w, int units, float fill) {
    for (int i = threadIdx.x; i < units * kPlanes; i += blockDim.x) {
      uint4 v;
      if (w != nullptr) {
        v = W32 ? static_cast<const uint4*>(w)[(i % units) * kPlanes + i / units] : static_cast<const uint4*>(w)[i];
      } else if (W32) {
        const uint32_t f = __float_as_uint(fill);
        v = make_uint4(f, f, f, f);
      } else {
        T* h = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int j = 0; j < E; ++j) h[j] = from_f<T>(fill);
      }
      dst[i] = v;
    }
  }
  __device__ static void load(const uint4* src, int units, int unit, Pair (&f)[E / 2]) {
    if (W32) {
#pragma unroll
      for (int q = 0; q < kPlanes; ++q) {
        const float4 v = reinterpret_cast<const float4*>(src)[q * units + unit];
        f[2 * q] = pair(v.x, v.y);
        f[2 * q + 1] = pair(v.z, v.w);
      }
    } else {
      unit_pairs<T>(src[unit], f);
    }
  }
};

// Backward of aligned rows of 8193 to 16384 values: a persistent CTA of 512 threads per row, 32 values
// per thread. The dw / db sums take 64 of the 128 registers that a thread can have, so x and dy stay
// in the ring's stage and are read twice, before and after the row's two sums, and w is staged in
// shared memory: 8000 x 16384 bf16 rows in 231 us, 298 in the kernels for any width.
constexpr int kBwdThreads = 512;
constexpr int kBwdValues = 32;

template <typename T, bool W32>
__global__ void __launch_bounds__(kBwdThreads, 1)
norm_bwd_kernel(const NormParams p) {
  using Affine = AffineStage<T, W32>;
  constexpr int E = Affine::E, NU = kBwdValues / E, kPairs = E / 2, kWarps = kBwdThreads / 32;
  extern __shared__ __align__(16) uint4 smem[];          // w, then [stage][x, dy][units]
  __shared__ __align__(8) uint64_t full[kRingMax];
  __shared__ __align__(8) uint64_t empty[kRingMax];
  __shared__ float2 red[2 * kWarps];
  const int warp = warp_id(), lane = lane_id();
  const int t = threadIdx.x;
  const int units = p.D / E;
  const uint32_t row_bytes = static_cast<uint32_t>(units) * 16;
  uint4* const ring = smem + units * Affine::kPlanes;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], kWarps); }
    fence_barrier_init();
  }
  pdl_enter();
  Affine::store(smem, p.w, units, 1.0f);
  __syncthreads();
  auto issue = [&](int stage, int64_t row) {              // thread 0
    uint4* dst = ring + static_cast<int64_t>(stage) * 2 * units;
    mbar_arrive_expect_tx(&full[stage], 2 * row_bytes);
    bulk_load(dst, x + row * p.ldx, row_bytes, &full[stage]);
    bulk_load(dst + units, dy + row * p.lddy, row_bytes, &full[stage]);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      const int64_t row = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
      if (row < p.M) issue(s, row);
    }
  }
  Pair sw[NU][kPairs], sb[NU][kPairs];
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < kPairs; ++j) { sw[i][j] = pair(0.f, 0.f); sb[i][j] = sw[i][j]; }
  const float inv = 1.0f / static_cast<float>(p.D);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  float next_mean = 0.f, next_rstd = 0.f;                // loaded a row ahead
  auto load_stats = [&](int64_t row) {
    next_mean = p.mean[row];
    next_rstd = p.rstd[row];
  };
  if (blockIdx.x < p.M) load_stats(blockIdx.x);
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const Pair nm = pair(-next_mean, -next_mean), rr = pair(next_rstd, next_rstd);
    if (row + gridDim.x < p.M) load_stats(row + gridDim.x);
    mbar_wait(&full[stage], phase, nullptr);
    __syncwarp();
    const uint4* xs = ring + static_cast<int64_t>(stage) * 2 * units;
    const uint4* ds = xs + units;
    Pair sa[2] = {pair(0.f, 0.f), pair(0.f, 0.f)}, sh[2] = {sa[0], sa[0]};
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = i * kBwdThreads + t;
      if (u < units) {
        Pair h[kPairs], d[kPairs], w[kPairs];
        unit_pairs<T>(xs[u], h);
        unit_pairs<T>(ds[u], d);
        Affine::load(smem, units, u, w);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const Pair c = (h[j] + nm) * rr;
          sw[i][j] = fma(d[j], c, sw[i][j]);
          sb[i][j] = sb[i][j] + d[j];
          const Pair a = d[j] * w[j];
          sa[j % 2] = sa[j % 2] + a;
          sh[j % 2] = fma(a, c, sh[j % 2]);
        }
      }
    }
    const float2 fa = split(sa[0] + sa[1]), fh = split(sh[0] + sh[1]);
    float2 s = make_float2(fa.x + fa.y, fh.x + fh.y);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    float2* sl = red + turn * kWarps;                    // two halves in turn: one barrier per row
    turn ^= 1;
    if (lane == 0) sl[warp] = s;
    __syncthreads();
    s = sl[lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.ldo);
    const Pair nma = pair(-s.x * inv, -s.x * inv), nmh = pair(-s.y * inv, -s.y * inv);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = i * kBwdThreads + t;
      if (u < units) {
        Pair h[kPairs], d[kPairs], w[kPairs];
        unit_pairs<T>(xs[u], h);
        unit_pairs<T>(ds[u], d);
        Affine::load(smem, units, u, w);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) d[j] = (fma((h[j] + nm) * rr, nmh, d[j] * w[j]) + nma) * rr;
        out[u] = pairs_unit<T>(d);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
    // Refill the stage of the step before: the other warps are past it or nearly so.
    if (threadIdx.x == 0 && row != blockIdx.x) {
      const int prev = stage == 0 ? p.stages - 1 : stage - 1;
      const int64_t next = row + static_cast<int64_t>(p.stages - 1) * gridDim.x;
      if (next < p.M && mbar_wait(&empty[prev], stage == 0 ? phase ^ 1 : phase, nullptr)) issue(prev, next);
    }
    __syncwarp();
    if (++stage == p.stages) { stage = 0; phase ^= 1; }
  }
  if (p.part_w == nullptr) return;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int c = (i * kBwdThreads + t) * E;
    if (c < p.D) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int64_t at = static_cast<int64_t>(blockIdx.x) * p.ldp + c + 2 * j;     // ldp is even
        *reinterpret_cast<float2*>(p.part_w + at) = split(sw[i][j]);
        *reinterpret_cast<float2*>(p.part_b + at) = split(sb[i][j]);
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
  pdl_enter();
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const float inv = 1.0f / static_cast<float>(p.D);
  float s = 0.f;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) s += to_f(x[c]);
  const float mean = row_sum2<kNormWide>(s, 0.f, red, turn).x * inv;
  s = 0.f;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) { const float d = to_f(x[c]) - mean; s += d * d; }
  const float rstd = rsqrtf(row_sum2<kNormWide>(s, 0.f, red, turn).x * inv + p.eps);
  if (threadIdx.x == 0 && p.mean != nullptr) { p.mean[row] = mean; p.rstd[row] = rstd; }
  T* y = static_cast<T*>(p.out) + row * p.ldo;
  for (int c = threadIdx.x; c < p.D; c += kNormWide) {
    float w = 1.f, b = 0.f;
    if (p.w != nullptr) load_w<T, 1>(p.w, c, p.w_f32, &w);
    if (p.b != nullptr) load_w<T, 1>(p.b, c, p.w_f32, &b);
    y[c] = from_f<T>((to_f(x[c]) - mean) * rstd * w + b);
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(kNormWide)
norm_dx_wide_kernel(const NormParams p) {
  __shared__ float2 red[2 * (kNormWide / 32)];
  pdl_enter();
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
  const float mean = p.mean[row], rstd = p.rstd[row];
  const float inv = 1.0f / static_cast<float>(p.D);
  float sa = 0.f, sh = 0.f;
#pragma unroll 4
  for (int c = threadIdx.x * E; c < p.D; c += kNormWide * E) {
    float xv[E], a[E], w[E];
    load_e<T, E>(x + c, xv);
    load_e<T, E>(dy + c, a);
    if (p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, w);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float v = __fmul_rn(a[j], p.w != nullptr ? w[j] : 1.f);
      sa += v;
      sh += v * ((xv[j] - mean) * rstd);
    }
  }
  const float2 s = row_sum2<kNormWide>(sa, sh, red, turn);
  const float ma = s.x * inv, mh = s.y * inv;
  T* dx = static_cast<T*>(p.out) + row * p.ldo;
#pragma unroll 4
  for (int c = threadIdx.x * E; c < p.D; c += kNormWide * E) {
    float xv[E], a[E], w[E], o[E];
    load_e<T, E>(x + c, xv);
    load_e<T, E>(dy + c, a);
    if (p.w != nullptr) load_w<T, E>(p.w, c, p.w_f32, w);
#pragma unroll
    for (int j = 0; j < E; ++j)
      o[j] = rstd * (__fmul_rn(a[j], p.w != nullptr ? w[j] : 1.f) - ma - (xv[j] - mean) * rstd * mh);
    store_e<T, E>(dx + c, o);
  }
}

// Partial dw / db of a row block: one thread per E columns.
template <typename T, int E>
__global__ void __launch_bounds__(128)
norm_dw_wide_kernel(const NormParams p, int rows_per_block) {
  pdl_enter();
  const int c = (blockIdx.x * 128 + threadIdx.x) * E;
  if (c >= p.D) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t r1 = min(p.M, r0 + rows_per_block);
  float sw[E], sb[E];
#pragma unroll
  for (int j = 0; j < E; ++j) { sw[j] = 0.f; sb[j] = 0.f; }
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    float d[E], xv[E];
    load_e<T, E>(static_cast<const T*>(p.dy) + r * p.lddy + c, d);
    load_e<T, E>(static_cast<const T*>(p.x) + r * p.ldx + c, xv);
    const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
    for (int j = 0; j < E; ++j) { sw[j] += d[j] * ((xv[j] - mean) * rstd); sb[j] += d[j]; }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) { p.part_w[blockIdx.y * p.ldp + c + j] = sw[j]; p.part_b[blockIdx.y * p.ldp + c + j] = sb[j]; }
}

}  // namespace dc
