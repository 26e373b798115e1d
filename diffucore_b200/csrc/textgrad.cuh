// Pointwise part of the projections' backward pass and the column sums of the weight, bias and
// norm gradients. All sums are fp32 in a fixed order: the row groups of a CTA add their rows in order
// and then one another's sums into one partial row per row block, and colsum_finish adds the partial
// rows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "hgemm.cuh"

namespace dc {

constexpr int kGradX = 64;                      // threads across the columns of a CTA, 8 columns each
constexpr int kGradY = 4;                       // row groups of a CTA
constexpr int kGradCols = 8 * kGradX;

struct ActGradParams {
  const uint16_t* dy;       // [M, N], row stride lddy
  int64_t lddy;
  const float* z0;          // kept pre-activations, row stride ldz (a multiple of 4); null: dz = dy
  const float* z1;          // gated: the up projection's
  int64_t ldz;
  uint16_t* dz0;            // outputs, row stride lddz (a multiple of 8); null: sums only
  uint16_t* dz1;
  int64_t lddz;
  float* part0;             // [row blocks, ldp] column sums of dz before rounding, or null
  float* part1;
  int64_t ldp;              // a multiple of 8
  int64_t M, N;
  int rows_per_block;
  int act, bf16, dy_vec;
};

// Eight 16-bit values (one vector access when `vec`), zero past `n` of them.
__device__ __forceinline__ uint4 load8_bits(const uint16_t* src, int n, bool vec) {
  if (vec && n >= 8) return __ldg(reinterpret_cast<const uint4*>(src));
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = i < n ? __ldg(src + i) : 0u;
  return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}
// Eight values at any even address as the words that hold them (WORDS), five where the first value is the
// second half of a word. Near the ends of the matrix [base, end), where a word could reach outside,
// and for fewer than 8 values they are read one by one into the same layout.
template <bool WORDS> struct Raw8 { uint4 w; };
template <> struct Raw8<true> { uint4 w; uint32_t last; };
__device__ __forceinline__ Raw8<true> load8_words(const uint16_t* src, int n, const uint16_t* base, const uint16_t* end) {
  Raw8<true> v;
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 2) >> 1);
  if (n >= 8 && (skip == 0 || (src > base && src + 9 <= end))) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(src - skip);
    v.w = make_uint4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
    v.last = skip ? __ldg(q + 4) : 0u;
    return v;
  }
  uint32_t h[9];
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const int k = i - skip;
    h[i] = k >= 0 && k < n && k < 8 ? __ldg(src + k) : 0u;
  }
  v.w = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
  v.last = h[8];
  return v;
}
template <bool WORDS>
__device__ __forceinline__ uint4 bits8(const Raw8<WORDS>& v, const uint16_t* src) {
  if constexpr (WORDS) {
    if (reinterpret_cast<uintptr_t>(src) & 2)
      return make_uint4(__funnelshift_r(v.w.x, v.w.y, 16), __funnelshift_r(v.w.y, v.w.z, 16), __funnelshift_r(v.w.z, v.w.w, 16),
                        __funnelshift_r(v.w.w, v.last, 16));
  }
  return v.w;
}

struct Float8 { float4 a, b; };
__device__ __forceinline__ Float8 load8_floats(const float* src, bool hi) {
  const float4* q = reinterpret_cast<const float4*>(src);
  return Float8{q[0], hi ? q[1] : make_float4(0.f, 0.f, 0.f, 0.f)};
}
__device__ __forceinline__ void pairs_of(const Float8& v, Pair (&f)[4]) {
  f[0] = pair(v.a.x, v.a.y); f[1] = pair(v.a.z, v.a.w); f[2] = pair(v.b.x, v.b.y); f[3] = pair(v.b.z, v.b.w);
}

// FORM 0: column sums of dy alone; 1: dz = dy act'(z); 2 (gated): dg = dy u act'(g), du = dy act(g).
// A thread owns 8 columns, a CTA 512 columns of a row block, its four row groups every fourth row.
// Bound by HBM: 2 B (dy) + 4 or 8 B (z) read and 2 or 4 B written per element. kAhead rows per thread
// are loaded, as they are in memory, ahead of their arithmetic: made into pairs where they are
// loaded they wait for each row in turn (57.3 us against 41.8 for 8192 x 4096 without an activation).
// dz is rounded to the 16 bits that the tensor core's operands have; the column sums are of dz before
// that. Against 64 bits it takes the relative error of dx and dw from 0.0017 (their own rounding to bf16) to
// 0.0023, from 0.00021 to 0.00029 in fp16; dz in two 16-bit halves would cost a second product each.
// Three CTAs per SM where registers allow it (gelu_tanh 45.7 us, 49.3 with two); at 8192 x 4096
// 41.8 us without an activation (6430 GB/s), 45.9 with GELU, 4.9 more with the bias's gradient;
// gated 4173 x 5464 with SiLU 51.6 us (6190 GB/s). Rows of dy that 16-byte accesses do not fit are read
// as words in the gated form (4173 x 5461 with biases 68.1 us, 77.5 by values); the other forms have no
// registers to spare for them (20000 x 1001 46.9 us, 43.7 by values).
template <int FORM, bool WORDS>
__global__ void __launch_bounds__(kGradX * kGradY, FORM == 2 ? 2 : 3)
act_grad_kernel(const ActGradParams p) {
  constexpr int kAhead = FORM == 0 ? 8 : FORM == 1 ? 3 : 2;
  __shared__ __align__(16) float red[FORM == 2 ? 2 : 1][kGradY][kGradCols];
  pdl_enter();
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kGradCols + threadIdx.x * 8;
  const int n = static_cast<int>(min(static_cast<int64_t>(8), p.N - col));      // may be <= 0
  const bool z_hi = n > 4;                  // z rows are padded to 4 values
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * p.rows_per_block;
  const int64_t r1 = min(p.M, r0 + p.rows_per_block);
  Pair s0[4], s1[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) s0[j] = s1[j] = both(0.f);
  if (n > 0) {
    for (int64_t rb = r0 + threadIdx.y; rb < r1; rb += kGradY * kAhead) {
      Raw8<WORDS> dv[kAhead];
      Float8 zv[kAhead], uv[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t r = rb + k * kGradY;
        if (r < r1) {
          const uint16_t* dy = p.dy + r * p.lddy + col;
          if constexpr (WORDS) dv[k] = load8_words(dy, n, p.dy, p.dy + (p.M - 1) * p.lddy + p.N);
          else dv[k].w = load8_bits(dy, n, p.dy_vec);
          if (FORM >= 1) zv[k] = load8_floats(p.z0 + r * p.ldz + col, z_hi);
          if (FORM == 2) uv[k] = load8_floats(p.z1 + r * p.ldz + col, z_hi);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t r = rb + k * kGradY;
        if (r >= r1) break;
        Pair d[4], z[4], u[4];
        unpack8(bits8<WORDS>(dv[k], p.dy + r * p.lddy + col), d, p.bf16);
        if (FORM >= 1) pairs_of(zv[k], z);
        if (FORM == 2) pairs_of(uv[k], u);
        if (FORM == 1) {
          act_grads(z, p.act, [&](int j, Pair, Pair da) { d[j] = d[j] * da; });
          *reinterpret_cast<uint4*>(p.dz0 + r * p.lddz + col) = pack8(d, p.bf16);     // rows are padded to 8
        }
        if (FORM == 2) {
          Pair e[4];
          act_grads(z, p.act, [&](int j, Pair a, Pair da) { e[j] = d[j] * a; d[j] = d[j] * u[j] * da; });
          *reinterpret_cast<uint4*>(p.dz0 + r * p.lddz + col) = pack8(d, p.bf16);
          *reinterpret_cast<uint4*>(p.dz1 + r * p.lddz + col) = pack8(e, p.bf16);
#pragma unroll
          for (int j = 0; j < 4; ++j) s1[j] = s1[j] + e[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s0[j] = s0[j] + d[j];
      }
    }
  }
  if (p.part0 == nullptr) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    *reinterpret_cast<float2*>(&red[0][threadIdx.y][threadIdx.x * 8 + 2 * j]) = split(s0[j]);
    if (FORM == 2) *reinterpret_cast<float2*>(&red[FORM == 2][threadIdx.y][threadIdx.x * 8 + 2 * j]) = split(s1[j]);
  }
  __syncthreads();
  for (int i = threadIdx.y * kGradX + threadIdx.x; i < kGradCols; i += kGradX * kGradY) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kGradCols + i;
    if (c >= p.N) continue;
    float a = red[0][0][i], b = FORM == 2 ? red[FORM == 2][0][i] : 0.f;
#pragma unroll
    for (int y = 1; y < kGradY; ++y) {
      a += red[0][y][i];
      if (FORM == 2) b += red[FORM == 2][y][i];
    }
    p.part0[blockIdx.y * p.ldp + c] = a;
    if (FORM == 2) p.part1[blockIdx.y * p.ldp + c] = b;
  }
}

__device__ __forceinline__ void store_as(void* dst, int64_t i, float v, int dtype) {
  if (dtype == DC_DTYPE_F32) static_cast<float*>(dst)[i] = v;
  else if (dtype == DC_DTYPE_BF16) static_cast<__nv_bfloat16*>(dst)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(dst)[i] = __float2half_rn(v);
}

// out[n] = sum of P partial rows. A CTA of 32 columns x 32 row groups: group g adds rows g, g + 32,
// ..., then the groups are added in order. Latency-bound (a few MB from L2), so every group's first
// loads are in flight at once. blockIdx.y picks one of two sums.
constexpr int kFinishGroups = 32;

__global__ void __launch_bounds__(32 * kFinishGroups)
colsum_finish_kernel(const float* __restrict__ part0, const float* __restrict__ part1, int64_t ldp, int P, int64_t N,
                     void* out0, void* out1, int dtype) {
  pdl_enter();
  const float* part = blockIdx.y ? part1 : part0;
  void* out = blockIdx.y ? out1 : out0;
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  __shared__ float red[kFinishGroups][33];
  float s = 0.f;
  if (col < N) {
#pragma unroll 8
    for (int r = g; r < P; r += kFinishGroups) s += part[r * ldp + col];
  }
  red[g][lane] = s;
  __syncthreads();
  if (g == 0 && col < N) {
#pragma unroll
    for (int i = 1; i < kFinishGroups; ++i) s += red[i][lane];
    store_as(out, col, s, dtype);
  }
}

}  // namespace dc
