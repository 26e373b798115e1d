// Pointwise part of the projections' backward pass and the column sums of the weight, bias and
// norm gradients. All sums are fp32 in a fixed order: each row block adds its rows in order into
// one partial row, and colsum_finish adds the partial rows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "hgemm.cuh"

namespace dc {

constexpr int kGradThreads = 128;
constexpr int kGradCols = 4 * kGradThreads;     // columns per block

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
  int64_t ldp;
  int64_t M, N;
  int rows_per_block;
  int act, bf16, dy_vec;
};

// dz = dy act'(z); gated: dg = dy u act'(g), du = dy act(g). One thread per 4 columns, a row
// block per CTA. Bound by HBM: 2 B (dy) + 4 or 8 B (z) read and 2 or 4 B written per element.
template <bool GATED>
__global__ void __launch_bounds__(kGradThreads)
act_grad_kernel(const ActGradParams p) {
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kGradCols + threadIdx.x * 4;
  const int n = static_cast<int>(min(static_cast<int64_t>(4), p.N - col));
  if (n <= 0) return;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * p.rows_per_block;
  const int64_t r1 = min(p.M, r0 + p.rows_per_block);
  float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 4;                 // rows whose loads are in flight at once
  for (int64_t rb = r0; rb < r1; rb += kAhead) {
    float4 d4[kAhead], z4[kAhead], u4[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t r = rb + k;
      if (r < r1) {
        d4[k] = load4(p.dy + r * p.lddy + col, n, p.dy_vec, p.bf16);
        if (p.z0 != nullptr) z4[k] = *reinterpret_cast<const float4*>(p.z0 + r * p.ldz + col);
        if (GATED) u4[k] = *reinterpret_cast<const float4*>(p.z1 + r * p.ldz + col);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t r = rb + k;
      if (r >= r1) break;
      float d[4] = {d4[k].x, d4[k].y, d4[k].z, d4[k].w};
      if (p.z0 != nullptr) {
        const float z[4] = {z4[k].x, z4[k].y, z4[k].z, z4[k].w};
        float e[4];
        if (GATED) {
          const float u[4] = {u4[k].x, u4[k].y, u4[k].z, u4[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 a = act_value_grad(z[j], p.act);
            e[j] = d[j] * a.x;
            d[j] *= u[j] * a.y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) d[j] *= act_value_grad(z[j], p.act).y;
        }
        // rows of dz are padded to 8 values, so a whole unit may be written
        *reinterpret_cast<uint2*>(p.dz0 + r * p.lddz + col) = make_uint2(pack_h2(d[0], d[1], p.bf16), pack_h2(d[2], d[3], p.bf16));
        if (GATED) {
          *reinterpret_cast<uint2*>(p.dz1 + r * p.lddz + col) = make_uint2(pack_h2(e[0], e[1], p.bf16), pack_h2(e[2], e[3], p.bf16));
#pragma unroll
          for (int j = 0; j < 4; ++j) s1[j] += e[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s0[j] += d[j];
    }
  }
  if (p.part0 != nullptr) {
    *reinterpret_cast<float4*>(p.part0 + blockIdx.y * p.ldp + col) = make_float4(s0[0], s0[1], s0[2], s0[3]);
    if (GATED) *reinterpret_cast<float4*>(p.part1 + blockIdx.y * p.ldp + col) = make_float4(s1[0], s1[1], s1[2], s1[3]);
  }
}

__device__ __forceinline__ void store_as(void* dst, int64_t i, float v, int dtype) {
  if (dtype == DC_DTYPE_F32) static_cast<float*>(dst)[i] = v;
  else if (dtype == DC_DTYPE_BF16) static_cast<__nv_bfloat16*>(dst)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(dst)[i] = __float2half_rn(v);
}

// out[n] = sum of P partial rows. A CTA of 32 columns x 8 row groups: group g adds rows g, g + 8,
// ..., then the groups are added in order. blockIdx.y picks one of two sums.
__global__ void __launch_bounds__(256)
colsum_finish_kernel(const float* __restrict__ part0, const float* __restrict__ part1, int64_t ldp, int P, int64_t N,
                     void* out0, void* out1, int dtype) {
  const float* part = blockIdx.y ? part1 : part0;
  void* out = blockIdx.y ? out1 : out0;
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  __shared__ float red[8][33];
  float s = 0.f;
  if (col < N) {
#pragma unroll 4
    for (int r = g; r < P; r += 8) s += part[r * ldp + col];
  }
  red[g][lane] = s;
  __syncthreads();
  if (g == 0 && col < N) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][lane];
    store_as(out, col, s, dtype);
  }
}

}  // namespace dc
