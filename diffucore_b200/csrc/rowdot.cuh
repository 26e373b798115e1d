// The projections of a few rows (decoded tokens, conditioning vectors): y = act(x . w^T + b) + r and
// the gated form for up to 16 rows. The weights, read once, are all the traffic that counts, so this
// kernel is built around that stream instead of shared-memory tiles.
//
// A warp owns 16 weight rows (16 output columns; gated: 8 columns, their gate rows and their up
// rows) and multiplies them as the 16 x k operand of mma.m16n8k16 with 8 rows of x as the k x 8
// operand, fp32 accumulators in registers. The contraction may visit k in any order as long as both
// operands agree, so each lane takes 16 consecutive bytes of its weight row and of its x row, which
// are its fragments of two instructions: no shared memory, no shuffles, four pieces of each stream in
// flight. The tensor pipe idles (at most 2 instructions per 1 KB of weights); the kernel is bound by
// HBM, and for narrow layers by latency, which is why `ks` warps divide the k of one group of rows.
// Their partial sums are added in a fixed order.
//
// Weights whose rows a 16-byte load cannot take are read by single values instead of being copied; so
// are aligned weights beside an x (of up to 8 rows) whose own rows are not aligned.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "hgemm.cuh"

namespace dc {

constexpr int kRowDotMax = 16;          // rows of x
constexpr int kRowDotWarps = 8;         // warps per CTA (16 when they all divide one group's k)

struct RowDotParams {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* w0;        // linear: w; gated: w_gate
  int64_t ldw0;
  const uint16_t* w1;        // gated: w_up
  int64_t ldw1;
  const uint16_t* bias0;
  const uint16_t* bias1;
  const uint16_t* residual;
  int64_t ldr;
  uint16_t* out;
  int64_t ldo;
  float* z0;
  float* z1;
  int64_t ldz;
  int M, N, K;
  int ks;                    // warps that divide the k of one column group: 1, 2, 4, 8 or 16
  int act;
};

__device__ __forceinline__ uint4 load_stream(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Eight values at row + k, zeros past K. STREAM: read once, kept out of L1.
template <bool VEC, bool STREAM>
__device__ __forceinline__ uint4 load_piece(const uint16_t* row, int k, int K) {
  if (VEC && k + 8 <= K) return STREAM ? load_stream(row + k) : __ldg(reinterpret_cast<const uint4*>(row + k));
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k < K) {
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = k + i < K ? __ldg(row + k + i) : 0u;
    v = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
  }
  return v;
}

// D += A . B on one warp: A 16 x 16 (a0..a3), B 16 x 8 (b0, b1).
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One value through an activation. A call of its own: inlined, its registers change the order of the
// main loop's loads (gated 4 x 2 x 10240 x 4096 33.8 us, 29.1 so).
__device__ __noinline__ float act_one(float z, int act) {
  Pair v[1] = {both(z)};
  act_values(v, act);
  return dc::split(v[0]).x;
}

// NT: blocks of 8 rows of x (1 or 2). kAhead: steps whose loads are in flight at once.
template <int NT, bool GATED, bool VEC, bool BF16, int kAhead>
__global__ void __launch_bounds__(512)
rowdot_kernel(const RowDotParams p) {
  constexpr int kCols = GATED ? 8 : 16;         // output columns per warp
  constexpr int kRows = 8 * NT;                 // rows of x, padded
  extern __shared__ float sums[];               // [warp][16 weight rows][kRows]
  pdl_enter();
  const int warp = warp_id(), lane = lane_id();
  const int warps = static_cast<int>(blockDim.x) >> 5;
  const int groups = warps / p.ks;              // column groups per CTA
  const int group = warp / p.ks, split = warp % p.ks;
  const int n0 = (static_cast<int>(blockIdx.x) * groups + group) * kCols;
  const int g = lane >> 2, t = lane & 3;        // weight row / x row of the fragments, piece of the quad
  if (n0 < p.N) {
    // Rows past N repeat the last one; their sums are never stored.
    const uint16_t* wa = p.w0 + static_cast<int64_t>(min(n0 + g, p.N - 1)) * p.ldw0;
    const uint16_t* wb = GATED ? p.w1 + static_cast<int64_t>(min(n0 + g, p.N - 1)) * p.ldw1
                               : p.w0 + static_cast<int64_t>(min(n0 + g + 8, p.N - 1)) * p.ldw0;
    const uint16_t* x[NT];
    bool live[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      live[i] = 8 * i + g < p.M;
      x[i] = p.x + static_cast<int64_t>(min(8 * i + g, p.M - 1)) * p.ldx;
    }
    float d[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) d[i][j] = 0.f;
    const int steps = (p.K + 31) >> 5;          // of 32 values: 8 per lane of a quad
    const int begin = static_cast<int>(static_cast<int64_t>(steps) * split / p.ks);
    const int end = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.ks);
    for (int s0 = begin; s0 < end; s0 += kAhead) {
      uint4 a[kAhead], b[kAhead], xv[kAhead][NT];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = s0 + u < end ? (s0 + u) * 32 + t * 8 : p.K;
        a[u] = load_piece<VEC, true>(wa, k, p.K);
        b[u] = load_piece<VEC, true>(wb, k, p.K);
#pragma unroll
        for (int i = 0; i < NT; ++i) xv[u][i] = load_piece<VEC, false>(x[i], live[i] ? k : p.K, p.K);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          mma_16816<BF16>(d[i], a[u].x, b[u].x, a[u].y, b[u].y, xv[u][i].x, xv[u][i].y);
          mma_16816<BF16>(d[i], a[u].z, b[u].z, a[u].w, b[u].w, xv[u][i].z, xv[u][i].w);
        }
    }
    float* mine = sums + warp * (16 * kRows);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      *reinterpret_cast<float2*>(mine + g * kRows + 8 * i + 2 * t) = make_float2(d[i][0], d[i][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * kRows + 8 * i + 2 * t) = make_float2(d[i][2], d[i][3]);
    }
  }
  __syncthreads();
  // Outputs of the CTA's groups, columns fastest.
  const int outs = groups * kCols * p.M;
  for (int i = static_cast<int>(threadIdx.x); i < outs; i += static_cast<int>(blockDim.x)) {
    const int j = i % kCols, q = i / kCols;
    const int m = q % p.M, grp = q / p.M;
    const int n = (static_cast<int>(blockIdx.x) * groups + grp) * kCols + j;
    if (n >= p.N) continue;
    const float* part = sums + grp * p.ks * (16 * kRows) + j * kRows + m;
    float z = 0.f, u = 0.f;
    for (int s = 0; s < p.ks; ++s) {
      z += part[s * (16 * kRows)];
      if (GATED) u += part[s * (16 * kRows) + 8 * kRows];
    }
    if (p.bias0 != nullptr) z += h_to_f(p.bias0[n], BF16);
    if (p.z0 != nullptr) p.z0[m * p.ldz + n] = z;
    float y = act_one(z, p.act);
    if (GATED) {
      if (p.bias1 != nullptr) u += h_to_f(p.bias1[n], BF16);
      if (p.z1 != nullptr) p.z1[m * p.ldz + n] = u;
      y *= u;
    } else if (p.residual != nullptr) {
      y += h_to_f(p.residual[m * p.ldr + n], BF16);
    }
    p.out[m * p.ldo + n] = static_cast<uint16_t>(pack_h2(y, y, BF16));
  }
}

}  // namespace dc
