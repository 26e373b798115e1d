// 16-bit GEMMs of the text operators on the sm_100a tensor core (bf16 / fp16 operands, fp32
// accumulators in TMEM):
//   forward   y[M, N]  = act(x[M, K] . w[N, K]^T + bias) + residual
//   gated     h[M, N]  = act(x . wg^T + bg) * (x . wu^T + bu)
//   d input   dx[M, K] = dz[M, N] . w[N, K]            (gated: dg . wg + du . wu, one accumulator)
//   d weight  dw[N, K] = dz[M, N]^T . x[M, K]          (gated: both weights in one launch)
// All four are one contraction D[m, n] = sum_k A(m, k) B(n, k); they differ in whether an operand
// is stored with k contiguous (K-major: x, w forward) or with its row index contiguous (MN-major:
// dz and x in the weight gradient, w in the input gradient). The tensor core reads either layout
// from 128-byte-swizzled tiles, so no operand is transposed in memory.
//
// Two kernels share the layouts and the epilogue arithmetic:
//   hgemm_pair_kernel     persistent, 256 x 256 tiles on a CTA pair (cta_group::2), two
//                         accumulators in TMEM so one tile's epilogue overlaps the next's MMAs
//   hgemm_cluster_kernel  128 x 128 tiles, two CTAs per SM, the contraction of a tile divided over
//                         a cluster of up to 8 CTAs whose fp32 partials meet in shared memory
// A gated tile's accumulator holds the gate in its first half of the columns and the up
// projection in the second (the pair's even CTA stages wg rows, the odd CTA wu rows), so both
// projections, the activation and the product are one pass over x.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "sm100.cuh"

namespace dc {

enum Act : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };
enum HEpi : int { kEpiLinear = 0, kEpiGated = 1 };

constexpr int kHBK = 64;                // contraction elements per swizzle atom (128 bytes)
constexpr int kHEpiWarps = 8;           // cluster kernel
constexpr int kHThreads = 64 + 32 * kHEpiWarps;
constexpr int kHAtom = 128 * 128;       // bytes of one operand atom: 128 rows (or columns) x 64 k

struct HGemmParams {
  int M, N;                // output rows and columns (gated: columns of h)
  int tiles_m, tiles_n, num_tiles, group_m;
  int bn;                  // pair kernel: accumulator columns per tile (128 .. 256, a multiple of 32)
  int kb0, kb1;            // k-blocks read from the operands' first and second maps
  int m_split;             // tiles with tm >= m_split read A's second map and write out1
  int splits;              // cluster kernel: CTAs per tile
  void* out;
  void* out1;
  int64_t ldo;
  const void* bias;        // [N] in the output dtype, or null
  const void* bias1;       // gated: the up projection's
  const void* residual;    // [M, N], or null
  int64_t ldr;
  float* z0;               // pre-activation values kept for the backward pass (fp32), or null
  float* z1;
  int64_t ldz;
  int act;
  int bf16;                // operands, bias, residual and output: bf16 (else fp16)
  int out_vec, res_vec;    // rows of out / residual are 16-byte aligned
  int a_rows;              // cluster kernel: rows of A one box loads
};

__device__ __forceinline__ float h_to_f(uint32_t bits, int bf16) {
  return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b, int bf16) {
  if (bf16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Two floats in one 64-bit register pair: the packed fp32 instructions of sm_100 do two operations per
// issue slot, and issue slots are what bounds the epilogues and the norms of 16-bit rows.
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Eight values, as four pairs, from and to 16-bit words; the type is decided once per block.
__device__ __forceinline__ void unpack8(const uint4& u, Pair (&f)[4], int bf16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if (bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[i] = pair(h.x, h.y);
    }
  }
}
__device__ __forceinline__ uint4 pack8(const Pair* f, int bf16) {
  uint32_t w[4];
  if (bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v = split(f[i]); w[i] = pack_h2(v.x, v.y, 1); }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v = split(f[i]); w[i] = pack_h2(v.x, v.y, 0); }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Activations in fp32, two values at a time. The tanh form of GELU is x * sigmoid(2 u) with
// u = sqrt(2/pi)(x + 0.044715 x^3) (0.5 (1 + tanh u) = sigmoid(2 u)), which loses nothing for
// negative x. The erf form takes the normal distribution's tail from Abramowitz and Stegun 7.1.26,
//   erfc(x) = (a1 t + a2 t^2 + ... + a5 t^5) exp(-x^2),  t = 1 / (1 + 0.3275911 x),  x >= 0,
// whose absolute error is at most 1.5e-7. Relative to a GELU of negative z that is 5e-5 at -3, 5e-4 at
// -4 and 3.6e-3 at -6, where 0.5 z (1 + erf) in fp32 cancels to 1e-6, 3e-4 and nothing; a rounding to
// bf16 is up to 4e-3, to fp16 up to 5e-4. Exponential and reciprocal are the instructions
// ex2.approx and rcp.approx, whose results are good to about 2 units in the last place; what they
// flush to zero is below 2^-126.
__device__ __forceinline__ Pair both(float a) { return pair(a, a); }
__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_ftz(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + 2^x) of both values.
__device__ __forceinline__ Pair logistic2(Pair x) {
  const float2 f = split(x);
  const float2 d = split(pair(ex2_ftz(f.x), ex2_ftz(f.y)) + both(1.0f));
  return pair(rcp_ftz(d.x), rcp_ftz(d.y));
}
__device__ __forceinline__ Pair silu_gate(Pair z) { return logistic2(z * both(-kLog2e)); }
__device__ __forceinline__ Pair tanh_gate(Pair z) {
  return logistic2(z * fma(z * z, both(-0.0713548162726f * kLog2e), both(-1.5957691216057308f * kLog2e)));
}
// P(X <= z) of a standard normal X, and e = exp(-z^2 / 2). |z| is cut at 40, where the tail has long
// been 0; within it the two values can share one reciprocal, 1/a = b / (a b).
__device__ __forceinline__ Pair normal_cdf(Pair z, Pair& e) {
  const float2 f = split(z);
  const Pair a = pair(fminf(fabsf(f.x), 40.0f), fminf(fabsf(f.y), 40.0f));
  const float2 d = split(fma(a, both(0.3275911f * 0.70710678f), both(1.0f)));
  const Pair t = pair(d.y, d.x) * both(rcp_ftz(d.x * d.y));
  const float2 x = split(a * a * both(-0.5f * kLog2e));
  e = pair(ex2_ftz(x.x), ex2_ftz(x.y));
  Pair q = fma(t, both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
  q = fma(t, q, both(0.5f * 1.421413741f));
  q = fma(t, q, both(0.5f * -0.284496736f));
  q = fma(t, q, both(0.5f * 0.254829592f));
  const Pair tail = q * t * e;
  const float2 lo = split(tail), hi = split(fma(tail, both(-1.0f), both(1.0f)));
  return pair(f.x < 0.0f ? lo.x : hi.x, f.y < 0.0f ? lo.y : hi.y);
}
__device__ __forceinline__ Pair relu_pair(Pair z) {
  const float2 f = split(z);
  return pair(f.x <= 0.0f ? 0.0f : f.x, f.y <= 0.0f ? 0.0f : f.y);      // NaN stays
}
template <int ACT>
__device__ __forceinline__ Pair act_pair(Pair z) {
  Pair e;
  if (ACT == kActRelu) return relu_pair(z);
  if (ACT == kActSilu) return z * silu_gate(z);
  if (ACT == kActGelu) return z * normal_cdf(z, e);
  if (ACT == kActGeluTanh) return z * tanh_gate(z);
  return z;
}
// Every value of a block through one activation; the switch stays outside the unrolled loops.
template <int ACT, int N>
__device__ __forceinline__ void each_pair(Pair (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = act_pair<ACT>(v[j]);
}
template <int N>
__device__ __forceinline__ void act_values(Pair (&v)[N], int act) {
  switch (act) {
    case kActRelu: each_pair<kActRelu>(v); break;
    case kActSilu: each_pair<kActSilu>(v); break;
    case kActGelu: each_pair<kActGelu>(v); break;
    case kActGeluTanh: each_pair<kActGeluTanh>(v); break;
    default: break;
  }
}

// Activation a and derivative da.
template <int ACT>
__device__ __forceinline__ void act_grad_pair(Pair z, Pair& a, Pair& da) {
  a = z;
  da = both(1.0f);
  if (ACT == kActRelu) {
    const float2 f = split(z);
    a = relu_pair(z);
    da = pair(f.x > 0.0f ? 1.0f : 0.0f, f.y > 0.0f ? 1.0f : 0.0f);
  } else if (ACT == kActSilu) {                 // s (1 + z (1 - s))
    const Pair s = silu_gate(z);
    a = z * s;
    da = s * fma(z, fma(s, both(-1.0f), both(1.0f)), both(1.0f));
  } else if (ACT == kActGelu) {                 // P(X <= z) + z phi(z)
    Pair e;
    const Pair c = normal_cdf(z, e);
    a = z * c;
    da = fma(z, e * both(0.39894228040143268f), c);
  } else if (ACT == kActGeluTanh) {             // s + z s (1 - s) (2 u)'
    const Pair s = tanh_gate(z);
    a = z * s;
    const Pair q = s * fma(s, both(-1.0f), both(1.0f));      // 0 for a large |z|, where (2 u)' may have overflowed
    const Pair du = fma(z * z, both(0.2140644488179f), both(1.5957691216057308f));
    const float2 qf = split(q), sf = split(s), g = split(fma(z * q, du, s));
    da = pair(qf.x == 0.0f ? sf.x : g.x, qf.y == 0.0f ? sf.y : g.y);
  }
}
// f(j, activation, derivative) for every pair of a block.
template <int ACT, int N, typename F>
__device__ __forceinline__ void each_grad(const Pair (&z)[N], F f) {
#pragma unroll
  for (int j = 0; j < N; ++j) { Pair a, da; act_grad_pair<ACT>(z[j], a, da); f(j, a, da); }
}
template <int N, typename F>
__device__ __forceinline__ void act_grads(const Pair (&z)[N], int act, F f) {
  switch (act) {
    case kActRelu: each_grad<kActRelu>(z, f); break;
    case kActSilu: each_grad<kActSilu>(z, f); break;
    case kActGelu: each_grad<kActGelu>(z, f); break;
    case kActGeluTanh: each_grad<kActGeluTanh>(z, f); break;
    default: each_grad<kActNone>(z, f); break;
  }
}

// ------------------------------------------------------------------ operand tiles

// TMA loads of one 64-deep atom. K-major: one box of 64 k x `rows` rows at (k, row). MN-major:
// boxes of 64 row indices x 64 k at (row + 64 i, k), 8 KB apart.
template <bool MN, bool PAIR>
__device__ __forceinline__ void load_atom(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t pair_bar,
                                          int k, int row, int rows) {
  if (MN) {
    for (int i = 0; 64 * i < rows; ++i) {
      if (PAIR) tma_load_2d_pair(dst + i * 8192, map, pair_bar, row + 64 * i, k);
      else tma_load_2d(dst + i * 8192, map, bar, row + 64 * i, k);
    }
  } else {
    if (PAIR) tma_load_2d_pair(dst, map, pair_bar, k, row);
    else tma_load_2d(dst, map, bar, k, row);
  }
}

// Descriptor of the 16-deep step `ks` of an atom. K-major: 32 bytes along the 128-byte rows,
// 8-row groups 1024 bytes apart. MN-major: 16 k-rows of 128 bytes further, 8-k groups 1024 bytes
// apart, the next 64 row indices 8192 bytes away.
template <bool MN>
__device__ __forceinline__ uint64_t atom_desc(uint32_t saddr, int ks) {
  return MN ? smem_desc(saddr + ks * 2048, 8192, 1024) : smem_desc(saddr + ks * 32, 16, 1024);
}

__host__ __device__ constexpr uint32_t idesc_h(int M, int N, bool a_mn, bool b_mn) {
  return idesc_f16(M, N, false, b_mn) | ((a_mn ? 1u : 0u) << 15);
}
constexpr uint32_t kIdescBF16 = (1u << 7) | (1u << 10);

// Column-grouped tile order: `group_m` tile rows at a time, all tile columns of a group before the
// next, rows fastest, so the tiles in flight share few A and B panels.
__device__ __forceinline__ void tile_coords(const HGemmParams& p, int tile, int& tm, int& tn) {
  const int per_group = p.group_m * p.tiles_n;
  const int g = tile / per_group, r = tile - g * per_group;
  const int first = g * p.group_m;
  const int gm = min(p.group_m, p.tiles_m - first);
  tm = first + r % gm;
  tn = r / gm;
}

// ------------------------------------------------------------------ pair kernel epilogue

// A warp's block of 32 rows x 32 bytes in shared memory, its two 16-byte units per row swapped in
// every other group of four rows, so that both the row-per-lane and the row-segment accesses spread
// over all banks.
__device__ __forceinline__ int block_unit(int row, int u) { return row * 2 + (u ^ ((row >> 2) & 1)); }

// Write the staged block to rows of `dst` (row pitch in bytes): `rows` rows, `bytes` of each row.
// ES is the element size for ragged edges and unaligned rows.
template <int ES>
__device__ __forceinline__ void block_store(const uint4* tile, uint8_t* dst, int64_t pitch, int rows, int bytes,
                                            bool vec) {
  const int lane = lane_id();
  if (vec && bytes == 32) {
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int rr = 16 * it + (lane >> 1), u = lane & 1;
      if (rr < rows) *reinterpret_cast<uint4*>(dst + rr * pitch + 16 * u) = tile[block_unit(rr, u)];
    }
  } else {
    constexpr int kPer = 32 / ES;               // elements per row of the block
    constexpr int kRows = 32 / kPer;            // rows per step
    const int e = lane % kPer, sub = lane / kPer;
    if (e * ES < bytes) {
      for (int r = sub; r < rows; r += kRows) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(&tile[block_unit(r, e * ES / 16)]) + e * ES % 16;
        if (ES == 2) *reinterpret_cast<uint16_t*>(dst + r * pitch + e * ES) = *reinterpret_cast<const uint16_t*>(src);
        else *reinterpret_cast<uint32_t*>(dst + r * pitch + e * ES) = *reinterpret_cast<const uint32_t*>(src);
      }
    }
  }
}

// A block of 16-bit values from rows of `src` to shared memory, in two steps: loaded to registers ahead
// of its use, so that its way from memory passes during other work, and put down later. 16 bytes per lane and
// load, or, at ragged edges and for unaligned rows, single values: 16 lanes per row, two rows per load.
struct BlockRegs { uint32_t w[8]; };
__device__ __forceinline__ void block_fetch16(BlockRegs& v, const uint8_t* src, int64_t pitch, int rows, int bytes, bool vec) {
  const int lane = lane_id();
#pragma unroll
  for (int i = 0; i < 8; ++i) v.w[i] = 0;
  if (vec && bytes == 32) {
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int rr = 16 * it + (lane >> 1);
      if (rr < rows) {
        const uint4 q = *reinterpret_cast<const uint4*>(src + rr * pitch + 16 * (lane & 1));
        v.w[4 * it] = q.x; v.w[4 * it + 1] = q.y; v.w[4 * it + 2] = q.z; v.w[4 * it + 3] = q.w;
      }
    }
  } else if ((lane & 15) * 2 < bytes) {
    const uint8_t* at = src + (lane >> 4) * pitch + (lane & 15) * 2;
    uint16_t h[16];
#pragma unroll
    for (int i = 0; i < 16; ++i, at += 2 * pitch) h[i] = 2 * i + (lane >> 4) < rows ? *reinterpret_cast<const uint16_t*>(at) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
  }
}
__device__ __forceinline__ void block_put16(uint4* tile, const BlockRegs& v, int bytes, bool vec) {
  const int lane = lane_id();
  if (vec && bytes == 32) {
#pragma unroll
    for (int it = 0; it < 2; ++it)
      tile[block_unit(16 * it + (lane >> 1), lane & 1)] = make_uint4(v.w[4 * it], v.w[4 * it + 1], v.w[4 * it + 2], v.w[4 * it + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      reinterpret_cast<uint16_t*>(&tile[block_unit(2 * i + (lane >> 4), (lane >> 3) & 1)])[lane & 7] =
          static_cast<uint16_t>(v.w[i / 2] >> (16 * (i & 1)));
  }
}

// 32 x 16 fp32 values (one row per lane) to `z`, 8 columns at a time.
__device__ __forceinline__ void store_z(uint4* tile, const Pair (&v)[8], float* z, int64_t ldz, int rows, int cols) {
  const int lane = lane_id();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (8 * h < cols) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float2 a = split(v[4 * h + 2 * u]), b = split(v[4 * h + 2 * u + 1]);
        tile[block_unit(lane, u)] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
      }
      __syncwarp();
      block_store<4>(tile, reinterpret_cast<uint8_t*>(z + 8 * h), ldz * 4, rows, min(32, 4 * (cols - 8 * h)), true);
      __syncwarp();
    }
  }
}

// Accumulator values and 16 biases (16-byte aligned, read by all lanes at once).
__device__ __forceinline__ void add_bias(Pair (&v)[8], const uint32_t (&r)[16], const float* bias) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 b = reinterpret_cast<const float4*>(bias)[j];
    v[2 * j] = pair(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1])) + pair(b.x, b.y);
    v[2 * j + 1] = pair(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])) + pair(b.z, b.w);
  }
}

// ------------------------------------------------------------------ pair kernel

constexpr int kPairBN = 256;                                       // widest tile; TMEM columns per accumulator
constexpr int kPairStages = 3;
constexpr int kPairAtoms = 2;                                      // 64-deep atoms per stage
constexpr int kPairStage = 2 * kPairAtoms * kHAtom;                // bytes per CTA: A and B atoms
constexpr int kPairSmem = kPairStages * kPairStage + 1024;
constexpr int kPairEpiWarps = 16;       // four per TMEM lane quarter
constexpr int kPairThreads = 64 + 32 * kPairEpiWarps;

template <bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(kPairThreads, 1)
hgemm_pair_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_a1,
                  const __grid_constant__ CUtensorMap map_b0, const __grid_constant__ CUtensorMap map_b1,
                  const HGemmParams p) {
  const int out_cols = EPI == kEpiGated ? p.bn / 2 : p.bn;             // output columns per tile
  const int b_rows = p.bn / 2;                                         // B rows staged by each CTA
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full_bar[kPairStages];
  __shared__ __align__(8) uint64_t empty_bar[kPairStages];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ __align__(16) float col_bias[kPairEpiWarps][64];          // two blocks' columns, or gate and up
  __shared__ __align__(16) uint4 epi_tile[kPairEpiWarps][64];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = warp_id(), lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  const int unit = static_cast<int>(blockIdx.x >> 1), units = static_cast<int>(gridDim.x >> 1);
  const int num_kb = p.kb0 + p.kb1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * kPairEpiWarps); }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&map_a0); tma_prefetch_desc(&map_b0); }
  if (warp == 1) { tmem_alloc_pair(&tmem_base_slot, 2 * kPairBN); tmem_relinquish_pair(); }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  pdl_enter();
  const uint32_t tmem_base = tmem_base_slot;
  volatile int* abort = &abort_flag;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t b_bytes = BMN ? (b_rows + 63) / 64 * 8192 : b_rows * 128;      // per atom
      const uint32_t stage_bytes = 2 * kPairAtoms * (kHAtom + b_bytes);             // both CTAs
      for (int tile = unit; tile < p.num_tiles && ok; tile += units) {
        int tm, tn;
        tile_coords(p, tile, tm, tn);
        const bool second = tm >= p.m_split;
        const int arow = (second ? tm - p.m_split : tm) * 256 + rank * 128;
        const int brow = EPI == kEpiGated ? tn * out_cols : tn * out_cols + rank * b_rows;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort)) { ok = false; break; }
          const bool seg = kb >= p.kb0;
          const CUtensorMap* ma = seg || second ? &map_a1 : &map_a0;
          const CUtensorMap* mb = (EPI == kEpiGated ? rank != 0 : seg) ? &map_b1 : &map_b0;
          uint8_t* sa = smem + stage * kPairStage;
          uint8_t* sb = sa + kPairAtoms * kHAtom;
          const uint32_t bar = cluster_addr(&full_bar[stage], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], stage_bytes);
#pragma unroll
          for (int at = 0; at < kPairAtoms; ++at) {
            const int k = (kb - (seg ? p.kb0 : 0)) * (kPairAtoms * kHBK) + at * kHBK;
            load_atom<AMN, true>(sa + at * kHAtom, ma, nullptr, bar, k, arow, 128);
            load_atom<BMN, true>(sb + at * kHAtom, mb, nullptr, bar, k, brow, b_rows);
          }
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);   // loads already issued land before the CTA exits
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (even CTA, lane 0)
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_h(256, p.bn, AMN, BMN) | (p.bf16 ? kIdescBF16 : 0u);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int tile = unit; tile < p.num_tiles && ok; tile += units, ++local) {
        const int buf = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!mbar_wait_cluster(&acc_empty[buf], acc_phase ^ 1, abort)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * kPairBN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kPairStage);
          const uint32_t sb = sa + kPairAtoms * kHAtom;
#pragma unroll
          for (int k = 0; k < kPairAtoms * 4; ++k) {
            const uint64_t ad = atom_desc<AMN>(sa + (k / 4) * kHAtom, k % 4);
            const uint64_t bd = atom_desc<BMN>(sb + (k / 4) * kHAtom, k % 4);
            mma_f16_ss_pair(d_tmem, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          mma_commit_pair_both(&empty_bar[stage]);
          if (kb == num_kb - 1) mma_commit_pair_both(&acc_full[buf]);
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
      mma_commit_pair(&drain_bar);
      mbar_wait(&drain_bar, 0, nullptr, 1000000);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue (16 warps)
    // A warp takes every fourth block of 32 output columns of its 32 rows, 16 columns at a time. Four
    // warps per scheduler: with two, the last tile's epilogue, which nothing overlaps, took 6 us of
    // 18.6 for a 1024 x 1024 x 1024 product with GELU.
    const int ew = warp - 2;
    const int quarter = warp & 3;               // TMEM lane quarter this warp may access
    const int group = ew >> 2;
    float* my_bias = col_bias[ew];
    uint4* tile_s = epi_tile[ew];
    const int blocks = (out_cols + 31) / 32;
    int local = 0;
    for (int tile = unit; tile < p.num_tiles; tile += units, ++local) {
      int tm, tn;
      tile_coords(p, tile, tm, tn);
      const int buf = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      __syncwarp();
      for (int b = group; b < blocks; b += 4) {
        // block b's biases at 32 (b / 4) (gated, at most one block: the up projection's 32 further)
        const int n = tn * out_cols + 32 * b + lane, at = 32 * (b >> 2) + lane;
        my_bias[at] = p.bias != nullptr && n < p.N ? h_to_f(reinterpret_cast<const uint16_t*>(p.bias)[n], p.bf16) : 0.0f;
        if (EPI == kEpiGated)
          my_bias[32 + at] =
              p.bias1 != nullptr && n < p.N ? h_to_f(reinterpret_cast<const uint16_t*>(p.bias1)[n], p.bf16) : 0.0f;
      }
      const bool second = tm >= p.m_split;
      const int64_t row0 = static_cast<int64_t>(second ? tm - p.m_split : tm) * 256 + rank * 128 + quarter * 32;
      const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.M - row0));   // may be <= 0
      // The residual of the 16 columns from c on, a block ahead (6580 x 3296 x 256: 39.7 us, 45.0 without).
      BlockRegs res;
      const uint8_t* res_row = reinterpret_cast<const uint8_t*>(p.residual) + row0 * p.ldr * 2;
      auto fetch_residual = [&](int c) {
        const int col0 = tn * out_cols + c, cols = min(min(16, out_cols - c), p.N - col0);
        if (cols > 0 && rows > 0) block_fetch16(res, res_row + col0 * 2ll, p.ldr * 2, rows, 2 * cols, p.res_vec);
      };
      if (EPI == kEpiLinear && p.residual != nullptr) fetch_residual(32 * group);
      __syncwarp();
      const bool ok = mbar_wait(&acc_full[buf], acc_phase, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kPairBN;
      uint8_t* out = reinterpret_cast<uint8_t*>(second ? p.out1 : p.out);
      // The accumulator goes back to the MMA thread once this warp's last block of it is in
      // registers, before that block's arithmetic and stores.
      bool returned = false;
      auto give_back = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(cluster_addr(&acc_empty[buf], 0));
        returned = true;
      };
#pragma unroll 1
      for (int b = group; b < blocks; b += 4) {
#pragma unroll 1
        for (int c = 32 * b, h = 0; h < 2; ++h, c += 16) {
          const int col0 = tn * out_cols + c, bias_at = 32 * (b >> 2) + 16 * h;
          const int cols = min(min(16, out_cols - c), p.N - col0);
          if (cols <= 0 || rows <= 0) continue;           // warp-uniform
          uint32_t r[16];
          tmem_ld16(taddr + c, r);
          Pair v[8];
          if (EPI == kEpiGated) {
            uint32_t ru[16];
            tmem_ld16(taddr + out_cols + c, ru);
            tmem_wait_ld();
            if (b + 4 >= blocks && h == 1) give_back();
            Pair u[8];
            add_bias(v, r, my_bias + bias_at);
            add_bias(u, ru, my_bias + 32 + bias_at);
            if (p.z0 != nullptr) {
              store_z(tile_s, v, p.z0 + row0 * p.ldz + col0, p.ldz, rows, cols);
              store_z(tile_s, u, p.z1 + row0 * p.ldz + col0, p.ldz, rows, cols);
            }
            act_values(v, p.act);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = v[j] * u[j];
          } else {
            tmem_wait_ld();
            if (b + 4 >= blocks && h == 1) give_back();
            add_bias(v, r, my_bias + bias_at);
            if (p.z0 != nullptr) store_z(tile_s, v, p.z0 + row0 * p.ldz + col0, p.ldz, rows, cols);
            act_values(v, p.act);
            if (p.residual != nullptr) {
              block_put16(tile_s, res, 2 * cols, p.res_vec);
              fetch_residual(h == 0 ? c + 16 : 32 * (b + 4));
              __syncwarp();
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                Pair f[4];
                unpack8(tile_s[block_unit(lane, u)], f, p.bf16);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * u + i] = v[4 * u + i] + f[i];
              }
              __syncwarp();
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) tile_s[block_unit(lane, u)] = pack8(v + 4 * u, p.bf16);
          __syncwarp();
          block_store<2>(tile_s, out + (row0 * p.ldo + col0) * 2, p.ldo * 2, rows, 2 * cols, p.out_vec);
          __syncwarp();
        }
      }
      if (!returned) give_back();
    }
  }

  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kPairBN);
  }
}

// ------------------------------------------------------------------ cluster kernel

constexpr int kClBN = 128;
constexpr int kClStages = 3;
constexpr int kClStage = 2 * kHAtom;
constexpr int kClSmem = kClStages * kClStage + 1024;
static_assert(kClStages * kClStage >= 128 * kClBN * 4, "the fp32 partial tile reuses the stages");

// Four 16-bit values at `src` (vector access when `vec`), zero past `n` of them.
__device__ __forceinline__ float4 load4(const uint16_t* src, int n, bool vec, int bf16) {
  uint32_t a = 0, b = 0;
  if (vec && n >= 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(src);
    a = u.x; b = u.y;
  } else {
    if (n > 0) a = src[0];
    if (n > 1) a |= static_cast<uint32_t>(src[1]) << 16;
    if (n > 2) b = src[2];
    if (n > 3) b |= static_cast<uint32_t>(src[3]) << 16;
  }
  return make_float4(h_to_f(a & 0xFFFFu, bf16), h_to_f(a >> 16, bf16), h_to_f(b & 0xFFFFu, bf16), h_to_f(b >> 16, bf16));
}

// fp32 partial tiles in the shared memory of a cluster's CTAs, added in the order of the CTAs (the
// same sums on every call) and finished: bias, pre-activations, activation, residual or gate, store.
// A partial row is kClUnits float4, unit u at u ^ (row & 7). Tile row 0 and column 0 are output
// (row0, col0); this CTA finishes rows [r_begin, r_end).
constexpr int kClUnits = kClBN / 4;

template <int EPI>
__device__ __forceinline__ void finish_tile(const HGemmParams& p, const float* part, int r_begin, int r_end, int64_t row0,
                                            int col0, uint16_t* out) {
  constexpr int kOutUnits = EPI == kEpiGated ? kClUnits / 2 : kClUnits;      // the gate's units, then the up projection's
  const uint32_t part_u = smem_u32(part);
  auto sum4 = [&](int r, int u) {
    const int off = r * kClUnits + (u ^ (r & 7));
    if (p.splits == 1) return reinterpret_cast<const float4*>(part)[off];
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < p.splits; ++c) {
      uint32_t a;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(part_u + off * 16), "r"(c));
      const float4 v = ld_cluster_f4(a);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    return s;
  };
  for (int i = r_begin * kOutUnits + static_cast<int>(threadIdx.x); i < r_end * kOutUnits; i += kHThreads) {
    const int r = i / kOutUnits, u = i % kOutUnits;
    const int col = col0 + 4 * u;
    const int n = p.N - col;                             // columns left, from this unit on
    if (n <= 0) continue;
    const int64_t row = row0 + r;
    float4 s = sum4(r, u);
    if (p.bias != nullptr) {
      const float4 b = load4(reinterpret_cast<const uint16_t*>(p.bias) + col, n, false, p.bf16);
      s.x += b.x; s.y += b.y; s.z += b.z; s.w += b.w;
    }
    if (p.z0 != nullptr) *reinterpret_cast<float4*>(p.z0 + row * p.ldz + col) = s;     // rows are padded to 4 floats
    Pair v[2] = {pair(s.x, s.y), pair(s.z, s.w)};
    act_values(v, p.act);
    if (EPI == kEpiGated) {
      float4 w = sum4(r, u + kOutUnits);
      if (p.bias1 != nullptr) {
        const float4 b = load4(reinterpret_cast<const uint16_t*>(p.bias1) + col, n, false, p.bf16);
        w.x += b.x; w.y += b.y; w.z += b.z; w.w += b.w;
      }
      if (p.z1 != nullptr) *reinterpret_cast<float4*>(p.z1 + row * p.ldz + col) = w;
      v[0] = v[0] * pair(w.x, w.y);
      v[1] = v[1] * pair(w.z, w.w);
    } else if (p.residual != nullptr) {
      const float4 b = load4(reinterpret_cast<const uint16_t*>(p.residual) + row * p.ldr + col, n, p.res_vec, p.bf16);
      v[0] = v[0] + pair(b.x, b.y);
      v[1] = v[1] + pair(b.z, b.w);
    }
    const float2 v0 = split(v[0]), v1 = split(v[1]);
    const uint32_t lo = pack_h2(v0.x, v0.y, p.bf16), hi = pack_h2(v1.x, v1.y, p.bf16);
    uint16_t* dst = out + row * p.ldo + col;
    if (p.out_vec && n >= 4) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    } else {
      dst[0] = static_cast<uint16_t>(lo);
      if (n > 1) dst[1] = static_cast<uint16_t>(lo >> 16);
      if (n > 2) dst[2] = static_cast<uint16_t>(hi);
      if (n > 3) dst[3] = static_cast<uint16_t>(hi >> 16);
    }
  }
}

// Columns [c, c + 32) of this warp's 32 TMEM lanes to the partial tile.
__device__ __forceinline__ void drain_block(uint32_t taddr, int c, float* part, int row) {
  uint32_t v[32];
  tmem_ld32(taddr + c, v);
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < 32; j += 4)
    reinterpret_cast<uint4*>(part)[row * kClUnits + (((c + j) >> 2) ^ (row & 7))] = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
}

// One CTA of a cluster computes its share of a tile's k-blocks and leaves its fp32 partials in shared
// memory; each CTA of the cluster finishes its share of the rows.
template <bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(kHThreads, 2)
hgemm_cluster_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_a1,
                     const __grid_constant__ CUtensorMap map_b0, const __grid_constant__ CUtensorMap map_b1,
                     const HGemmParams p) {
  constexpr int kOutCols = EPI == kEpiGated ? kClBN / 2 : kClBN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full_bar[kClStages];
  __shared__ __align__(8) uint64_t empty_bar[kClStages];
  __shared__ __align__(8) uint64_t acc_full;
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = warp_id(), lane = lane_id();
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  int tm, tn;
  tile_coords(p, static_cast<int>(blockIdx.x) / p.splits, tm, tn);
  const bool second = tm >= p.m_split;
  const int row0 = (second ? tm - p.m_split : tm) * 128;
  const int num_kb = p.kb0 + p.kb1;
  const int kb_begin = static_cast<int>(static_cast<int64_t>(num_kb) * rank / p.splits);
  const int kb_end = static_cast<int>(static_cast<int64_t>(num_kb) * (rank + 1) / p.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kClStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(&acc_full, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&map_a0); tma_prefetch_desc(&map_b0); }
  if (warp == 1) { tmem_alloc(&tmem_base_slot, kClBN); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_enter();
  const uint32_t tmem_base = tmem_base_slot;
  volatile int* abort = &abort_flag;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t a_bytes = AMN ? kHAtom : static_cast<uint32_t>(p.a_rows) * 128;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort)) { ok = false; break; }
        const bool seg = kb >= p.kb0;
        const CUtensorMap* ma = seg || second ? &map_a1 : &map_a0;
        const int k = (kb - (seg ? p.kb0 : 0)) * kHBK;
        uint8_t* sa = smem + stage * kClStage;
        uint8_t* sb = sa + kHAtom;
        mbar_arrive_expect_tx(&full_bar[stage], a_bytes + kHAtom);
        load_atom<AMN, false>(sa, ma, &full_bar[stage], 0, k, row0, 128);
        if (EPI == kEpiGated) {
          load_atom<BMN, false>(sb, &map_b0, &full_bar[stage], 0, k, tn * kOutCols, kOutCols);
          load_atom<BMN, false>(sb + kHAtom / 2, &map_b1, &full_bar[stage], 0, k, tn * kOutCols, kOutCols);
        } else {
          load_atom<BMN, false>(sb, seg ? &map_b1 : &map_b0, &full_bar[stage], 0, k, tn * kClBN, kClBN);
        }
        if (++stage == kClStages) { stage = 0; phase ^= 1; }
      }
      if (!ok) {
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_h(128, kClBN, AMN, BMN) | (p.bf16 ? kIdescBF16 : 0u);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * kClStage);
        const uint32_t sb = sa + kHAtom;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16_ss(tmem_base, atom_desc<AMN>(sa, k), atom_desc<BMN>(sb, k), idesc,
                     (kb != kb_begin || k != 0) ? 1u : 0u);
        mma_commit(&empty_bar[stage]);
        if (++stage == kClStages) { stage = 0; phase ^= 1; }
      }
      mma_commit(&acc_full);
    }
    __syncwarp();
  }
  // Every thread: the accumulator is complete, and with it every load and every MMA of this CTA.
  bool ok = mbar_wait(&acc_full, 0, nullptr);
  ok = __all_sync(0xffffffffu, ok && *abort == 0);
  tc_fence_after();
  float* part = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
    for (int c = half * (kClBN / 2); c < (half + 1) * (kClBN / 2); c += 32) drain_block(taddr, c, part, quarter * 32 + lane);
  }
  tc_fence_before();
  if (p.splits > 1) cluster_sync();
  else __syncthreads();
  if (ok) {
    const int rows = min(128, p.M - row0);
    const int per = (rows + p.splits - 1) / p.splits;
    const int r_begin = min(rows, rank * per);
    finish_tile<EPI>(p, part, r_begin, min(rows, r_begin + per), row0, tn * kOutCols,
                     reinterpret_cast<uint16_t*>(second ? p.out1 : p.out));
  }
  // No CTA leaves while another may still read its partials.
  if (p.splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kClBN);
  }
}

}  // namespace dc
