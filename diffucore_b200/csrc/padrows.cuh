// Operands of the projections whose rows a tile load cannot take (an odd width, a view that starts
// between 16-byte boundaries) copied to rows of a multiple of 16 bytes: up to three matrices of
// 16-bit values in one launch, since a call's operands usually share their width.
//
// Bound by HBM, 2 B read and written per value. A thread makes one 16-byte unit. Its source lies at
// any even address, so it is read as 32-bit words, five of them shifted by half a word where the unit starts in
// the middle of one; where a word would reach outside the matrix (its first and last values) the
// unit is read value by value.
#pragma once
#include <cstdint>
#include "sm100.cuh"

namespace dc {

constexpr int kPadMatrices = 3;
constexpr int kPadThreads = 256;

struct PadMatrix {
  const uint16_t* src;
  uint16_t* dst;
  int64_t ld, ldd;          // in values; ldd a multiple of 8
  int64_t rows;
  int cols;
  int64_t first;            // units of the matrices before this one
};
struct PadParams {
  PadMatrix m[kPadMatrices];
  int count;
  int64_t units;
};

__global__ void __launch_bounds__(kPadThreads)
pad_rows_kernel(const PadParams p) {
  pdl_enter();
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kPadThreads + threadIdx.x; i < p.units;
       i += static_cast<int64_t>(gridDim.x) * kPadThreads) {
    PadMatrix m = p.m[0];
#pragma unroll
    for (int k = 1; k < kPadMatrices; ++k) {
      if (k < p.count && i >= p.m[k].first) m = p.m[k];
    }
    const int per_row = static_cast<int>(m.ldd / 8);
    const int64_t at = i - m.first;
    int64_t r;
    if (at <= UINT32_MAX) r = static_cast<uint32_t>(at) / static_cast<uint32_t>(per_row);     // a 64-bit division costs as much as the copy
    else r = at / per_row;
    const int c = static_cast<int>(at - r * per_row) * 8;
    const uint16_t* src = m.src + r * m.ld + c;
    const uint16_t* end = m.src + (m.rows - 1) * m.ld + m.cols;
    uint32_t w[4];
    const bool odd = (reinterpret_cast<uintptr_t>(src) & 2) != 0;
    if (c + 8 <= m.cols && !odd) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint32_t*>(src) + j);
    } else if (c + 8 <= m.cols && src > m.src && src + 9 <= end) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(src - 1);
      uint32_t v[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) v[j] = __ldg(q + j);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < m.cols ? src[2 * j] : 0u, hi = c + 2 * j + 1 < m.cols ? src[2 * j + 1] : 0u;
        w[j] = lo | (hi << 16);
      }
    }
    *reinterpret_cast<uint4*>(m.dst + r * m.ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace dc
