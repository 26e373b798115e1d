// Token embedding: y[t] = scale * table[id[t]], and the table's gradient
//   dtable[v] = scale * sum over t with id[t] = v of dy[t], in the order of t,
// rounded once from fp32. A token id outside the table gives a zero row and takes no part in the
// gradient, and sets the device error word (kErrTokenId); the padding id takes no part in it
// either.
//
// The gradient is summed over tokens sorted by id (stable, so equal ids keep their order and the
// sums are the same on every call, without float atomics):
//   sort    up to 8192 tokens: each token's place is the number of smaller (id, t) keys, counted
//           against all keys in shared memory, one launch; more: least-significant-digit radix
//           passes of up to 9 bits (histogram per tile, scan, stable scatter)
//   sum     a CTA per chunk of sorted places and slab of columns adds up runs of equal ids; runs
//           inside the chunk go to the table, the first and last may continue in the
//           neighbouring chunks and leave fp32 partials
//   join    the chunk in which such a run starts adds its partials in order
// Chunks of equal length keep a frequent token from falling to one CTA.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "norm.cuh"

namespace dc {

struct EmbedIds {
  const void* ids;
  int i64;
  int64_t T;
  int64_t V;
  int64_t padding;          // id that gets no gradient, or -1
};

__device__ __forceinline__ int64_t id_at(const EmbedIds& e, int64_t t) {
  return e.i64 ? static_cast<const int64_t*>(e.ids)[t] : static_cast<int64_t>(static_cast<const int32_t*>(e.ids)[t]);
}
// Sort key: the id, or V for a token without a gradient.
__device__ __forceinline__ uint32_t key_at(const EmbedIds& e, int64_t t) {
  const int64_t id = id_at(e, t);
  return id >= 0 && id < e.V && id != e.padding ? static_cast<uint32_t>(id) : static_cast<uint32_t>(e.V);
}

// Bound by HBM: one read and one write of a row per token. blockDim (x: vectors of a row, y: tokens).
template <typename T, int E>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const EmbedIds ids, const T* __restrict__ table, int64_t ldt, T* __restrict__ out, int64_t ldo,
                 int D, float scale) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= ids.T) return;
  const int64_t id = id_at(ids, t);
  const bool ok = id >= 0 && id < ids.V;
  if (!ok && threadIdx.x == 0) record_error(kErrTokenId);
  const T* src = table + (ok ? id : 0) * ldt;
  T* dst = out + t * ldo;
#pragma unroll 4
  for (int c = threadIdx.x * E; c < D; c += blockDim.x * E) {
    float f[E];
    if (ok) load_e<T, E>(src + c, f);
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = ok ? f[j] * scale : 0.f;
    store_e<T, E>(dst + c, f);
  }
}

// ------------------------------------------------------------------ sort

constexpr int kRankMax = 8192;          // tokens of the counting sort: (id, t) fit 19 + 13 bits
constexpr int kRankItems = 32;          // tokens per CTA
constexpr int kRankWarps = 8;

__global__ void __launch_bounds__(32 * kRankWarps)
embed_rank_kernel(const EmbedIds ids, uint32_t* __restrict__ skey, uint32_t* __restrict__ sidx) {
  __shared__ __align__(16) uint32_t keys[kRankMax];
  __shared__ int count[kRankWarps][32];
  const int T = static_cast<int>(ids.T);
  const int Tp = (T + 4 * kRankWarps - 1) / (4 * kRankWarps) * (4 * kRankWarps);
  for (int t = threadIdx.x; t < Tp; t += 32 * kRankWarps)
    keys[t] = t < T ? (key_at(ids, t) << 13) | static_cast<uint32_t>(t) : 0xFFFFFFFFu;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int item = blockIdx.x * kRankItems + lane;
  const uint32_t mine = item < T ? keys[item] : 0u;
  const int per = Tp / kRankWarps;
  int n = 0;
  for (int t = warp * per; t < (warp + 1) * per; t += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(keys + t);
    n += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
  }
  count[warp][lane] = n;
  __syncthreads();
  if (warp == 0 && item < T) {
    n = 0;
#pragma unroll
    for (int w = 0; w < kRankWarps; ++w) n += count[w][lane];
    const uint32_t key = mine >> 13;
    skey[n] = key;
    sidx[n] = static_cast<uint32_t>(item);
  }
}

constexpr int kRadixTile = 2048;
constexpr int kRadixWarps = 8;
constexpr int kRadixBits = 9;
constexpr int kRadixDigits = 1 << kRadixBits;

// Digit counts of each tile: hist[digit * tiles + tile]. The first pass reads the ids.
template <bool FIRST>
__global__ void __launch_bounds__(32 * kRadixWarps)
radix_hist_kernel(const EmbedIds ids, const uint32_t* __restrict__ keys, uint32_t* __restrict__ hist, int shift,
                  int bits) {
  __shared__ uint32_t h[kRadixDigits];
  const int digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += blockDim.x) h[d] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kRadixTile;
  for (int i = threadIdx.x; i < kRadixTile; i += blockDim.x) {
    const int64_t t = base + i;
    if (t < ids.T) atomicAdd(&h[((FIRST ? key_at(ids, t) : keys[t]) >> shift) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += blockDim.x) hist[static_cast<int64_t>(d) * gridDim.x + blockIdx.x] = h[d];
}

// Exclusive scan of n counts in place, one CTA; each thread scans a run of 16 per step.
constexpr int kScanPer = 16;
__global__ void __launch_bounds__(1024)
radix_scan_kernel(uint32_t* __restrict__ hist, int64_t n) {
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t total;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t carry = 0;
  for (int64_t base = 0; base < n; base += 1024 * kScanPer) {
    const int64_t at = base + static_cast<int64_t>(threadIdx.x) * kScanPer;
    uint32_t v[kScanPer], s = 0;
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) { v[i] = at + i < n ? hist[at + i] : 0u; }
#pragma unroll
    for (int i = 0; i < kScanPer; ++i) { const uint32_t x = v[i]; v[i] = s; s += x; }
    uint32_t incl = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      const uint32_t own = warp_sum[lane];
      uint32_t x = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      warp_sum[lane] = x - own;
      if (lane == 31) total = x;
    }
    __syncthreads();
    const uint32_t off = carry + warp_sum[warp] + incl - s;
#pragma unroll
    for (int i = 0; i < kScanPer; ++i)
      if (at + i < n) hist[at + i] = off + v[i];
    carry += total;
    __syncthreads();
  }
}

// Stable scatter of a tile. Warp w owns keys [256 w, 256 w + 256) of the tile, 32 at a time; a
// key's place is the digit's base for the tile + equal digits in earlier warps + in earlier rounds
// of its warp + in lower lanes.
template <bool FIRST>
__global__ void __launch_bounds__(32 * kRadixWarps)
radix_scatter_kernel(const EmbedIds ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ idx,
                     const uint32_t* __restrict__ base_of, uint32_t* __restrict__ keys_out,
                     uint32_t* __restrict__ idx_out, int shift, int bits) {
  __shared__ uint32_t cnt[kRadixWarps][kRadixDigits];
  constexpr int kRounds = kRadixTile / (32 * kRadixWarps);
  const int digits = 1 << bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kRadixWarps * kRadixDigits; i += blockDim.x) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kRadixTile + warp * (32 * kRounds);
  uint32_t key[kRounds], place[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t t = base + r * 32 + lane;
    const bool in = t < ids.T;
    key[r] = in ? (FIRST ? key_at(ids, t) : keys[t]) : 0u;
    const uint32_t d = (key[r] >> shift) & (digits - 1);
    // lanes past the end form a group of their own (digit count is at most 512)
    const uint32_t peers = __match_any_sync(0xffffffffu, in ? d : 0xFFFFu);
    place[r] = __popc(peers & ((1u << lane) - 1u));
    uint32_t before = 0;
    if (in) before = cnt[warp][d];
    __syncwarp();
    if (in && place[r] == 0) cnt[warp][d] = before + __popc(peers);
    __syncwarp();
    place[r] += before;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += blockDim.x) {
    uint32_t s = base_of[static_cast<int64_t>(d) * gridDim.x + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kRadixWarps; ++w) { const uint32_t c = cnt[w][d]; cnt[w][d] = s; s += c; }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t t = base + r * 32 + lane;
    if (t < ids.T) {
      const uint32_t to = cnt[warp][(key[r] >> shift) & (digits - 1)] + place[r];
      keys_out[to] = key[r];
      idx_out[to] = FIRST ? static_cast<uint32_t>(t) : idx[t];
    }
  }
}

// ------------------------------------------------------------------ sums over sorted tokens

constexpr int kSumThreads = 128;
constexpr int kSumChunkMax = 128;

struct EmbedSumParams {
  const uint32_t* skey;
  const uint32_t* sidx;
  int64_t T;
  int64_t V;
  const void* dy;
  int64_t lddy;
  void* out;                // [V, D] contiguous
  float* part;              // [chunks][2][D]: runs that came from before / continue behind the chunk
  int D;
  int chunk;                // sorted places per chunk
  float scale;
};

template <typename T, int E>
__global__ void __launch_bounds__(kSumThreads)
embed_sum_kernel(const EmbedSumParams p) {
  __shared__ uint32_t key[kSumChunkMax + 2];
  __shared__ uint32_t idx[kSumChunkMax];
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.chunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.chunk), p.T - begin));
  const uint32_t none = 0xFFFFFFFFu;      // never a key
  for (int i = threadIdx.x; i < n + 2; i += kSumThreads) {
    const int64_t t = begin + i - 1;
    key[i] = t >= 0 && t < p.T ? p.skey[t] : none;
    if (i < n) idx[i] = p.sidx[begin + i];
  }
  __syncthreads();
  const int c = (blockIdx.y * kSumThreads + threadIdx.x) * E;
  if (c >= p.D || key[1] == static_cast<uint32_t>(p.V)) return;
  const T* dy = static_cast<const T*>(p.dy) + c;
  float acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.f;
  bool from_before = key[0] == key[1];
  constexpr int kAhead = 8;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float v[kAhead][E];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u < n) load_e<T, E>(dy + static_cast<int64_t>(idx[i0 + u]) * p.lddy, v[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      const uint32_t k = key[i + 1];
      if (k == static_cast<uint32_t>(p.V)) return;
#pragma unroll
      for (int j = 0; j < E; ++j) acc[j] += v[u][j];
      const bool ends = key[i + 2] != k;
      if (ends || i == n - 1) {
        if (ends && !from_before) {
#pragma unroll
          for (int j = 0; j < E; ++j) acc[j] *= p.scale;
          store_e<T, E>(static_cast<T*>(p.out) + static_cast<int64_t>(k) * p.D + c, acc);
        } else {
          float* q = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (from_before ? 0 : 1)) * p.D + c;
#pragma unroll
          for (int j = 0; j < E; ++j) q[j] = acc[j];
        }
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = 0.f;
        from_before = false;
      }
    }
  }
}

// The run that starts in this chunk and continues in the next ones, if there is one.
template <typename T, int E>
__global__ void __launch_bounds__(kSumThreads)
embed_join_kernel(const EmbedSumParams p) {
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.chunk;
  const int64_t end = begin + p.chunk;
  if (end >= p.T) return;
  const uint32_t k = p.skey[end - 1];
  if (k == static_cast<uint32_t>(p.V) || p.skey[end] != k) return;
  if (p.skey[begin] == k && begin > 0 && p.skey[begin - 1] == k) return;    // it started before
  // last place of the run: keys are sorted
  int64_t lo = end, hi = p.T;               // skey[lo] == k, skey[hi] > k (or hi == T)
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.skey[mid] == k) lo = mid; else hi = mid;
  }
  const int64_t last = lo / p.chunk;
  const int c = (blockIdx.y * kSumThreads + threadIdx.x) * E;
  if (c >= p.D) return;
  float acc[E];
  const float* q = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + 1) * p.D + c;
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = q[j];
#pragma unroll 4
  for (int64_t ch = blockIdx.x + 1; ch <= last; ++ch) {
    const float* s = p.part + ch * 2 * p.D + c;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] += s[j];
  }
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] *= p.scale;
  store_e<T, E>(static_cast<T*>(p.out) + static_cast<int64_t>(k) * p.D + c, acc);
}

}  // namespace dc
