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
//           passes of up to 9 bits (histogram per tile, for many tiles their prefix sums, stable scatter)
//   sum     a CTA per chunk of sorted places and slab of columns adds up the runs of equal ids that
//           start in its chunk; a run that covers a whole chunk leaves fp32 partials per chunk
//   join    adds the partials of those runs in order
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

// Bound by HBM: one read and one write of a row per token. blockDim (x: vectors of a row, y: rows);
// a row of threads takes kTokens tokens, whose loads are in flight together: four where a thread has
// one vector of a row and tokens are many (500000 x 256 bf16 84 us, 134 with one), else one (65536 x
// 2048 76 us, 80 with four).
template <typename T, int E, int kTokens>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const EmbedIds ids, const T* __restrict__ table, int64_t ldt, T* __restrict__ out, int64_t ldo,
                 int D, float scale) {
  pdl_enter();
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y) * kTokens;
  const T* src[kTokens];
  bool ok[kTokens];
#pragma unroll
  for (int k = 0; k < kTokens; ++k) {
    const int64_t id = t0 + k < ids.T ? id_at(ids, t0 + k) : 0;
    ok[k] = id >= 0 && id < ids.V;
    if (!ok[k] && threadIdx.x == 0) record_error(kErrTokenId);
    src[k] = table + (ok[k] ? id : 0) * ldt;
  }
#pragma unroll 4
  for (int c = threadIdx.x * E; c < D; c += blockDim.x * E) {
    float f[kTokens][E];
#pragma unroll
    for (int k = 0; k < kTokens; ++k)
      if (t0 + k < ids.T) load_e<T, E>(src[k] + c, f[k]);
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      if (t0 + k < ids.T) {
#pragma unroll
        for (int j = 0; j < E; ++j) f[k][j] = ok[k] ? f[k][j] * scale : 0.f;
        store_e<T, E>(out + (t0 + k) * ldo + c, f[k]);
      }
    }
  }
}

// ------------------------------------------------------------------ zero fill

// The gradient's rows start as zeros. The sorting kernels keep few SMs busy and wait on latency, so
// each launch of theirs carries extra CTAs that zero a slice of the table.
struct FillSlice {
  uint8_t* p;               // 16-byte aligned up to `tail`
  int64_t bytes;
  int ctas;                 // CTAs of the launch that fill (the first ones sort)
};

constexpr int kFillCta = 64 << 10;      // bytes per filling CTA, about

__device__ __forceinline__ void fill_slice(const FillSlice& f, int cta) {
  const int64_t units = f.bytes >> 4;
  const int64_t stride = static_cast<int64_t>(f.ctas) * blockDim.x;
  uint4* q = reinterpret_cast<uint4*>(f.p);
#pragma unroll 4
  for (int64_t i = static_cast<int64_t>(cta) * blockDim.x + threadIdx.x; i < units; i += stride) q[i] = make_uint4(0, 0, 0, 0);
  if (cta == 0) {
    for (int64_t i = (units << 4) + threadIdx.x; i < f.bytes; i += blockDim.x) f.p[i] = 0;
  }
}

// ------------------------------------------------------------------ sort

constexpr int kRankMax = 8192;          // tokens of the counting sort: (id, t) fit 19 + 13 bits
constexpr int kRankItems = 32;          // tokens per CTA
constexpr int kRankWarps = 8;

__global__ void __launch_bounds__(32 * kRankWarps)
embed_rank_kernel(const EmbedIds ids, uint32_t* __restrict__ skey, uint32_t* __restrict__ sidx, int ctas,
                  const FillSlice fill) {
  pdl_enter();
  if (static_cast<int>(blockIdx.x) >= ctas) {
    fill_slice(fill, static_cast<int>(blockIdx.x) - ctas);
    return;
  }
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

constexpr int kRadixTile = 1024;
constexpr int kRadixWarps = 8;
constexpr int kRadixBits = 9;
constexpr int kRadixDigits = 1 << kRadixBits;

// Digit counts of each tile: hist[tile * digits + digit]. The first pass reads the ids.
template <bool FIRST>
__global__ void __launch_bounds__(32 * kRadixWarps)
radix_hist_kernel(const EmbedIds ids, const uint32_t* __restrict__ keys, uint32_t* __restrict__ hist, int shift,
                  int bits, int tiles, const FillSlice fill) {
  pdl_enter();
  if (static_cast<int>(blockIdx.x) >= tiles) {
    fill_slice(fill, static_cast<int>(blockIdx.x) - tiles);
    return;
  }
  __shared__ uint32_t h[kRadixDigits];
  const int digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += blockDim.x) h[d] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kRadixTile;
#pragma unroll
  for (int i = 0; i < kRadixTile / (32 * kRadixWarps); ++i) {
    const int64_t t = base + i * (32 * kRadixWarps) + threadIdx.x;
    if (t < ids.T) atomicAdd(&h[((FIRST ? key_at(ids, t) : keys[t]) >> shift) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += blockDim.x) hist[static_cast<int64_t>(blockIdx.x) * digits + d] = h[d];
}

// In place, the counts of the tiles before each tile, and the digits' totals behind the last tile's
// counts: for many tiles, where adding up every tile's counts in every CTA of the scatter would grow
// with their square. A CTA takes 32 digits, its warps equal ranges of tiles, each read twice.
constexpr int kScanWarps = 32;

__global__ void __launch_bounds__(32 * kScanWarps)
radix_scan_kernel(uint32_t* __restrict__ hist, int digits, int tiles) {
  pdl_enter();
  __shared__ uint32_t sums[kScanWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * warp / kScanWarps);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (warp + 1) / kScanWarps);
  uint32_t s = 0;
  if (d < digits) {
#pragma unroll 16
    for (int i = t0; i < t1; ++i) s += hist[static_cast<int64_t>(i) * digits + d];
  }
  sums[warp][lane] = s;
  __syncthreads();
  s = 0;
  for (int w = 0; w < warp; ++w) s += sums[w][lane];
  if (d >= digits) return;
  constexpr int kAhead = 16;                    // loads in flight before their stores
  for (int i0 = t0; i0 < t1; i0 += kAhead) {
    uint32_t c[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) c[j] = i0 + j < t1 ? hist[static_cast<int64_t>(i0 + j) * digits + d] : 0u;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j < t1) hist[static_cast<int64_t>(i0 + j) * digits + d] = s;
      s += c[j];
    }
  }
  if (warp == kScanWarps - 1) hist[static_cast<int64_t>(tiles) * digits + d] = s;
}

// Stable scatter of a tile. Warp w owns keys [32 kRounds w, 32 kRounds (w + 1)) of the tile, 32 at a
// time; a key's place is the number of smaller digits + equal digits in earlier tiles (both summed
// here from the tiles' counts, or taken from their prefix sums: SCANNED) + in earlier warps + in earlier
// rounds of its warp + in lower lanes.
template <bool FIRST, bool SCANNED>
__global__ void __launch_bounds__(32 * kRadixWarps)
radix_scatter_kernel(const EmbedIds ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ idx,
                     const uint32_t* __restrict__ hist, uint32_t* __restrict__ keys_out,
                     uint32_t* __restrict__ idx_out, int shift, int bits, int tiles, const FillSlice fill) {
  pdl_enter();
  if (static_cast<int>(blockIdx.x) >= tiles) {
    fill_slice(fill, static_cast<int>(blockIdx.x) - tiles);
    return;
  }
  __shared__ uint32_t cnt[kRadixWarps][kRadixDigits];
  __shared__ uint32_t below[kRadixWarps];
  constexpr int kRounds = kRadixTile / (32 * kRadixWarps);
  constexpr int kPerThread = kRadixDigits / (32 * kRadixWarps);   // digits per thread
  const int digits = 1 << bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kRadixTile + warp * (32 * kRounds);
  uint32_t key[kRounds], val[kRounds], place[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t t = base + r * 32 + lane;
    key[r] = t < ids.T ? (FIRST ? key_at(ids, t) : keys[t]) : 0u;
    val[r] = t < ids.T ? (FIRST ? static_cast<uint32_t>(t) : idx[t]) : 0u;
  }
  for (int i = threadIdx.x; i < kRadixWarps * kRadixDigits; i += blockDim.x) (&cnt[0][0])[i] = 0;
  // Digits kPerThread * threadIdx.x, ...: counts of all tiles and of the tiles before this one.
  uint32_t total[kPerThread], before_tile[kPerThread], mine = 0;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int d = threadIdx.x * kPerThread + j;
    total[j] = 0; before_tile[j] = 0;
    if (SCANNED && d < digits) {
      total[j] = hist[static_cast<int64_t>(tiles) * digits + d];
      before_tile[j] = hist[static_cast<int64_t>(blockIdx.x) * digits + d];
    } else if (d < digits) {
#pragma unroll 16
      for (int i = 0; i < tiles; ++i) {
        const uint32_t c = hist[static_cast<int64_t>(i) * digits + d];
        total[j] += c;
        if (i < static_cast<int>(blockIdx.x)) before_tile[j] += c;
      }
    }
    mine += total[j];
  }
  uint32_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) below[warp] = incl;
  __syncthreads();                          // cnt is zero, below is complete
  uint32_t smaller = incl - mine;           // keys with a smaller digit than this thread's first
#pragma unroll
  for (int w = 0; w < kRadixWarps; ++w) smaller += w < warp ? below[w] : 0u;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool in = base + r * 32 + lane < ids.T;
    const uint32_t d = (key[r] >> shift) & (digits - 1);
    // lanes past the end form a group of their own (digits are below 512)
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
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int d = threadIdx.x * kPerThread + j;
    if (d < digits) {
      uint32_t s = smaller + before_tile[j];
#pragma unroll
      for (int w = 0; w < kRadixWarps; ++w) { const uint32_t c = cnt[w][d]; cnt[w][d] = s; s += c; }
    }
    smaller += total[j];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (base + r * 32 + lane < ids.T) {
      const uint32_t to = cnt[warp][(key[r] >> shift) & (digits - 1)] + place[r];
      keys_out[to] = key[r];
      idx_out[to] = val[r];
    }
  }
}

// ------------------------------------------------------------------ sums over sorted tokens

// A run of equal keys that covers no whole chunk is summed by the CTA of the chunk it starts in, at
// most one chunk past its end. A longer run leaves one partial row per chunk (its first chunk in slot
// 1, the others in slot 0) for the join.
constexpr int kSumThreads = 128;
constexpr int kSumChunkMax = 64;

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
  pdl_enter();
  constexpr uint32_t kNone = 0xFFFFFFFFu;       // never a key
  using Unit = typename NormUnit<T, (E > 1)>::type;
  __shared__ uint32_t key[2 * kSumChunkMax + 2];
  __shared__ uint32_t idx[2 * kSumChunkMax];
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.chunk;
  const int chunk = p.chunk;
  // places of this chunk and the next one, and one on either side
  for (int i = threadIdx.x; i < 2 * chunk + 2; i += kSumThreads) {
    const int64_t t = begin + i - 1;
    key[i] = t >= 0 && t < p.T ? p.skey[t] : kNone;
    if (i < 2 * chunk && begin + i < p.T) idx[i] = p.sidx[begin + i];
  }
  const uint32_t before_chunk = begin - chunk - 1 >= 0 ? p.skey[begin - chunk - 1] : kNone;
  __syncthreads();
  const int n = static_cast<int>(min(static_cast<int64_t>(chunk), p.T - begin));
  const uint32_t first = key[1], last = key[n];
  const int i_own = static_cast<int>(threadIdx.x);
  const int lead = __syncthreads_count(i_own < n && key[i_own + 1] == first);
  const int tail = __syncthreads_count(i_own < chunk && n == chunk && key[n + i_own + 1] == last);
  // A leading run that began in the previous chunk and covers neither chunk belongs to that one.
  const int s0 = key[0] == first && before_chunk != first && key[chunk + 1] != first ? lead : 0;
  // The last run goes on into the next chunk: to its end, unless it covers that chunk (or this one).
  const int e0 = n == chunk && s0 < n && key[2 * chunk + 1] != last && !(first == last && key[0] == last) ? n + tail : n;
  const int c = (blockIdx.y * kSumThreads + threadIdx.x) * E;
  if (c >= p.D || s0 >= e0) return;
  const T* dy = static_cast<const T*>(p.dy) + c;
  float acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.f;
  bool from_before = s0 == 0 && key[0] == key[1];
  constexpr int kAhead = 8;
  for (int i0 = s0; i0 < e0; i0 += kAhead) {
    if (key[i0 + 1] == static_cast<uint32_t>(p.V)) return;         // sorted last: nothing follows
    // Kept packed until they are added: widened at the load they would take twice the registers, and
    // the compiler would not keep all of them in flight.
    Unit v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      v[u] = *reinterpret_cast<const Unit*>(dy + static_cast<int64_t>(idx[min(i0 + u, e0 - 1)]) * p.lddy);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i >= e0) break;
      const uint32_t k = key[i + 1];
      if (k == static_cast<uint32_t>(p.V)) return;
      const T* h = reinterpret_cast<const T*>(&v[u]);
#pragma unroll
      for (int j = 0; j < E; ++j) acc[j] += to_f(h[j]);
      const bool ends = key[i + 2] != k;
      if (ends || i == e0 - 1) {
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

// Runs that cover a whole chunk. A CTA looks at 4 chunks for one that such a run starts in, and adds
// the run's partial rows: four groups of threads take a quarter of them each, then the quarters are
// added in order.
constexpr int kJoinGroups = 4;
constexpr int kJoinChunks = 4;

template <typename T, int E>
__global__ void __launch_bounds__(kSumThreads * kJoinGroups)
embed_join_kernel(const EmbedSumParams p) {
  pdl_enter();
  __shared__ float part[kJoinGroups][E][kSumThreads];
  __shared__ uint32_t found;
  if (threadIdx.x < 32) {
    const int64_t ch = static_cast<int64_t>(blockIdx.x) * kJoinChunks + threadIdx.x;
    const int64_t begin = ch * p.chunk, end = begin + p.chunk;
    bool starts = false;
    if (threadIdx.x < kJoinChunks && end + p.chunk < p.T) {
      const uint32_t k = p.skey[end - 1];
      // covers the next chunk whole, and began in this one
      starts = k != static_cast<uint32_t>(p.V) && p.skey[end + p.chunk] == k &&
               !(p.skey[begin] == k && begin > 0 && p.skey[begin - 1] == k);
    }
    const uint32_t m = __ballot_sync(0xffffffffu, starts);
    if (threadIdx.x == 0) found = m;
  }
  __syncthreads();
  const int t = threadIdx.x % kSumThreads, g = threadIdx.x / kSumThreads;
  const int c = (blockIdx.y * kSumThreads + t) * E;
  for (uint32_t m = found; m != 0; m &= m - 1) {
    const int which = __ffs(m) - 1;
    const int64_t ch0 = static_cast<int64_t>(blockIdx.x) * kJoinChunks + which;
    // The run's last place: keys are sorted, all threads narrow its range together.
    const uint32_t k = p.skey[(ch0 + 1) * p.chunk];
    // The first round looks at single places, so only runs beyond 512 more take a second.
    constexpr int64_t kProbes = kSumThreads * kJoinGroups;
    int64_t lo = (ch0 + 2) * p.chunk, hi = p.T, step = 1; // skey[lo] == k, skey[hi] > k (or hi == T)
    while (hi - lo > 1) {
      const int64_t at = lo + (static_cast<int64_t>(threadIdx.x) + 1) * step;
      const int64_t below = __syncthreads_count(at < hi && p.skey[at] == k);
      lo += below * step;
      if (below < kProbes) hi = min(hi, lo + step);
      step = (hi - lo + kProbes - 1) / kProbes;
    }
    const int64_t n = lo / p.chunk - ch0;                 // its chunks after the first
    float acc[E];
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = 0.f;
    if (c < p.D) {
      if (g == 0) {
        const float* q = p.part + (ch0 * 2 + 1) * p.D + c;
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = q[j];
      }
      const int64_t c1 = ch0 + 1 + n * (g + 1) / kJoinGroups;
#pragma unroll 8
      for (int64_t ch = ch0 + 1 + n * g / kJoinGroups; ch < c1; ++ch) {
        const float* q = p.part + ch * 2 * p.D + c;
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] += q[j];
      }
    }
#pragma unroll
    for (int j = 0; j < E; ++j) part[g][j][t] = acc[j];
    __syncthreads();
    if (g == 0 && c < p.D) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
#pragma unroll
        for (int i = 1; i < kJoinGroups; ++i) acc[j] += part[i][j][t];
        acc[j] *= p.scale;
      }
      store_e<T, E>(static_cast<T*>(p.out) + static_cast<int64_t>(k) * p.D + c, acc);
    }
    __syncthreads();
  }
}

}  // namespace dc
