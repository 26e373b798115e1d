// C entry points of the text operators: dense and gated projections, layer norm and token
// embedding with their gradients. Same conventions as dc_api.cu: an int status, caller-owned outputs
// and workspaces, every launch on the caller's stream, nothing synchronizes.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "host.cuh"
#include "sm100.cuh"
#include "hgemm.cuh"
#include "padrows.cuh"
#include "rowdot.cuh"
#include "textgrad.cuh"
#include "norm.cuh"
#include "embed.cuh"

namespace dc {
int text_device_error(unsigned int* code, int clear) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code));
  if (e != cudaSuccess) return cuda_fail(e, "reading the device error word");
  if (clear && *code) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
    if (e != cudaSuccess) return cuda_fail(e, "clearing the device error word");
  }
  return DC_OK;
}
}  // namespace dc

namespace {

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t elem_size(int dtype) { return dtype == DC_DTYPE_F32 ? 4 : 2; }

// Every kernel of this file is launched with programmatic stream serialization (see pdl_wait), in
// clusters of `cluster` CTAs where that is above 0.
template <typename... P, typename... A>
int launch(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster,
           const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster); attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e != cudaSuccess ? cuda_fail(e, what) : DC_OK;
}

// ------------------------------------------------------------------------------ projections

// An operand of the contraction as the tensor core sees it: `rows` row indices x `k` contraction
// indices; mn: stored [k][rows] (the row index contiguous), else [rows][k].
struct Operand {
  const void* p = nullptr;
  int64_t ld = 0;
  int64_t rows = 0, k = 0;
};

int operand_map(CUtensorMap* map, const Operand& o, bool mn, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(mn ? o.rows : o.k), static_cast<uint64_t>(mn ? o.k : o.rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(o.ld) * 2};
  const uint32_t box[2] = {64, static_cast<uint32_t>(mn ? 64 : box_rows)};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, o.p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int check_operand(const char* what, const char* name, const void* p, int64_t ld, int64_t cols) {
  if (p == nullptr) return fail("%s: %s is null", what, name);
  if (!aligned(p, 16) || ld % 8) return fail("%s: %s needs a 16-byte aligned base and rows of a multiple of 16 bytes", what, name);
  if (ld < cols) return fail("%s: leading dimension of %s smaller than its row", what, name);
  return DC_OK;
}

int check_dims(const char* what, int dtype, int64_t M, int64_t N, int64_t K) {
  if (dtype != DC_DTYPE_BF16 && dtype != DC_DTYPE_F16) return fail("%s: dtype must be bf16 or fp16", what);
  if (M < 0 || N <= 0 || K <= 0) return fail("%s: bad shape M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
  if (M > (1ll << 30) || N > (1ll << 30) || K > (1ll << 30)) return fail("%s: dimension above 2^30", what);
  return DC_OK;
}

int check_act(const char* what, int act) {
  if (act < dc::kActNone || act > dc::kActGeluTanh) return fail("%s: unknown activation %d", what, act);
  return DC_OK;
}

// DC_HGEMM_PAIR = "0" / "1": force the cluster / the pair kernel (both compute every shape).
int pair_override() {
  const char* env = getenv("DC_HGEMM_PAIR");
  if (env == nullptr || (env[0] != '0' && env[0] != '1') || env[1] != 0) return -1;
  return env[0] - '0';
}

// Kernel and tile of a product: the smallest estimate of its time on the GPU. Both kernels are bound by
// what their CTAs read from L2, 128 bytes per row of A or B and 64-deep k-block; in nanoseconds,
// measured with the operands in L2,
//   pair      5400 + 4 bn + waves * k-blocks * 0.605 (256 + bn)
//   cluster   5200 + (S > 1: 900 + 200 S rows / 128) + load * k-blocks / S * 1.29 (rows + 128)
// with bn the pair's tile width, S the CTAs that divide a cluster tile's k-blocks, rows the tile's
// rows of A (at most 128), and load the CTAs per SM (at least one; two are resident, so a second
// wave counts as two more). Measured (M x N x K, one captured graph of calls, operands in L2 / from HBM)
// against the estimate, us; the choice first: 300 x 4096 x 4096 cluster S = 2 20.2 / 21.4 (20.2), pair 128
// wide 20.5 / 21.0 (20.9); 700 x 5120 x 1280 pair 12.2 / 12.8, cluster 14.5 / 15.3; 256 x 1024 x 4096 cluster
// 10.5 / 11.4, pair 19.4 / 20.4; 512 x 512 x 8192 cluster S = 8 13.2 / 14.5 (13.0), pair 34 / 36; 64 x 1024 x 1024
// cluster S = 8 5.1 / 5.6 (7.4), pair 7.8 / 8.3. Near its crossings the choice can be the slower one by a tenth:
// 1024^3 cluster S = 2 8.7 / 9.6 (9.1), pair 128 wide 8.4 / 8.8 (9.6).
struct HChoice { bool pair; int bn, splits; };

HChoice choose_hgemm(int64_t M, int stack, int64_t cols, int64_t k, int sms) {
  HChoice best = {true, 256, 1};
  double best_ns = 1e30;
  const int forced = pair_override();
  const double kb = static_cast<double>(ceil_div(k, dc::kHBK));
  if (forced != 0) {
    const int64_t m_tiles = ceil_div(M, 256) * stack;
    for (int bn = 256; bn >= 128; bn -= 32) {
      const double waves = static_cast<double>(ceil_div(m_tiles * ceil_div(cols, bn), sms / 2));
      const double ns = 5400 + 4.0 * bn + waves * kb * 0.605 * (256 + bn);
      if (ns < best_ns) { best = {true, bn, 1}; best_ns = ns; }
    }
  }
  if (forced != 1) {
    const double tiles = static_cast<double>(ceil_div(M, 128) * stack * ceil_div(cols, dc::kClBN));
    const double rows = static_cast<double>(std::min<int64_t>(M, 128));
    for (int s = 1; s <= 8 && (s == 1 || kb >= 2 * s); s *= 2) {
      const double ctas = tiles * s;
      const double load = ctas <= 2 * sms ? std::max(1.0, ctas / sms) : 2 * std::ceil(ctas / (2 * sms));
      const double ns = 5200 + (s > 1 ? 900 + 200 * s * rows / 128 : 0) + load * (kb / s) * 1.29 * (rows + 128);
      if (ns < best_ns) { best = {false, 256, s}; best_ns = ns; }
    }
  }
  return best;
}

// One contraction: A rows x B rows, over one or two segments of k (a0 . b0 + a1 . b1), or, with
// `stacked`, two A operands of equal shape whose rows follow one another (their products go to
// p.out and p.out1).
template <bool AMN, bool BMN, int EPI>
int launch_hgemm(const Operand& a0, const Operand& a1, const Operand& b0, const Operand& b1, bool stacked,
                 dc::HGemmParams p, cudaStream_t st) {
  const int sms = sm_count(), stack = stacked ? 2 : 1;
  const int64_t cols = EPI == dc::kEpiGated ? 2 * static_cast<int64_t>(p.N) : p.N;        // accumulator columns
  const int64_t k_all = a0.k + (!stacked && a1.p != nullptr ? a1.k : 0);
  const HChoice choice = choose_hgemm(p.M, stack, cols, k_all, sms);
  const bool pair = choice.pair;
  p.bn = choice.bn;
  p.splits = choice.splits;
  const int tile_m = pair ? 256 : 128;
  const int tile_n = (pair ? p.bn : dc::kClBN) / (EPI == dc::kEpiGated ? 2 : 1);
  const int bk = pair ? dc::kPairAtoms * dc::kHBK : dc::kHBK;
  const int half_m = static_cast<int>(ceil_div(p.M, tile_m));
  p.tiles_m = half_m * (stacked ? 2 : 1);
  p.tiles_n = static_cast<int>(ceil_div(p.N, tile_n));
  p.m_split = stacked ? half_m : INT32_MAX;
  p.group_m = 8;
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  if (tiles * 8 > INT32_MAX) return fail("projection: too many tiles");
  p.num_tiles = static_cast<int>(tiles);
  p.kb0 = static_cast<int>(ceil_div(a0.k, bk));
  p.kb1 = !stacked && a1.p != nullptr ? static_cast<int>(ceil_div(a1.k, bk)) : 0;
  p.a_rows = static_cast<int>(std::min<int64_t>(128, round_up(std::min<int64_t>(p.M, 128), 8)));
  p.out_vec = aligned(p.out, 16) && (p.out1 == nullptr || aligned(p.out1, 16)) && p.ldo % 8 == 0;
  p.res_vec = p.residual != nullptr && aligned(p.residual, 16) && p.ldr % 8 == 0;
  const int box_a = pair ? 128 : p.a_rows;
  const int box_b = pair ? p.bn / 2 : EPI == dc::kEpiGated ? dc::kClBN / 2 : dc::kClBN;
  CUtensorMap ma0, ma1, mb0, mb1;
  int r;
  if ((r = operand_map(&ma0, a0, AMN, box_a))) return r;
  if ((r = operand_map(&mb0, b0, BMN, box_b))) return r;
  if (a1.p == nullptr) ma1 = ma0;
  else if ((r = operand_map(&ma1, a1, AMN, box_a))) return r;
  if (b1.p == nullptr) mb1 = mb0;
  else if ((r = operand_map(&mb1, b1, BMN, box_b))) return r;

  if (pair) {
    auto kernel = dc::hgemm_pair_kernel<AMN, BMN, EPI>;
    if ((r = set_smem(kernel, dc::kPairSmem))) return r;
    return launch("projection launch", kernel, dim3(2 * static_cast<unsigned>(std::min(p.num_tiles, sms / 2))),
                  dim3(dc::kPairThreads), dc::kPairSmem, st, 2, ma0, ma1, mb0, mb1, p);
  }
  auto kernel = dc::hgemm_cluster_kernel<AMN, BMN, EPI>;
  if ((r = set_smem(kernel, dc::kClSmem))) return r;
  return launch("projection launch", kernel, dim3(static_cast<unsigned>(tiles * p.splits)), dim3(dc::kHThreads), dc::kClSmem, st,
                p.splits, ma0, ma1, mb0, mb1, p);
}

template <int NT, bool GATED, int AHEAD>
int launch_rowdot_rows(const dc::RowDotParams& p, bool vec, bool bf16, unsigned ctas, unsigned threads, cudaStream_t st) {
  const size_t smem = threads / 32 * 16 * 8 * NT * sizeof(float);     // at most 16 KB
  auto go = [&](auto kernel) { return launch("projection launch", kernel, ctas, threads, smem, st, 0, p); };
  if (vec) return bf16 ? go(dc::rowdot_kernel<NT, GATED, true, true, AHEAD>) : go(dc::rowdot_kernel<NT, GATED, true, false, AHEAD>);
  return bf16 ? go(dc::rowdot_kernel<NT, GATED, false, true, 4>) : go(dc::rowdot_kernel<NT, GATED, false, false, 4>);
}

template <bool GATED>
int launch_rowdot(dc::RowDotParams p, bool bf16, cudaStream_t st) {
  const bool vec = aligned(p.x, 16) && aligned(p.w0, 16) && (p.N == 1 || p.ldw0 % 8 == 0) && (p.M == 1 || p.ldx % 8 == 0) &&
                   (!GATED || (aligned(p.w1, 16) && (p.N == 1 || p.ldw1 % 8 == 0)));
  // Eight warps divide the k of a column group, 16 where one group per SM is all there is, fewer for
  // a short k. Measured, 8 rows: 4096 x 4096 14.2 / 11.6 / 12.4 us with 4 / 8 / 16 warps, gated
  // 2 x 512 x 4096 12.4 / 8.3 / 7.8, 640 x 640 4.9 / 5.0 / 5.9.
  const int64_t groups = ceil_div(p.N, GATED ? 8 : 16), steps = ceil_div(p.K, 32);
  p.ks = groups <= 148 && steps >= 64 ? 16 : 8;
  while (p.ks > 1 && steps < 2 * p.ks) p.ks /= 2;
  const int warps = std::max(p.ks, dc::kRowDotWarps);
  const unsigned ctas = static_cast<unsigned>(ceil_div(groups, warps / p.ks)), threads = 32 * warps;
  // Up to two CTAs per SM there are registers for eight steps in flight instead of four: 10.2 us
  // against 11.6 at 4096 x 4096; with more CTAs they cost occupancy (gated 2 x 10240 x 4096: 34.8
  // against 29.9).
  if (p.M > 8) return launch_rowdot_rows<2, GATED, 4>(p, vec, bf16, ctas, threads, st);
  if (ctas <= 2 * 148) return launch_rowdot_rows<1, GATED, 8>(p, vec, bf16, ctas, threads, st);
  return launch_rowdot_rows<1, GATED, 4>(p, vec, bf16, ctas, threads, st);
}

// Operands of the few-row path: any rows with element alignment.
int check_few_rows(const char* what, const char* name, const void* p, int64_t ld, int64_t cols) {
  if (p == nullptr) return fail("%s: %s is null", what, name);
  if (!aligned(p, 2)) return fail("%s: %s must be aligned to its element size", what, name);
  if (ld < cols) return fail("%s: leading dimension of %s smaller than its row", what, name);
  return DC_OK;
}

// Which projections take the few-row kernel (DC_HGEMM_PAIR picks among the tiled kernels only).
// Up to 8 rows it reads x once per step and weights always dominate: 4096 x 4096 11.6 us against 14.4
// for the cluster kernel, gated 2 x 10240 x 4096 29.9 against 38.8. At 9 to 16 rows the second
// block of x costs as many L1 accesses as the weights: 12.4 against 14.4, but 45 against 40 us.
bool few_rows(int64_t M, int64_t weights) {
  return (M <= 8 || (M <= dc::kRowDotMax && weights <= (32 << 20))) && pair_override() < 0;
}

int check_z(const char* what, const float* z, int64_t ldz, int64_t N) {
  if (z == nullptr) return DC_OK;
  if (!aligned(z, 16) || ldz % 4 || ldz < round_up(N, 4))
    return fail("%s: kept pre-activations need 16-byte aligned rows of at least N rounded up to 4", what);
  return DC_OK;
}

}  // namespace

extern "C" {

int dc_pad_rows(int count, const void* const* src, const int64_t* ld, const int64_t* rows, const int64_t* cols,
                void* const* dst, const int64_t* ldd, void* stream) {
  if (count < 1 || count > dc::kPadMatrices) return fail("pad_rows: 1 to %d matrices", dc::kPadMatrices);
  if (src == nullptr || ld == nullptr || rows == nullptr || cols == nullptr || dst == nullptr || ldd == nullptr)
    return fail("pad_rows: null array");
  dc::PadParams p = {};
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 0 || cols[i] <= 0 || rows[i] > (1ll << 30) || cols[i] > (1ll << 30))
      return fail("pad_rows: bad shape %lld x %lld", (long long)rows[i], (long long)cols[i]);
    if (rows[i] == 0) continue;
    if (src[i] == nullptr || dst[i] == nullptr) return fail("pad_rows: null pointer");
    if (!aligned(src[i], 2) || !aligned(dst[i], 16)) return fail("pad_rows: src must be aligned to its element size, dst to 16 bytes");
    if (ld[i] < 0 || ldd[i] % 8 || ldd[i] < cols[i] || ldd[i] > (1ll << 31) - 8) return fail("pad_rows: bad leading dimension");
    p.m[p.count++] = {static_cast<const uint16_t*>(src[i]), static_cast<uint16_t*>(dst[i]), ld[i], ldd[i], rows[i],
                      static_cast<int>(cols[i]), p.units};
    p.units += rows[i] * (ldd[i] / 8);
  }
  if (p.count == 0) return DC_OK;
  if (int r = check_sm100()) return r;
  const int64_t ctas = std::min<int64_t>(ceil_div(p.units, dc::kPadThreads), 148 * 32);
  return launch("pad_rows launch", dc::pad_rows_kernel, static_cast<unsigned>(ctas), dc::kPadThreads, 0, as_stream(stream), 0, p);
}

int dc_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
              int64_t ldr, void* y, int64_t ldy, float* z, int64_t ldz, int dtype, int64_t M, int64_t N, int64_t K,
              int act, void* stream) {
  int r;
  if ((r = check_dims("linear", dtype, M, N, K)) || (r = check_act("linear", act))) return r;
  if (M == 0) return DC_OK;
  const bool few = few_rows(M, N * K);
  const auto check = few ? check_few_rows : check_operand;
  if ((r = check("linear", "x", x, ldx, K)) || (r = check("linear", "w", w, ldw, K))) return r;
  if (y == nullptr) return fail("linear: y is null");
  if (!aligned(y, 2) || !aligned(bias, 2) || !aligned(residual, 2)) return fail("linear: pointers must be aligned to their element size");
  if (ldy < N || (residual != nullptr && ldr < 0)) return fail("linear: leading dimension smaller than the row");
  if ((r = check_z("linear", z, ldz, N)) || (r = check_sm100())) return r;
  if (few) {
    dc::RowDotParams d = {};
    d.x = static_cast<const uint16_t*>(x); d.ldx = ldx;
    d.w0 = static_cast<const uint16_t*>(w); d.ldw0 = ldw;
    d.bias0 = static_cast<const uint16_t*>(bias);
    d.residual = static_cast<const uint16_t*>(residual); d.ldr = ldr;
    d.out = static_cast<uint16_t*>(y); d.ldo = ldy; d.z0 = z; d.ldz = ldz;
    d.M = static_cast<int>(M); d.N = static_cast<int>(N); d.K = static_cast<int>(K); d.act = act;
    return launch_rowdot<false>(d, dtype == DC_DTYPE_BF16, as_stream(stream));
  }
  dc::HGemmParams p = {};
  p.M = static_cast<int>(M); p.N = static_cast<int>(N);
  p.out = y; p.ldo = ldy; p.bias = bias; p.residual = residual; p.ldr = ldr;
  p.z0 = z; p.ldz = ldz; p.act = act; p.bf16 = dtype == DC_DTYPE_BF16;
  return launch_hgemm<false, false, dc::kEpiLinear>({x, ldx, M, K}, {}, {w, ldw, N, K}, {}, false, p, as_stream(stream));
}

int dc_gated_linear(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                    const void* b_gate, const void* b_up, void* h, int64_t ldh, float* z_gate, float* z_up,
                    int64_t ldz, int dtype, int64_t M, int64_t N, int64_t K, int act, void* stream) {
  int r;
  if ((r = check_dims("gated_linear", dtype, M, N, K)) || (r = check_act("gated_linear", act))) return r;
  if (M == 0) return DC_OK;
  const bool few = few_rows(M, 2 * N * K);
  const auto check = few ? check_few_rows : check_operand;
  if ((r = check("gated_linear", "x", x, ldx, K)) || (r = check("gated_linear", "w_gate", w_gate, ldwg, K)) ||
      (r = check("gated_linear", "w_up", w_up, ldwu, K)))
    return r;
  if (h == nullptr) return fail("gated_linear: h is null");
  if (!aligned(h, 2) || !aligned(b_gate, 2) || !aligned(b_up, 2)) return fail("gated_linear: pointers must be aligned to their element size");
  if (ldh < N) return fail("gated_linear: leading dimension smaller than the row");
  if ((z_gate == nullptr) != (z_up == nullptr)) return fail("gated_linear: z_gate and z_up go together");
  if ((r = check_z("gated_linear", z_gate, ldz, N)) || (r = check_z("gated_linear", z_up, ldz, N)) || (r = check_sm100())) return r;
  if (few) {
    dc::RowDotParams d = {};
    d.x = static_cast<const uint16_t*>(x); d.ldx = ldx;
    d.w0 = static_cast<const uint16_t*>(w_gate); d.ldw0 = ldwg;
    d.w1 = static_cast<const uint16_t*>(w_up); d.ldw1 = ldwu;
    d.bias0 = static_cast<const uint16_t*>(b_gate); d.bias1 = static_cast<const uint16_t*>(b_up);
    d.out = static_cast<uint16_t*>(h); d.ldo = ldh; d.z0 = z_gate; d.z1 = z_up; d.ldz = ldz;
    d.M = static_cast<int>(M); d.N = static_cast<int>(N); d.K = static_cast<int>(K); d.act = act;
    return launch_rowdot<true>(d, dtype == DC_DTYPE_BF16, as_stream(stream));
  }
  dc::HGemmParams p = {};
  p.M = static_cast<int>(M); p.N = static_cast<int>(N);
  p.out = h; p.ldo = ldh; p.bias = b_gate; p.bias1 = b_up;
  p.z0 = z_gate; p.z1 = z_up; p.ldz = ldz; p.act = act; p.bf16 = dtype == DC_DTYPE_BF16;
  return launch_hgemm<false, false, dc::kEpiGated>({x, ldx, M, K}, {}, {w_gate, ldwg, N, K}, {w_up, ldwu, N, K}, false,
                                                   p, as_stream(stream));
}

int dc_linear_dx(const void* dz, const void* dz1, int64_t lddz, const void* w, int64_t ldw, const void* w1, int64_t ldw1,
                 void* dx, int64_t lddx, int dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  int r;
  if ((r = check_dims("linear_dx", dtype, M, N, K))) return r;
  if (M == 0) return DC_OK;
  if ((r = check_operand("linear_dx", "dz", dz, lddz, N)) || (r = check_operand("linear_dx", "w", w, ldw, K))) return r;
  if ((dz1 == nullptr) != (w1 == nullptr)) return fail("linear_dx: dz1 and w1 go together");
  if (dz1 != nullptr && ((r = check_operand("linear_dx", "dz1", dz1, lddz, N)) || (r = check_operand("linear_dx", "w1", w1, ldw1, K)))) return r;
  if (dx == nullptr || !aligned(dx, 2)) return fail("linear_dx: dx is null or not aligned to its element size");
  if (lddx < K) return fail("linear_dx: leading dimension smaller than the row");
  if ((r = check_sm100())) return r;
  dc::HGemmParams p = {};
  p.M = static_cast<int>(M); p.N = static_cast<int>(K);
  p.out = dx; p.ldo = lddx; p.bf16 = dtype == DC_DTYPE_BF16;
  return launch_hgemm<false, true, dc::kEpiLinear>({dz, lddz, M, N}, {dz1, lddz, M, N}, {w, ldw, K, N}, {w1, ldw1, K, N},
                                                   false, p, as_stream(stream));
}

int dc_linear_dw(const void* dz, const void* dz1, int64_t lddz, const void* x, int64_t ldx, void* dw, void* dw1,
                 int64_t lddw, int dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  int r;
  if ((r = check_dims("linear_dw", dtype, M, N, K))) return r;
  if (M == 0) return fail("linear_dw: no rows to sum (M = 0): the gradient is zero");
  if ((r = check_operand("linear_dw", "dz", dz, lddz, N)) || (r = check_operand("linear_dw", "x", x, ldx, K))) return r;
  if ((dz1 == nullptr) != (dw1 == nullptr)) return fail("linear_dw: dz1 and dw1 go together");
  if (dz1 != nullptr && (r = check_operand("linear_dw", "dz1", dz1, lddz, N))) return r;
  if (dw == nullptr || !aligned(dw, 2) || !aligned(dw1, 2)) return fail("linear_dw: dw is null or not aligned to its element size");
  if (lddw < K) return fail("linear_dw: leading dimension smaller than the row");
  if ((r = check_sm100())) return r;
  dc::HGemmParams p = {};
  p.M = static_cast<int>(N); p.N = static_cast<int>(K);
  p.out = dw; p.out1 = dw1; p.ldo = lddw; p.bf16 = dtype == DC_DTYPE_BF16;
  return launch_hgemm<true, true, dc::kEpiLinear>({dz, lddz, N, M}, {dz1, lddz, N, M}, {x, ldx, K, M}, {}, dz1 != nullptr,
                                                  p, as_stream(stream));
}

}  // extern "C"

namespace {

// Row blocks of the column sums: about eight CTAs per SM, at least 16 rows each.
int64_t grad_row_blocks(int64_t M, int64_t N) {
  const int64_t col_blocks = ceil_div(N, dc::kGradCols);
  return std::max<int64_t>(1, std::min<int64_t>({148 * 8 / col_blocks, ceil_div(M, 16), 65535}));
}

int colsum_finish(const float* p0, const float* p1, int64_t ldp, int64_t P, int64_t N, void* o0, void* o1, int dtype,
                  cudaStream_t st) {
  return launch("column sums launch", dc::colsum_finish_kernel, dim3(static_cast<unsigned>(ceil_div(N, 32)), o1 != nullptr ? 2 : 1),
                32 * dc::kFinishGroups, 0, st, 0, p0, p1, ldp, static_cast<int>(P), N, o0, o1, dtype);
}

}  // namespace

extern "C" {

int dc_act_grad_workspace(int64_t M, int64_t N, size_t* bytes) {
  if (M < 0 || N <= 0 || bytes == nullptr) return fail("act_grad: bad shape M=%lld N=%lld", (long long)M, (long long)N);
  *bytes = static_cast<size_t>(grad_row_blocks(M, N)) * round_up(N, 8) * 2 * sizeof(float);
  return DC_OK;
}

int dc_act_grad(const void* dy, int64_t lddy, const float* z, const float* z1, int64_t ldz, void* dz, void* dz1,
                int64_t lddz, void* db, void* db1, void* workspace, size_t workspace_bytes, int dtype, int64_t M,
                int64_t N, int act, void* stream) {
  int r;
  if ((r = check_dims("act_grad", dtype, M, N, 1)) || (r = check_act("act_grad", act))) return r;
  if (M == 0) return fail("act_grad: no rows (M = 0): every gradient is empty or zero");
  if (dy == nullptr || !aligned(dy, 2) || lddy < N) return fail("act_grad: dy is null, misaligned or its rows overlap");
  if (z == nullptr && (z1 != nullptr || dz != nullptr)) return fail("act_grad: dz needs the kept pre-activations");
  if (z == nullptr && db == nullptr) return fail("act_grad: nothing to compute");
  if ((r = check_z("act_grad", z, ldz, N)) || (r = check_z("act_grad", z1, ldz, N))) return r;
  if (z != nullptr) {
    if ((r = check_operand("act_grad", "dz", dz, lddz, N))) return r;
    if (z1 != nullptr && (r = check_operand("act_grad", "dz1", dz1, lddz, N))) return r;
  }
  if (db1 != nullptr && (z1 == nullptr || db == nullptr)) return fail("act_grad: db1 needs z1 and db");
  const int64_t blocks = grad_row_blocks(M, N), ldp = round_up(N, 8);
  if (db != nullptr) {
    size_t need = 0;
    dc_act_grad_workspace(M, N, &need);
    if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need)
      return fail("act_grad: workspace below %zu bytes or misaligned", need);
    if (!aligned(db, 2) || !aligned(db1, 2)) return fail("act_grad: db must be aligned to its element size");
  }
  if ((r = check_sm100())) return r;
  dc::ActGradParams p = {};
  p.dy = static_cast<const uint16_t*>(dy); p.lddy = lddy;
  p.z0 = z; p.z1 = z1; p.ldz = ldz;
  p.dz0 = static_cast<uint16_t*>(dz); p.dz1 = static_cast<uint16_t*>(dz1); p.lddz = lddz;
  p.part0 = db != nullptr ? static_cast<float*>(workspace) : nullptr;
  p.part1 = db != nullptr ? static_cast<float*>(workspace) + blocks * ldp : nullptr;
  p.ldp = ldp; p.M = M; p.N = N;
  p.rows_per_block = static_cast<int>(ceil_div(M, blocks));
  p.act = act; p.bf16 = dtype == DC_DTYPE_BF16;
  p.dy_vec = aligned(dy, 16) && lddy % 8 == 0;
  const cudaStream_t st = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(ceil_div(N, dc::kGradCols)), static_cast<unsigned>(blocks));
  const dim3 block(dc::kGradX, dc::kGradY);
  const auto kernel = z1 != nullptr ? (p.dy_vec ? dc::act_grad_kernel<2, false> : dc::act_grad_kernel<2, true>)
                      : z != nullptr ? dc::act_grad_kernel<1, false> : dc::act_grad_kernel<0, false>;
  if ((r = launch("act_grad launch", kernel, grid, block, 0, st, 0, p))) return r;
  if (db != nullptr) return colsum_finish(p.part0, p.part1, ldp, blocks, N, db, db1, dtype, st);
  return DC_OK;
}

}  // extern "C"

// ------------------------------------------------------------------------------ layer norm

namespace {

int64_t norm_wide_blocks(int64_t M, int64_t D) {
  return std::max<int64_t>(1, std::min<int64_t>({ceil_div(148 * 16, ceil_div(D, 512)), ceil_div(M, 16), 65535}));
}
// The ring kernel's launch shape: threads per row, values per thread, stages and persistent CTAs, as
// many per SM as its registers and 200 KB of shared memory allow with at least two stages each; no
// shape (ctas 0) where the row is too wide for it.
struct RingPlan { int tpr, ept, slot, stages, smem; int64_t ctas; };

RingPlan ring_plan(int64_t M, int64_t D, size_t es, bool vec, bool bwd) {
  // 32 values per thread: the sums over a row cost each warp as much as 16 values' arithmetic
  // (32768 x 4096 bf16: 96 us forward against 117 with 16 values, 167 against 171 backward). Rows read
  // by single values need more threads' loads in flight at 2048 (10007 x 2047: 39 against 45 us).
  RingPlan n = {};
  n.tpr = D <= 1024 ? 32 : D <= 2048 ? 64 : D <= 4096 ? 128 : D <= 8192 ? 256 : 512;
  n.ept = D <= 256 ? 8 : D <= 512 ? 16 : 32;
  if (!vec && n.tpr == 64) { n.tpr = 128; n.ept = 16; }
  // 16-bit rows of up to three quarters of a shape: the issue slots of absent values are what they
  // wait for (19660 x 2560 bf16 46.9 us forward and 77.9 backward, 54.5 and 92.4 with 32).
  if (es == 2 && n.ept == 32 && D <= n.tpr * 24) n.ept = 24;
  if (D > 16384 || (bwd && D > 8192)) return n;
  const int threads = std::max(128, n.tpr), rows = threads / n.tpr;
  const bool shared_w = bwd && n.ept == 32 && (es == 4 || n.tpr < 128);       // RingCta::kSharedW
  const int sm_threads = n.ept > 16 ? (!bwd ? 512 : shared_w || n.ept == 24 ? 384 : 256) : (bwd ? 512 : 768);
  const int64_t w_bytes = shared_w ? n.tpr * n.ept * 4 : 0;
  n.slot = static_cast<int>(round_up(D * static_cast<int64_t>(es), 16)) + (vec ? 0 : 16);
  const int64_t stage = static_cast<int64_t>(rows) * (bwd ? 2 : 1) * n.slot;
  constexpr int64_t kSm = 200 << 10;
  int per_sm = std::max(1, sm_threads / threads);
  while (per_sm > 0 && (w_bytes + 2 * stage) * per_sm > kSm) --per_sm;
  if (per_sm == 0) return n;
  n.stages = static_cast<int>(std::min<int64_t>(dc::kRingMax, (kSm / per_sm - w_bytes) / stage));
  const int64_t sums = rows > 1 ? 2 * n.tpr * n.ept * 4 : 0;
  n.smem = static_cast<int>(w_bytes + std::max(n.stages * stage, sums));
  n.ctas = std::min<int64_t>(ceil_div(M, rows), 148 * per_sm);
  return n;
}

// norm_bwd_kernel's stages and shared memory; no shape (stages 0) where fewer than two stages fit.
struct NormBwdPlan { int stages, smem; };

NormBwdPlan norm_bwd_plan(int64_t D, size_t es, bool w32) {
  NormBwdPlan n = {};
  if (D > dc::kBwdThreads * dc::kBwdValues) return n;
  const int64_t w = D * static_cast<int64_t>(w32 ? 4 : es), stage = 2 * D * static_cast<int64_t>(es);
  constexpr int64_t kSm = 200 << 10;
  n.stages = static_cast<int>(std::min<int64_t>(dc::kRingMax, (kSm - w) / stage));
  if (n.stages < 2) n.stages = 0;
  n.smem = static_cast<int>(w + n.stages * stage);
  return n;
}

template <typename T>
int launch_norm_bwd(dc::NormParams p, const NormBwdPlan& n, cudaStream_t st) {
  p.stages = n.stages;
  auto go = [&](auto kernel) {
    if (int r = set_smem(kernel, n.smem)) return r;
    return launch("layer_norm_grad launch", kernel, static_cast<unsigned>(p.parts), dc::kBwdThreads, n.smem, st, 0, p);
  };
  if constexpr (sizeof(T) == 2) {
    if (p.w_f32) return go(dc::norm_bwd_kernel<T, true>);
  }
  return go(dc::norm_bwd_kernel<T, false>);
}

template <typename T, int E, int EPT, int TPR, bool BWD>
int launch_ring(dc::NormParams p, const RingPlan& n, cudaStream_t st) {
  p.slot = n.slot;
  p.stages = n.stages;
  auto kernel = dc::norm_ring_kernel<T, E, EPT, TPR, BWD>;
  if (int r = set_smem(kernel, n.smem)) return r;
  return launch("layer_norm launch", kernel, static_cast<unsigned>(n.ctas), dc::RingCta<T, TPR, EPT, BWD>::kThreads, n.smem, st, 0, p);
}

template <typename T, int E, bool BWD>
int launch_ring_rows(const dc::NormParams& p, const RingPlan& n, cudaStream_t st) {
  switch (n.tpr * 100 + n.ept) {
    case 3232: return launch_ring<T, E, 32, 32, BWD>(p, n, st);
    case 12832: return launch_ring<T, E, 32, 128, BWD>(p, n, st);
    case 25632: return launch_ring<T, E, 32, 256, BWD>(p, n, st);
  }
  if constexpr (E != 8) {                                 // narrower aligned rows: norm_narrow_kernel
    if (n.ept == 16 && n.tpr == 32) return launch_ring<T, E, 16, 32, BWD>(p, n, st);
  }
  if constexpr (sizeof(T) == 2) {
    switch (n.tpr * 100 + n.ept) {
      case 3224: return launch_ring<T, E, 24, 32, BWD>(p, n, st);
      case 12824: return launch_ring<T, E, 24, 128, BWD>(p, n, st);
      case 25624: return launch_ring<T, E, 24, 256, BWD>(p, n, st);
    }
    if constexpr (E == 8) {
      if (n.tpr == 64 && n.ept == 24) return launch_ring<T, E, 24, 64, BWD>(p, n, st);
    }
    if constexpr (!BWD) {
      if (n.tpr == 512 && n.ept == 24) return launch_ring<T, E, 24, 512, BWD>(p, n, st);
    }
  }
  if constexpr (E == 1) {
    if (n.ept == 8) return launch_ring<T, E, 8, 32, BWD>(p, n, st);
    if (n.tpr == 128) return launch_ring<T, E, 16, 128, BWD>(p, n, st);
  } else {
    if (n.tpr == 64) return launch_ring<T, E, 32, 64, BWD>(p, n, st);
  }
  if constexpr (!BWD) return launch_ring<T, E, 32, 512, BWD>(p, n, st);
  return fail("layer_norm: no kernel for rows of %d values", p.D);
}

// Narrow rows: threads per row of norm_narrow_kernel (0: too wide for it) and its CTAs.
int narrow_threads(int64_t D, size_t es) {
  const int64_t units = ceil_div(D * static_cast<int64_t>(es), 16);
  for (int tpr = 4; tpr <= 32; tpr *= 2) {
    if (units <= tpr * dc::kNarrowUnits) return tpr;
  }
  return 0;
}
int64_t narrow_ctas(int64_t M, int tpr, int per_sm) {
  return std::min<int64_t>(ceil_div(M * tpr, dc::kNarrowThreads), 148 * per_sm);
}
template <typename T, bool BWD>
int launch_narrow(const dc::NormParams& p, int tpr, cudaStream_t st) {
  const unsigned ctas = static_cast<unsigned>(narrow_ctas(p.M, tpr, dc::NormNarrow<BWD>::kPerSm));
  const auto kernel = tpr == 4 ? dc::norm_narrow_kernel<T, 4, BWD> : tpr == 8 ? dc::norm_narrow_kernel<T, 8, BWD>
                    : tpr == 16 ? dc::norm_narrow_kernel<T, 16, BWD> : dc::norm_narrow_kernel<T, 32, BWD>;
  return launch("layer_norm launch", kernel, ctas, dc::kNarrowThreads, 0, st, 0, p);
}

template <typename T, int E>
int launch_norm_grad_wide(const dc::NormParams& p, cudaStream_t st) {
  if (int status = launch("layer_norm_grad launch", dc::norm_dx_wide_kernel<T, E>, static_cast<unsigned>(p.M), dc::kNormWide, 0, st, 0, p)) return status;
  if (p.part_w == nullptr) return DC_OK;
  return launch("layer_norm_grad launch", dc::norm_dw_wide_kernel<T, E>, dim3(static_cast<unsigned>(ceil_div(p.D, 128 * E)), static_cast<unsigned>(p.parts)), 128, 0, st, 0, p, static_cast<int>(ceil_div(p.M, p.parts)));
}

// The forward register kernel, for few rows that are not narrow: the fewest threads per row that hold
// it in two units (eight single values) each, up to 512 threads and eight units (32 values). Wider rows
// take the kernel for any width.
template <typename T, bool VEC>
int launch_norm_reg(const dc::NormParams& p, cudaStream_t st) {
  constexpr int E = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  const int64_t units = ceil_div(p.D, E);
  constexpr int most = VEC ? 2 : 8, top = VEC ? 8 : 32;
  const int tpr = units <= 32 * most ? 32 : units <= 128 * most ? 128 : 512;
  const int64_t nu = ceil_div(units, tpr);
  auto go = [&](auto kernel, int threads, int rows) {
    return launch("layer_norm launch", kernel, static_cast<unsigned>(ceil_div(p.M, rows)), threads, 0, st, 0, p);
  };
  if constexpr (!VEC) {                                   // aligned rows of so few units are narrow
    if (tpr == 32) return go(dc::norm_fwd_kernel<T, VEC, most, 32>, dc::NormCta<32>::kThreads, 8);
  }
  if (tpr == 128) return go(dc::norm_fwd_kernel<T, VEC, most, 128>, 128, 1);
  if (nu <= most) return go(dc::norm_fwd_kernel<T, VEC, most, 512>, 512, 1);
  if (nu <= top) return go(dc::norm_fwd_kernel<T, VEC, top, 512>, 512, 1);
  return go(dc::norm_fwd_wide_kernel<T>, dc::kNormWide, 1);
}

// Which kernel a gradient runs in, and its partial rows: the one for narrow aligned rows; the ring, for
// unaligned rows where the window of a row lies inside its neighbours; the kernel for wide aligned
// rows; else the ones for any width.
enum NormGradPath { kNormGradNarrow, kNormGradRing, kNormGradLong, kNormGradWide };
NormGradPath norm_grad_path(const dc::NormParams& p, bool vec, size_t es, int64_t* parts) {
  if (const int tpr = vec ? narrow_threads(p.D, es) : 0) {
    *parts = narrow_ctas(p.M, tpr, dc::NormNarrow<true>::kPerSm);
    return kNormGradNarrow;
  }
  const RingPlan r = ring_plan(p.M, p.D, es, vec, true);
  if (r.ctas > 0 && (vec || (p.ldx >= p.D && p.lddy >= p.D && p.D * es >= 16))) { *parts = r.ctas; return kNormGradRing; }
  if (vec && norm_bwd_plan(p.D, es, p.w_f32).stages > 0) { *parts = std::min<int64_t>(p.M, 148); return kNormGradLong; }
  *parts = norm_wide_blocks(p.M, p.D);
  return kNormGradWide;
}

template <typename T, bool BWD>
int launch_norm(const dc::NormParams& p, bool vec, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const RingPlan n = ring_plan(p.M, p.D, sizeof(T), vec, BWD);
  if constexpr (BWD) {
    int64_t parts;
    switch (norm_grad_path(p, vec, sizeof(T), &parts)) {
      case kNormGradNarrow: return launch_narrow<T, true>(p, narrow_threads(p.D, sizeof(T)), st);
      case kNormGradRing: return vec ? launch_ring_rows<T, E, true>(p, n, st) : launch_ring_rows<T, 1, true>(p, n, st);
      case kNormGradLong: return launch_norm_bwd<T>(p, norm_bwd_plan(p.D, sizeof(T), p.w_f32), st);
      default: return vec ? launch_norm_grad_wide<T, E>(p, st) : launch_norm_grad_wide<T, 1>(p, st);
    }
  } else {
    if (const int tpr = vec ? narrow_threads(p.D, sizeof(T)) : 0) return launch_narrow<T, false>(p, tpr, st);
    // Many wider rows through the ring: 30000 x 2048 bf16 53 us against 66 in the register kernel.
    const bool apart = p.ldx >= p.D && p.D * sizeof(T) >= 16;
    if (p.M >= 148 * 8 && n.ctas > 0) {
      if (vec) return launch_ring_rows<T, E, false>(p, n, st);
      if (!vec && apart) return launch_ring_rows<T, 1, false>(p, n, st);
    }
    return vec ? launch_norm_reg<T, true>(p, st) : launch_norm_reg<T, false>(p, st);
  }
}

template <bool BWD>
int dispatch_norm(const dc::NormParams& p, int dtype, bool vec, cudaStream_t st) {
  switch (dtype) {
    case DC_DTYPE_F32: return launch_norm<float, BWD>(p, vec, st);
    case DC_DTYPE_F16: return launch_norm<__half, BWD>(p, vec, st);
    default: return launch_norm<__nv_bfloat16, BWD>(p, vec, st);
  }
}

int check_norm(const char* what, int dtype, int w_dtype, int64_t M, int64_t D) {
  if (dtype != DC_DTYPE_F32 && dtype != DC_DTYPE_F16 && dtype != DC_DTYPE_BF16) return fail("%s: unsupported dtype %d", what, dtype);
  if (w_dtype != dtype && w_dtype != DC_DTYPE_F32) return fail("%s: the weight must be in x's type or fp32", what);
  if (M < 0 || D <= 0 || M > INT32_MAX || D > (1 << 30)) return fail("%s: bad shape M=%lld D=%lld", what, (long long)M, (long long)D);
  return DC_OK;
}

}  // namespace

extern "C" {

int dc_layer_norm(const void* x, int64_t ldx, const void* w, const void* b, int w_dtype, void* y, int64_t ldy,
                  float* mean, float* rstd, int dtype, int64_t M, int64_t D, float eps, void* stream) {
  int r;
  if ((r = check_norm("layer_norm", dtype, w_dtype, M, D))) return r;
  if (M == 0) return DC_OK;
  const size_t es = elem_size(dtype), ws = elem_size(w_dtype);
  if (x == nullptr || y == nullptr) return fail("layer_norm: null pointer");
  if (!aligned(x, es) || !aligned(y, es) || !aligned(w, ws) || !aligned(b, ws) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail("layer_norm: pointers must be aligned to their element size");
  if (ldx < 0 || ldy < D) return fail("layer_norm: leading dimension smaller than the row");
  if ((mean == nullptr) != (rstd == nullptr)) return fail("layer_norm: mean and rstd go together");
  if ((r = check_sm100())) return r;
  dc::NormParams p = {};
  p.x = x; p.ldx = ldx; p.w = w; p.b = b; p.out = y; p.ldo = ldy; p.mean = mean; p.rstd = rstd;
  p.M = M; p.D = static_cast<int>(D); p.eps = eps; p.w_f32 = w_dtype == DC_DTYPE_F32;
  const int64_t e = 16 / static_cast<int64_t>(es);
  const bool vec = D % e == 0 && ldx % e == 0 && ldy % e == 0 && aligned(x, 16) && aligned(y, 16) && aligned(w, 16) && aligned(b, 16);
  return dispatch_norm<false>(p, dtype, vec, as_stream(stream));
}

int dc_layer_norm_grad_workspace(int64_t M, int64_t D, size_t* bytes) {
  if (M < 0 || D <= 0 || bytes == nullptr) return fail("layer_norm_grad: bad shape M=%lld D=%lld", (long long)M, (long long)D);
  // Enough for every path: up to six persistent CTAs per SM, or the wide kernel's row blocks.
  *bytes = static_cast<size_t>(std::max<int64_t>(norm_wide_blocks(M, D), std::min<int64_t>(M, 6 * 148))) * round_up(D, 4) * 2 *
           sizeof(float);
  return DC_OK;
}

int dc_layer_norm_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int w_dtype,
                       const float* mean, const float* rstd, void* dx, int64_t lddx, void* dw, void* db,
                       void* workspace, size_t workspace_bytes, int dtype, int64_t M, int64_t D, void* stream) {
  int r;
  if ((r = check_norm("layer_norm_grad", dtype, w_dtype, M, D))) return r;
  if (M == 0) return fail("layer_norm_grad: no rows (M = 0): every gradient is empty or zero");
  const size_t es = elem_size(dtype), ws = elem_size(w_dtype);
  if (dy == nullptr || x == nullptr || dx == nullptr || mean == nullptr || rstd == nullptr) return fail("layer_norm_grad: null pointer");
  if (!aligned(x, es) || !aligned(dy, es) || !aligned(dx, es) || !aligned(w, ws) || !aligned(dw, ws) || !aligned(db, ws) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return fail("layer_norm_grad: pointers must be aligned to their element size");
  if (ldx < 0 || lddy < 0 || lddx < D) return fail("layer_norm_grad: leading dimension smaller than the row");
  if (dw == nullptr && db != nullptr) return fail("layer_norm_grad: db is computed with dw");
  size_t need = 0;
  dc_layer_norm_grad_workspace(M, D, &need);
  if (dw != nullptr && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need))
    return fail("layer_norm_grad: workspace below %zu bytes or misaligned", need);
  if ((r = check_sm100())) return r;
  dc::NormParams p = {};
  p.x = x; p.ldx = ldx; p.dy = dy; p.lddy = lddy; p.w = w; p.out = dx; p.ldo = lddx;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.ldp = round_up(D, 4);
  p.M = M; p.D = static_cast<int>(D); p.w_f32 = w_dtype == DC_DTYPE_F32;
  const int64_t e = 16 / static_cast<int64_t>(es);
  const bool vec = D % e == 0 && ldx % e == 0 && lddy % e == 0 && lddx % e == 0 && aligned(x, 16) && aligned(dy, 16) &&
                   aligned(dx, 16) && aligned(w, 16);
  int64_t parts;
  norm_grad_path(p, vec, es, &parts);
  p.parts = static_cast<int>(parts);
  if (dw != nullptr) { p.part_w = static_cast<float*>(workspace); p.part_b = p.part_w + p.parts * p.ldp; }
  const cudaStream_t st = as_stream(stream);
  if ((r = dispatch_norm<true>(p, dtype, vec, st))) return r;
  if (dw != nullptr) return colsum_finish(p.part_w, p.part_b, p.ldp, p.parts, D, dw, db, w_dtype, st);
  return DC_OK;
}

}  // extern "C"

// ------------------------------------------------------------------------------ embedding

namespace {

int check_embed(const char* what, int dtype, int64_t T, int64_t V, int64_t D) {
  if (dtype != DC_DTYPE_F32 && dtype != DC_DTYPE_F16 && dtype != DC_DTYPE_BF16) return fail("%s: unsupported dtype %d", what, dtype);
  if (T < 0 || V <= 0 || D <= 0 || T > INT32_MAX - 4096 || V >= INT32_MAX || D > (1 << 30))
    return fail("%s: bad shape T=%lld V=%lld D=%lld", what, (long long)T, (long long)V, (long long)D);
  return DC_OK;
}

template <typename T, int E>
int launch_embed_fwd(const dc::EmbedIds& ids, const void* table, int64_t ldt, void* out, int64_t ldo, int64_t D, float scale,
                     cudaStream_t st) {
  const int64_t vecs = ceil_div(D, E);
  unsigned bx = 8;
  while (bx < 128 && bx < vecs) bx *= 2;
  const unsigned by = 128 / bx;
  auto go = [&](auto kernel, unsigned tokens) {
    return launch("embedding launch", kernel, static_cast<unsigned>(ceil_div(ids.T, by * tokens)), dim3(bx, by), 0, st, 0, ids,
                  static_cast<const T*>(table), ldt, static_cast<T*>(out), ldo, static_cast<int>(D), scale);
  };
  return vecs <= bx && ids.T >= 148 * 16 * static_cast<int64_t>(by) ? go(dc::embed_fwd_kernel<T, E, 4>, 4)
                                                                    : go(dc::embed_fwd_kernel<T, E, 1>, 1);
}

// Workspace of the gradient: two (key, index) pairs of arrays, the radix histogram, the partials.
struct EmbedPlan {
  bool rank;                // counting sort in one launch
  int passes, bits;         // radix
  bool scan;                // the tiles' counts are made into prefix sums by a launch of its own
  int64_t tiles, chunk, chunks;
  size_t keys[2], idx[2], hist, part, total;
};

// Tiles of 1024 tokens from which on the scatter's counts are summed by a launch of their own. The whole
// gradient, 32128 x 8 fp32, without / with it: 64 tiles 39.9 / 43.1 us, 96 46.4 / 45.0, 128 61.8 / 49.3, 512 168 /
// 92, 4096 3580 / 584.
constexpr int64_t kScanTiles = 96;

EmbedPlan embed_plan(int64_t T, int64_t V, int64_t D) {
  EmbedPlan e = {};
  e.rank = T <= dc::kRankMax && V < (1 << 19);
  int nbits = 1;
  while ((V >> nbits) != 0) ++nbits;             // keys are 0 .. V
  e.passes = e.rank ? 0 : (nbits + dc::kRadixBits - 1) / dc::kRadixBits;
  e.bits = e.rank ? 0 : (nbits + e.passes - 1) / e.passes;
  e.tiles = e.rank ? 0 : ceil_div(T, dc::kRadixTile);
  const int64_t slabs = ceil_div(D, 8 * dc::kSumThreads);
  e.chunk = 8;
  while (e.chunk < dc::kSumChunkMax && ceil_div(T, 2 * e.chunk) * slabs >= 16 * 148) e.chunk *= 2;
  e.chunks = ceil_div(T, e.chunk);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t a = at; at += (n + 255) / 256 * 256; return a; };
  for (int i = 0; i < (e.rank ? 1 : 2); ++i) { e.keys[i] = take(T * 4); e.idx[i] = take(T * 4); }
  e.scan = e.tiles >= kScanTiles;
  e.hist = take((static_cast<size_t>(e.tiles + (e.scan ? 1 : 0)) << e.bits) * 4);
  e.part = take(static_cast<size_t>(e.chunks) * 2 * D * 4);
  e.total = at;
  return e;
}

template <typename T, int E>
int launch_embed_sum(const dc::EmbedSumParams& p, int64_t chunks, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(ceil_div(p.D, E * dc::kSumThreads)));
  if (grid.y > 65535) return fail("embedding_grad: rows of %d values are too wide", p.D);
  if (int status = launch("embedding_grad sum launch", dc::embed_sum_kernel<T, E>, grid, dc::kSumThreads, 0, st, 0, p)) return status;
  if (chunks <= 2) return DC_OK;             // no run can go on behind the chunk after its first
  const dim3 join(static_cast<unsigned>(ceil_div(chunks, dc::kJoinChunks)), grid.y);
  return launch("embedding_grad join launch", dc::embed_join_kernel<T, E>, join, dc::kSumThreads * dc::kJoinGroups, 0, st, 0, p);
}

}  // namespace

extern "C" {

int dc_embedding(const void* ids, int ids_i64, int64_t T, const void* table, int64_t ldt, int64_t V, int64_t D,
                 float scale, void* out, int64_t ldo, int dtype, void* stream) {
  int r;
  if ((r = check_embed("embedding", dtype, T, V, D))) return r;
  if (T == 0) return DC_OK;
  const size_t es = elem_size(dtype);
  if (ids == nullptr || table == nullptr || out == nullptr) return fail("embedding: null pointer");
  if (!aligned(ids, ids_i64 ? 8 : 4) || !aligned(table, es) || !aligned(out, es))
    return fail("embedding: pointers must be aligned to their element size");
  if (ldt < D || ldo < D) return fail("embedding: leading dimension smaller than the row");
  if ((r = check_sm100())) return r;
  const dc::EmbedIds e = {ids, ids_i64 != 0, T, V, -1};
  const int64_t n = 16 / static_cast<int64_t>(es);
  const bool vec = D % n == 0 && ldt % n == 0 && ldo % n == 0 && aligned(table, 16) && aligned(out, 16);
  const cudaStream_t st = as_stream(stream);
  switch (dtype) {
    case DC_DTYPE_F32: return vec ? launch_embed_fwd<float, 4>(e, table, ldt, out, ldo, D, scale, st)
                                  : launch_embed_fwd<float, 1>(e, table, ldt, out, ldo, D, scale, st);
    case DC_DTYPE_F16: return vec ? launch_embed_fwd<__half, 8>(e, table, ldt, out, ldo, D, scale, st)
                                  : launch_embed_fwd<__half, 1>(e, table, ldt, out, ldo, D, scale, st);
    default: return vec ? launch_embed_fwd<__nv_bfloat16, 8>(e, table, ldt, out, ldo, D, scale, st)
                        : launch_embed_fwd<__nv_bfloat16, 1>(e, table, ldt, out, ldo, D, scale, st);
  }
}

int dc_embedding_grad_workspace(int64_t T, int64_t V, int64_t D, size_t* bytes) {
  int r;
  if ((r = check_embed("embedding_grad", DC_DTYPE_F32, T, V, D))) return r;
  if (bytes == nullptr) return fail("embedding_grad: null pointer");
  *bytes = embed_plan(T, V, D).total;
  return DC_OK;
}

int dc_embedding_grad(const void* dy, int64_t lddy, const void* ids, int ids_i64, int64_t T, int64_t V, int64_t D,
                      int64_t padding_idx, float scale, void* dtable, void* workspace, size_t workspace_bytes, int dtype,
                      void* stream) {
  int r;
  if ((r = check_embed("embedding_grad", dtype, T, V, D))) return r;
  const size_t es = elem_size(dtype);
  if (dtable == nullptr || !aligned(dtable, es)) return fail("embedding_grad: dtable is null or not aligned to its element size");
  if (T > 0 && (dy == nullptr || ids == nullptr)) return fail("embedding_grad: null pointer");
  if (!aligned(ids, ids_i64 ? 8 : 4) || !aligned(dy, es)) return fail("embedding_grad: pointers must be aligned to their element size");
  if (lddy < 0) return fail("embedding_grad: negative leading dimension");
  const EmbedPlan plan = embed_plan(T, V, D);
  if (T > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < plan.total))
    return fail("embedding_grad: workspace below %zu bytes or misaligned", plan.total);
  if ((r = check_sm100())) return r;
  const cudaStream_t st = as_stream(stream);
  uint8_t* const table = static_cast<uint8_t*>(dtable);
  const int64_t table_bytes = V * D * static_cast<int64_t>(es);
  // Up to the first 16-byte boundary of an unaligned table, or all of it when there are no tokens.
  const int64_t head = T == 0 ? table_bytes : std::min<int64_t>(table_bytes, (16 - reinterpret_cast<uintptr_t>(table) % 16) % 16);
  if (head > 0) {
    cudaError_t ce = cudaMemsetAsync(table, 0, static_cast<size_t>(head), st);
    if (ce != cudaSuccess) return cuda_fail(ce, "embedding_grad zero fill");
  }
  if (T == 0) return DC_OK;

  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto u32 = [&](size_t off) { return reinterpret_cast<uint32_t*>(ws + off); };
  const dc::EmbedIds e = {ids, ids_i64 != 0, T, V, padding_idx};
  // Slice `i` of the launches that share the zero fill.
  const int launches = plan.rank ? 1 : 2 * plan.passes;
  const int64_t slice_bytes = round_up(ceil_div(table_bytes - head, launches), 16);
  auto slice = [&](int i) {
    const int64_t lo = std::min(table_bytes, head + i * slice_bytes), hi = std::min(table_bytes, lo + slice_bytes);
    dc::FillSlice f = {table + lo, hi - lo, 0};
    f.ctas = static_cast<int>(std::min<int64_t>(4 * 148, ceil_div(hi - lo, dc::kFillCta)));
    return f;
  };
  int cur = 0;
  if (plan.rank) {
    const dc::FillSlice fill = slice(0);
    const int ctas = static_cast<int>(ceil_div(T, dc::kRankItems));
    if (int status = launch("embedding_grad sort launch", dc::embed_rank_kernel, ctas + fill.ctas, 32 * dc::kRankWarps, 0, st, 0, e, u32(plan.keys[0]), u32(plan.idx[0]), ctas, fill)) return status;
  } else {
    const int tiles = static_cast<int>(plan.tiles);
    const unsigned threads = 32 * dc::kRadixWarps;
    for (int pass = 0; pass < plan.passes; ++pass) {
      const int shift = pass * plan.bits, out = pass & 1, in = out ^ 1;
      uint32_t* hist = u32(plan.hist);
      const dc::FillSlice f0 = slice(2 * pass), f1 = slice(2 * pass + 1);
      const unsigned g0 = tiles + f0.ctas, g1 = tiles + f1.ctas;
      // the first pass reads the ids, whatever the key arrays hold
      const auto count = pass == 0 ? dc::radix_hist_kernel<true> : dc::radix_hist_kernel<false>;
      const auto scatter = plan.scan ? (pass == 0 ? dc::radix_scatter_kernel<true, true> : dc::radix_scatter_kernel<false, true>)
                                     : (pass == 0 ? dc::radix_scatter_kernel<true, false> : dc::radix_scatter_kernel<false, false>);
      if ((r = launch("embedding_grad sort launch", count, g0, threads, 0, st, 0, e, u32(plan.keys[in]), hist, shift, plan.bits,
                      tiles, f0)))
        return r;
      if (plan.scan) {
        const int digits = 1 << plan.bits;
        if ((r = launch("embedding_grad sort launch", dc::radix_scan_kernel, static_cast<unsigned>(ceil_div(digits, 32)),
                        32 * dc::kScanWarps, 0, st, 0, hist, digits, tiles)))
          return r;
      }
      if ((r = launch("embedding_grad sort launch", scatter, g1, threads, 0, st, 0, e, u32(plan.keys[in]), u32(plan.idx[in]), hist,
                      u32(plan.keys[out]), u32(plan.idx[out]), shift, plan.bits, tiles, f1)))
        return r;
      cur = out;
    }
  }
  dc::EmbedSumParams p = {};
  p.skey = u32(plan.keys[cur]); p.sidx = u32(plan.idx[cur]);
  p.T = T; p.V = V; p.dy = dy; p.lddy = lddy; p.out = dtable; p.part = reinterpret_cast<float*>(ws + plan.part);
  p.D = static_cast<int>(D); p.chunk = static_cast<int>(plan.chunk); p.scale = scale;
  const int64_t n = 16 / static_cast<int64_t>(es);
  const bool vec = D % n == 0 && lddy % n == 0 && aligned(dy, 16) && aligned(dtable, 16);
  switch (dtype) {
    case DC_DTYPE_F32: return vec ? launch_embed_sum<float, 4>(p, plan.chunks, st) : launch_embed_sum<float, 1>(p, plan.chunks, st);
    case DC_DTYPE_F16: return vec ? launch_embed_sum<__half, 8>(p, plan.chunks, st) : launch_embed_sum<__half, 1>(p, plan.chunks, st);
    default: return vec ? launch_embed_sum<__nv_bfloat16, 8>(p, plan.chunks, st) : launch_embed_sum<__nv_bfloat16, 1>(p, plan.chunks, st);
  }
}

}  // extern "C"
