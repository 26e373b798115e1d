// Torch binding of the text operators: argument checks, outputs and workspaces from the caching
// allocator, the C entry points on the current stream of the tensors' device, and the autograd nodes.
// Native because an operator on a few tokens takes the GPU a few microseconds: the same steps in
// Python cost 10 to 15 us a call, and 60 us more for each backward node.
//
// Nothing here falls back to another implementation. A non-zero status of the library is raised with
// its message.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <initializer_list>
#include <string>
#include <utility>

#include "../../include/diffucore_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
template <typename... A>
std::string cat(const A&... a) { return c10::str(a...); }
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

void check(int status) {
  if (status != DC_OK) throw std::runtime_error(std::string("diffucore_b200: ") + dc_last_error());
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DC_DTYPE_F32;
    case at::kHalf: return DC_DTYPE_F16;
    case at::kBFloat16: return DC_DTYPE_BF16;
    default: return -1;
  }
}

using Named = std::pair<const char*, const OptTensor*>;

// A forward-mode tangent would not reach the result: the kernels see the primal values alone.
void refuse_tangent(const char* what, const Tensor& t) {
  if (t._fw_grad(0).defined())
    throw std::runtime_error(cat("diffucore_b200: ", what, " has no forward-mode derivative (an argument is a dual tensor); differentiate it in "
                                 "reverse mode"));
}
void refuse_tangents(const char* what, std::initializer_list<const OptTensor*> ts) {
  for (const OptTensor* t : ts)
    if (has(*t)) refuse_tangent(what, **t);
}

// dtype code of `lead`, a CUDA tensor in bf16 or fp16 (or fp32 where `floats`); the others share its
// type and device. No tensor carries a forward-mode tangent.
int check_text(const char* what, const Tensor& lead, bool floats, std::initializer_list<Named> others = {}) {
  refuse_tangent(what, lead);
  for (const Named& n : others)
    if (has(*n.second)) refuse_tangent(what, **n.second);
  if (!lead.is_cuda())
    throw std::runtime_error(cat("diffucore_b200 kernels run on CUDA tensors only (got a ", c10::DeviceTypeName(lead.device().type(), true),
                                 " tensor); there is no CPU path"));
  const int code = dtype_code(lead.scalar_type());
  if (code < 0 || (code == DC_DTYPE_F32 && !floats)) throw py::type_error(cat(what, ": unsupported dtype ", lead.scalar_type()));
  for (const Named& n : others) {
    const OptTensor& t = *n.second;
    if (has(t) && (t->scalar_type() != lead.scalar_type() || t->device() != lead.device()))
      throw py::type_error(cat(what, ": ", n.first, " is ", t->scalar_type(), " on ", t->device(), ", expected ",
                               lead.scalar_type(), " on ", lead.device()));
  }
  return code;
}

// The device of a call made current, and its current stream.
struct Launch {
  explicit Launch(const Tensor& t) : guard(t.device()), stream(at::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
  c10::cuda::CUDAGuard guard;
  void* stream;
};

// t with its values as they are in memory: a negated view (the imaginary part of a conjugate) is
// materialised, a zero tensor without memory too. Everything else is t itself.
Tensor plain(const Tensor& t) {
  if (!t.defined()) return t;
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}
OptTensor plain(const OptTensor& t) { return has(t) ? OptTensor(plain(*t)) : std::nullopt; }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const OptTensor& t) { return has(t) ? t->data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
Tensor workspace(const Tensor& like, size_t bytes) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}
int64_t pad(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
// Rows of the tensors that only the kernels see (kept pre-activations, dz) start on 64 bytes: rows on
// 16 split the kernels' 32-byte accesses over two sectors (6580 x 3291 x 256 with z kept 51.8 us,
// 75.2 on 16 bytes).
constexpr int64_t kZPad = 16, kDzPad = 32;

// Whether a TMA tile load takes the rows of t [R, C]: unit inner stride, 16-byte aligned rows that do
// not overlap.
bool tile_loadable(const Tensor& t) {
  return t.stride(1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         (t.size(0) == 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)));
}
// t itself, or a copy with padded rows.
Tensor matrix_operand(const Tensor& t) {
  if (tile_loadable(t)) return t;
  return at::empty({t.size(0), pad(t.size(1), 8)}, t.options()).narrow(1, 0, t.size(1)).copy_(t);
}
// Leading dimension of a matrix operand (any multiple of 8 will do for a single row).
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : pad(t.size(1), 8); }

// The same for a call's operands, in place; those that need padding are copied by one launch (a fourth
// by torch).
void matrix_operands(std::initializer_list<Tensor*> ts) {
  const void* src[3];
  void* dst[3];
  int64_t ld_src[3], rows[3], cols[3], ld_dst[3];
  int n = 0;
  Tensor lead;
  for (Tensor* t : ts) {
    if (!t->defined() || tile_loadable(*t)) continue;
    const bool same = !lead.defined() || lead.device() == t->device();
    if (!t->is_cuda() || t->element_size() != 2 || t->stride(1) != 1 || !same || n == 3) {
      *t = matrix_operand(*t);
      continue;
    }
    if (!lead.defined()) lead = *t;
    src[n] = t->data_ptr();
    ld_src[n] = t->size(0) > 1 ? t->stride(0) : t->size(1);
    rows[n] = t->size(0);
    cols[n] = t->size(1);
    ld_dst[n] = pad(cols[n], 8);
    Tensor copy = at::empty({rows[n], ld_dst[n]}, t->options());
    dst[n] = copy.data_ptr();
    *t = copy.narrow(1, 0, cols[n]);
    ++n;
  }
  if (n == 0) return;
  Launch at_(lead);
  check(dc_pad_rows(n, src, ld_src, rows, cols, dst, ld_dst, at_.stream));
}

constexpr int64_t kFewRows = 8;         // rows of x up to which the projections read any layout in place

// Forward operands for `rows` rows of x. DC_HGEMM_PAIR forces the tiled kernels.
void projection_operands(std::initializer_list<Tensor*> ts, int64_t rows) {
  bool in_place = rows <= kFewRows;
  for (const Tensor* t : ts) in_place = in_place && t->stride(1) == 1 && (t->size(0) == 1 || t->stride(0) >= t->size(1));
  if (in_place && getenv("DC_HGEMM_PAIR") == nullptr) return;
  matrix_operands(ts);
}

// t [R, C] with unit inner stride, and its row stride (one row: its width).
Tensor unit_rows(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

OptTensor vector_arg(const char* what, const char* name, const OptTensor& t, int64_t n) {
  if (!has(t)) return std::nullopt;
  if (t->dim() != 1 || t->size(0) != n)
    throw py::value_error(cat(what, ": ", name, " must have shape (", n, ",), got ", shape_of(*t)));
  return plain(*t).contiguous();
}

int64_t rows_of(const Tensor& t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  return n;
}
void check_width(const char* what, const Tensor& x, int64_t width) {
  if (x.dim() < 1 || x.size(-1) != width)
    throw py::value_error(cat(what, ": expected inputs of width ", width, ", got ", shape_of(x)));
}
Tensor flat(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({rows_of(t), t.size(-1)}); }
Tensor unflat(const Tensor& y, const Tensor& like, int64_t width) {
  if (like.dim() == 2) return y;
  std::vector<int64_t> s = like.sizes().vec();
  s.back() = width;
  return y.view(s);
}
bool wants_grad(std::initializer_list<const OptTensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor* t : ts)
    if (has(*t) && (*t)->requires_grad()) return true;
  return false;
}

// ------------------------------------------------------------------ operators on flat tensors

std::pair<Tensor, Tensor> linear_raw(const Tensor& x_, const Tensor& w_, const OptTensor& bias_, int act,
                                     const OptTensor& residual_, bool keep_z) {
  const OptTensor wo(w_);
  const int dt = check_text("linear", x_, false, {{"w", &wo}, {"bias", &bias_}, {"residual", &residual_}});
  if (x_.dim() != 2 || w_.dim() != 2 || x_.size(1) != w_.size(1))
    throw py::value_error(cat("linear: x ", shape_of(x_), " does not match w ", shape_of(w_)));
  const int64_t M = x_.size(0), K = x_.size(1), N = w_.size(0);
  const OptTensor bias = vector_arg("linear", "bias", bias_, N);
  Tensor residual;
  if (has(residual_)) {
    if (residual_->dim() != 2 || residual_->size(0) != M || residual_->size(1) != N)
      throw py::value_error(cat("linear: residual must have shape (", M, ", ", N, "), got ", shape_of(*residual_)));
    residual = unit_rows(plain(*residual_));
  }
  Launch at_(x_);
  Tensor x = plain(x_), w = plain(w_);
  projection_operands({&x, &w}, M);
  Tensor y = at::empty({M, N}, x.options()), z;
  if (keep_z) z = at::empty({M, pad(N, kZPad)}, x.options().dtype(at::kFloat));
  check(dc_linear(ptr(x), ld(x), ptr(w), ld(w), ptr(bias), ptr(residual), residual.defined() ? residual.stride(0) : 0, ptr(y), N,
                  fptr(z), keep_z ? z.size(1) : 0, dt, M, N, K, act, at_.stream));
  return {y, z};
}

std::tuple<Tensor, Tensor, Tensor> gated_raw(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const OptTensor& bg_,
                                             const OptTensor& bu_, int act, bool keep_z) {
  const OptTensor go(wg_), uo(wu_);
  const int dt = check_text("gated_linear", x_, false, {{"w_gate", &go}, {"w_up", &uo}, {"b_gate", &bg_}, {"b_up", &bu_}});
  if (x_.dim() != 2 || wg_.dim() != 2 || wg_.sizes() != wu_.sizes() || x_.size(1) != wg_.size(1))
    throw py::value_error(cat("gated_linear: shapes of x ", shape_of(x_), ", w_gate ", shape_of(wg_), " and w_up ", shape_of(wu_),
                              " do not match"));
  const int64_t M = x_.size(0), K = x_.size(1), N = wg_.size(0);
  const OptTensor bg = vector_arg("gated_linear", "b_gate", bg_, N), bu = vector_arg("gated_linear", "b_up", bu_, N);
  Launch at_(x_);
  Tensor x = plain(x_), wg = plain(wg_), wu = plain(wu_);
  projection_operands({&x, &wg, &wu}, M);
  Tensor h = at::empty({M, N}, x.options()), zg, zu;
  const int64_t ldz = pad(N, kZPad);
  if (keep_z) {
    zg = at::empty({M, ldz}, x.options().dtype(at::kFloat));
    zu = at::empty({M, ldz}, x.options().dtype(at::kFloat));
  }
  check(dc_gated_linear(ptr(x), ld(x), ptr(wg), ld(wg), ptr(wu), ld(wu), ptr(bg), ptr(bu), ptr(h), N, fptr(zg), fptr(zu), ldz, dt,
                        M, N, K, act, at_.stream));
  return {h, zg, zu};
}

struct ActGrad { Tensor dz, dz1, db, db1; };

// A kept pre-activation of dy [M, N]: fp32 rows whose memory holds N rounded up to 4 values, as the
// kernels read it.
void check_kept(const char* name, const Tensor& z, const Tensor& dy) {
  if (!z.defined()) return;
  if (z.scalar_type() != at::kFloat || z.device() != dy.device())
    throw py::type_error(cat("act_grad: ", name, " is ", z.scalar_type(), " on ", z.device(), ", expected fp32 on ", dy.device()));
  const int64_t M = dy.size(0), N = dy.size(1);
  if (z.dim() != 2 || z.size(0) != M || z.size(1) < N || (z.size(1) > 1 && z.stride(1) != 1) || z.is_neg() || z._is_zerotensor())
    throw py::value_error(cat("act_grad: ", name, " ", shape_of(z), " is not the kept pre-activation of dy ", shape_of(dy)));
  const int64_t room = static_cast<int64_t>(z.storage().nbytes() / sizeof(float)) - z.storage_offset();
  if (M > 0 && (M - 1) * z.stride(0) + pad(N, 4) > room)
    throw py::value_error(cat("act_grad: the rows of ", name, " must hold ", pad(N, 4), " values, ", N, " rounded up to 4"));
}

// dz (dy itself without z), dz1, db and db1 from dy and the kept pre-activations.
ActGrad act_grad_raw(const Tensor& dy_, const Tensor& z, const Tensor& z1, int act, bool bias, bool bias1) {
  check_text("act_grad", dy_, false);
  if (dy_.dim() != 2) throw py::value_error(cat("act_grad: dy must be [M, N], got ", shape_of(dy_)));
  if (z1.defined() && !z.defined()) throw py::value_error("act_grad: z1 goes with z");
  if (bias1 && !z1.defined()) throw py::value_error("act_grad: the second bias gradient needs z1");
  check_kept("z", z, dy_);
  check_kept("z1", z1, dy_);
  if (z1.defined() && z1.stride(0) != z.stride(0) && z.size(0) > 1)
    throw py::value_error("act_grad: z and z1 must have the same row stride");
  ActGrad g;
  if (!z.defined() && !bias) {
    g.dz = dy_;
    return g;
  }
  const int64_t M = dy_.size(0), N = dy_.size(1), lddz = pad(N, kDzPad);
  Launch at_(dy_);
  Tensor dy = unit_rows(plain(dy_));
  if (M > 1 && dy.stride(0) < N) dy = dy.contiguous();
  if (z.defined()) g.dz = at::empty({M, lddz}, dy.options()).narrow(1, 0, N);
  if (z1.defined()) g.dz1 = at::empty({M, lddz}, dy.options()).narrow(1, 0, N);
  Tensor ws;
  size_t bytes = 0;
  if (bias || bias1) {
    g.db = at::empty({N}, dy.options());
    if (bias1) g.db1 = at::empty({N}, dy.options());
    check(dc_act_grad_workspace(M, N, &bytes));
    ws = workspace(dy, bytes);
  }
  check(dc_act_grad(ptr(dy), row_stride(dy), fptr(z), fptr(z1), z.defined() ? z.stride(0) : 0, ptr(g.dz), ptr(g.dz1), lddz,
                    ptr(g.db), ptr(g.db1), ptr(ws), bytes, dtype_code(dy.scalar_type()), M, N, act, at_.stream));
  if (!z.defined()) g.dz = dy_;
  return g;
}

// dz and w (or x) of a backward product, and dz's twin: 2-D tensors of one type on one device.
void check_product(const char* what, const Tensor& dz, const char* name, const Tensor& t, const Tensor& dz1) {
  const OptTensor to(t), d1(dz1);
  check_text(what, dz, false, {{name, &to}, {"dz1", &d1}});
  if (dz.dim() != 2 || t.dim() != 2) throw py::value_error(cat(what, ": dz ", shape_of(dz), " and ", name, " ", shape_of(t), " must be matrices"));
  if (dz1.defined() && dz1.sizes() != dz.sizes()) throw py::value_error(cat(what, ": dz1 ", shape_of(dz1), " does not match dz ", shape_of(dz)));
}
// dz and dz1 as matrix operands with one leading dimension.
void same_rows(Tensor& dz, Tensor& dz1) {
  if (!dz1.defined() || ld(dz) == ld(dz1)) return;
  for (Tensor* t : {&dz, &dz1}) *t = at::empty({t->size(0), pad(t->size(1), 8)}, t->options()).narrow(1, 0, t->size(1)).copy_(*t);
}

Tensor linear_dx_raw(const Tensor& dz_, const Tensor& w_, const Tensor& dz1_, const Tensor& w1_) {
  check_product("linear_dx", dz_, "w", w_, dz1_);
  if (dz1_.defined() != w1_.defined()) throw py::value_error("linear_dx: dz1 and w1 go together");
  if (w1_.defined()) {
    check_product("linear_dx", dz_, "w1", w1_, dz1_);
    if (w1_.sizes() != w_.sizes()) throw py::value_error(cat("linear_dx: w1 ", shape_of(w1_), " does not match w ", shape_of(w_)));
  }
  if (dz_.size(1) != w_.size(0)) throw py::value_error(cat("linear_dx: dz ", shape_of(dz_), " does not match w ", shape_of(w_)));
  Launch at_(dz_);
  Tensor dz = plain(dz_), w = plain(w_), dz1 = plain(dz1_), w1 = plain(w1_);
  matrix_operands({&dz, &w, &dz1, &w1});
  same_rows(dz, dz1);
  const int64_t M = dz.size(0), N = dz.size(1), K = w.size(1);
  Tensor dx = at::empty({M, K}, dz.options());
  check(dc_linear_dx(ptr(dz), ptr(dz1), ld(dz), ptr(w), ld(w), ptr(w1), w1.defined() ? ld(w1) : 0, ptr(dx), K,
                     dtype_code(dz.scalar_type()), M, N, K, at_.stream));
  return dx;
}

std::pair<Tensor, Tensor> linear_dw_raw(const Tensor& dz_, const Tensor& x_, const Tensor& dz1_) {
  check_product("linear_dw", dz_, "x", x_, dz1_);
  if (dz_.size(0) != x_.size(0)) throw py::value_error(cat("linear_dw: dz ", shape_of(dz_), " does not match x ", shape_of(x_)));
  Launch at_(dz_);
  Tensor dz = plain(dz_), x = plain(x_), dz1 = plain(dz1_);
  matrix_operands({&dz, &x, &dz1});
  same_rows(dz, dz1);
  const int64_t M = dz.size(0), N = dz.size(1), K = x.size(1);
  Tensor dw = at::empty({N, K}, x.options()), dw1;
  if (dz1.defined()) dw1 = at::empty({N, K}, x.options());
  check(dc_linear_dw(ptr(dz), ptr(dz1), ld(dz), ptr(x), ld(x), ptr(dw), ptr(dw1), K, dtype_code(dz.scalar_type()), M, N, K,
                     at_.stream));
  return {dw, dw1};
}

// The affine vectors in one type the kernels take.
at::ScalarType norm_affine(const char* what, const Tensor& x, OptTensor& w, OptTensor& b) {
  const int64_t D = x.size(-1);
  std::optional<at::ScalarType> kind;
  for (auto& [name, t] : {std::pair<const char*, OptTensor*>{"weight", &w}, {"bias", &b}}) {
    if (!has(*t)) continue;
    refuse_tangent(what, **t);
    if ((*t)->device() != x.device() || ((*t)->scalar_type() != x.scalar_type() && (*t)->scalar_type() != at::kFloat))
      throw py::type_error(cat(what, ": ", name, " is ", (*t)->scalar_type(), " on ", (*t)->device(), ", expected ",
                               x.scalar_type(), " or fp32 on ", x.device()));
    if ((*t)->dim() != 1 || (*t)->size(0) != D)
      throw py::value_error(cat(what, ": ", name, " must have shape (", D, ",), got ", shape_of(**t)));
    kind = !kind || *kind == (*t)->scalar_type() ? (*t)->scalar_type() : at::kFloat;
  }
  const at::ScalarType k = kind.value_or(x.scalar_type());
  if (has(w)) w = plain(*w).to(k).contiguous();
  if (has(b)) b = plain(*b).to(k).contiguous();
  return k;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_raw(const Tensor& x_, OptTensor w, OptTensor b, double eps, bool keep_stats) {
  const int dt = check_text("layer_norm", x_, true);
  if (x_.dim() != 2) throw py::value_error(cat("layer_norm: x must be [M, D], got ", shape_of(x_)));
  Launch at_(x_);
  const at::ScalarType kind = norm_affine("layer_norm", x_, w, b);
  const Tensor x = unit_rows(plain(x_));
  const int64_t M = x.size(0), D = x.size(1);
  Tensor y = at::empty({M, D}, x.options()), mean, rstd;
  if (keep_stats) {
    mean = at::empty({M}, x.options().dtype(at::kFloat));
    rstd = at::empty({M}, x.options().dtype(at::kFloat));
  }
  check(dc_layer_norm(ptr(x), row_stride(x), ptr(w), ptr(b), dtype_code(kind), ptr(y), D, fptr(mean), fptr(rstd), dt, M, D,
                      static_cast<float>(eps), at_.stream));
  return {y, mean, rstd};
}

// A row statistic [M] that layer_norm_raw kept.
Tensor kept_stat(const char* name, const Tensor& t, const Tensor& x) {
  if (t.scalar_type() != at::kFloat || t.device() != x.device())
    throw py::type_error(cat("layer_norm_grad: ", name, " is ", t.scalar_type(), " on ", t.device(), ", expected fp32 on ", x.device()));
  if (t.dim() != 1 || t.size(0) != x.size(0))
    throw py::value_error(cat("layer_norm_grad: ", name, " must have shape (", x.size(0), ",), got ", shape_of(t)));
  return plain(t).contiguous();
}

// dw and db come in `kind` (x's type or fp32), computed in fp32 where w is fp32.
std::tuple<Tensor, Tensor, Tensor> layer_norm_grad_raw(const Tensor& dy_, const Tensor& x_, const OptTensor& w_, const Tensor& mean_,
                                                       const Tensor& rstd_, bool weight, bool bias, at::ScalarType kind) {
  const OptTensor xo(x_);
  const int dt = check_text("layer_norm_grad", dy_, true, {{"x", &xo}});
  if (x_.dim() != 2 || dy_.sizes() != x_.sizes())
    throw py::value_error(cat("layer_norm_grad: dy ", shape_of(dy_), " does not match x ", shape_of(x_), ", [M, D]"));
  Launch at_(x_);
  OptTensor w = w_, none;
  at::ScalarType sums = norm_affine("layer_norm_grad", x_, w, none);
  if (kind != x_.scalar_type() && kind != at::kFloat)
    throw py::type_error(cat("layer_norm_grad: gradients in ", kind, ", expected ", x_.scalar_type(), " or fp32"));
  if (kind == at::kFloat) sums = kind;
  if (has(w)) w = w->to(sums);
  const Tensor mean = kept_stat("mean", mean_, x_), rstd = kept_stat("rstd", rstd_, x_);
  const Tensor dy = unit_rows(plain(dy_)), x = unit_rows(plain(x_));
  const int64_t M = x.size(0), D = x.size(1);
  Tensor dx = at::empty({M, D}, x.options()), dw, db, ws;
  size_t bytes = 0;
  if (weight || bias) {
    dw = at::empty({D}, x.options().dtype(sums));
    if (bias) db = at::empty({D}, x.options().dtype(sums));
    check(dc_layer_norm_grad_workspace(M, D, &bytes));
    ws = workspace(x, bytes);
  }
  check(dc_layer_norm_grad(ptr(dy), row_stride(dy), ptr(x), row_stride(x), ptr(w), dtype_code(sums), fptr(mean), fptr(rstd), ptr(dx),
                           D, ptr(dw), ptr(db), ptr(ws), bytes, dt, M, D, at_.stream));
  dw = weight ? dw.to(kind) : Tensor();
  if (bias) db = db.to(kind);
  return {dx, dw, db};
}

// Flat contiguous ids.
Tensor check_ids(const char* what, const Tensor& ids, const Tensor& like) {
  if ((ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt) || ids.device() != like.device())
    throw py::type_error(cat(what, ": ids must be int64 or int32 on ", like.device(), ", got ", ids.scalar_type(), " on ", ids.device()));
  return plain(ids.dim() == 1 ? ids : ids.reshape({-1})).contiguous();
}

Tensor embedding_raw(const Tensor& ids_, const Tensor& table_, double scale) {
  const int dt = check_text("embedding", table_, true);
  if (table_.dim() != 2) throw py::value_error(cat("embedding: table must be [V, D], got ", shape_of(table_)));
  const Tensor ids = check_ids("embedding", ids_, table_);
  Launch at_(table_);
  const int64_t V = table_.size(0), D = table_.size(1), T = ids.size(0);
  Tensor table = unit_rows(plain(table_));
  if (V > 1 && table.stride(0) < D) table = table.contiguous();
  Tensor out = at::empty({T, D}, table.options());
  check(dc_embedding(ptr(ids), ids.scalar_type() == at::kLong, T, ptr(table), row_stride(table), V, D, static_cast<float>(scale),
                     ptr(out), D, dt, at_.stream));
  return out;
}

Tensor embedding_grad_raw(const Tensor& dy_, const Tensor& ids_, int64_t V, double scale, int64_t padding) {
  const int dt = check_text("embedding_grad", dy_, true);
  if (dy_.dim() != 2) throw py::value_error(cat("embedding_grad: dy must be [T, D], got ", shape_of(dy_)));
  const Tensor ids = check_ids("embedding_grad", ids_, dy_);
  const int64_t T = dy_.size(0), D = dy_.size(1);
  if (ids.size(0) != T) throw py::value_error(cat("embedding_grad: ", ids.size(0), " ids for ", T, " rows"));
  Launch at_(dy_);
  const Tensor dy = unit_rows(plain(dy_));
  size_t bytes = 0;
  check(dc_embedding_grad_workspace(T, V, D, &bytes));
  const Tensor ws = workspace(dy, bytes);
  Tensor out = at::empty({V, D}, dy.options());
  check(dc_embedding_grad(ptr(dy), row_stride(dy), ptr(ids), ids.scalar_type() == at::kLong, T, V, D, padding,
                          static_cast<float>(scale), ptr(out), ptr(ws), bytes, dt, at_.stream));
  return out;
}

// ------------------------------------------------------------------ autograd

// Gradients of a node run under create_graph: usable, but differentiating them again is an error. The
// node that raises it hangs on the inputs of the differentiated node and on its incoming gradient `dy`,
// so the engine comes through it wherever a second derivative would go, also for a loss that reaches the
// same input by another way.
variable_list grads_once(bool create_graph, const Tensor& dy, variable_list grads) {
  if (!create_graph) return grads;
  torch::autograd::edge_list edges = torch::autograd::get_current_node()->next_edges();
  if (dy.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(dy));
  const auto node = std::make_shared<torch::autograd::Error>("a diffucore_b200 text operator cannot be differentiated twice",
                                                             std::move(edges));
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    g = g.detach();
    torch::autograd::set_history(g, node);
  }
  return grads;
}

// Which of the node's inputs want a gradient. Absent optional inputs have no edge.
struct Wants {
  Wants(AutogradContext* ctx, std::initializer_list<bool> present) {
    size_t edge = 0, i = 0;
    for (bool p : present) want[i++] = p && ctx->needs_input_grad(edge++);
  }
  bool operator[](size_t i) const { return want[i]; }
  bool want[8] = {};
};

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const OptTensor& bias, const OptTensor& residual,
                        int64_t act) {
    Tensor x = plain(x_), w = plain(w_);
    matrix_operands({&x, &w});                                       // padded once for both passes
    const bool keep = act != DC_ACT_NONE && (x_.requires_grad() || w_.requires_grad() || (has(bias) && bias->requires_grad()));
    auto [y, z] = linear_raw(x, w, bias, static_cast<int>(act), residual, keep);
    ctx->save_for_backward({x, w, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = has(bias);
    ctx->saved_data["residual"] = has(residual);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool create = at::GradMode::is_enabled();
    at::AutoGradMode off(false);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &z = saved[2], &dy = grads[0];
    const Wants want(ctx, {true, true, ctx->saved_data["bias"].toBool(), ctx->saved_data["residual"].toBool()});
    Tensor dx, dw, db;
    if (dy.size(0) == 0) {
      if (want[0]) dx = at::zeros(x.sizes(), x.options());
      if (want[1]) dw = at::zeros(w.sizes(), w.options());
      if (want[2]) db = at::zeros({w.size(0)}, w.options());
    } else if (want[0] || want[1] || want[2]) {
      const ActGrad g = act_grad_raw(dy, z, Tensor(), static_cast<int>(ctx->saved_data["act"].toInt()), want[2], false);
      db = g.db;
      if (want[0] || want[1]) {
        Tensor dz = plain(g.dz);
        matrix_operands({&dz});
        if (want[0]) dx = linear_dx_raw(dz, w, Tensor(), Tensor());
        if (want[1]) dw = linear_dw_raw(dz, x, Tensor()).first;
      }
    }
    return grads_once(create, dy, {dx, dw, db, want[3] ? plain(dy) : Tensor(), Tensor()});
  }
};

struct GatedNode : torch::autograd::Function<GatedNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const OptTensor& bg,
                        const OptTensor& bu, int64_t act) {
    Tensor x = plain(x_), wg = plain(wg_), wu = plain(wu_);
    matrix_operands({&x, &wg, &wu});
    auto [h, zg, zu] = gated_raw(x, wg, wu, bg, bu, static_cast<int>(act), true);
    ctx->save_for_backward({x, wg, wu, zg, zu});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bg"] = has(bg);
    ctx->saved_data["bu"] = has(bu);
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool create = at::GradMode::is_enabled();
    at::AutoGradMode off(false);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &dh = grads[0];
    const Wants want(ctx, {true, true, true, ctx->saved_data["bg"].toBool(), ctx->saved_data["bu"].toBool()});
    Tensor dx, dwg, dwu, dbg, dbu;
    if (dh.size(0) == 0) {
      if (want[0]) dx = at::zeros(x.sizes(), x.options());
      if (want[1]) dwg = at::zeros(wg.sizes(), wg.options());
      if (want[2]) dwu = at::zeros(wu.sizes(), wu.options());
      if (want[3]) dbg = at::zeros({wg.size(0)}, wg.options());
      if (want[4]) dbu = at::zeros({wg.size(0)}, wg.options());
    } else {
      const ActGrad g = act_grad_raw(dh, saved[3], saved[4], static_cast<int>(ctx->saved_data["act"].toInt()), want[3] || want[4],
                                     want[4]);
      if (want[3]) dbg = g.db;
      dbu = g.db1;
      if (want[0]) dx = linear_dx_raw(g.dz, wg, g.dz1, wu);
      if (want[1] && want[2]) std::tie(dwg, dwu) = linear_dw_raw(g.dz, x, g.dz1);
      else if (want[1]) dwg = linear_dw_raw(g.dz, x, Tensor()).first;
      else if (want[2]) dwu = linear_dw_raw(g.dz1, x, Tensor()).first;
    }
    return grads_once(create, dh, {dx, dwg, dwu, dbg, dbu, Tensor()});
  }
};

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    auto [y, mean, rstd] = layer_norm_raw(x, w, b, eps, true);
    ctx->save_for_backward({x, has(w) ? *w : Tensor(), mean, rstd});
    ctx->saved_data["w"] = has(w) ? static_cast<int64_t>(w->scalar_type()) : -1;
    ctx->saved_data["b"] = has(b) ? static_cast<int64_t>(b->scalar_type()) : -1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool create = at::GradMode::is_enabled();
    at::AutoGradMode off(false);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &dy = grads[0];
    const int64_t wk = ctx->saved_data["w"].toInt(), bk = ctx->saved_data["b"].toInt();
    const Wants want(ctx, {true, wk >= 0, bk >= 0});
    Tensor dx, dw, db;
    if (dy.size(0) == 0) {
      const int64_t D = x.size(1);
      dx = at::zeros(x.sizes(), x.options());
      if (want[1]) dw = at::zeros({D}, x.options().dtype(static_cast<at::ScalarType>(wk)));
      if (want[2]) db = at::zeros({D}, x.options().dtype(static_cast<at::ScalarType>(bk)));
    } else {
      // both sums in one type: fp32 when either vector is
      const int64_t f32 = static_cast<int64_t>(at::kFloat);
      const at::ScalarType kind = wk == f32 || bk == f32 ? at::kFloat : x.scalar_type();
      std::tie(dx, dw, db) = layer_norm_grad_raw(dy, x, w.defined() ? OptTensor(w) : std::nullopt, saved[2], saved[3], want[1],
                                                 want[2], kind);
      if (want[1]) dw = dw.to(static_cast<at::ScalarType>(wk));
      if (want[2]) db = db.to(static_cast<at::ScalarType>(bk));
    }
    return grads_once(create, dy, {dx, dw, db, Tensor()});
  }
};

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embedding_raw(ids, table, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool create = at::GradMode::is_enabled();
    at::AutoGradMode off(false);
    const Tensor d = embedding_grad_raw(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                                        ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt());
    return grads_once(create, grads[0], {Tensor(), d, Tensor(), Tensor()});
  }
};

// ------------------------------------------------------------------ public functions

Tensor linear(const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t act, const OptTensor& residual) {
  if (w.dim() != 2) throw py::value_error(cat("linear: weight must be [N, K], got ", shape_of(w)));
  check_width("linear", x, w.size(1));
  const int64_t N = w.size(0);
  OptTensor res;
  if (has(residual)) {
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = N;
    if (residual->sizes() != at::IntArrayRef(s))
      throw py::value_error(cat("linear: residual must have shape ", at::IntArrayRef(s), ", got ", shape_of(*residual)));
    res = flat(*residual);
  }
  const OptTensor xo(x), wo(w);
  refuse_tangents("linear", {&xo, &wo, &bias, &residual});
  const Tensor x2 = flat(x);
  const Tensor y = wants_grad({&xo, &wo, &bias, &residual})
                       ? LinearNode::apply(x2, w, bias, res, act)
                       : linear_raw(x2, w, bias, static_cast<int>(act), res, false).first;
  return unflat(y, x, N);
}

Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptTensor& bg, const OptTensor& bu, int64_t act) {
  if (wg.dim() != 2) throw py::value_error(cat("gated_linear: w_gate must be [N, K], got ", shape_of(wg)));
  check_width("gated_linear", x, wg.size(1));
  const OptTensor xo(x), go(wg), uo(wu);
  refuse_tangents("gated_linear", {&xo, &go, &uo, &bg, &bu});
  const Tensor x2 = flat(x);
  const Tensor h = wants_grad({&xo, &go, &uo, &bg, &bu})
                       ? GatedNode::apply(x2, wg, wu, bg, bu, act)
                       : std::get<0>(gated_raw(x2, wg, wu, bg, bu, static_cast<int>(act), false));
  return unflat(h, x, wg.size(0));
}

Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  if (x.dim() < 1) throw py::value_error("layer_norm: expected at least one dimension");
  const OptTensor xo(x);
  refuse_tangents("layer_norm", {&xo, &w, &b});
  const Tensor x2 = flat(x);
  const Tensor y = wants_grad({&xo, &w, &b}) ? LayerNormNode::apply(x2, w, b, eps) : std::get<0>(layer_norm_raw(x2, w, b, eps, false));
  return unflat(y, x, x.size(-1));
}

Tensor embedding(const Tensor& ids, const Tensor& table, double scale, std::optional<int64_t> padding) {
  if (table.dim() != 2) throw py::value_error(cat("embedding: table must be [V, D], got ", shape_of(table)));
  const int64_t V = table.size(0);
  int64_t pad_id = -1;
  if (padding) {
    if (*padding < -V || *padding >= V)
      throw py::value_error(cat("embedding: padding_idx ", *padding, " outside a table of ", V, " rows"));
    pad_id = *padding < 0 ? *padding + V : *padding;
  }
  const OptTensor to(table);
  refuse_tangents("embedding", {&to});
  const Tensor flat_ids = ids.dim() == 1 ? ids : ids.reshape({-1});
  const Tensor y = wants_grad({&to}) ? EmbeddingNode::apply(flat_ids, table, scale, pad_id) : embedding_raw(flat_ids, table, scale);
  if (ids.dim() == 1) return y;
  std::vector<int64_t> s = ids.sizes().vec();
  s.push_back(table.size(1));
  return y.view(s);
}

Tensor or_none(const OptTensor& t) { return has(t) ? *t : Tensor(); }
py::object none_if_undefined(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

}  // namespace

PYBIND11_MODULE(_text_ext, m) {
  using Free = py::call_guard<py::gil_scoped_release>;
  m.def("linear", &linear, Free());
  m.def("gated_linear", &gated_linear, Free());
  m.def("layer_norm", &layer_norm, Free());
  m.def("embedding", &embedding, Free());
  m.def("matrix_operand", [](Tensor t) {
    if (t.dim() != 2) throw py::value_error(cat("matrix_operand: expected a matrix, got ", shape_of(t)));
    t = plain(t);
    matrix_operands({&t});
    return t;
  });
  m.def("linear_raw", [](const Tensor& x, const Tensor& w, const OptTensor& b, int act, const OptTensor& r, bool keep) {
    auto [y, z] = linear_raw(x, w, b, act, r, keep);
    return py::make_tuple(y, none_if_undefined(z));
  });
  m.def("gated_linear_raw", [](const Tensor& x, const Tensor& wg, const Tensor& wu, const OptTensor& bg, const OptTensor& bu, int act,
                               bool keep) {
    auto [h, zg, zu] = gated_raw(x, wg, wu, bg, bu, act, keep);
    return py::make_tuple(h, none_if_undefined(zg), none_if_undefined(zu));
  });
  m.def("act_grad_raw", [](const Tensor& dy, const OptTensor& z, const OptTensor& z1, int act, bool bias, bool bias1) {
    const ActGrad g = act_grad_raw(dy, or_none(z), or_none(z1), act, bias, bias1);
    return py::make_tuple(g.dz, none_if_undefined(g.dz1), none_if_undefined(g.db), none_if_undefined(g.db1));
  });
  m.def("linear_dx_raw", [](const Tensor& dz, const Tensor& w, const OptTensor& dz1, const OptTensor& w1) {
    return linear_dx_raw(dz, w, or_none(dz1), or_none(w1));
  });
  m.def("linear_dw_raw", [](const Tensor& dz, const Tensor& x, const OptTensor& dz1) {
    auto [dw, dw1] = linear_dw_raw(dz, x, or_none(dz1));
    return py::make_tuple(dw, none_if_undefined(dw1));
  });
  m.def("layer_norm_raw", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, bool keep) {
    auto [y, mean, rstd] = layer_norm_raw(x, w, b, eps, keep);
    return py::make_tuple(y, none_if_undefined(mean), none_if_undefined(rstd));
  });
  m.def("layer_norm_grad_raw", [](const Tensor& dy, const Tensor& x, const OptTensor& w, const Tensor& mean, const Tensor& rstd,
                                  bool weight, bool bias, at::ScalarType kind) {
    auto [dx, dw, db] = layer_norm_grad_raw(dy, x, w, mean, rstd, weight, bias, kind);
    return py::make_tuple(dx, none_if_undefined(dw), none_if_undefined(db));
  });
  m.def("embedding_raw", &embedding_raw);
  m.def("embedding_grad_raw", &embedding_grad_raw);
}
