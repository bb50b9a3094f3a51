// torch.library registration of the layer norm, the 8-bit activation checkpoints and the linear layer
// that keeps one (layer_norm_*.hip, ckpt8.hip, linear_ckpt8_*.hip).  The two differentiable ones have their
// autograd node here, not in Python: a training step of a small layer is bound by the host, and the
// Python nodes cost 30 us of the 125 us that forward and backward of 32 x 256 x 256 took.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <limits>
#include <utility>

#include "rtseg_launch.h"
#include "rtseg_ops.h"

namespace rtseg {
namespace {

constexpr int64_t kBlock = 32;
constexpr int64_t kMaxChannels = 1 << 20;  // the kernels' tile counts along channels are grid.y / int
int64_t padded(int64_t c) { return (c + kBlock - 1) / kBlock * kBlock; }

bool float_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
bool float_type(const at::Tensor& t) { return float_type(t.scalar_type()); }
int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }

// contiguous fp32 / bf16 / fp16 [rows, C] on the GPU
void check_rows(const at::Tensor& t, const char* op, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.is_contiguous() && float_type(t), "rtseg.", op, ": ", what,
              " must be a contiguous [rows, channels] fp32/bf16/fp16 GPU tensor");
  TORCH_CHECK(t.size(1) >= 1 && t.size(1) <= kMaxChannels, "rtseg.", op, ": ", what, " needs 1 .. ", kMaxChannels,
              " channels, got ", t.size(1));
  TORCH_CHECK(t.size(0) < std::numeric_limits<int>::max(), "rtseg.", op, ": too many rows (", t.size(0), ")");
}

void check_ckpt(const at::Tensor& codes, const at::Tensor& scales, int64_t rows, int64_t C, const at::Tensor& like,
                const char* op) {
  const int64_t Cp = padded(C);
  TORCH_CHECK(codes.is_cuda() && codes.device() == like.device() && codes.scalar_type() == at::kChar &&
                  codes.is_contiguous() && codes.dim() == 2 && codes.size(0) == rows && codes.size(1) == Cp,
              "rtseg.", op, ": codes must be contiguous int8 [", rows, ", ", Cp, "] on the same GPU");
  TORCH_CHECK(scales.is_cuda() && scales.device() == like.device() && scales.scalar_type() == at::kByte &&
                  scales.is_contiguous() && scales.dim() == 2 && scales.size(0) == rows && scales.size(1) == Cp / kBlock,
              "rtseg.", op, ": scales must be contiguous uint8 [", rows, ", ", Cp / kBlock, "] on the same GPU");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0, "rtseg.", op, ": codes must be 16-byte aligned");
}

std::pair<at::Tensor, at::Tensor> new_ckpt(int64_t rows, int64_t C, const at::Tensor& like) {
  const int64_t Cp = padded(C);
  return {at::empty({rows, Cp}, like.options().dtype(at::kChar)),
          at::empty({rows, Cp / kBlock}, like.options().dtype(at::kByte))};
}

// a weight or bias vector / matrix: x's type or fp32, contiguous, on x's device
void check_param(const at::Tensor& t, at::IntArrayRef sizes, const at::Tensor& like, const char* op, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.is_contiguous() && t.sizes() == sizes &&
                  (t.scalar_type() == like.scalar_type() || t.scalar_type() == at::kFloat),
              "rtseg.", op, ": ", what, " must be a contiguous ", sizes, " tensor of the input's type or fp32 on its device");
}

const void* opt_ptr(const std::optional<at::Tensor>& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

// ------------------------------ 8-bit checkpoints -------------------------------
std::tuple<at::Tensor, at::Tensor> ckpt8_pack(const at::Tensor& x) {
  check_rows(x, "ckpt8_pack", "x");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto [codes, scales] = new_ckpt(x.size(0), x.size(1), x);
  launch_ckpt8_pack(x.data_ptr(), dtype_code(x), codes.data_ptr<int8_t>(), scales.data_ptr<uint8_t>(), x.size(0),
                    static_cast<int>(x.size(1)), cur_stream());
  return {codes, scales};
}

// held: the type of the tensor that was packed
at::Tensor ckpt8_unpack(const at::Tensor& codes, const at::Tensor& scales, int64_t C, at::ScalarType dtype, at::ScalarType held) {
  TORCH_CHECK(codes.dim() == 2 && C >= 1 && C <= kMaxChannels,
              "rtseg.ckpt8_unpack: codes must be [rows, padded channels] with 1 .. ", kMaxChannels, " channels");
  TORCH_CHECK(codes.size(0) < std::numeric_limits<int>::max(), "rtseg.ckpt8_unpack: too many rows");
  check_ckpt(codes, scales, codes.size(0), C, codes, "ckpt8_unpack");
  for (const at::ScalarType t : {dtype, held})
    TORCH_CHECK(float_type(t), "rtseg.ckpt8_unpack: fp32, bf16 or fp16 expected, got ", t);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
  at::Tensor x = at::empty({codes.size(0), C}, codes.options().dtype(dtype));
  launch_ckpt8_unpack(codes.data_ptr<int8_t>(), scales.data_ptr<uint8_t>(), x.data_ptr(), dtype_code(x), type_code(held),
                      x.size(0), static_cast<int>(C), cur_stream());
  return x;
}

// ------------------------------ layer norm --------------------------------------
void check_ln_types(int x, int y, const char* op) {
  TORCH_CHECK(y == x || y == 0 || x == 0, "rtseg.", op, ": the output is of the input's type, fp32, or 16 bits behind fp32");
}

// keep: 0 nothing, 1 mean / rstd ([2, rows]), 2 those and the 8-bit checkpoint.  -> (sum or empty, y, stats, codes,
// scales), the first two of `shape` (x's rows as the caller has them: a result that is a view could not be changed in place)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> layer_norm_fwd(
    const at::Tensor& x, const std::optional<at::Tensor>& r, const std::optional<at::Tensor>& w,
    const std::optional<at::Tensor>& b, double eps, at::ScalarType out, int64_t keep, bool want_sum, at::IntArrayRef shape) {
  check_rows(x, "layer_norm", "x");
  const int64_t rows = x.size(0), C = x.size(1);
  TORCH_CHECK(C <= layer_norm_max_channels(), "rtseg.layer_norm: at most ", layer_norm_max_channels(), " channels");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  LnFwdArgs a{};
  a.x = x.data_ptr();
  a.x_dtype = dtype_code(x);
  at::Tensor s, y = at::empty(shape, x.options().dtype(out));
  a.y = y.data_ptr();
  a.y_dtype = dtype_code(y);
  check_ln_types(a.x_dtype, a.y_dtype, "layer_norm");
  if (r.has_value()) {
    check_rows(*r, "layer_norm", "residual");
    TORCH_CHECK(r->sizes() == x.sizes() && r->device() == x.device(), "rtseg.layer_norm: residual must match x");
    a.r = r->data_ptr();
    a.r_dtype = dtype_code(*r);
    TORCH_CHECK(a.r_dtype == a.x_dtype || a.x_dtype == 0,
                "rtseg.layer_norm: residual must be of x's type, or 16 bits beside an fp32 x");
    if (want_sum) {
      s = at::empty(shape, x.options());
      a.s = s.data_ptr();
    }
  }
  for (const auto* p : {&w, &b})
    if (p->has_value())
      TORCH_CHECK((*p)->is_cuda() && (*p)->device() == x.device() && (*p)->scalar_type() == at::kFloat &&
                      (*p)->is_contiguous() && (*p)->dim() == 1 && (*p)->size(0) == C,
                  "rtseg.layer_norm: weight and bias must be contiguous fp32 [", C, "] on x's device");
  a.w = static_cast<const float*>(opt_ptr(w));
  a.b = static_cast<const float*>(opt_ptr(b));
  at::Tensor stats, codes, scales;
  if (keep > 0) {
    stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    a.mean = stats.data_ptr<float>();
    a.rstd = a.mean + rows;
  }
  if (keep > 1) {
    std::tie(codes, scales) = new_ckpt(rows, C, x);
    a.codes = codes.data_ptr<int8_t>();
    a.scales = scales.data_ptr<uint8_t>();
  }
  a.rows = rows;
  a.C = static_cast<int>(C);
  a.Cp = padded(C);
  a.eps = static_cast<float>(eps);
  launch_layer_norm_fwd(a, cur_stream());
  return {s, y, stats, codes, scales};
}

// -> (dx or empty, dr, dw, db or empty).  dr is written only where the branch's type is not the
// stream's: where it is, its gradient is dx.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> layer_norm_bwd(
    const at::Tensor& dy, const std::optional<at::Tensor>& ds, const std::optional<at::Tensor>& x,
    const std::optional<at::Tensor>& codes, const std::optional<at::Tensor>& scales, const at::Tensor& stats,
    const std::optional<at::Tensor>& w, at::ScalarType x_dtype,
    std::optional<at::ScalarType> r_dtype, bool want_dx, bool want_dr, bool want_w) {
  check_rows(dy, "layer_norm_bwd", "grad");
  const int64_t rows = dy.size(0), C = dy.size(1);
  TORCH_CHECK(C <= layer_norm_max_channels(), "rtseg.layer_norm_bwd: at most ", layer_norm_max_channels(), " channels");
  TORCH_CHECK(x.has_value() != (codes.has_value() && scales.has_value()),
              "rtseg.layer_norm_bwd: one of the normalised tensor and its checkpoint");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  LnBwdArgs a{};
  const at::TensorOptions opt = dy.options();
  at::Tensor dx = at::empty({want_dx ? rows : 0, C}, opt.dtype(x_dtype));
  a.x_dtype = dtype_code(dx);
  a.y_dtype = dtype_code(dy);
  check_ln_types(a.x_dtype, a.y_dtype, "layer_norm_bwd");
  a.dy = dy.data_ptr();
  if (x.has_value()) {
    check_rows(*x, "layer_norm_bwd", "x");
    TORCH_CHECK(x->sizes() == dy.sizes() && x->device() == dy.device() && x->scalar_type() == x_dtype,
                "rtseg.layer_norm_bwd: x must match the gradient");
    a.x = x->data_ptr();
  } else {
    check_ckpt(*codes, *scales, rows, C, dy, "layer_norm_bwd");
    a.codes = codes->data_ptr<int8_t>();
    a.scales = scales->data_ptr<uint8_t>();
  }
  if (ds.has_value()) {
    check_rows(*ds, "layer_norm_bwd", "gradient of the sum");
    TORCH_CHECK(ds->sizes() == dy.sizes() && ds->device() == dy.device() && ds->scalar_type() == x_dtype,
                "rtseg.layer_norm_bwd: the gradient of the sum must be of the sum's shape and type");
    a.ds = ds->data_ptr();
  }
  TORCH_CHECK(stats.is_cuda() && stats.device() == dy.device() && stats.scalar_type() == at::kFloat &&
                  stats.is_contiguous() && stats.numel() == 2 * rows,
              "rtseg.layer_norm_bwd: mean and rstd must be contiguous fp32 [2, rows]");
  a.mean = stats.data_ptr<float>();
  a.rstd = a.mean + rows;
  if (w.has_value()) {
    TORCH_CHECK(w->is_cuda() && w->device() == dy.device() && w->scalar_type() == at::kFloat && w->is_contiguous() &&
                    w->dim() == 1 && w->size(0) == C,
                "rtseg.layer_norm_bwd: weight must be contiguous fp32 [", C, "]");
    a.w = w->data_ptr<float>();
  }
  a.rows = rows;
  a.C = static_cast<int>(C);
  a.Cp = padded(C);
  at::Tensor dr, dw, db, part;
  if (want_dr) {
    TORCH_CHECK(r_dtype.has_value(), "rtseg.layer_norm_bwd: no residual to give a gradient to");
    TORCH_CHECK(x_dtype == at::kFloat && *r_dtype != x_dtype,
                "rtseg.layer_norm_bwd: a residual gradient of its own is 16 bits beside an fp32 stream");
    dr = at::empty({rows, C}, opt.dtype(*r_dtype));
    a.r_dtype = dtype_code(dr);
    a.dr = dr.data_ptr();
  }
  if (want_dx) a.dx = dx.data_ptr();
  if (want_w) {
    dw = at::empty({C}, opt.dtype(at::kFloat));
    db = at::empty({C}, opt.dtype(at::kFloat));
    part = at::empty({layer_norm_bwd_blocks(rows, a.C), 2, C}, opt.dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  launch_layer_norm_bwd(a, want_w ? dw.data_ptr<float>() : nullptr, want_w ? db.data_ptr<float>() : nullptr, cur_stream());
  return {want_dx ? dx : at::Tensor(), dr, dw, db};
}

// ------------------------------ linear --------------------------------------------
int act_code(int64_t act) {
  TORCH_CHECK(act == kCkptNone || act == kCkptGelu, "rtseg.linear_ckpt8: bad activation code ", act);
  return static_cast<int>(act);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_ckpt8_fwd(const at::Tensor& x, const at::Tensor& w,
                                                                const std::optional<at::Tensor>& b, int64_t act, bool keep,
                                                                at::IntArrayRef shape) {
  check_rows(x, "linear_ckpt8", "x");
  TORCH_CHECK(w.dim() == 2 && w.size(0) >= 1 && w.size(0) <= kMaxChannels && w.scalar_type() == x.scalar_type(),
              "rtseg.linear_ckpt8: weight must be [out, in] of x's type with 1 .. ", kMaxChannels, " outputs");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  check_param(w, {N, K}, x, "linear_ckpt8", "weight");
  if (b.has_value()) check_param(*b, {N}, x, "linear_ckpt8", "bias");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  at::Tensor y = at::empty(shape, x.options()), codes, scales;
  LinFwdArgs a{};
  if (keep) {
    std::tie(codes, scales) = new_ckpt(M, K, x);
    a.codes = codes.data_ptr<int8_t>();
    a.scales = scales.data_ptr<uint8_t>();
  }
  a.x = x.data_ptr();
  a.w = w.data_ptr();
  a.b = opt_ptr(b);
  a.y = y.data_ptr();
  a.dtype = dtype_code(x);
  a.b_dtype = b.has_value() ? dtype_code(*b) : a.dtype;
  a.act = act_code(act);
  a.M = M;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  launch_lin_fwd(a, cur_stream());
  return {y, codes, scales};
}

at::Tensor linear_ckpt8_dgrad(const at::Tensor& dy, const at::Tensor& w, const std::optional<at::Tensor>& codes,
                              const std::optional<at::Tensor>& scales, int64_t act) {
  check_rows(dy, "linear_ckpt8_dgrad", "grad");
  TORCH_CHECK(w.dim() == 2 && w.size(1) >= 1 && w.size(1) <= kMaxChannels,
              "rtseg.linear_ckpt8_dgrad: weight must be [out, in]");
  const int64_t M = dy.size(0), N = dy.size(1), K = w.size(1);
  check_param(w, {N, K}, dy, "linear_ckpt8_dgrad", "weight");
  TORCH_CHECK(w.scalar_type() == dy.scalar_type(), "rtseg.linear_ckpt8_dgrad: the weight must be of the gradient's type");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  at::Tensor dx = at::empty({M, K}, dy.options());
  LinDgradArgs a{};
  a.act = act_code(act);
  if (a.act != kCkptNone) {
    TORCH_CHECK(codes.has_value() && scales.has_value(), "rtseg.linear_ckpt8_dgrad: the activation needs the checkpoint");
    check_ckpt(*codes, *scales, M, K, dy, "linear_ckpt8_dgrad");
    a.codes = codes->data_ptr<int8_t>();
    a.scales = scales->data_ptr<uint8_t>();
  }
  if (M == 0) return dx;
  a.dy = dy.data_ptr();
  a.w = w.data_ptr();
  a.dx = dx.data_ptr();
  a.dtype = dtype_code(dy);
  a.M = M;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  launch_lin_dgrad(a, cur_stream());
  return dx;
}

std::tuple<at::Tensor, at::Tensor> linear_ckpt8_wgrad(const at::Tensor& dy, const at::Tensor& codes, const at::Tensor& scales,
                                                      int64_t K, int64_t act, at::ScalarType w_dtype, bool want_db) {
  check_rows(dy, "linear_ckpt8_wgrad", "grad");
  TORCH_CHECK(K >= 1 && K <= kMaxChannels, "rtseg.linear_ckpt8_wgrad: bad input width");
  const int64_t M = dy.size(0), N = dy.size(1);
  check_ckpt(codes, scales, M, K, dy, "linear_ckpt8_wgrad");
  TORCH_CHECK(w_dtype == dy.scalar_type() || w_dtype == at::kFloat,
              "rtseg.linear_ckpt8_wgrad: the weight is of the gradient's type or fp32");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  at::Tensor dw = at::empty({N, K}, dy.options().dtype(w_dtype)), db;
  if (want_db) db = at::empty({N}, dw.options());
  LinWgradArgs a{};
  a.dy = dy.data_ptr();
  a.codes = codes.data_ptr<int8_t>();
  a.scales = scales.data_ptr<uint8_t>();
  a.dw = dw.data_ptr();
  a.db = want_db ? db.data_ptr() : nullptr;
  a.dtype = dtype_code(dy);
  a.w_dtype = dtype_code(dw);
  a.act = act_code(act);
  a.M = M;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  at::Tensor ws = at::empty({lin_wgrad_ws_elems(M, a.N, a.K, a.act)}, dy.options().dtype(at::kFloat));
  a.ws = ws.data_ptr<float>();
  launch_lin_wgrad(a, cur_stream());
  return {dw, db};
}

at::Tensor linear_ckpt8_bgrad(const at::Tensor& dy, at::ScalarType dtype) {
  check_rows(dy, "linear_ckpt8_bgrad", "grad");
  TORCH_CHECK(dtype == dy.scalar_type() || dtype == at::kFloat,
              "rtseg.linear_ckpt8_bgrad: the bias is of the gradient's type or fp32");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  at::Tensor db = at::empty({dy.size(1)}, dy.options().dtype(dtype));
  at::Tensor ws = at::empty({lin_colsum_splits(dy.size(0)) * dy.size(1)}, dy.options().dtype(at::kFloat));
  launch_lin_colsum(dy.data_ptr(), dtype_code(dy), ws.data_ptr<float>(), db.data_ptr(), dtype_code(db), dy.size(0),
                    static_cast<int>(dy.size(1)), cur_stream());
  return db;
}

// ------------------------------ autograd ------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor rows_of(const at::Tensor& t) {
  return t.dim() == 2 && t.is_contiguous() ? t : t.reshape({-1, t.size(-1)}).contiguous();
}
at::Tensor shaped(const at::Tensor& t, at::IntArrayRef sizes) { return t.sizes() == sizes ? t : t.view(sizes); }

// The gradients are kernels' outputs without a graph of their own: under create_graph any further use
// of them raises instead of passing for a constant.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto err = std::make_shared<torch::autograd::DelayedError>(
      "rtseg: this gradient cannot be differentiated again (the operator is differentiable once)",
      static_cast<int>(grads.size()));
  return (*err)(std::move(grads));
}

bool wants(const at::Tensor& t) { return t.requires_grad(); }
bool wants(const std::optional<at::Tensor>& t) { return t.has_value() && t->defined() && t->requires_grad(); }
std::optional<at::Tensor> maybe(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }

struct LinearCkpt8Fn : torch::autograd::Function<LinearCkpt8Fn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const std::optional<at::Tensor>& b, int64_t act, bool need_x, bool need_w, bool need_b) {
    // fp32 weights beside 16-bit operands are cast once, for the forward and the data gradient, as autocast casts
    // them (what that costs in digits: rtseg_linear_dev.h)
    const at::Tensor x2 = rows_of(x), wc = w.to(x.scalar_type()).contiguous();
    auto shape = x.sizes().vec();
    if (need_x) ctx->saved_data["shape"] = shape;
    shape.back() = w.size(0);
    auto [y, codes, scales] = linear_ckpt8_fwd(x2, wc, b, act, need_w || (need_x && act != kCkptNone), shape);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({codes, scales, need_x ? wc : at::Tensor()});
    ctx->saved_data["call"] = std::vector<int64_t>{x2.size(1), act, need_x, need_w, need_b, static_cast<int64_t>(w.scalar_type())};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const auto call = ctx->saved_data["call"].toIntVector();
    const int64_t k = call[0], act = call[1];
    const bool need_x = call[2] != 0, need_w = call[3] != 0, need_b = call[4] != 0;
    const auto wt = static_cast<at::ScalarType>(call[5]);
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor dy = rows_of(grads[0]);
    if (need_x)
      out[0] = shaped(linear_ckpt8_dgrad(dy, saved[2], maybe(saved[0]), maybe(saved[1]), act),
                      ctx->saved_data["shape"].toIntVector());
    if (need_w) std::tie(out[1], out[2]) = linear_ckpt8_wgrad(dy, saved[0], saved[1], k, act, wt, need_b);
    else if (need_b) out[2] = linear_ckpt8_bgrad(dy, wt);
    return once(std::move(out));
  }
};

at::Tensor linear_ckpt8(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& b, int64_t act) {
  const at::Tensor x2 = rows_of(x);
  auto shape = x.sizes().vec();
  shape.back() = w.size(0);
  return std::get<0>(linear_ckpt8_fwd(x2, w.to(x.scalar_type()).contiguous(), b, act, false, shape));
}
at::Tensor linear_ckpt8_autograd(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& b, int64_t act) {
  const bool on = at::GradMode::is_enabled();
  const bool nx = on && wants(x), nw = on && wants(w), nb = on && wants(b);
  if (!(nx || nw || nb)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_ckpt8(x, w, b, act);
  }
  return LinearCkpt8Fn::apply(x, w, b, act, nx, nw, nb);
}

// x, residual, weight, bias -> {y} or {x + residual, y}; `sum`: the sum is wanted by the caller
struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& r,
                               const std::optional<at::Tensor>& w, const std::optional<at::Tensor>& b, double eps,
                               at::ScalarType out, bool ckpt, bool sum, int64_t need) {
    const at::Tensor x2 = rows_of(x);
    std::optional<at::Tensor> r2, wf, bf;
    if (r.has_value()) r2 = rows_of(*r);
    if (w.has_value()) wf = w->to(at::kFloat).contiguous();
    if (b.has_value()) bf = b->to(at::kFloat).contiguous();
    // without a checkpoint the backward normalises the sum again, so it is kept even if unwanted
    auto [s, y, stats, codes, scales] = layer_norm_fwd(x2, r2, wf, bf, eps, out, need == 0 ? 0 : ckpt ? 2 : 1, sum || !ckpt,
                                                      x.sizes());
    auto st = [](const std::optional<at::Tensor>& t, at::ScalarType other) {
      return static_cast<int64_t>(t.has_value() ? t->scalar_type() : other);
    };
    variable_list got;
    if (sum) got.push_back(s);
    got.push_back(y);
    // the tensor that the caller holds, where there is one, not a view of it: a change in place has to be noticed
    const at::Tensor kept = ckpt ? codes : r.has_value() ? s : x.is_contiguous() ? x : x2;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({kept, scales, stats, wf.has_value() ? *wf : at::Tensor()});
    ctx->saved_data["call"] = std::vector<int64_t>{need, ckpt, sum, static_cast<int64_t>(x.scalar_type()), st(r, x.scalar_type()),
                                                   st(w, at::kFloat), st(b, at::kFloat)};
    ctx->saved_data["shape"] = x.sizes().vec();
    return got;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(9);
    const auto call = ctx->saved_data["call"].toIntVector();
    const int64_t need = call[0];
    const bool need_x = need & 1, need_r = need & 2, need_w = need & 4, need_b = need & 8, ckpt = call[1] != 0, sum = call[2] != 0;
    auto type = [&](int i) { return static_cast<at::ScalarType>(call[i]); };
    const at::ScalarType xt = type(3), rt = type(4);
    const at::Tensor ds = sum ? grads[0] : at::Tensor(), dy = grads.back();
    if (!dy.defined()) {  // the norm's output is unused: only the sum carries a gradient
      if (ds.defined() && need_x) out[0] = ds;
      if (ds.defined() && need_r) out[1] = ds.to(rt);
      return out;
    }
    const variable_list saved = ctx->get_saved_variables();
    const bool own_r = need_r && rt != xt;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::optional<at::Tensor> ds2, x2;
      if (ds.defined()) ds2 = rows_of(ds);
      if (!ckpt) x2 = rows_of(saved[0]);
      auto [dx, dr, dw, db] = layer_norm_bwd(rows_of(dy), ds2, x2, ckpt ? maybe(saved[0]) : std::nullopt,
                                             ckpt ? maybe(saved[1]) : std::nullopt, saved[2], maybe(saved[3]), xt, rt,
                                             need_x || (need_r && !own_r), own_r, need_w || need_b);
      const auto shape = ctx->saved_data["shape"].toIntVector();
      if (dx.defined()) dx = shaped(dx, shape);
      // one tensor, not two views of it: whoever accumulates into the one then knows that it is shared
      if (need_x) out[0] = dx;
      if (need_r) out[1] = own_r ? shaped(dr, shape) : dx;
      if (need_w) out[2] = dw.to(type(5));
      if (need_b) out[3] = db.to(type(6));
    }
    return once(std::move(out));
  }
};

std::vector<at::Tensor> layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& r, const std::optional<at::Tensor>& w,
                                   const std::optional<at::Tensor>& b, double eps, at::ScalarType out, bool, bool sum) {
  std::optional<at::Tensor> r2, wf, bf;
  if (r.has_value()) r2 = rows_of(*r);
  if (w.has_value()) wf = w->to(at::kFloat).contiguous();
  if (b.has_value()) bf = b->to(at::kFloat).contiguous();
  auto got = layer_norm_fwd(rows_of(x), r2, wf, bf, eps, out, 0, sum, x.sizes());
  if (sum) return {std::get<0>(got), std::get<1>(got)};
  return {std::get<1>(got)};
}
std::vector<at::Tensor> layer_norm_autograd(const at::Tensor& x, const std::optional<at::Tensor>& r,
                                            const std::optional<at::Tensor>& w, const std::optional<at::Tensor>& b, double eps,
                                            at::ScalarType out, bool ckpt, bool sum) {
  TORCH_CHECK(!sum || r.has_value(), "rtseg.layer_norm: no residual, no sum");
  const int64_t need = !at::GradMode::is_enabled() ? 0 : wants(x) | wants(r) << 1 | wants(w) << 2 | wants(b) << 3;
  if (need == 0) {
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm(x, r, w, b, eps, out, ckpt, sum);
  }
  return LayerNormFn::apply(x, r, w, b, eps, out, ckpt, sum, need);
}

}  // namespace
}  // namespace rtseg

TORCH_LIBRARY_FRAGMENT(rtseg, m) {
  m.def("ckpt8_pack(Tensor x) -> (Tensor, Tensor)");
  m.def("ckpt8_unpack(Tensor codes, Tensor scales, int channels, ScalarType dtype, ScalarType held) -> Tensor");
  // -> [y], or [x + r, y] with sum
  m.def("layer_norm(Tensor x, Tensor? r, Tensor? w, Tensor? b, float eps, ScalarType out, bool ckpt8, bool sum) -> Tensor[]");
  m.def("linear_ckpt8(Tensor x, Tensor w, Tensor? b, int act) -> Tensor");
}

TORCH_LIBRARY_IMPL(rtseg, CUDA, m) {
  m.impl("ckpt8_pack", &rtseg::ckpt8_pack);
  m.impl("ckpt8_unpack", &rtseg::ckpt8_unpack);
  m.impl("layer_norm", &rtseg::layer_norm);
  m.impl("linear_ckpt8", &rtseg::linear_ckpt8);
}

TORCH_LIBRARY_IMPL(rtseg, AutogradCUDA, m) {
  m.impl("layer_norm", &rtseg::layer_norm_autograd);
  m.impl("linear_ckpt8", &rtseg::linear_ckpt8_autograd);
}
