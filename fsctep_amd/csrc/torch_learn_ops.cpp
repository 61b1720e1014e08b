// torch.ops.fsctep.* of the training step: layer norm, lookups and the optimiser's step on the C ABI of layer_norm.hip,
// embedding.hip and adamw.hip.  Each op has device and Meta kernels; calls run on the current stream of their tensors'
// device, allocate outputs and workspaces from the caching allocator and never wait for the GPU.  layer_norm
// differentiates twice (its backward is an op with a backward), embedding to any order.

#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <cmath>

#include "torch_args.h"

namespace {

// ============================================================== layer norm
int32_t weight_code(const Tensor& t, const Tensor& x, const char* op, const char* name) {
  if (!t.defined()) return FSC_F32;
  const int32_t c = code_of(t.scalar_type(), name);
  TORCH_CHECK(c == FSC_F32 || t.scalar_type() == x.scalar_type(), op, ": ", name, " must be float32 or of x's type");
  TORCH_CHECK(t.dim() == 1 && t.sym_size(0) == x.sym_size(1), op, ": ", name, " must be (", x.sym_size(1), ",)");
  return c;
}

// the weight's code, the bias' where there is no weight
int32_t check_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t act, const char* op) {
  TORCH_CHECK(x.dim() == 2, op, ": x must be (rows, width), got ", x.dim(), " dimensions");
  code_of(x.scalar_type(), "x");
  TORCH_CHECK(x.sym_size(1) >= 1 && x.sym_size(1) <= (1 << 20), op, ": the width must be 1 to 2^20");
  TORCH_CHECK(act == FSC_ACT_NONE || act == FSC_ACT_SILU, op, ": unknown activation ", act);
  TORCH_CHECK(eps >= 0 && std::isfinite(eps), op, ": eps must be finite and not negative, got ", eps);
  const int32_t wc = weight_code(w, x, op, "weight"), bc = weight_code(b, x, op, "bias");
  TORCH_CHECK(!w.defined() || !b.defined() || wc == bc, op, ": weight and bias must have one type");
  return w.defined() ? wc : bc;
}

void check_rows_like(const Tensor& t, const Tensor& x, const char* op, const char* name) {
  if (!t.defined()) return;
  TORCH_CHECK(t.sym_sizes() == x.sym_sizes() && t.scalar_type() == x.scalar_type(), op, ": ", name,
              " must have the rows' shape and type");
}

void check_stats(const Tensor& x, const Tensor& mean, const Tensor& rstd, const char* op) {
  TORCH_CHECK(mean.dim() == 1 && mean.sym_size(0) == x.sym_size(0) && mean.scalar_type() == at::kDouble && rstd.dim() == 1 &&
                  rstd.sym_size(0) == x.sym_size(0) && rstd.scalar_type() == at::kFloat,
              op, ": mean (float64) and rstd (float32) must be (", x.sym_size(0), ",)");
}

Tensor flat(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
int64_t stride_or_0(const Tensor& t) { return t.defined() ? stride_of(t) : 0; }

// (y, mean, rstd); the statistics are empty unless they are to be kept
std::tuple<Tensor, Tensor, Tensor> layer_norm(const Tensor& x_, const optional<Tensor>& w_, const optional<Tensor>& b_,
                                              double eps, int64_t act, bool keep) {
  require_gpu({x_, some(w_), some(b_)}, "layer_norm");
  const int32_t wt = check_norm(x_, some(w_), some(b_), eps, act, "layer_norm");
  const c10::OptionalDeviceGuard device(x_.device());
  const Tensor x = rows2d(x_, "x"), w = flat(some(w_)), b = flat(some(b_));
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor mean = at::empty({keep ? x.size(0) : 0}, x.options().dtype(at::kDouble));
  Tensor rstd = at::empty({keep ? x.size(0) : 0}, x.options().dtype(at::kFloat));
  check(fsc_layer_norm_forward(x.size(0), (int32_t)x.size(1), code_of(x.scalar_type(), "x"), wt, (int32_t)act,
                               stride_of(x), ptr(x), ptr(w), ptr(b), (float)eps, mptr(y), (double*)mptr(mean),
                               (float*)mptr(rstd), stream_of(x)),
        "fsc_layer_norm_forward");
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_meta(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                                   double eps, int64_t act, bool keep) {
  check_norm(x, some(w), some(b), eps, act, "layer_norm");
  const c10::SymInt n = keep ? x.sym_size(0) : c10::SymInt(0);
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint({n}, x.options().dtype(at::kDouble)),
          at::empty_symint({n}, x.options().dtype(at::kFloat))};
}

struct NormGrad {
  Tensor x, w, b, ws;
  int32_t dt, wt;
};
Tensor out_if(bool want, const Tensor& like) {
  return want ? at::empty_symint(like.sym_sizes(), like.options()) : at::empty({0}, like.options());
}
void check_wanted(const Tensor& w, const Tensor& b, bool want_w, bool want_b, const char* op) {
  TORCH_CHECK((!want_w || w.defined()) && (!want_b || b.defined()), op, ": no gradient of a weight or bias that is not there");
}
NormGrad norm_grad(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t act, bool sums, const char* op) {
  NormGrad g{rows2d(x, "x"), flat(w), flat(b), Tensor(), code_of(x.scalar_type(), "x"), check_norm(x, w, b, eps, act, op)};
  int64_t n = 0;
  check(fsc_layer_norm_workspace(x.size(0), (int32_t)x.size(1), &n), "fsc_layer_norm_workspace");
  g.ws = at::empty({sums ? n : 0}, x.options().dtype(at::kFloat));
  return g;
}

// (dx + plus, dweight, dbias), empty where not wanted.  `through` has x's shape and no values: the gradient of x takes its way
// where it is given (LayerNormFn).
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& dy_, const Tensor& x_, const optional<Tensor>& w_,
                                                       const optional<Tensor>& b_, const Tensor& mean_, const Tensor& rstd_,
                                                       double eps, int64_t act, bool want_x, bool want_w, bool want_b,
                                                       const optional<Tensor>& plus_, const optional<Tensor>&) {
  const char* op = "layer_norm_backward";
  require_gpu({x_, dy_, some(w_), some(b_), mean_, rstd_, some(plus_)}, op);
  check_rows_like(some(plus_), x_, op, "plus");
  check_norm(x_, some(w_), some(b_), eps, act, op);
  check_rows_like(dy_, x_, op, "dy");
  check_stats(x_, mean_, rstd_, op);
  check_wanted(some(w_), some(b_), want_w, want_b, op);
  const c10::OptionalDeviceGuard device(x_.device());
  NormGrad g = norm_grad(x_, some(w_), some(b_), eps, act, want_w || want_b, op);
  const Tensor dy = rows2d(dy_, "dy"), mean = mean_.contiguous(), rstd = rstd_.contiguous();
  const Tensor plus = plus_.has_value() ? rows2d(*plus_, "plus") : Tensor();
  Tensor dx = out_if(want_x, g.x);
  Tensor dw = out_if(want_w, want_w ? g.w : g.x), db = out_if(want_b, want_b ? g.b : g.x);
  check(fsc_layer_norm_backward(g.x.size(0), (int32_t)g.x.size(1), g.dt, g.wt, (int32_t)act, stride_of(g.x), stride_of(dy),
                                stride_or_0(plus), ptr(g.x), ptr(g.w), ptr(g.b), (float)eps, (const double*)ptr(mean),
                                (const float*)ptr(rstd), ptr(dy), ptr(plus), want_x ? mptr(dx) : nullptr, want_w ? mptr(dw) : nullptr,
                                want_b ? mptr(db) : nullptr, (float*)mptr(g.ws), stream_of(g.x)),
        "fsc_layer_norm_backward");
  return {dx, dw, db};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_meta(const Tensor& dy, const Tensor& x, const optional<Tensor>& w,
                                                            const optional<Tensor>& b, const Tensor& mean, const Tensor& rstd,
                                                            double eps, int64_t act, bool want_x, bool want_w, bool want_b,
                                                            const optional<Tensor>& plus, const optional<Tensor>&) {
  const char* op = "layer_norm_backward";
  check_norm(x, some(w), some(b), eps, act, op);
  check_rows_like(dy, x, op, "dy");
  check_rows_like(some(plus), x, op, "plus");
  check_stats(x, mean, rstd, op);
  check_wanted(some(w), some(b), want_w, want_b, op);
  return {out_if(want_x, x), out_if(want_w, want_w ? some(w) : x), out_if(want_b, want_b ? some(b) : x)};
}

// (grad_x, grad_dy, grad_weight, grad_bias) from cotangents of dx, dweight and dbias
std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm_backward_twice(
    const optional<Tensor>& v_, const optional<Tensor>& vw_, const optional<Tensor>& vb_, const Tensor& dy_, const Tensor& x_,
    const optional<Tensor>& w_, const optional<Tensor>& b_, const Tensor& mean_, const Tensor& rstd_, double eps, int64_t act,
    bool want_x, bool want_dy, bool want_w, bool want_b) {
  const char* op = "layer_norm_backward_twice";
  require_gpu({x_, dy_, some(w_), some(b_), mean_, rstd_, some(v_), some(vw_), some(vb_)}, op);
  const int32_t wt = check_norm(x_, some(w_), some(b_), eps, act, op);
  check_rows_like(dy_, x_, op, "dy");
  check_rows_like(some(v_), x_, op, "v");
  check_stats(x_, mean_, rstd_, op);
  check_wanted(some(w_), some(b_), want_w, want_b, op);
  for (const Tensor& t : {some(vw_), some(vb_)})
    TORCH_CHECK(!t.defined() || (code_of(t.scalar_type(), "v") == wt && t.dim() == 1 && t.size(0) == x_.size(1)), op,
                ": cotangents of weight and bias must have their shape and type");
  const c10::OptionalDeviceGuard device(x_.device());
  NormGrad g = norm_grad(x_, some(w_), some(b_), eps, act, want_w || want_b, op);
  const Tensor dy = rows2d(dy_, "dy"), v = v_.has_value() ? rows2d(*v_, "v") : Tensor();
  const Tensor vw = flat(some(vw_)), vb = flat(some(vb_)), mean = mean_.contiguous(), rstd = rstd_.contiguous();
  Tensor gx = out_if(want_x, g.x), gdy = out_if(want_dy, g.x);
  Tensor gw = out_if(want_w, want_w ? g.w : g.x), gb = out_if(want_b, want_b ? g.b : g.x);
  check(fsc_layer_norm_backward_twice(g.x.size(0), (int32_t)g.x.size(1), g.dt, wt, (int32_t)act, stride_of(g.x),
                                      stride_of(dy), stride_or_0(v), ptr(g.x), ptr(g.w), ptr(g.b), (float)eps,
                                      (const double*)ptr(mean), (const float*)ptr(rstd), ptr(dy), ptr(v), ptr(vw), ptr(vb),
                                      want_x ? mptr(gx) : nullptr, want_dy ? mptr(gdy) : nullptr,
                                      want_w ? mptr(gw) : nullptr, want_b ? mptr(gb) : nullptr, (float*)mptr(g.ws),
                                      stream_of(g.x)),
        "fsc_layer_norm_backward_twice");
  return {gx, gdy, gw, gb};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm_backward_twice_meta(
    const optional<Tensor>& v, const optional<Tensor>&, const optional<Tensor>&, const Tensor& dy, const Tensor& x,
    const optional<Tensor>& w, const optional<Tensor>& b, const Tensor& mean, const Tensor& rstd, double eps, int64_t act,
    bool want_x, bool want_dy, bool want_w, bool want_b) {
  const char* op = "layer_norm_backward_twice";
  check_norm(x, some(w), some(b), eps, act, op);
  check_rows_like(dy, x, op, "dy");
  check_rows_like(some(v), x, op, "v");
  check_stats(x, mean, rstd, op);
  check_wanted(some(w), some(b), want_w, want_b, op);
  return {out_if(want_x, x), out_if(want_dy, x), out_if(want_w, want_w ? some(w) : x), out_if(want_b, want_b ? some(b) : x)};
}

auto& layer_norm_op() {
  static auto op = op_handle<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const optional<Tensor>&, const optional<Tensor>&,
                                                                double, int64_t, bool)>("fsctep::layer_norm");
  return op;
}
auto& layer_norm_backward_op() {
  static auto op = op_handle<std::tuple<Tensor, Tensor, Tensor>(
      const Tensor&, const Tensor&, const optional<Tensor>&, const optional<Tensor>&, const Tensor&, const Tensor&, double,
      int64_t, bool, bool, bool, const optional<Tensor>&, const optional<Tensor>&)>("fsctep::layer_norm_backward");
  return op;
}
optional<Tensor> opt(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

// The backward as a function of dy, x, weight and bias (the statistics are x's own), and of plus: its backward is an op without
// one.
struct LayerNormBackwardFn : public torch::autograd::Function<LayerNormBackwardFn> {
  static variable_list forward(AutogradContext* ctx, Tensor dy, Tensor x, optional<Tensor> w, optional<Tensor> b, Tensor mean,
                               Tensor rstd, double eps, int64_t act, bool want_x, bool want_w, bool want_b,
                               optional<Tensor> plus, optional<Tensor> through) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [dx, dw, db] =
        layer_norm_backward_op().call(dy, x, w, b, mean, rstd, eps, act, want_x, want_w, want_b, plus, std::nullopt);
    ctx->save_for_backward({dy, x, some(w), some(b), mean, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    ctx->saved_data["plus"] = plus.has_value();
    ctx->saved_data["through"] = through.has_value();
    ctx->set_materialize_grads(false);
    variable_list none;
    if (!want_x) none.push_back(dx);
    if (!want_w) none.push_back(dw);
    if (!want_b) none.push_back(db);
    ctx->mark_non_differentiable(none);
    return {dx, dw, db};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(13);
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return out;
    auto s = ctx->get_saved_variables();
    static auto op = op_handle<std::tuple<Tensor, Tensor, Tensor, Tensor>(
        const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, const Tensor&, const Tensor&,
        const optional<Tensor>&, const optional<Tensor>&, const Tensor&, const Tensor&, double, int64_t, bool, bool, bool, bool)>(
        "fsctep::layer_norm_backward_twice");
    // needs_input_grad counts the tensors there are: dy, x, weight, bias, mean, rstd, plus, through
    const bool has_w = s[2].defined(), has_b = s[3].defined();
    const bool has_plus = ctx->saved_data["plus"].toBool(), has_through = ctx->saved_data["through"].toBool();
    const size_t at_plus = 4 + has_w + has_b, at_through = at_plus + has_plus;
    const bool want_dy = ctx->needs_input_grad(0);
    const bool want_x = has_through ? ctx->needs_input_grad(at_through) : ctx->needs_input_grad(1);
    const bool want_w = has_w && ctx->needs_input_grad(2), want_b = has_b && ctx->needs_input_grad(2 + has_w);
    if (has_plus && ctx->needs_input_grad(at_plus)) out[11] = grads[0];
    if (!want_dy && !want_x && !want_w && !want_b) return out;
    BackwardGuard guard;
    auto [gx, gdy, gw, gb] =
        op.call(opt(grads[0]), opt(grads[1]), opt(grads[2]), s[0], s[1], opt(s[2]), opt(s[3]), s[4], s[5],
                ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt(), want_x, want_dy, want_w, want_b);
    if (want_dy) out[0] = gdy;
    if (want_x) out[has_through ? 12 : 1] = gx;
    if (want_w) out[2] = gw;
    if (want_b) out[3] = gb;
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_autograd(const Tensor& dy, const Tensor& x, const optional<Tensor>& w,
                                                                const optional<Tensor>& b, const Tensor& mean,
                                                                const Tensor& rstd, double eps, int64_t act, bool want_x,
                                                                bool want_w, bool want_b, const optional<Tensor>& plus,
                                                                const optional<Tensor>& through) {
  if (differentiates({dy, x, some(w), some(b), some(plus), some(through)})) {
    auto r = LayerNormBackwardFn::apply(dy, x, w, b, mean, rstd, eps, act, want_x, want_w, want_b, plus, through);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return layer_norm_backward_op().call(dy, x, w, b, mean, rstd, eps, act, want_x, want_w, want_b, plus, through);
}

// A force loss sends two gradients to x, one through y and one through the backward's own backward.  The second comes to this
// function's node as the gradient of `through`, an output of x's shape that holds nothing, and the kernel that makes the first
// adds it (`plus`): a pass over x less than autograd's addition takes.  A run of the node that only passes the second one on
// reads nothing that the node keeps, and leaves it (release_variables below).
struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
  static variable_list forward(AutogradContext* ctx, Tensor x, optional<Tensor> w, optional<Tensor> b, double eps,
                               int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, mean, rstd] = layer_norm_op().call(x, w, b, eps, act, true);
    Tensor through = at::empty_strided_symint(x.sym_sizes(), {0, 0}, x.options());
    ctx->save_for_backward({x, some(w), some(b), mean, rstd, through});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    ctx->saved_data["passed"] = false;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({mean, rstd});
    return {y, mean, rstd, through};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    const bool want_x = ctx->needs_input_grad(0);
    ctx->saved_data["passed"] = !grads[0].defined();
    if (!grads[0].defined()) {
      if (want_x) out[0] = grads[3];
      return out;
    }
    auto s = ctx->get_saved_variables();
    const bool want_w = s[1].defined() && ctx->needs_input_grad(1);
    const bool want_b = s[2].defined() && ctx->needs_input_grad(s[1].defined() ? 2 : 1);    // counts the tensors there are
    auto [dx, dw, db] = layer_norm_backward_op().call(
        grads[0], s[0], opt(s[1]), opt(s[2]), s[3], s[4], ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt(),
        want_x, want_w, want_b, want_x ? opt(grads[3]) : std::nullopt,
        want_x && at::GradMode::is_enabled() ? opt(s[5]) : std::nullopt);
    if (want_x) out[0] = dx;
    if (want_w) out[1] = dw;
    if (want_b) out[2] = db;
    return out;
  }
};

}  // namespace

// The engine calls this after a node's run unless the graph is to be kept.  x's second gradient alone comes through LayerNormFn's
// node without using it up: y can still be differentiated, as where the second gradient goes straight to x.
template <>
void torch::autograd::CppNode<LayerNormFn>::release_variables() {
  std::lock_guard<std::mutex> lock(mutex_);
  if (ctx_.saved_data["passed"].toBool()) return;
  ctx_.saved_variables_.clear();
  ctx_.has_freed_buffers_ = true;
}

namespace {

std::tuple<Tensor, Tensor, Tensor> layer_norm_autograd(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                                       double eps, int64_t act, bool keep) {
  if (differentiates({x, some(w), some(b)})) {
    auto r = LayerNormFn::apply(x, w, b, eps, act);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return layer_norm_op().call(x, w, b, eps, act, keep);
}

// ============================================================== lookup
int32_t check_index(const Tensor& index, const char* op) {
  TORCH_CHECK(index.dim() == 1, op, ": index must have one dimension, got ", index.dim());
  TORCH_CHECK(index.scalar_type() == at::kInt || index.scalar_type() == at::kLong, op, ": index must be int32 or int64, got ",
              index.scalar_type());
  return index.scalar_type() == at::kInt ? 32 : 64;
}
// the C entry's width has 32 bits
void check_width(const c10::SymInt& width, const char* op) {
  TORCH_CHECK(width <= (1 << 20), op, ": the width must be at most 2^20, got ", width);
}
void check_scale(double scale, const char* op) {
  TORCH_CHECK(std::isfinite((float)scale), op, ": scale must be finite, got ", scale);
}

Tensor embedding(const Tensor& table_, const Tensor& index_, double scale, double outside) {
  require_gpu({table_, index_}, "embedding");
  TORCH_CHECK(table_.dim() == 2, "embedding: table must be (rows, width), got ", table_.dim(), " dimensions");
  const int32_t dt = code_of(table_.scalar_type(), "table"), bits = check_index(index_, "embedding");
  check_scale(scale, "embedding");
  check_width(table_.sym_size(1), "embedding");
  const c10::OptionalDeviceGuard device(table_.device());
  const Tensor table = rows2d(table_, "table"), index = index_.contiguous();
  Tensor out = at::empty({index.size(0), table.size(1)}, table.options());
  if (out.numel() == 0) return out;
  check(fsc_embedding_forward_or(index.size(0), (int32_t)table.size(1), table.size(0), dt, bits, stride_of(table), ptr(table),
                                 ptr(index), (float)scale, (float)outside, mptr(out), stream_of(table)),
        "fsc_embedding_forward_or");
  return out;
}

Tensor embedding_meta(const Tensor& table, const Tensor& index, double scale, double) {
  TORCH_CHECK(table.dim() == 2, "embedding: table must be (rows, width), got ", table.dim(), " dimensions");
  code_of(table.scalar_type(), "table");
  check_index(index, "embedding");
  check_scale(scale, "embedding");
  check_width(table.sym_size(1), "embedding");
  return at::empty_symint({index.sym_size(0), table.sym_size(1)}, table.options());
}

Tensor embedding_backward(const Tensor& dy_, const Tensor& index_, c10::SymInt table_rows_, double scale) {
  const char* op = "embedding_backward";
  require_gpu({dy_, index_}, op);
  TORCH_CHECK(dy_.dim() == 2 && dy_.size(0) == index_.size(0), op, ": dy must be (tokens, width)");
  const int32_t dt = code_of(dy_.scalar_type(), "dy"), bits = check_index(index_, op);
  const int64_t table_rows = table_rows_.expect_int();
  TORCH_CHECK(table_rows >= 0, op, ": negative table rows");
  check_scale(scale, op);
  check_width(dy_.sym_size(1), op);
  const c10::OptionalDeviceGuard device(dy_.device());
  const Tensor dy = rows2d(dy_, "dy"), index = index_.contiguous();
  Tensor out = at::empty({table_rows, dy.size(1)}, dy.options());
  if (out.numel() == 0) return out;
  int64_t bytes = 0;
  check(fsc_embedding_workspace(index.size(0), (int32_t)dy.size(1), table_rows, &bytes), "fsc_embedding_workspace");
  Tensor ws = at::empty({bytes}, dy.options().dtype(at::kByte));
  check(fsc_embedding_backward(index.size(0), (int32_t)dy.size(1), table_rows, dt, bits, stride_of(dy), ptr(dy), ptr(index),
                               (float)scale, mptr(out), mptr(ws), stream_of(dy)),
        "fsc_embedding_backward");
  return out;
}

Tensor embedding_backward_meta(const Tensor& dy, const Tensor& index, c10::SymInt table_rows, double scale) {
  TORCH_CHECK(dy.dim() == 2 && dy.sym_size(0) == index.sym_size(0), "embedding_backward: dy must be (tokens, width)");
  code_of(dy.scalar_type(), "dy");
  check_index(index, "embedding_backward");
  check_scale(scale, "embedding_backward");
  check_width(dy.sym_size(1), "embedding_backward");
  return at::empty_symint({table_rows, dy.sym_size(1)}, dy.options());
}

auto& embedding_op() {
  static auto op = op_handle<Tensor(const Tensor&, const Tensor&, double, double)>("fsctep::embedding");
  return op;
}
auto& embedding_backward_op() {
  static auto op = op_handle<Tensor(const Tensor&, const Tensor&, c10::SymInt, double)>("fsctep::embedding_backward");
  return op;
}

// Linear in the table, and the gradient linear in dy: each is the other's backward.
struct EmbeddingBackwardFn : public torch::autograd::Function<EmbeddingBackwardFn> {
  static variable_list forward(AutogradContext* ctx, Tensor dy, Tensor index, c10::SymInt table_rows, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({index});
    ctx->saved_data["scale"] = scale;
    return {embedding_backward_op().call(dy, index, table_rows, scale)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (ctx->needs_input_grad(0))
      out[0] = embedding_op().call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["scale"].toDouble(), 0.0);
    return out;
  }
};

Tensor embedding_backward_autograd(const Tensor& dy, const Tensor& index, c10::SymInt table_rows, double scale) {
  if (differentiates({dy})) return EmbeddingBackwardFn::apply(dy, index, table_rows, scale)[0];
  at::AutoDispatchBelowADInplaceOrView guard;
  return embedding_backward_op().call(dy, index, table_rows, scale);
}

struct EmbeddingFn : public torch::autograd::Function<EmbeddingFn> {
  static variable_list forward(AutogradContext* ctx, Tensor table, Tensor index, double scale, double outside) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({index});
    ctx->saved_data["rows"] = table.sym_size(0);
    ctx->saved_data["scale"] = scale;
    return {embedding_op().call(table, index, scale, outside)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (ctx->needs_input_grad(0))
      out[0] = embedding_backward_op().call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toSymInt(),
                                            ctx->saved_data["scale"].toDouble());
    return out;
  }
};

Tensor embedding_autograd(const Tensor& table, const Tensor& index, double scale, double outside) {
  if (differentiates({table})) return EmbeddingFn::apply(table, index, scale, outside)[0];
  at::AutoDispatchBelowADInplaceOrView guard;
  return embedding_op().call(table, index, scale, outside);
}

// ============================================================== optimiser
constexpr int64_t kGroup = 256;      // values that share a scale

// One list of an optimiser step: as long as the parameters, each of a type and of as many values as `values` says.
template <typename N>
void check_list(at::TensorList list, at::TensorList params, at::ScalarType type, N&& values, const char* op, const char* name) {
  TORCH_CHECK(list.size() == params.size(), op, ": ", list.size(), " ", name, " for ", params.size(), " parameters");
  for (size_t i = 0; i < list.size(); ++i) {
    TORCH_CHECK(list[i].device() == params[0].device(), op, ": ", name, " ", i, " is on ", list[i].device(),
                ", the parameters are on ", params[0].device());
    TORCH_CHECK(list[i].scalar_type() == type, op, ": ", name, " ", i, " must be ", type, ", got ", list[i].scalar_type());
    TORCH_CHECK(list[i].numel() == values(i) && list[i].is_contiguous(), op, ": ", name, " ", i, " must be contiguous and of ",
                values(i), " values");
  }
}

// Checks parameters (and what else is stepped) and gradients; gradients that are not contiguous are copied.
std::vector<Tensor> check_params(at::TensorList params, at::TensorList grads, const char* op) {
  TORCH_CHECK(params.size() == grads.size(), op, ": ", grads.size(), " gradients for ", params.size(), " parameters");
  TORCH_CHECK(!params.empty(), op, ": no parameters");
  std::vector<Tensor> out;
  out.reserve(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor &p = params[i], &g = grads[i];
    TORCH_CHECK(p.layout() == at::kStrided && g.layout() == at::kStrided, op, ": tensor ", i, " is not strided");
    TORCH_CHECK(p.device() == params[0].device() && g.device() == p.device(), op, ": tensors on ", params[0].device(), " and ",
                p.device(), ", ", g.device());
    code_of(p.scalar_type(), "parameters");
    TORCH_CHECK(p.is_contiguous(), op, ": parameter ", i, " is not contiguous");
    TORCH_CHECK(g.sizes() == p.sizes() && g.scalar_type() == p.scalar_type(), op, ": gradient ", i,
                " must have its parameter's shape and type");
    out.push_back(g.contiguous());
  }
  return out;
}

Tensor grad_norm(at::TensorList grads) {
  TORCH_CHECK(!grads.empty(), "grad_norm: no gradients");
  std::vector<FscAdamTensor> t(grads.size());
  std::vector<Tensor> keep;
  for (size_t i = 0; i < grads.size(); ++i) {
    require_gpu({grads[0], grads[i]}, "grad_norm");
    TORCH_CHECK(grads[i].layout() == at::kStrided, "grad_norm: tensor ", i, " is not strided");
    keep.push_back(grads[i].contiguous());
    t[i] = FscAdamTensor{};
    t[i].n = grads[i].numel();
    t[i].dtype = code_of(grads[i].scalar_type(), "gradients");
    t[i].g = ptr(keep[i]);
  }
  const c10::OptionalDeviceGuard device(grads[0].device());
  int64_t step = 0, bytes = 0;
  check(fsc_adamw_workspace((int32_t)t.size(), t.data(), &step, &bytes), "fsc_adamw_workspace");
  Tensor ws = at::empty({bytes}, grads[0].options().dtype(at::kByte)), norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  check(fsc_grad_norm((int32_t)t.size(), t.data(), mptr(ws), (float*)mptr(norm), stream_of(norm)), "fsc_grad_norm");
  return norm;
}

Tensor grad_norm_meta(at::TensorList grads) {
  TORCH_CHECK(!grads.empty(), "grad_norm: no gradients");
  for (const Tensor& g : grads) code_of(g.scalar_type(), "gradients");
  return at::empty({}, grads[0].options().dtype(at::kFloat));
}

// The step of a list of tensors, in place; m_scales empty: states in 32 bits.
void adamw_check(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList m_scales, at::TensorList v,
                 at::TensorList v_scales, at::TensorList steps, at::TensorList masters, const optional<Tensor>& norm,
                 const optional<Tensor>& lr_tensor, bool q8, const char* op, std::vector<Tensor>& g) {
  g = check_params(params, grads, op);
  const auto values = [&](size_t i) { return params[i].numel(); };
  const auto groups = [&](size_t i) { return (params[i].numel() + kGroup - 1) / kGroup; };
  const auto one = [](size_t) { return int64_t(1); };
  check_list(m, params, q8 ? at::kByte : at::kFloat, values, op, "first moments");
  check_list(v, params, q8 ? at::kByte : at::kFloat, values, op, q8 ? "roots" : "second moments");
  check_list(steps, params, at::kFloat, one, op, "step counts");
  if (q8) {
    check_list(m_scales, params, at::kFloat, groups, op, "first moments' scales");
    check_list(v_scales, params, at::kFloat, groups, op, "roots' scales");
  }
  bool half = false;
  for (const Tensor& p : params) half |= p.scalar_type() == at::kBFloat16;
  TORCH_CHECK(masters.size() == params.size() || (masters.empty() && !half), op,
              ": bfloat16 parameters need their float32 copies (masters), as many as parameters");
  for (size_t i = 0; i < params.size() && half; ++i)
    TORCH_CHECK(params[i].scalar_type() == at::kFloat ||
                    (masters[i].scalar_type() == at::kFloat && masters[i].sizes() == params[i].sizes() &&
                     masters[i].is_contiguous() && masters[i].device() == params[i].device()),
                op, ": master ", i, " must be contiguous, float32 and of its parameter's shape");
  for (const Tensor& t : {some(norm), some(lr_tensor)})
    TORCH_CHECK(!t.defined() || (t.numel() == 1 && t.scalar_type() == at::kFloat && t.device() == params[0].device()), op,
                ": norm and lr are single float32 values on the parameters' device");
  // a value that two of them hold would depend on the order in which it is written (and gradients on what was written before)
  struct Range { const char *from, *to; bool written; };
  std::vector<Range> ranges;
  ranges.reserve(8 * params.size());
  const auto add = [&](const Tensor& x, bool written) {
    if (x.is_meta() || !x.numel()) return;
    const char* from = (const char*)x.const_data_ptr();
    ranges.push_back({from, from + x.nbytes(), written});
  };
  for (const at::TensorList list : {params, m, v, m_scales, v_scales, steps})
    for (const Tensor& x : list) add(x, true);
  for (size_t i = 0; i < params.size() && half; ++i)
    if (params[i].scalar_type() == at::kBFloat16) add(masters[i], true);
  for (const Tensor& x : g) add(x, false);
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
  const char *end = nullptr, *written_end = nullptr;     // of the ranges so far
  for (const Range& r : ranges) {
    TORCH_CHECK(r.from >= (r.written ? end : written_end), op, ": a tensor is given twice, or two tensors overlap");
    end = std::max(end, r.to);
    if (r.written) written_end = std::max(written_end, r.to);
  }
}

void adamw_any(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList m_scales, at::TensorList v,
               at::TensorList v_scales, at::TensorList steps, at::TensorList masters, const optional<Tensor>& norm,
               const optional<Tensor>& lr_tensor, double lr, double beta1, double beta2, double eps, double weight_decay,
               double max_norm, bool q8, const char* op) {
  std::vector<Tensor> g;
  for (const Tensor& p : params) TORCH_CHECK(p.is_cuda(), op, ": fsctep ops run on the GPU only (HIP kernels); got a ", p.device(), " tensor");
  adamw_check(params, grads, m, m_scales, v, v_scales, steps, masters, norm, lr_tensor, q8, op, g);
  std::vector<FscAdamTensor> t(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    const bool half = params[i].scalar_type() == at::kBFloat16;
    t[i] = FscAdamTensor{};
    t[i].n = params[i].numel();
    t[i].dtype = half ? FSC_BF16 : FSC_F32;
    t[i].step = (float*)steps[i].data_ptr();
    if (t[i].n == 0) continue;
    t[i].p = params[i].data_ptr();
    t[i].g = ptr(g[i]);
    t[i].m = m[i].data_ptr();
    t[i].v = v[i].data_ptr();
    if (q8) {
      t[i].m_scale = (float*)m_scales[i].data_ptr();
      t[i].v_scale = (float*)v_scales[i].data_ptr();
    }
    if (half) t[i].master = (float*)masters[i].data_ptr();
  }
  const c10::OptionalDeviceGuard device(params[0].device());
  int64_t bytes = 0, other = 0;
  check(fsc_adamw_workspace((int32_t)t.size(), t.data(), &bytes, &other), "fsc_adamw_workspace");
  Tensor ws = at::empty({bytes}, params[0].options().dtype(at::kByte));
  FscAdamSettings k{};
  k.lr = lr; k.beta1 = beta1; k.beta2 = beta2; k.eps = eps; k.weight_decay = weight_decay; k.max_norm = max_norm;
  k.lr_tensor = (const float*)ptr(some(lr_tensor));
  k.norm = (const float*)ptr(some(norm));
  k.bits = q8 ? 8 : 32;
  check(fsc_adamw_step((int32_t)t.size(), t.data(), &k, mptr(ws), stream_of(params[0])), "fsc_adamw_step");
  // autograd sees that they changed
  for (const at::TensorList list : {params, m, v, m_scales, v_scales, steps, masters})
    for (const Tensor& x : list)
      if (x.defined() && !x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

void adamw_(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList v, at::TensorList steps,
            at::TensorList masters, const optional<Tensor>& norm, const optional<Tensor>& lr_tensor, double lr, double beta1,
            double beta2, double eps, double weight_decay, double max_norm) {
  adamw_any(params, grads, m, {}, v, {}, steps, masters, norm, lr_tensor, lr, beta1, beta2, eps, weight_decay, max_norm, false,
            "adamw_");
}
void adamw_q8_(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList m_scales, at::TensorList v,
               at::TensorList v_scales, at::TensorList steps, at::TensorList masters, const optional<Tensor>& norm,
               const optional<Tensor>& lr_tensor, double lr, double beta1, double beta2, double eps, double weight_decay,
               double max_norm) {
  adamw_any(params, grads, m, m_scales, v, v_scales, steps, masters, norm, lr_tensor, lr, beta1, beta2, eps, weight_decay,
            max_norm, true, "adamw_q8_");
}
void adamw_meta(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList v, at::TensorList steps,
                at::TensorList masters, const optional<Tensor>& norm, const optional<Tensor>& lr_tensor, double, double, double,
                double, double, double) {
  std::vector<Tensor> g;
  adamw_check(params, grads, m, {}, v, {}, steps, masters, norm, lr_tensor, false, "adamw_", g);
}
void adamw_q8_meta(at::TensorList params, at::TensorList grads, at::TensorList m, at::TensorList m_scales, at::TensorList v,
                   at::TensorList v_scales, at::TensorList steps, at::TensorList masters, const optional<Tensor>& norm,
                   const optional<Tensor>& lr_tensor, double, double, double, double, double, double) {
  std::vector<Tensor> g;
  adamw_check(params, grads, m, m_scales, v, v_scales, steps, masters, norm, lr_tensor, true, "adamw_q8_", g);
}

void check_values(const Tensor& codes, const Tensor& scale) {
  TORCH_CHECK(codes.scalar_type() == at::kByte, "adamw_values: codes must be uint8, got ", codes.scalar_type());
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.dim() == 1 && scale.size(0) == (codes.numel() + kGroup - 1) / kGroup,
              "adamw_values: scale must be float32 of ", (codes.numel() + kGroup - 1) / kGroup, " values");
}
Tensor adamw_values(const Tensor& codes_, const Tensor& scale_, bool root) {
  require_gpu({codes_, scale_}, "adamw_values");
  check_values(codes_, scale_);
  const c10::OptionalDeviceGuard device(codes_.device());
  const Tensor codes = codes_.contiguous(), scale = scale_.contiguous();
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(at::kFloat));
  check(fsc_adamw_values(codes.numel(), root, (const uint8_t*)ptr(codes), (const float*)ptr(scale), (float*)mptr(out),
                         stream_of(codes)),
        "fsc_adamw_values");
  return out;
}
Tensor adamw_values_meta(const Tensor& codes, const Tensor& scale, bool) {
  check_values(codes, scale);
  return at::empty(codes.sizes(), codes.options().dtype(at::kFloat));
}

const char* const kNames[] = {"layer_norm", "layer_norm_backward", "layer_norm_backward_twice", "embedding",
                              "embedding_backward", "grad_norm", "adamw_", "adamw_q8_", "adamw_values"};

}  // namespace

TORCH_LIBRARY_FRAGMENT(fsctep, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, int activation, bool keep)"
        " -> (Tensor y, Tensor mean, Tensor rstd)");
  m.def("layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor mean, Tensor rstd, float eps,"
        " int activation, bool want_x, bool want_weight, bool want_bias, Tensor? plus=None, Tensor? through=None)"
        " -> (Tensor dx, Tensor dweight, Tensor dbias)");
  m.def("layer_norm_backward_twice(Tensor? v, Tensor? v_weight, Tensor? v_bias, Tensor dy, Tensor x, Tensor? weight,"
        " Tensor? bias, Tensor mean, Tensor rstd, float eps, int activation, bool want_x, bool want_dy, bool want_weight,"
        " bool want_bias) -> (Tensor grad_x, Tensor grad_dy, Tensor grad_weight, Tensor grad_bias)");
  m.def("embedding(Tensor table, Tensor index, float scale, float outside=0.) -> Tensor");
  m.def("embedding_backward(Tensor dy, Tensor index, SymInt table_rows, float scale) -> Tensor");
  m.def("grad_norm(Tensor[] grads) -> Tensor");
  m.def("adamw_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, Tensor(d!)[] steps,"
        " Tensor(e!)[] masters, Tensor? norm, Tensor? lr_tensor, float lr, float beta1, float beta2, float eps,"
        " float weight_decay, float max_norm) -> ()");
  m.def("adamw_q8_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_scale, Tensor(d!)[] root,"
        " Tensor(e!)[] root_scale, Tensor(f!)[] steps, Tensor(g!)[] masters, Tensor? norm, Tensor? lr_tensor, float lr,"
        " float beta1, float beta2, float eps, float weight_decay, float max_norm) -> ()");
  m.def("adamw_values(Tensor codes, Tensor scale, bool root) -> Tensor");
}

TORCH_LIBRARY_IMPL(fsctep, CUDA, m) {
  m.impl("layer_norm", layer_norm);
  m.impl("layer_norm_backward", layer_norm_backward);
  m.impl("layer_norm_backward_twice", layer_norm_backward_twice);
  m.impl("embedding", embedding);
  m.impl("embedding_backward", embedding_backward);
  m.impl("grad_norm", grad_norm);
  m.impl("adamw_", adamw_);
  m.impl("adamw_q8_", adamw_q8_);
  m.impl("adamw_values", adamw_values);
}

TORCH_LIBRARY_IMPL(fsctep, Meta, m) {
  m.impl("layer_norm", layer_norm_meta);
  m.impl("layer_norm_backward", layer_norm_backward_meta);
  m.impl("layer_norm_backward_twice", layer_norm_backward_twice_meta);
  m.impl("embedding", embedding_meta);
  m.impl("embedding_backward", embedding_backward_meta);
  m.impl("grad_norm", grad_norm_meta);
  m.impl("adamw_", adamw_meta);
  m.impl("adamw_q8_", adamw_q8_meta);
  m.impl("adamw_values", adamw_values_meta);
}

TORCH_LIBRARY_IMPL(fsctep, Autograd, m) {
  m.impl("layer_norm", layer_norm_autograd);
  m.impl("layer_norm_backward", layer_norm_backward_autograd);
  m.impl("embedding", embedding_autograd);
  m.impl("embedding_backward", embedding_backward_autograd);
  // a gradient of these is refused when it is asked for
  for (const char* name : {"layer_norm_backward_twice", "grad_norm", "adamw_values"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(fsctep, CPU, m) {
  for (const char* name : kNames) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse<kGpuOnly>>());
}
