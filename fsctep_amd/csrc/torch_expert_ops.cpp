// torch.ops.fsctep.* of the expert readout: norm, router and the experts' products on the C ABI of
// rms_norm.hip, expert_route.hip, expert_plan.hip and expert_mlp.hip.  Each op has device, Meta and, where it
// has a gradient, autograd kernels; calls run on the current stream, allocate their outputs and workspaces from
// the caching allocator and never wait for the GPU.  The backward ops have no gradient of their own: a double
// backward raises (fsctep_amd.train_ops has the twice differentiable forms).

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include <cmath>

#include "fsctep.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc, const char* name) { TORCH_CHECK(rc == 0, name, " failed (", rc, "): ", fsc_last_error()); }

const Tensor& some(const optional<Tensor>& t) {
  static const Tensor none;
  return t.has_value() ? *t : none;
}

void require_gpu(std::initializer_list<std::reference_wrapper<const Tensor>> ts, const char* name) {
  const Tensor& first = ts.begin()->get();
  for (const Tensor& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK(t.is_cuda(), name, ": fsctep ops run on the GPU only (HIP kernels); got a ", t.device(), " tensor");
    TORCH_CHECK(t.device() == first.device(), name, ": tensors on ", first.device(), " and ", t.device());
  }
}

int32_t code_of(at::ScalarType t, const char* name) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16, name, " must be float32 or bfloat16, got ", t);
  return t == at::kFloat ? FSC_F32 : FSC_BF16;
}

// (rows, width) with a contiguous last dimension; rows may lie at any non-negative stride.
Tensor rows2d(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be (rows, width), got ", t.dim(), " dimensions");
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= 0) ? t : t.contiguous();
}
int64_t stride_of(const Tensor& t) { return t.size(0) <= 1 ? 0 : t.stride(0); }
// the row stride of a single row is of no meaning: 0 keeps it aligned
const void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.const_data_ptr() : nullptr; }
void* mptr(Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

template <typename Sig>
auto op_handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

// Whether a call goes through its autograd function: a gradient is wanted, or an input carries a forward-mode tangent,
// which the function refuses (below autograd it would be lost).
bool differentiates(std::initializer_list<std::reference_wrapper<const Tensor>> ts) {
  for (const Tensor& t : ts)
    if (t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined())) return true;
  return false;
}

// A backward op's call: below autograd unless a gradient of the gradient may be asked for, which then raises.
struct BackwardGuard {
  optional<at::AutoDispatchBelowADInplaceOrView> below;
  BackwardGuard() {
    if (!at::GradMode::is_enabled()) below.emplace();
  }
};

// ============================================================== norm
struct NormDims {
  int64_t rows, width;
  int32_t dt, wt;
};

NormDims norm_dims(const Tensor& x, const Tensor& weight, const Tensor& residual, const char* name) {
  TORCH_CHECK(x.dim() == 2, name, ": x must be (rows, width), got ", x.dim(), " dimensions");
  TORCH_CHECK(x.size(1) >= 1, name, ": the width must be at least 1");
  const int32_t dt = code_of(x.scalar_type(), "x"), wt = code_of(weight.scalar_type(), "weight");
  TORCH_CHECK(wt == FSC_F32 || wt == dt, name, ": weight must be float32 or of x's type");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(1), name, ": weight must be (", x.size(1), ",)");
  if (residual.defined()) {
    TORCH_CHECK(residual.sizes() == x.sizes(), name, ": residual must have x's shape");
    TORCH_CHECK(residual.scalar_type() == x.scalar_type(), name, ": residual must have x's type");
  }
  return {x.size(0), x.size(1), dt, wt};
}

// (y, z, rstd); z is empty without a residual (it would be x)
std::tuple<Tensor, Tensor, Tensor> rms_norm(const Tensor& x_, const Tensor& weight_, const optional<Tensor>& residual_,
                                            double eps) {
  require_gpu({x_, weight_, some(residual_)}, "rms_norm");
  const NormDims d = norm_dims(x_, weight_, some(residual_), "rms_norm");
  const Tensor x = rows2d(x_, "x"), w = weight_.contiguous();
  const Tensor r = residual_.has_value() ? rows2d(*residual_, "residual") : Tensor();
  Tensor y = at::empty(x.sizes(), x.options()), z = at::empty(r.defined() ? x.sizes() : at::IntArrayRef({0}), x.options());
  Tensor rstd = at::empty({d.rows}, x.options().dtype(at::kFloat));
  check(fsc_rms_norm_forward(d.rows, (int32_t)d.width, d.dt, d.wt, stride_of(x), r.defined() ? stride_of(r) : 0, ptr(x),
                             ptr(r), ptr(w), (float)eps, mptr(y), mptr(z), (float*)mptr(rstd), stream_of(x)),
        "fsc_rms_norm_forward");
  return {y, z, rstd};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_meta(const Tensor& x, const Tensor& weight, const optional<Tensor>& residual,
                                                 double) {
  norm_dims(x, weight, some(residual), "rms_norm");
  return {at::empty_symint(x.sym_sizes(), x.options()),
          residual.has_value() ? at::empty_symint(x.sym_sizes(), x.options()) : at::empty({0}, x.options()),
          at::empty_symint({x.sym_size(0)}, x.options().dtype(at::kFloat))};
}

// (codes, scales, z)
std::tuple<Tensor, Tensor, Tensor> rms_norm_q8(const Tensor& x_, const Tensor& weight_,
                                               const optional<Tensor>& residual_, double eps) {
  require_gpu({x_, weight_, some(residual_)}, "rms_norm_q8");
  const NormDims d = norm_dims(x_, weight_, some(residual_), "rms_norm_q8");
  const Tensor x = rows2d(x_, "x"), w = weight_.contiguous();
  const Tensor r = residual_.has_value() ? rows2d(*residual_, "residual") : Tensor();
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
  Tensor z = at::empty(r.defined() ? x.sizes() : at::IntArrayRef({0}), x.options());
  Tensor scale = at::empty({d.rows}, x.options().dtype(at::kFloat));
  check(fsc_rms_norm_q8(d.rows, (int32_t)d.width, d.dt, d.wt, stride_of(x), r.defined() ? stride_of(r) : 0, ptr(x),
                        ptr(r), ptr(w), (float)eps, (int8_t*)mptr(q), (float*)mptr(scale), mptr(z), stream_of(x)),
        "fsc_rms_norm_q8");
  return {q, scale, z};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_q8_meta(const Tensor& x, const Tensor& weight,
                                                    const optional<Tensor>& residual, double) {
  norm_dims(x, weight, some(residual), "rms_norm_q8");
  return {at::empty_symint(x.sym_sizes(), x.options().dtype(at::kChar)),
          at::empty_symint({x.sym_size(0)}, x.options().dtype(at::kFloat)),
          residual.has_value() ? at::empty_symint(x.sym_sizes(), x.options()) : at::empty({0}, x.options())};
}

// (dx, dweight) from dy and, with a residual, dz; empty where not wanted
std::tuple<Tensor, Tensor> rms_norm_backward(const Tensor& dy_, const optional<Tensor>& dz_, const Tensor& z_,
                                             const Tensor& weight_, const Tensor& rstd, double eps, bool want_dx, bool want_dw) {
  require_gpu({z_, weight_, rstd, dy_, some(dz_)}, "rms_norm_backward");
  const NormDims d = norm_dims(z_, weight_, some(dz_), "rms_norm_backward");
  TORCH_CHECK(dy_.sizes() == z_.sizes() && dy_.scalar_type() == z_.scalar_type(),
              "rms_norm_backward: dy must have the rows' shape and type");
  const Tensor z = rows2d(z_, "z"), dy = rows2d(dy_, "dy"), w = weight_.contiguous();
  const Tensor dz = dz_.has_value() ? rows2d(*dz_, "dz") : Tensor();
  Tensor dx = want_dx ? at::empty(z.sizes(), z.options()) : at::empty({0}, z.options());
  Tensor dw = want_dw ? at::empty(w.sizes(), w.options()) : at::empty({0}, w.options());
  int64_t n = 0;
  check(fsc_rms_norm_workspace(d.rows, (int32_t)d.width, &n), "fsc_rms_norm_workspace");
  Tensor ws = at::empty({want_dw ? n : 0}, z.options().dtype(at::kFloat));
  check(fsc_rms_norm_backward(d.rows, (int32_t)d.width, d.dt, d.wt, stride_of(z), stride_of(dy),
                              dz.defined() ? stride_of(dz) : 0, ptr(z), ptr(w), (const float*)ptr(rstd), (float)eps, ptr(dy), ptr(dz),
                              mptr(dx), want_dw ? mptr(dw) : nullptr, (float*)mptr(ws), stream_of(z)),
        "fsc_rms_norm_backward");
  return {dx, dw};
}

std::tuple<Tensor, Tensor> rms_norm_backward_meta(const Tensor&, const optional<Tensor>&, const Tensor& z,
                                                  const Tensor& weight, const Tensor&, double, bool want_dx, bool want_dw) {
  return {want_dx ? at::empty_symint(z.sym_sizes(), z.options()) : at::empty({0}, z.options()),
          want_dw ? at::empty_symint(weight.sym_sizes(), weight.options()) : at::empty({0}, weight.options())};
}

auto& rms_norm_op() {
  static auto op = op_handle<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const optional<Tensor>&,
                                                                double)>("fsctep::rms_norm");
  return op;
}

struct RmsNormFn : public torch::autograd::Function<RmsNormFn> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, optional<Tensor> residual, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, z, rstd] = rms_norm_op().call(x, weight, residual, eps);
    ctx->save_for_backward({residual.has_value() ? z : x, weight, rstd});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    if (residual.has_value()) ctx->mark_non_differentiable({rstd});
    else ctx->mark_non_differentiable({z, rstd});
    return {y, z, rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto s = ctx->get_saved_variables();
    const bool res = ctx->saved_data["residual"].toBool();
    const bool want_x = ctx->needs_input_grad(0) || (res && ctx->needs_input_grad(2));
    const bool want_w = ctx->needs_input_grad(1);
    variable_list out(4);
    if (!grads[0].defined()) {       // nothing reached y: the sum's own gradient passes
      if (res && grads[1].defined()) out[0] = out[2] = grads[1];
      return out;
    }
    static auto op = op_handle<std::tuple<Tensor, Tensor>(const Tensor&, const optional<Tensor>&, const Tensor&,
                                                          const Tensor&, const Tensor&, double, bool, bool)>(
        "fsctep::rms_norm_backward");
    const optional<Tensor> dz = res && grads[1].defined() ? optional<Tensor>(grads[1]) : std::nullopt;
    BackwardGuard guard;
    auto [dx, dw] = op.call(grads[0], dz, s[0], s[1], s[2], ctx->saved_data["eps"].toDouble(), want_x, want_w);
    if (want_x) {
      out[0] = dx;
      if (res) out[2] = dx;
    }
    if (want_w) out[1] = dw;
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> rms_norm_autograd(const Tensor& x, const Tensor& weight,
                                                     const optional<Tensor>& residual, double eps) {
  if (differentiates({x, weight, some(residual)})) {
    auto r = RmsNormFn::apply(x, weight, residual, eps);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return rms_norm_op().call(x, weight, residual, eps);
}

// ============================================================== router
// What the router takes, the same on the GPU and on Meta tensors.
void check_route(const Tensor& l, const Tensor& bias, int64_t k, int64_t score, int64_t groups, int64_t kept, int64_t best,
                 double scale) {
  TORCH_CHECK(l.dim() == 2, "route_experts: logits must be (rows, experts), got ", l.dim(), " dimensions");
  code_of(l.scalar_type(), "logits");
  const auto experts = l.sym_size(1);
  TORCH_CHECK(experts >= 1 && experts <= 512, "route_experts: 1 to 512 experts, got ", experts);
  if (bias.defined()) {
    TORCH_CHECK(bias.dim() == 1 && bias.sym_size(0) == experts, "route_experts: bias must be (", experts, ",)");
    TORCH_CHECK(bias.scalar_type() == at::kFloat, "route_experts: bias must be float32, got ", bias.scalar_type());
  }
  TORCH_CHECK(score == 0 || score == 1, "route_experts: score is 0 (softmax) or 1 (sigmoid), got ", score);
  TORCH_CHECK(k >= 1 && k <= 16 && experts >= k, "route_experts: k must be 1 to 16 and at most the experts, got ", k);
  TORCH_CHECK(groups >= 1 && groups <= 128 && kept >= 1 && kept <= groups,
              "route_experts: groups must be 1 to 128 and groups_kept 1 to groups, got ", groups, " and ", kept);
  TORCH_CHECK(experts % groups == 0, "route_experts: groups must divide the experts, got ", groups, " and ", experts);
  TORCH_CHECK(experts / groups * kept >= k, "route_experts: k is more than the kept groups' experts, got ", k);
  TORCH_CHECK(best == 1 || best == 2, "route_experts: group_best is 1 or 2, got ", best);
  TORCH_CHECK(scale > 0 && std::isfinite((float)scale), "route_experts: scale must be positive and finite, got ", scale);
}

std::tuple<Tensor, Tensor> route_experts(const Tensor& logits_, const optional<Tensor>& bias_, int64_t k, int64_t score,
                                         int64_t groups, int64_t groups_kept, int64_t group_best, bool renormalise,
                                         double scale) {
  require_gpu({logits_, some(bias_)}, "route_experts");
  check_route(logits_, some(bias_), k, score, groups, groups_kept, group_best, scale);
  const Tensor l = rows2d(logits_, "logits"), b = bias_.has_value() ? bias_->contiguous() : Tensor();
  const int32_t dt = code_of(l.scalar_type(), "logits");
  Tensor index = at::empty({l.size(0), k}, l.options().dtype(at::kInt));
  Tensor weight = at::empty({l.size(0), k}, l.options().dtype(at::kFloat));
  check(fsc_route_experts(l.size(0), (int32_t)l.size(1), dt, stride_of(l), ptr(l), (const float*)ptr(b), (int32_t)k,
                          (int32_t)score, (int32_t)groups, (int32_t)groups_kept, (int32_t)group_best, renormalise,
                          (float)scale, (int32_t*)mptr(index), (float*)mptr(weight), stream_of(l)),
        "fsc_route_experts");
  return {index, weight};
}

std::tuple<Tensor, Tensor> route_experts_meta(const Tensor& l, const optional<Tensor>& bias, int64_t k, int64_t score,
                                              int64_t groups, int64_t kept, int64_t best, bool, double scale) {
  check_route(l, some(bias), k, score, groups, kept, best, scale);
  return {at::empty_symint({l.sym_size(0), k}, l.options().dtype(at::kInt)),
          at::empty_symint({l.sym_size(0), k}, l.options().dtype(at::kFloat))};
}

Tensor route_experts_backward(const Tensor& dweight_, const Tensor& logits_, const Tensor& index, const Tensor& weight,
                              int64_t score, bool renormalise, double scale) {
  require_gpu({logits_, index, weight, dweight_}, "route_experts_backward");
  const Tensor l = rows2d(logits_, "logits");
  const int32_t dt = code_of(l.scalar_type(), "logits");
  TORCH_CHECK(index.dim() == 2 && index.size(0) == l.size(0) && index.scalar_type() == at::kInt &&
                  weight.sizes() == index.sizes() && weight.scalar_type() == at::kFloat &&
                  dweight_.sizes() == index.sizes(),
              "route_experts_backward: index (int32), weight and dweight (float32) must be (rows, k)");
  const Tensor i = index.contiguous(), w = weight.contiguous(), dw = dweight_.to(at::kFloat).contiguous();
  Tensor dl = at::empty(l.sizes(), l.options());
  check(fsc_route_experts_backward(l.size(0), (int32_t)l.size(1), dt, stride_of(l), ptr(l), (const int32_t*)ptr(i),
                                   (const float*)ptr(w), (const float*)ptr(dw), (int32_t)i.size(1), (int32_t)score,
                                   renormalise, (float)scale, mptr(dl), stream_of(l)),
        "fsc_route_experts_backward");
  return dl;
}

Tensor route_experts_backward_meta(const Tensor&, const Tensor& l, const Tensor&, const Tensor&, int64_t, bool, double) {
  return at::empty_symint(l.sym_sizes(), l.options());
}

auto& route_op() {
  static auto op = op_handle<std::tuple<Tensor, Tensor>(const Tensor&, const optional<Tensor>&, int64_t, int64_t, int64_t,
                                                        int64_t, int64_t, bool, double)>("fsctep::route_experts");
  return op;
}

struct RouteFn : public torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, Tensor logits, optional<Tensor> bias, int64_t k, int64_t score,
                               int64_t groups, int64_t kept, int64_t best, bool renormalise, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [index, weight] = route_op().call(logits, bias, k, score, groups, kept, best, renormalise, scale);
    ctx->save_for_backward({logits, index, weight});
    ctx->saved_data["score"] = score;
    ctx->saved_data["renormalise"] = renormalise;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({index});
    return {index, weight};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    // the bias chooses and does not weigh: it has no gradient
    if (!grads[1].defined() || !ctx->needs_input_grad(0)) return out;
    auto s = ctx->get_saved_variables();
    static auto op = op_handle<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, bool, double)>(
        "fsctep::route_experts_backward");
    BackwardGuard guard;
    out[0] = op.call(grads[1], s[0], s[1], s[2], ctx->saved_data["score"].toInt(),
                     ctx->saved_data["renormalise"].toBool(), ctx->saved_data["scale"].toDouble());
    return out;
  }
};

std::tuple<Tensor, Tensor> route_experts_autograd(const Tensor& logits, const optional<Tensor>& bias, int64_t k,
                                                  int64_t score, int64_t groups, int64_t kept, int64_t best,
                                                  bool renormalise, double scale) {
  if (differentiates({logits})) {
    auto r = RouteFn::apply(logits, bias, k, score, groups, kept, best, renormalise, scale);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return route_op().call(logits, bias, k, score, groups, kept, best, renormalise, scale);
}

// ============================================================== the experts' products
struct Sizes {
  int64_t plan = 0, saved = 0, fwd = 0, bwd = 0;
};

// What the products take, the same on the GPU and on Meta tensors (of sizes that a trace does not know yet, too).
void check_products(const Tensor& x, const Tensor& index, const Tensor& weight, const Tensor& w_in, const Tensor& w_out,
                    const char* name, bool q8 = false) {
  TORCH_CHECK(x.dim() == 2, name, ": x must be (rows, width), got ", x.dim(), " dimensions");
  if (q8) {
    TORCH_CHECK(x.scalar_type() == at::kChar, name, ": x must be int8 codes, got ", x.scalar_type());
  } else {
    code_of(x.scalar_type(), "x");
  }
  const auto rows = x.sym_size(0), width = x.sym_size(1);
  TORCH_CHECK(w_out.dim() == 3 && w_out.sym_size(1) == width, name, ": w_out must be (experts, ", width, ", hidden)");
  const auto experts = w_out.sym_size(0), hidden = w_out.sym_size(2);
  TORCH_CHECK(w_in.dim() == 3 && w_in.sym_size(0) == experts && w_in.sym_size(1) == hidden * 2 && w_in.sym_size(2) == width,
              name, ": w_in must be (", experts, ", ", hidden * 2, ", ", width, ")");
  TORCH_CHECK(index.dim() == 2 && index.sym_size(0) == rows && index.sym_size(1) >= 1, name, ": index must be (", rows, ", k)");
  TORCH_CHECK(index.scalar_type() == at::kInt, name, ": index must be int32, got ", index.scalar_type());
  TORCH_CHECK(weight.sym_sizes() == index.sym_sizes(), name, ": weight must have index's shape");
  TORCH_CHECK(weight.scalar_type() == at::kFloat, name, ": weight must be float32, got ", weight.scalar_type());
  TORCH_CHECK(w_in.scalar_type() == x.scalar_type() && w_out.scalar_type() == x.scalar_type(), name,
              ": x, w_in and w_out must have one type");
  TORCH_CHECK(width >= 1 && width <= (1 << 17) && hidden >= 1 && hidden <= (1 << 17), name,
              ": width and hidden must be 1 to 2^17");
  TORCH_CHECK(experts >= 1 && experts <= 512, name, ": 1 to 512 experts, got ", experts);
  TORCH_CHECK(index.sym_size(1) <= 64, name, ": at most 64 slots a row, got ", index.sym_size(1));
}

FscExpertDims expert_dims(const Tensor& x, const Tensor& index, const Tensor& weight, const Tensor& w_in,
                          const Tensor& w_out, const char* name, bool q8 = false) {
  check_products(x, index, weight, w_in, w_out, name, q8);
  const int32_t dt = q8 ? FSC_I8 : code_of(x.scalar_type(), "x");
  return {x.size(0), (int32_t)x.size(1), (int32_t)w_out.size(2), (int32_t)w_out.size(0), (int32_t)index.size(1), dt};
}

Sizes sizes_of(const FscExpertDims& d) {
  Sizes s;
  check(fsc_expert_sizes(&d, &s.plan, &s.saved, &s.fwd, &s.bwd), "fsc_expert_sizes");
  return s;
}

// Rows of the products by tiles (those with a plan).  fp32 rows that lie too far apart for one buffer of 32-bit offsets
// would be read value by value: packed first where that brings them into one (10,000 rows of 640 over 4 GB, two of eight
// experts: forward 247 us against 528).  16- and 8-bit rows are copied by the products themselves.
Tensor product_rows(const Tensor& t, const char* name, const Sizes& s) {
  constexpr int64_t kReach = 0xF0000000;
  const Tensor r = rows2d(t, name);
  if (s.plan == 0 || r.scalar_type() != at::kFloat || r.numel() * 4 >= kReach) return r;
  return ((r.size(0) - 1) * r.stride(0) + r.size(1)) * 4 < kReach ? r : r.contiguous();
}

// (y, plan, saved): plan and saved are what the backward takes; saved is empty without `keep`
std::tuple<Tensor, Tensor, Tensor> expert_mlp_forward(const Tensor& x_, const Tensor& index_, const Tensor& weight_,
                                                      const Tensor& w_in_, const Tensor& w_out_, bool keep) {
  require_gpu({x_, index_, weight_, w_in_, w_out_}, "expert_mlp");
  const FscExpertDims d = expert_dims(x_, index_, weight_, w_in_, w_out_, "expert_mlp");
  const Sizes s = sizes_of(d);
  const Tensor x = product_rows(x_, "x", s), index = index_.contiguous(), weight = weight_.contiguous();
  const Tensor w_in = w_in_.contiguous(), w_out = w_out_.contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor plan = at::empty({s.plan}, index.options());
  Tensor saved = at::empty({keep ? s.saved : 0}, weight.options());
  Tensor ws = at::empty({s.fwd}, x.options().dtype(at::kByte));
  check(fsc_expert_plan(&d, (const int32_t*)ptr(index), (int32_t*)mptr(plan), stream_of(x)), "fsc_expert_plan");
  check(fsc_expert_mlp_forward(&d, stride_of(x), ptr(x), (const int32_t*)ptr(index), (const int32_t*)ptr(plan),
                               (const float*)ptr(weight), ptr(w_in), ptr(w_out), (float*)mptr(saved), mptr(ws), mptr(y), stream_of(x)),
        "fsc_expert_mlp_forward");
  return {y, plan, saved};
}

std::tuple<Tensor, Tensor, Tensor> expert_mlp_forward_meta(const Tensor& x, const Tensor& index, const Tensor& weight,
                                                           const Tensor& w_in, const Tensor& w_out, bool keep) {
  const FscExpertDims d = expert_dims(x, index, weight, w_in, w_out, "expert_mlp");
  const Sizes s = sizes_of(d);
  return {at::empty(x.sizes(), x.options()), at::empty({s.plan}, index.options()),
          at::empty({keep ? s.saved : 0}, weight.options())};
}

// (dx, dweight, dw_in, dw_out), empty where not wanted
std::tuple<Tensor, Tensor, Tensor, Tensor> expert_mlp_backward(const Tensor& dy_, const Tensor& x_, const Tensor& index_,
                                                               const Tensor& weight_, const Tensor& w_in_,
                                                               const Tensor& w_out_, const Tensor& plan,
                                                               const Tensor& saved, bool want_x, bool want_weight,
                                                               bool want_in, bool want_out) {
  require_gpu({x_, dy_, index_, weight_, w_in_, w_out_, plan, saved}, "expert_mlp_backward");
  const FscExpertDims d = expert_dims(x_, index_, weight_, w_in_, w_out_, "expert_mlp_backward");
  TORCH_CHECK(dy_.sizes() == x_.sizes() && dy_.scalar_type() == x_.scalar_type(),
              "expert_mlp_backward: dy must have x's shape and type");
  const Sizes s = sizes_of(d);
  const Tensor x = product_rows(x_, "x", s), dy = product_rows(dy_, "dy", s);
  const Tensor index = index_.contiguous(), weight = weight_.contiguous(), w_in = w_in_.contiguous(), w_out = w_out_.contiguous();
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.is_contiguous() && plan.numel() == s.plan &&
                  saved.scalar_type() == at::kFloat && saved.is_contiguous() && saved.numel() == s.saved,
              "expert_mlp_backward: plan and saved must be the forward's (with keep)");
  auto out = [](bool want, const Tensor& like) {
    return want ? at::empty(like.sizes(), like.options()) : at::empty({0}, like.options());
  };
  Tensor dx = out(want_x, x), dweight = out(want_weight, weight), dw_in = out(want_in, w_in), dw_out = out(want_out, w_out);
  Tensor ws = at::empty({s.bwd}, x.options().dtype(at::kByte));
  check(fsc_expert_mlp_backward(&d, stride_of(x), stride_of(dy), ptr(dy), ptr(x), (const int32_t*)ptr(index), (const int32_t*)ptr(plan),
                                (const float*)ptr(weight), ptr(w_in), ptr(w_out), (const float*)ptr(saved), mptr(ws),
                                mptr(dx), (float*)mptr(dweight), mptr(dw_in), mptr(dw_out), stream_of(x)),
        "fsc_expert_mlp_backward");
  return {dx, dweight, dw_in, dw_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> expert_mlp_backward_meta(const Tensor&, const Tensor& x, const Tensor&,
                                                                    const Tensor& weight, const Tensor& w_in,
                                                                    const Tensor& w_out, const Tensor&, const Tensor&,
                                                                    bool want_x, bool want_weight, bool want_in,
                                                                    bool want_out) {
  auto out = [](bool want, const Tensor& like) {
    return want ? at::empty(like.sizes(), like.options()) : at::empty({0}, like.options());
  };
  return {out(want_x, x), out(want_weight, weight), out(want_in, w_in), out(want_out, w_out)};
}

using ForwardSig = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                      const Tensor&, bool);

struct ExpertMlpFn : public torch::autograd::Function<ExpertMlpFn> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor index, Tensor weight, Tensor w_in, Tensor w_out) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = op_handle<ForwardSig>("fsctep::expert_mlp_forward");
    auto [y, plan, saved] = op.call(x, index, weight, w_in, w_out, true);
    ctx->save_for_backward({x, index, weight, w_in, w_out, plan, saved});
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    auto s = ctx->get_saved_variables();
    static auto op = op_handle<std::tuple<Tensor, Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
        const Tensor&, bool, bool, bool, bool)>("fsctep::expert_mlp_backward");
    const bool want[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(2), ctx->needs_input_grad(3),
                          ctx->needs_input_grad(4)};
    BackwardGuard guard;
    auto [dx, dweight, dw_in, dw_out] =
        op.call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], want[0], want[1], want[2], want[3]);
    if (want[0]) out[0] = dx;
    if (want[1]) out[2] = dweight;
    if (want[2]) out[3] = dw_in;
    if (want[3]) out[4] = dw_out;
    return out;
  }
};

Tensor expert_mlp(const Tensor& x, const Tensor& index, const Tensor& weight, const Tensor& w_in, const Tensor& w_out) {
  static auto op = op_handle<ForwardSig>("fsctep::expert_mlp_forward");
  return std::get<0>(op.call(x, index, weight, w_in, w_out, false));
}

// The values before the activation are kept only where a gradient will ask for them.
Tensor expert_mlp_autograd(const Tensor& x, const Tensor& index, const Tensor& weight, const Tensor& w_in,
                           const Tensor& w_out) {
  if (differentiates({x, weight, w_in, w_out}))
    return ExpertMlpFn::apply(x, index, weight, w_in, w_out)[0];
  at::AutoDispatchBelowADInplaceOrView guard;
  return expert_mlp(x, index, weight, w_in, w_out);
}

// A scale for each row of codes.
void check_scales(const Tensor& scale, const Tensor& codes, const char* name) {
  const auto shape = codes.sym_sizes().slice(0, codes.dim() - 1);
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.sym_sizes() == shape, "expert_mlp_q8: ", name,
              " must be float32 of shape ", shape);
}

Tensor expert_mlp_q8(const Tensor& x_, const Tensor& x_scale_, const Tensor& index_, const Tensor& weight_,
                     const Tensor& w_in_, const Tensor& w_in_scale_, const Tensor& w_out_, const Tensor& w_out_scale_) {
  require_gpu({x_, x_scale_, index_, weight_, w_in_, w_in_scale_, w_out_, w_out_scale_}, "expert_mlp_q8");
  const FscExpertDims d = expert_dims(x_, index_, weight_, w_in_, w_out_, "expert_mlp_q8", true);
  check_scales(x_scale_, x_, "x_scale");
  check_scales(w_in_scale_, w_in_, "w_in_scale");
  check_scales(w_out_scale_, w_out_, "w_out_scale");
  const Tensor xs = x_scale_.contiguous(), is = w_in_scale_.contiguous(), os = w_out_scale_.contiguous();
  const Tensor x = rows2d(x_, "x"), index = index_.contiguous(), weight = weight_.contiguous();
  const Tensor w_in = w_in_.contiguous(), w_out = w_out_.contiguous();
  const Sizes s = sizes_of(d);
  Tensor y = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
  Tensor plan = at::empty({s.plan}, index.options());
  Tensor ws = at::empty({s.fwd}, x.options().dtype(at::kByte));
  check(fsc_expert_plan(&d, (const int32_t*)ptr(index), (int32_t*)mptr(plan), stream_of(x)), "fsc_expert_plan");
  check(fsc_expert_mlp_q8(&d, stride_of(x), (const int8_t*)ptr(x), (const float*)ptr(xs), (const int32_t*)ptr(index), (const int32_t*)ptr(plan),
                          (const float*)ptr(weight), (const int8_t*)ptr(w_in), (const float*)ptr(is),
                          (const int8_t*)ptr(w_out), (const float*)ptr(os), mptr(ws), mptr(y), stream_of(x)),
        "fsc_expert_mlp_q8");
  return y;
}

Tensor expert_mlp_q8_meta(const Tensor& x, const Tensor& x_scale, const Tensor& index, const Tensor& weight,
                          const Tensor& w_in, const Tensor& w_in_scale, const Tensor& w_out, const Tensor& w_out_scale) {
  check_products(x, index, weight, w_in, w_out, "expert_mlp_q8", true);
  check_scales(x_scale, x, "x_scale");
  check_scales(w_in_scale, w_in, "w_in_scale");
  check_scales(w_out_scale, w_out, "w_out_scale");
  return at::empty_symint(x.sym_sizes(), x.options().dtype(at::kBFloat16));
}

Tensor expert_mlp_meta(const Tensor& x, const Tensor& index, const Tensor& weight, const Tensor& w_in, const Tensor& w_out) {
  check_products(x, index, weight, w_in, w_out, "expert_mlp");
  return at::empty_symint(x.sym_sizes(), x.options());
}

template <const char* const& NAME>
void refuse(const c10::OperatorHandle& op, torch::jit::Stack*) {
  TORCH_CHECK(false, op.schema().name(), ": ", NAME);
}
const char* const kGpuOnly = "fsctep ops run on the GPU only (HIP kernels)";

}  // namespace

TORCH_LIBRARY_FRAGMENT(fsctep, m) {
  m.def("rms_norm(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor y, Tensor z, Tensor rstd)");
  m.def("rms_norm_backward(Tensor dy, Tensor? dz, Tensor z, Tensor weight, Tensor rstd, float eps, bool want_dx,"
        " bool want_dw)"
        " -> (Tensor dx, Tensor dweight)");
  m.def("rms_norm_q8(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor codes, Tensor scale, Tensor z)");
  m.def("route_experts(Tensor logits, Tensor? bias, int k, int score, int groups, int groups_kept, int group_best,"
        " bool renormalise, float scale) -> (Tensor index, Tensor weight)");
  m.def("route_experts_backward(Tensor dweight, Tensor logits, Tensor index, Tensor weight, int score,"
        " bool renormalise, float scale) -> Tensor");
  m.def("expert_mlp(Tensor x, Tensor index, Tensor weight, Tensor w_in, Tensor w_out) -> Tensor");
  m.def("expert_mlp_forward(Tensor x, Tensor index, Tensor weight, Tensor w_in, Tensor w_out, bool keep)"
        " -> (Tensor y, Tensor plan, Tensor saved)");
  m.def("expert_mlp_backward(Tensor dy, Tensor x, Tensor index, Tensor weight, Tensor w_in, Tensor w_out, Tensor plan,"
        " Tensor saved, bool want_x, bool want_weight, bool want_in, bool want_out)"
        " -> (Tensor dx, Tensor dweight, Tensor dw_in, Tensor dw_out)");
  m.def("expert_mlp_q8(Tensor x, Tensor x_scale, Tensor index, Tensor weight, Tensor w_in, Tensor w_in_scale,"
        " Tensor w_out, Tensor w_out_scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(fsctep, CUDA, m) {
  m.impl("rms_norm", rms_norm);
  m.impl("rms_norm_backward", rms_norm_backward);
  m.impl("rms_norm_q8", rms_norm_q8);
  m.impl("route_experts", route_experts);
  m.impl("route_experts_backward", route_experts_backward);
  m.impl("expert_mlp", expert_mlp);
  m.impl("expert_mlp_forward", expert_mlp_forward);
  m.impl("expert_mlp_backward", expert_mlp_backward);
  m.impl("expert_mlp_q8", expert_mlp_q8);
}

TORCH_LIBRARY_IMPL(fsctep, Meta, m) {
  m.impl("rms_norm", rms_norm_meta);
  m.impl("rms_norm_backward", rms_norm_backward_meta);
  m.impl("rms_norm_q8", rms_norm_q8_meta);
  m.impl("route_experts", route_experts_meta);
  m.impl("route_experts_backward", route_experts_backward_meta);
  m.impl("expert_mlp", expert_mlp_meta);
  m.impl("expert_mlp_forward", expert_mlp_forward_meta);
  m.impl("expert_mlp_backward", expert_mlp_backward_meta);
  m.impl("expert_mlp_q8", expert_mlp_q8_meta);
}

TORCH_LIBRARY_IMPL(fsctep, Autograd, m) {
  m.impl("rms_norm", rms_norm_autograd);
  m.impl("route_experts", route_experts_autograd);
  m.impl("expert_mlp", expert_mlp_autograd);
  // a gradient of these is refused when it is asked for
  for (const char* name : {"rms_norm_backward", "rms_norm_q8", "route_experts_backward", "expert_mlp_forward",
                           "expert_mlp_backward", "expert_mlp_q8"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

TORCH_LIBRARY_IMPL(fsctep, CPU, m) {
  for (const char* name : {"rms_norm", "rms_norm_backward", "rms_norm_q8", "route_experts", "route_experts_backward",
                           "expert_mlp", "expert_mlp_forward", "expert_mlp_backward", "expert_mlp_q8"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse<kGpuOnly>>());
}
