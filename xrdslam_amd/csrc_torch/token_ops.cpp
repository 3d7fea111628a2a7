// torch.ops.xrdslam.{plan, lookup, linear}: the token and grouped-product entry
// points (xrd_token_*, xrd_lookup_*, xrd_grouped_*) as differentiable torch
// operators.  Host code only: allocation, the autograd node and the C calls.
// (As Python autograd functions over ctypes a forward and backward pass of a
// layer cost 103 us of host time, more than the kernels of a mapping batch.)
//
// Every launch sits behind an operator of its own under the device's dispatch
// key (lookup_grads and linear_grads are those of the backward passes), the
// nodes under the autograd key: whatever works by dispatch - tracing, negated
// views, function transforms - sees the operators and not their allocations.
// Forward-mode tangents have no formula here and are refused.
//
// Arguments are checked by xrdslam_amd/engine/{tokens,grouped}.py, the only
// callers; a status other than XRD_OK becomes a RuntimeError.  Every buffer,
// workspaces included, comes from torch's allocator on the current stream.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "xrdslam_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check(int status, const char* what) {
  if (status == XRD_OK) return;
  const char* kind = status == XRD_ERR_ARG           ? "bad argument"
                     : status == XRD_ERR_UNSUPPORTED ? "unsupported configuration"
                                                     : "HIP launch/runtime error";
  TORCH_CHECK(false, what, ": ", kind,
              status == XRD_ERR_LAUNCH ? " (" : "",
              status == XRD_ERR_LAUNCH ? xrd_last_error() : "",
              status == XRD_ERR_LAUNCH ? ")" : "");
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return XRD_F32;
    case at::kBFloat16: return XRD_BF16;
    case at::kHalf: return XRD_F16;
    default: return -1;
  }
}

// columns side by side, rows apart by up to a million elements (the kernels'
// 32-bit offsets)
Tensor dense_rows(const Tensor& t) {
  if (t.is_contiguous()) return t;
  const bool rows = t.stride(0) >= 0 && t.stride(0) <= (1 << 20) &&
                    (t.stride(1) == 1 || t.size(1) == 1);
  return rows ? t : t.contiguous();
}

Tensor workspace(int64_t n, const Tensor& like, at::ScalarType type) {
  return at::empty({n}, like.options().dtype(type));
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* address(const optional<Tensor>& t) {
  return t.has_value() && t->defined() ? t->data_ptr() : nullptr;
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const optional<Tensor>& t) {
  return t.has_value() && wants_grad(*t);
}

optional<Tensor> given(const Tensor& t) {
  return t.defined() ? optional<Tensor>(t) : std::nullopt;
}

// The C entry points count k, columns and groups in 32 bits: a size that does
// not fit would arrive there as another one.  (Checked in front of anything that
// copies: an expanded tensor of that size holds one element.)
void refuse_wide(const char* what, std::initializer_list<int64_t> sizes) {
  for (int64_t s : sizes)
    if (s > INT32_MAX) check(XRD_ERR_UNSUPPORTED, what);
}

// a derivative of the operator along a direction would be needed: without this
// a dual tensor would lose its tangent and its derivative read as zero
void refuse_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK(!torch::autograd::isFwGradDefined(t), what,
              ": forward-mode derivatives are not supported");
}
void refuse_tangent(const char* what, const optional<Tensor>& t) {
  if (t.has_value()) refuse_tangent(what, *t);
}

// the operator of that name, to be called below the autograd keys
template <typename F>
c10::TypedOperatorHandle<F> operator_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// the results of a backward pass that has none of its own: differentiating
// them raises instead of giving wrong numbers
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (auto& g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that can be differentiated "
      "once",
      (int64_t)some.size());
  some = error->apply(std::move(some));
  size_t next = 0;
  for (auto& g : grads)
    if (g.defined()) g = some[next++];
  return grads;
}

// ------------------------------------------------------------------- plan
int64_t plan_words(int64_t n, int64_t n_groups) {
  const int64_t words = xrd_token_plan_ws_ints(n, n_groups);
  if (words < 0) check(XRD_ERR_UNSUPPORTED, "xrd_token_plan");
  return words;
}

std::tuple<Tensor, Tensor, Tensor> plan(const Tensor& ids_, int64_t n_groups,
                                        bool want_rank) {
  const c10::DeviceGuard guard(ids_.device());
  const Tensor ids = ids_.contiguous();
  const int64_t n = ids.numel();
  const Tensor ws = workspace(plan_words(n, n_groups), ids, at::kInt);
  Tensor order = workspace(n, ids, at::kInt);
  Tensor starts = workspace(n_groups + 1, ids, at::kInt);
  Tensor rank = workspace(want_rank ? n : 0, ids, at::kInt);
  check(xrd_token_plan(n, n_groups, ids.data_ptr(), (int)ids.element_size(),
                       order.data_ptr<int>(), starts.data_ptr<int>(),
                       want_rank ? rank.data_ptr<int>() : nullptr,
                       ws.data_ptr<int>(), stream_of(ids)),
        "xrd_token_plan");
  return {order, starts, rank};
}

// ------------------------------------------------------------------ lookup
Tensor plain_weights(const Tensor& w) { return w.to(at::kFloat).contiguous(); }

Tensor lookup(const Tensor& table_, const Tensor& ids_,
              const optional<Tensor>& weights_, double scale,
              const optional<Tensor>&, const optional<Tensor>&) {
  refuse_wide("xrd_lookup_fwd",
              {table_.size(1), weights_.has_value() ? ids_.size(-1) : 1});
  const c10::DeviceGuard guard(table_.device());
  const Tensor table = dense_rows(table_), ids = ids_.contiguous();
  Tensor weights;
  int64_t k = 1;
  auto shape = ids.sizes().vec();
  if (weights_.has_value()) {
    weights = plain_weights(*weights_);
    k = shape.back();
    shape.pop_back();
  }
  const int64_t n = ids.numel() / k, dim = table.size(1);
  shape.push_back(dim);
  Tensor out = at::empty(shape, table.options());
  check(xrd_lookup_fwd(dtype_of(table), n, (int)k, table.size(0), (int)dim,
                       table.data_ptr(), table.stride(0), ids.data_ptr(),
                       (int)ids.element_size(), (const float*)address(weights),
                       (float)scale, out.data_ptr(), stream_of(table)),
        "xrd_lookup_fwd");
  return out;
}

// the gradients of the table (from the ids' plan, made here if none is given)
// and of the weights (from the table); undefined where not needed
std::tuple<Tensor, Tensor> lookup_grads(
    const Tensor& dout_, const optional<Tensor>& table_, const Tensor& ids_,
    const optional<Tensor>& weights_, double scale,
    const optional<Tensor>& order_, const optional<Tensor>& starts_,
    int64_t rows, bool need_table, bool need_weights) {
  const c10::DeviceGuard guard(dout_.device());
  const Tensor ids = ids_.contiguous();
  Tensor weights;
  int64_t k = 1;
  if (weights_.has_value()) {
    weights = plain_weights(*weights_);
    k = ids.size(-1);
  }
  const int64_t n = ids.numel() / k, dim = dout_.size(-1);
  const Tensor dout = dense_rows(dout_.reshape({n, dim}));
  const int dtype = dtype_of(dout), id_bytes = (int)ids.element_size();
  const int32_t* order = (const int32_t*)address(order_);
  const int32_t* starts = (const int32_t*)address(starts_);
  Tensor table, dtable, dw, ws;   // ws: partial sums, then the plan if none
  if (need_table) {               // was given (an allocation costs 1 us)
    const int64_t sums = xrd_lookup_bwd_ws_floats(n, (int)k, (int)dim);
    if (sums < 0) check(XRD_ERR_UNSUPPORTED, "xrd_lookup_bwd");
    if (order_.has_value()) {
      ws = workspace(sums, dout, at::kInt);
    } else {
      const int64_t groups = rows > 0 ? rows : 1, t = ids.numel();
      ws = workspace(sums + t + groups + 1 + plan_words(t, groups), dout,
                     at::kInt);
      int* const o = ws.data_ptr<int>() + sums;
      check(xrd_token_plan(t, groups, ids.data_ptr(), id_bytes, o, o + t,
                           nullptr, o + t + groups + 1, stream_of(dout)),
            "xrd_token_plan");
      order = o, starts = o + t;
    }
    dtable = at::empty({rows, dim}, dout.options());
  }
  if (need_weights) {
    table = dense_rows(*table_);
    dw = at::empty(weights.sizes(), weights.options());
  }
  check(xrd_lookup_bwd(
            dtype, n, (int)k, rows, (int)dim, address(table),
            need_weights ? table.stride(0) : 0, ids.data_ptr(), id_bytes,
            (const float*)address(weights), dout.data_ptr(), dout.stride(0),
            order, starts, (float)scale,
            need_table ? dtable.data_ptr() : nullptr, (float*)address(dw),
            (float*)address(ws), stream_of(dout)),
        "xrd_lookup_bwd");
  return {dtable, dw};
}

class Lookup : public torch::autograd::Function<Lookup> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& table,
                        const Tensor& ids, const optional<Tensor>& weights,
                        double scale, const optional<Tensor>& order,
                        const optional<Tensor>& starts) {
    static const auto op = operator_of<decltype(lookup)>("xrdslam::lookup");
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rows"] = table.size(0);
    // the table is needed for the weights' gradient alone
    ctx->save_for_backward({wants_grad(weights) ? table : Tensor(), ids,
                            weights.value_or(Tensor()),
                            order.value_or(Tensor()),
                            starts.value_or(Tensor())});
    const at::AutoDispatchBelowADInplaceOrView below;
    return op.call(table, ids, weights, scale, order, starts);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op =
        operator_of<decltype(lookup_grads)>("xrdslam::lookup_grads");
    refuse_tangent("xrd_lookup_bwd", grads[0]);
    const auto saved = ctx->get_saved_variables();
    // (numbered by the tensors that were given: ids is 1, weights 2)
    const bool need_table = ctx->needs_input_grad(0);
    const bool need_w = saved[2].defined() && ctx->needs_input_grad(2);
    Tensor dtable, dw;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dtable, dw) = op.call(
          grads[0], given(saved[0]), saved[1], given(saved[2]),
          ctx->saved_data["scale"].toDouble(), given(saved[3]),
          given(saved[4]), ctx->saved_data["rows"].toInt(), need_table, need_w);
    }
    return once({dtable, Tensor(), dw, Tensor(), Tensor(), Tensor()});
  }
};

Tensor lookup_autograd(const Tensor& table, const Tensor& ids_,
                       const optional<Tensor>& weights_, double scale,
                       const optional<Tensor>& order,
                       const optional<Tensor>& starts) {
  static const auto op = operator_of<decltype(lookup)>("xrdslam::lookup");
  refuse_wide("xrd_lookup_fwd",
              {table.size(1), weights_.has_value() ? ids_.size(-1) : 1});
  refuse_tangent("xrd_lookup_fwd", table);
  refuse_tangent("xrd_lookup_fwd", weights_);
  if (at::GradMode::is_enabled() &&
      (wants_grad(table) || wants_grad(weights_))) {
    const Tensor ids = ids_.contiguous();
    optional<Tensor> weights;
    if (weights_.has_value()) weights = plain_weights(*weights_);
    return Lookup::apply(table, ids, weights, scale, order, starts);
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(table, ids_, weights_, scale, order, starts);
}

// ------------------------------------------------------------------ linear
Tensor linear(const Tensor& x_, const Tensor& weight_, const Tensor& starts,
              const optional<Tensor>& bias_, bool relu) {
  refuse_wide("xrd_grouped_fwd",
              {weight_.size(0), weight_.size(1), weight_.size(2)});
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = dense_rows(x_), weight = weight_.contiguous();
  Tensor bias;
  if (bias_.has_value()) bias = bias_->contiguous();
  const int64_t m = x.size(0), n_out = weight.size(1);
  Tensor y = at::empty({m, n_out}, x.options());
  check(xrd_grouped_fwd(dtype_of(x), m, (int)weight.size(0), (int)x.size(1),
                        (int)n_out, x.data_ptr(), x.stride(0),
                        weight.data_ptr(), address(bias),
                        starts.data_ptr<int>(), relu, y.data_ptr(),
                        stream_of(x)),
        "xrd_grouped_fwd");
  return y;
}

// the gradients of x (from the weight), of the weight and of the bias (from
// x); y: the result, if a ReLU was applied.  Undefined where not needed.
std::tuple<Tensor, Tensor, Tensor> linear_grads(
    const Tensor& dout, const optional<Tensor>& x_,
    const optional<Tensor>& weight_, const Tensor& starts,
    const optional<Tensor>& y, int64_t n_groups, int64_t in, bool need_x,
    bool need_w, bool need_b) {
  const c10::DeviceGuard guard(dout.device());
  Tensor dz = dense_rows(dout), dx, dw, db;
  const int dtype = dtype_of(dz);
  const auto options = dz.options();
  const int64_t m = dz.size(0);
  const int e = (int)n_groups, n_in = (int)in, n_out = (int)dz.size(1);
  void* st = stream_of(dz);
  const int* sp = starts.data_ptr<int>();
  if (y.has_value()) {
    const Tensor result = y->contiguous();
    Tensor masked = at::empty({m, n_out}, options);
    check(xrd_grouped_relu_grad(dtype, m, n_out, result.data_ptr(),
                                dz.data_ptr(), dz.stride(0),
                                masked.data_ptr(), st),
          "xrd_grouped_relu_grad");
    dz = masked;
  }
  if (need_x) {
    const Tensor weight = weight_->contiguous();
    dx = at::empty({m, n_in}, options);
    check(xrd_grouped_bwd_x(dtype, m, e, n_in, n_out, dz.data_ptr(),
                            dz.stride(0), weight.data_ptr(), sp, dx.data_ptr(),
                            st),
          "xrd_grouped_bwd_x");
  }
  if (need_w || need_b) {
    const Tensor x = dense_rows(*x_);
    const int64_t words = xrd_grouped_ws_floats(dtype, m, e, n_in, n_out);
    if (words < 0) check(XRD_ERR_UNSUPPORTED, "xrd_grouped_bwd_w");
    const Tensor ws = workspace(words, dz, at::kFloat);
    dw = at::empty({e, n_out, n_in}, options);
    if (need_b) db = at::empty({e, n_out}, options);
    check(xrd_grouped_bwd_w(dtype, m, e, n_in, n_out, x.data_ptr(),
                            x.stride(0), dz.data_ptr(), dz.stride(0), sp,
                            dw.data_ptr(), address(db),
                            words > 0 ? ws.data_ptr<float>() : nullptr, st),
          "xrd_grouped_bwd_w");
    if (!need_w) dw = Tensor();
  }
  return {dx, dw, db};
}

class Linear : public torch::autograd::Function<Linear> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& weight, const Tensor& starts,
                        const optional<Tensor>& bias, bool relu) {
    static const auto op = operator_of<decltype(linear)>("xrdslam::linear");
    ctx->saved_data["groups"] = weight.size(0);
    ctx->saved_data["in"] = weight.size(2);
    ctx->saved_data["bias"] = bias.has_value();
    const bool need_x = wants_grad(x);
    const bool need_w = wants_grad(weight) || wants_grad(bias);
    Tensor y;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      y = op.call(x, weight, starts, bias, relu);
    }
    ctx->save_for_backward({need_w ? x : Tensor(), need_x ? weight : Tensor(),
                            starts, relu ? y : Tensor()});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op =
        operator_of<decltype(linear_grads)>("xrdslam::linear_grads");
    refuse_tangent("xrd_grouped_bwd", grads[0]);
    const auto saved = ctx->get_saved_variables();
    const bool need_b =
        ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
    Tensor dx, dw, db;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dx, dw, db) = op.call(
          grads[0], given(saved[0]), given(saved[1]), saved[2],
          given(saved[3]), ctx->saved_data["groups"].toInt(),
          ctx->saved_data["in"].toInt(), ctx->needs_input_grad(0),
          ctx->needs_input_grad(1), need_b);
    }
    return once({dx, dw, Tensor(), db, Tensor()});
  }
};

Tensor linear_autograd(const Tensor& x, const Tensor& weight,
                       const Tensor& starts, const optional<Tensor>& bias,
                       bool relu) {
  static const auto op = operator_of<decltype(linear)>("xrdslam::linear");
  refuse_wide("xrd_grouped_fwd", {weight.size(0), weight.size(1), weight.size(2)});
  refuse_tangent("xrd_grouped_fwd", x);
  refuse_tangent("xrd_grouped_fwd", weight);
  refuse_tangent("xrd_grouped_fwd", bias);
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return Linear::apply(x, weight, starts, bias, relu);
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, starts, bias, relu);
}

}  // namespace

TORCH_LIBRARY(xrdslam, m) {
  m.def("plan(Tensor ids, int n_groups, bool rank) -> (Tensor, Tensor, Tensor)");
  m.def(
      "lookup(Tensor table, Tensor ids, Tensor? weights, float scale, "
      "Tensor? order, Tensor? starts) -> Tensor");
  m.def(
      "lookup_grads(Tensor dout, Tensor? table, Tensor ids, Tensor? weights, "
      "float scale, Tensor? order, Tensor? starts, int rows, bool need_table, "
      "bool need_weights) -> (Tensor, Tensor)");
  m.def(
      "linear(Tensor x, Tensor weight, Tensor starts, Tensor? bias, bool relu)"
      " -> Tensor");
  m.def(
      "linear_grads(Tensor dout, Tensor? x, Tensor? weight, Tensor starts, "
      "Tensor? y, int n_groups, int n_in, bool need_x, bool need_w, "
      "bool need_b) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(xrdslam, CUDA, m) {
  m.impl("plan", &plan);
  m.impl("lookup", &lookup);
  m.impl("lookup_grads", &lookup_grads);
  m.impl("linear", &linear);
  m.impl("linear_grads", &linear_grads);
}

TORCH_LIBRARY_IMPL(xrdslam, Autograd, m) {
  m.impl("plan", torch::CppFunction::makeFallthrough());    // whole numbers
  m.impl("lookup", &lookup_autograd);
  m.impl("linear", &linear_autograd);
}
