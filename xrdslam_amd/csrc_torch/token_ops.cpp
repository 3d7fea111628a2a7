// torch.ops.xrdslam.{plan, lookup, linear}: the token and grouped-product entry
// points (xrd_token_*, xrd_lookup_*, xrd_grouped_*) as differentiable torch
// operators.  Host code only: allocation, the autograd node and the C calls.
// (As Python autograd functions over ctypes a forward and backward pass of a
// layer cost 103 us of host time, more than the kernels of a mapping batch.)
//
// Arguments are checked by xrdslam_amd/engine/{tokens,grouped}.py, the only
// callers; a status other than XRD_OK becomes a RuntimeError.  Every buffer,
// workspaces included, comes from torch's allocator on the current stream.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
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
  at::NoGradGuard no_grad;
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
// ids [n * k], weights [n * k] f32 or undefined, both dense
Tensor lookup_forward(const Tensor& table_, const Tensor& ids,
                      const Tensor& weights, int64_t k, double scale) {
  const c10::DeviceGuard guard(table_.device());
  const Tensor table = dense_rows(table_);
  const int64_t n = ids.numel() / k, dim = table.size(1);
  Tensor out = at::empty({n, dim}, table.options());
  check(xrd_lookup_fwd(dtype_of(table), n, (int)k, table.size(0), (int)dim,
                       table.data_ptr(), table.stride(0), ids.data_ptr(),
                       (int)ids.element_size(), (const float*)address(weights),
                       (float)scale, out.data_ptr(), stream_of(table)),
        "xrd_lookup_fwd");
  return out;
}

class Lookup : public torch::autograd::Function<Lookup> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& table,
                        const Tensor& ids, const optional<Tensor>& weights_,
                        int64_t k, double scale,
                        const optional<Tensor>& order,
                        const optional<Tensor>& starts) {
    const Tensor weights = weights_.value_or(Tensor());
    ctx->saved_data["k"] = k;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rows"] = table.size(0);
    const bool need_w = wants_grad(weights);
    // the table is needed for the weights' gradient alone
    ctx->save_for_backward(
        {need_w ? table : Tensor(), ids, weights, order.value_or(Tensor()),
         starts.value_or(Tensor())});
    return lookup_forward(table, ids, weights, k, scale);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &table = saved[0], &ids = saved[1], &weights = saved[2];
    const int64_t k = ctx->saved_data["k"].toInt();
    const int64_t rows = ctx->saved_data["rows"].toInt();
    const float scale = (float)ctx->saved_data["scale"].toDouble();
    // (numbered by the tensors that were given: ids is 1, weights 2)
    const bool need_table = ctx->needs_input_grad(0);
    const bool need_w = weights.defined() && ctx->needs_input_grad(2);
    Tensor dtable, dw;
    {
      at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(grads[0].device());
      const Tensor dout = dense_rows(grads[0]);
      const int dtype = dtype_of(dout), id_bytes = (int)ids.element_size();
      const int64_t n = ids.numel() / k, dim = dout.size(1);
      const int32_t* order = (const int32_t*)address(saved[3]);
      const int32_t* starts = (const int32_t*)address(saved[4]);
      Tensor tab = table, ws;       // ws: partial sums, then the plan if none
      if (need_table) {             // was given (an allocation costs 1 us)
        const int64_t sums = xrd_lookup_bwd_ws_floats(n, (int)k, (int)dim);
        if (sums < 0) check(XRD_ERR_UNSUPPORTED, "xrd_lookup_bwd");
        if (order != nullptr) {
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
      if (need_w) {
        tab = dense_rows(table);
        dw = at::empty(weights.sizes(), weights.options());
      }
      check(xrd_lookup_bwd(
                dtype, n, (int)k, rows, (int)dim, address(tab),
                need_w ? tab.stride(0) : 0, ids.data_ptr(), id_bytes,
                (const float*)address(weights), dout.data_ptr(),
                dout.stride(0), order, starts, scale,
                need_table ? dtable.data_ptr() : nullptr,
                (float*)address(dw), (float*)address(ws), stream_of(dout)),
            "xrd_lookup_bwd");
    }
    return once({dtable, Tensor(), dw, Tensor(), Tensor(), Tensor(),
                 Tensor()});
  }
};

Tensor lookup(const Tensor& table, const Tensor& ids_,
              const optional<Tensor>& weights_, double scale,
              const optional<Tensor>& order, const optional<Tensor>& starts) {
  const bool bag = weights_.has_value();
  const int64_t k = bag ? ids_.size(-1) : 1;
  const Tensor ids = ids_.contiguous();
  optional<Tensor> weights;
  if (bag) weights = weights_->to(at::kFloat).contiguous();
  Tensor out;
  if (at::GradMode::is_enabled() && (wants_grad(table) || wants_grad(weights)))
    out = Lookup::apply(table, ids, weights, k, scale, order, starts);
  else
    out = lookup_forward(table, ids, weights.value_or(Tensor()), k, scale);
  auto shape = ids_.sizes().vec();
  if (bag) shape.pop_back();
  if (shape.size() == 1) return out;
  shape.push_back(table.size(1));
  return out.view(shape);
}

// ------------------------------------------------------------------ linear
Tensor linear_forward(const Tensor& x_, const Tensor& weight_,
                      const Tensor& starts, const Tensor& bias_, bool relu) {
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = dense_rows(x_), weight = weight_.contiguous();
  Tensor bias;
  if (bias_.defined()) bias = bias_.contiguous();
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

class Linear : public torch::autograd::Function<Linear> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& weight, const Tensor& starts,
                        const optional<Tensor>& bias, bool relu) {
    Tensor y =
        linear_forward(x, weight, starts, bias.value_or(Tensor()), relu);
    ctx->saved_data["relu"] = relu;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["sizes"] = std::vector<int64_t>{
        x.size(0), weight.size(0), x.size(1), weight.size(1)};
    const bool need_x = wants_grad(x);
    const bool need_w = wants_grad(weight) || wants_grad(bias);
    ctx->save_for_backward({need_w ? x : Tensor(), need_x ? weight : Tensor(),
                            starts, relu ? y : Tensor()});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& starts = saved[2];
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t m = sizes[0];
    const int e = (int)sizes[1], n_in = (int)sizes[2], n_out = (int)sizes[3];
    const bool need_x = ctx->needs_input_grad(0);
    const bool need_w = ctx->needs_input_grad(1);
    const bool need_b =
        ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
    Tensor dx, dw, db;
    {
      at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(grads[0].device());
      Tensor dz = dense_rows(grads[0]);
      const int dtype = dtype_of(dz);
      const auto options = dz.options();
      void* st = stream_of(dz);
      int* sp = starts.data_ptr<int>();
      if (ctx->saved_data["relu"].toBool()) {
        Tensor masked = at::empty({m, n_out}, options);
        check(xrd_grouped_relu_grad(dtype, m, n_out, saved[3].data_ptr(),
                                    dz.data_ptr(), dz.stride(0),
                                    masked.data_ptr(), st),
              "xrd_grouped_relu_grad");
        dz = masked;
      }
      if (need_x) {
        const Tensor weight = saved[1].contiguous();
        dx = at::empty({m, n_in}, options);
        check(xrd_grouped_bwd_x(dtype, m, e, n_in, n_out, dz.data_ptr(),
                                dz.stride(0), weight.data_ptr(), sp,
                                dx.data_ptr(), st),
              "xrd_grouped_bwd_x");
      }
      if (need_w || need_b) {
        const Tensor x = dense_rows(saved[0]);
        const int64_t words =
            xrd_grouped_ws_floats(dtype, m, e, n_in, n_out);
        if (words < 0) check(XRD_ERR_UNSUPPORTED, "xrd_grouped_bwd_w");
        const Tensor ws = workspace(words, dz, at::kFloat);
        dw = at::empty({e, n_out, n_in}, options);
        if (need_b) db = at::empty({e, n_out}, options);
        check(xrd_grouped_bwd_w(dtype, m, e, n_in, n_out, x.data_ptr(),
                                x.stride(0), dz.data_ptr(), dz.stride(0), sp,
                                dw.data_ptr(), address(db),
                                words > 0 ? ws.data_ptr<float>() : nullptr,
                                st),
              "xrd_grouped_bwd_w");
        if (!need_w) dw = Tensor();
      }
    }
    return once({dx, dw, Tensor(), db, Tensor()});
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const Tensor& starts,
              const optional<Tensor>& bias, bool relu) {
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return Linear::apply(x, weight, starts, bias, relu);
  return linear_forward(x, weight, starts, bias.value_or(Tensor()), relu);
}

}  // namespace

TORCH_LIBRARY(xrdslam, m) {
  m.def("plan(Tensor ids, int n_groups, bool rank) -> (Tensor, Tensor, Tensor)",
        &plan);
  m.def(
      "lookup(Tensor table, Tensor ids, Tensor? weights, float scale, "
      "Tensor? order, Tensor? starts) -> Tensor",
      &lookup);
  m.def(
      "linear(Tensor x, Tensor weight, Tensor starts, Tensor? bias, bool relu)"
      " -> Tensor",
      &linear);
}
