// Host side of the group norm + activation op and of the teacher's top logits
// and their distillation: checks, allocation, autograd. The kernels are in
// group_norm.hip and distill.hip.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <string>

#include "common.h"
#include "distill.h"
#include "group_norm.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

GnType gn_type(const at::Tensor& x, const char* who) {
  switch (x.scalar_type()) {
    case at::kFloat: return GnType::kF32;
    case at::kBFloat16: return GnType::kBf16;
    case at::kHalf: return GnType::kF16;
    default:
      TORCH_CHECK_TYPE(false, who, ": float32, bfloat16 or float16 expected, got ",
                       x.scalar_type());
  }
}

void check_launch(hipError_t e, const char* who) {
  TORCH_CHECK(e != hipErrorInvalidConfiguration, who, ": too large for one launch");
  TORCH_CHECK(e == hipSuccess, who, ": ", hipGetErrorString(e));
}

const float* f32_or_null(const at::Tensor& t) {
  return t.defined() ? t.data_ptr<float>() : nullptr;
}

struct GroupNormAct : public torch::autograd::Function<GroupNormAct> {
  // A small call waits for its allocations and for what autograd keeps:
  // 1x1632x10x10 fp16 without a gradient takes 7.7 us, and 9.3 through apply()
  // with two allocations more.
  static at::Tensor run(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias,
                        const at::Tensor& residual, const at::Tensor& drop, int64_t groups,
                        double eps, int64_t act, at::Tensor& stats) {
    auto y = at::empty_like(x);
    auto opts = x.options().dtype(at::kFloat);
    stats = at::empty({2, x.size(0), groups}, opts);  // mean, rstd
    GnArgs a = args(x, weight, bias, drop, stats, groups, act);
    a.eps = (float)eps;
    a.residual = residual.defined() ? residual.data_ptr() : nullptr;
    a.y = y.data_ptr();
    if (x.numel() > 0) {
      at::Tensor ws;
      if (const long long floats = gn_fwd_ws(a)) {
        ws = at::empty({floats}, opts);
        a.ws = ws.data_ptr<float>();
      }
      check_launch(gn_fwd(a, at::hip::getCurrentHIPStream().stream()), "group_norm_act");
    }
    return y;
  }

  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, OptTensor weight_opt,
                            OptTensor bias_opt, OptTensor residual_opt, OptTensor drop_opt,
                            int64_t groups, double eps, int64_t act) {
    const auto weight = weight_opt.value_or(at::Tensor()), bias = bias_opt.value_or(at::Tensor()),
               residual = residual_opt.value_or(at::Tensor()),
               drop = drop_opt.value_or(at::Tensor());
    at::Tensor stats;
    auto y = run(x, weight, bias, residual, drop, groups, eps, act, stats);
    ctx->save_for_backward({x, weight, bias, drop, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = residual.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "group_norm_act: gradients of gradients are not supported");
    auto saved = ctx->get_saved_variables();
    const auto &x = saved[0], &weight = saved[1], &bias = saved[2], &drop = saved[3],
               &stats = saved[4];
    const c10::DeviceGuard guard(x.device());
    auto opts = x.options().dtype(at::kFloat);
    at::Tensor dx, dweight, dbias, dres;
    // the tensors that were given, in the order of forward's arguments
    size_t input = 0;
    if (ctx->needs_input_grad(input++)) dx = at::empty_like(x);
    if (weight.defined() && ctx->needs_input_grad(input++)) dweight = at::empty({x.size(1)}, opts);
    if (bias.defined() && ctx->needs_input_grad(input++)) dbias = at::empty({x.size(1)}, opts);
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(input++)) dres = grads[0];
    if (x.numel() == 0) {
      if (dweight.defined()) dweight.zero_();
      if (dbias.defined()) dbias.zero_();
    } else if (dx.defined() || dweight.defined() || dbias.defined()) {
      auto dy = grads[0].to(x.scalar_type()).contiguous(at::MemoryFormat::ChannelsLast);
      GnArgs a = args(x, weight, bias, drop, stats, ctx->saved_data["groups"].toInt(),
                      ctx->saved_data["act"].toInt());
      a.dy = dy.data_ptr();
      a.dx = dx.defined() ? dx.data_ptr() : nullptr;
      a.dweight = dweight.defined() ? dweight.data_ptr<float>() : nullptr;
      a.dbias = dbias.defined() ? dbias.data_ptr<float>() : nullptr;
      auto ws = at::empty({gn_bwd_ws(a)}, opts);
      a.ws = ws.data_ptr<float>();
      check_launch(gn_bwd(a, at::hip::getCurrentHIPStream().stream()),
                   "group_norm_act backward");
    }
    return {dx, dweight, dbias, dres, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }

  static GnArgs args(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias,
                     const at::Tensor& drop, const at::Tensor& stats, int64_t groups,
                     int64_t act) {
    GnArgs a = {};
    a.n = x.size(0);
    a.hw = x.size(2) * x.size(3);
    a.c = (int)x.size(1);
    a.groups = (int)groups;
    a.type = gn_type(x, "group_norm_act");
    a.act = (int)act;
    a.x = x.data_ptr();
    const at::Tensor& param = weight.defined() ? weight : bias;
    a.ptype = param.defined() ? gn_type(param, "group_norm_act: parameters") : GnType::kF32;
    a.weight = weight.defined() ? weight.data_ptr() : nullptr;
    a.bias = bias.defined() ? bias.data_ptr() : nullptr;
    a.drop = f32_or_null(drop);
    a.mean = stats.data_ptr<float>();
    a.rstd = a.mean + a.n * a.groups;
    return a;
  }
};

LogitType logit_type(const at::Tensor& x, const char* who) {
  return static_cast<LogitType>(gn_type(x, who));
}
static_assert((int)LogitType::kBf16 == (int)GnType::kBf16 &&
                  (int)LogitType::kF16 == (int)GnType::kF16,
              "one numbering of types");

// t as `sizes`, itself if it has them: a view is a node more for the backward
// pass, which the host of a small step waits for (26x2 logits, 61 us forward
// and backward with two views, 49 without).
at::Tensor sized(const at::Tensor& t, at::IntArrayRef sizes) {
  return t.sizes() == sizes ? t : t.reshape(sizes);
}

// [..., classes] as [rows, classes] with unit stride in a row: a view where
// the rows are evenly spaced, or else a copy.
at::Tensor as_rows(const at::Tensor& x, const char* who) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1, who, ": CUDA logits expected");
  const int64_t classes = x.size(-1);
  // a block's threads step past the last class by less than 4096, in 32 bits
  TORCH_CHECK(classes >= 1 && classes <= INT_MAX - 4096, who, ": ", classes, " classes");
  auto rows = x.dim() == 2 ? x : x.reshape({-1, classes});
  TORCH_CHECK(rows.size(0) <= INT_MAX, who, ": too many rows");
  return rows.stride(1) == 1 || classes == 1 ? rows : rows.contiguous();
}

struct DistillTopk : public torch::autograd::Function<DistillTopk> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor logits, at::Tensor values,
                            at::Tensor indices, OptTensor rest_opt, double temperature) {
    const auto rest = rest_opt.value_or(at::Tensor());
    const int64_t rows = logits.size(0);
    auto opts = logits.options().dtype(at::kFloat);
    auto loss = at::empty({rows}, opts);
    auto stats = at::empty({rows, kDistillStats}, opts);
    DistillArgs a = args(logits, values, indices, stats, temperature);
    a.rest = f32_or_null(rest);
    a.loss = loss.data_ptr<float>();
    if (rows > 0)
      check_launch(distill_fwd(a, at::hip::getCurrentHIPStream().stream()), "distill_topk");
    ctx->save_for_backward({logits, values, indices, stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "distill_topk: gradients of gradients are not supported");
    auto saved = ctx->get_saved_variables();
    const auto &logits = saved[0], &values = saved[1], &indices = saved[2], &stats = saved[3];
    const c10::DeviceGuard guard(logits.device());
    auto grad = at::empty(logits.sizes(), logits.options());
    auto up = grads[0].to(at::kFloat);
    DistillArgs a = args(logits, values, indices, stats, ctx->saved_data["temperature"].toDouble());
    a.upstream = up.data_ptr<float>();
    a.upstream_stride = up.stride(0);
    a.grad = grad.data_ptr();
    if (a.rows > 0)
      check_launch(distill_bwd(a, at::hip::getCurrentHIPStream().stream()),
                   "distill_topk backward");
    return {grad, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }

  static DistillArgs args(const at::Tensor& logits, const at::Tensor& values,
                          const at::Tensor& indices, const at::Tensor& stats,
                          double temperature) {
    DistillArgs a = {};
    a.logits = logits.data_ptr();
    a.rows = logits.size(0);
    a.row_stride = logits.stride(0);
    a.classes = (int)logits.size(1);
    a.k = (int)values.size(1);
    a.type = logit_type(logits, "distill_topk");
    a.vtype = logit_type(values, "distill_topk: values");
    a.temperature = (float)temperature;
    a.values = values.data_ptr();
    a.indices = reinterpret_cast<const long long*>(indices.data_ptr<int64_t>());
    a.stats = stats.data_ptr<float>();
    return a;
  }
};

}  // namespace

std::vector<at::Tensor> topk_logits(at::Tensor logits, int64_t k, double temperature) {
  const char* who = "topk_logits";
  const LogitType type = logit_type(logits, who);
  const c10::DeviceGuard guard(logits.device());
  const at::Tensor x = as_rows(logits.detach(), who);
  TORCH_CHECK(k >= 1 && k <= kMaxTopK && k <= x.size(1), who, ": k is ", k);
  auto shape = logits.sizes().vec();
  shape.back() = k;
  auto values = at::empty(shape, logits.options());
  auto indices = at::empty(shape, logits.options().dtype(at::kLong));
  shape.pop_back();
  auto rest = at::empty(shape, logits.options().dtype(at::kFloat));
  TopkArgs a = {};
  a.logits = x.data_ptr();
  a.rows = x.size(0);
  a.row_stride = x.stride(0);
  a.classes = (int)x.size(1);
  a.k = (int)k;
  a.type = type;
  a.temperature = (float)temperature;
  a.values = values.data_ptr();
  a.indices = reinterpret_cast<long long*>(indices.data_ptr<int64_t>());
  a.rest = rest.data_ptr<float>();
  if (a.rows > 0)
    check_launch(topk_logits_launch(a, at::hip::getCurrentHIPStream().stream()), who);
  return {values, indices, rest};
}

at::Tensor distill_topk(at::Tensor logits, at::Tensor values, at::Tensor indices,
                        OptTensor rest_opt, double temperature) {
  const char* who = "distill_topk";
  logit_type(logits, who);
  logit_type(values, "distill_topk: values");
  const c10::DeviceGuard guard(logits.device());
  const at::Tensor x = as_rows(logits, who);
  const int64_t rows = x.size(0), k = values.size(-1);
  TORCH_CHECK(x.size(1) <= kMaxDistillClasses, who, ": ", x.size(1), " classes");
  TORCH_CHECK(k >= 1 && k <= kMaxTopK, who, ": k is ", k);
  TORCH_CHECK(values.numel() == rows * k && indices.numel() == rows * k, who,
              ": values and indices must be [rows, k]");
  TORCH_CHECK(values.device() == x.device() && indices.device() == x.device(), who,
              ": the teacher's answer must be on the device of the logits");
  auto rest = rest_opt.has_value() && rest_opt->defined() ? *rest_opt : at::Tensor();
  if (rest.defined()) {
    TORCH_CHECK(rest.numel() == rows && rest.device() == x.device(), who,
                ": rest must be [rows], on the device of the logits");
    rest = sized(rest.detach().to(at::kFloat), {rows}).contiguous();
  }
  auto loss = DistillTopk::apply(
      x, sized(values.detach(), {rows, k}).contiguous(),
      sized(indices.to(at::kLong), {rows, k}).contiguous(),
      rest.defined() ? OptTensor(rest) : c10::nullopt, temperature);
  return sized(loss, logits.sizes().slice(0, logits.dim() - 1));
}

at::Tensor group_norm_act(at::Tensor x, OptTensor weight_opt,
                          OptTensor bias_opt, int64_t groups, double eps,
                          std::string act_s, OptTensor residual_opt,
                          OptTensor drop_opt) {
  const char* who = "group_norm_act";
  TORCH_CHECK(x.is_cuda() && x.dim() == 4, who, ": 4D CUDA tensor expected");
  gn_type(x, who);
  const int64_t c = x.size(1);
  TORCH_CHECK(c <= 1 << 18, who, ": more than 2^18 channels");
  TORCH_CHECK(groups > 0 && c % groups == 0, who, ": ", c, " channels are not a multiple of ",
              groups, " groups");
  TORCH_CHECK(c / groups <= kGnMaxGroupChannels, who, ": more than 2^14 channels in a group");
  Act act = Act::kNone;
  if (act_s == "relu") act = Act::kRelu;
  else if (act_s == "silu") act = Act::kSilu;
  else TORCH_CHECK(act_s == "none", who, ": unknown activation '", act_s, "'");
  auto param = [&](const OptTensor& t, const char* name) {
    if (!t.has_value() || !t->defined()) return at::Tensor();
    TORCH_CHECK(t->dim() == 1 && t->size(0) == c && t->device() == x.device(), who, ": ", name,
                " must be [", c, "] on the device of x");
    return t->contiguous();
  };
  const c10::DeviceGuard guard(x.device());
  auto weight = param(weight_opt, "weight"), bias = param(bias_opt, "bias");
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) {
    weight = weight.to(at::kFloat);
    bias = bias.to(at::kFloat);
  }
  at::Tensor residual, drop;
  if (residual_opt.has_value() && residual_opt->defined()) {
    TORCH_CHECK(residual_opt->sizes() == x.sizes() && residual_opt->device() == x.device(),
                who, ": residual must have the shape and device of x");
    residual = residual_opt->to(x.scalar_type()).contiguous(at::MemoryFormat::ChannelsLast);
  }
  if (drop_opt.has_value() && drop_opt->defined()) {
    TORCH_CHECK(drop_opt->numel() == x.size(0) && drop_opt->device() == x.device(), who,
                ": drop_path_mask must have one value for each image, on the device of x");
    TORCH_CHECK(!drop_opt->requires_grad(), who, ": drop_path_mask has no gradient");
    drop = drop_opt->to(at::kFloat).contiguous();
  }
  const at::Tensor cl = x.contiguous(at::MemoryFormat::ChannelsLast);
  auto learns = [](const at::Tensor& t) {
    return t.defined() && (t.requires_grad() ? at::GradMode::is_enabled()
                                             : t._fw_grad(/*level=*/0).defined());
  };
  if (!(learns(cl) || learns(weight) || learns(bias) || learns(residual))) {
    at::Tensor stats;
    return GroupNormAct::run(cl, weight, bias, residual, drop, groups, eps, (int64_t)act, stats);
  }
  auto given = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; };
  return GroupNormAct::apply(cl, given(weight), given(bias), given(residual), given(drop), groups,
                             eps, (int64_t)act);
}
