// torch_scatter::expert_{topk,sort,dispatch,combine}: a router's choice of experts, the stable sort of tokens by expert,
// and the rows' way to the experts and back.  Not part of upstream's operator set.  Argument checks and autograd here,
// the data-touching halves are operators of their own (see ops_common.h).
#include "ops_common.h"

namespace tsb_ops {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- expert_topk ----------------------------------------------------------------------------------

std::tuple<torch::Tensor, torch::Tensor> topk_fw_impl(torch::Tensor logits_, int64_t k, bool normalize) {
  c10::cuda::CUDAGuard guard(logits_.device());
  auto logits = logits_.contiguous();
  auto sizes = logits.sizes().vec();
  const int64_t E = sizes.back(), T = E > 0 ? logits.numel() / E : 0;
  sizes.back() = k;
  auto weight = torch::empty(sizes, logits.options().dtype(torch::kFloat32));
  auto index = torch::empty(sizes, logits.options().dtype(torch::kInt64));
  check_status(tsb_expert_topk(logits.data_ptr(), weight.data_ptr<float>(), index.data_ptr<int64_t>(), T, E, k, normalize,
                               dtype_enum(logits), current_stream()),
               "tsb_expert_topk");
  return std::make_tuple(weight, index);
}

torch::Tensor topk_bw_impl(torch::Tensor grad_, torch::Tensor logits_, torch::Tensor weight_, torch::Tensor index_, bool normalize) {
  c10::cuda::CUDAGuard guard(logits_.device());
  auto grad = grad_.contiguous(), logits = logits_.contiguous(), weight = weight_.contiguous(), index = index_.contiguous();
  auto out = torch::empty_like(logits);
  const int64_t E = logits.size(-1), T = E > 0 ? logits.numel() / E : 0;
  check_status(tsb_expert_topk_backward(logits.data_ptr(), weight.data_ptr<float>(), index.data_ptr<int64_t>(),
                                        grad.data_ptr<float>(), out.data_ptr(), T, E, index.size(-1), normalize,
                                        dtype_enum(logits), current_stream()),
               "tsb_expert_topk_backward");
  return out;
}

std::tuple<torch::Tensor, torch::Tensor> topk_fw(const torch::Tensor &logits, int64_t k, bool normalize) {
  static auto op = internal_op<std::tuple<torch::Tensor, torch::Tensor>(torch::Tensor, int64_t, bool)>("torch_scatter::_expert_topk_fw");
  return op.call(logits, k, normalize);
}

class ExpertTopk : public torch::autograd::Function<ExpertTopk> {
public:
  static variable_list forward(AutogradContext *ctx, Variable logits, int64_t k, bool normalize) {
    auto r = topk_fw(logits, k, normalize);
    ctx->saved_data["normalize"] = normalize;
    ctx->save_for_backward({logits, std::get<0>(r), std::get<1>(r)});
    ctx->mark_non_differentiable({std::get<1>(r)});
    return {std::get<0>(r), std::get<1>(r)};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad_outs) {
    static auto op = internal_op<torch::Tensor(torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, bool)>("torch_scatter::_expert_topk_bw");
    auto saved = ctx->get_saved_variables();
    auto grad = op.call(grad_outs[0], saved[0], saved[1], saved[2], ctx->saved_data["normalize"].toBool());
    return first_order({grad, Variable(), Variable()}, {grad_outs[0], saved[0]});
  }
};

std::tuple<torch::Tensor, torch::Tensor> expert_topk(torch::Tensor logits, int64_t k, bool normalize) {
  TSB_CHECK_CUDA(logits);
  const auto s = logits.scalar_type();
  TORCH_CHECK(s == at::ScalarType::Float || s == at::ScalarType::Half || s == at::ScalarType::BFloat16,
              "expert_topk: logits must be a float32, float16 or bfloat16 tensor, got ", s);
  TORCH_CHECK(logits.dim() >= 1, "expert_topk: logits must have a last dimension of experts");
  TORCH_CHECK(logits.size(-1) >= 1 && logits.size(-1) <= 1024, "expert_topk: 1 to 1024 experts are supported, got ", std::to_string(logits.size(-1)));
  TORCH_CHECK(k >= 1 && k <= logits.size(-1), "expert_topk: k must be between 1 and the number of experts (", std::to_string(logits.size(-1)), "), got ", std::to_string(k));
  if (no_grad_for({logits})) return topk_fw(logits, k, normalize);
  auto r = ExpertTopk::apply(logits, k, normalize);
  return std::make_tuple(r[0], r[1]);
}

// ---- expert_sort ----------------------------------------------------------------------------------

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> sort_impl(torch::Tensor index_, int64_t num_experts) {
  c10::cuda::CUDAGuard guard(index_.device());
  auto index = index_.contiguous();
  const int64_t n = index.numel();
  auto slot = torch::empty_like(index);
  auto order = torch::empty({n}, index.options());
  auto indptr = torch::empty({num_experts + 1}, index.options());
  const size_t ws_bytes = tsb_expert_sort_workspace_bytes(n, num_experts);
  auto workspace = torch::empty({(int64_t)ws_bytes}, index.options().dtype(torch::kUInt8));
  check_status(tsb_expert_sort(index.data_ptr<int64_t>(), slot.data_ptr<int64_t>(), order.data_ptr<int64_t>(),
                               indptr.data_ptr<int64_t>(), n, num_experts, workspace.data_ptr(), ws_bytes, current_stream()),
               "tsb_expert_sort");
  return std::make_tuple(slot, order, indptr);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> expert_sort(torch::Tensor index, int64_t num_experts) {
  TSB_CHECK_CUDA(index);
  check_index_dtype(index, "index");
  TORCH_CHECK(num_experts >= 1 && num_experts <= 4096, "expert_sort: 1 to 4096 experts are supported, got ", std::to_string(num_experts));
  static auto op = internal_op<std::tuple<torch::Tensor, torch::Tensor, torch::Tensor>(torch::Tensor, int64_t)>("torch_scatter::_expert_sort");
  return op.call(index, num_experts);
}

// ---- expert_dispatch / expert_combine ---------------------------------------------------------------

int64_t features_of(const torch::Tensor &x, int64_t from) {
  int64_t K = 1;
  for (int64_t i = from; i < x.dim(); i++) K *= x.size(i);
  return K;
}

// (many, dot or a placeholder): few [*, ...] -> many [M, ...]
std::tuple<torch::Tensor, torch::Tensor> spread_impl(torch::Tensor few_, torch::Tensor slot_, torch::Tensor indptr_,
                                                     std::optional<torch::Tensor> weight_, std::optional<torch::Tensor> rows_) {
  c10::cuda::CUDAGuard guard(few_.device());
  auto few = few_.contiguous(), slot = slot_.contiguous(), indptr = indptr_.contiguous();
  auto weight = opt_contiguous(weight_), rows = opt_contiguous(rows_);
  const int64_t lead = slot.dim() - 1, k = slot.size(-1), T = k > 0 ? slot.numel() / k : 0, K = features_of(few, lead);
  std::vector<int64_t> sizes{slot.numel()};
  for (int64_t i = lead; i < few.dim(); i++) sizes.push_back(few.size(i));
  auto many = torch::empty(sizes, few.options());
  auto dot = rows.has_value() ? torch::empty(slot.sizes(), few.options().dtype(acc_dtype(few))) : no_tensor(few);
  if (slot.numel() > 0)
    check_status(tsb_expert_spread(few.data_ptr(), slot.data_ptr<int64_t>(), indptr.data_ptr<int64_t>() + (indptr.numel() - 1),
                                   opt_ptr(weight), opt_ptr(rows), many.data_ptr(), rows.has_value() ? dot.data_ptr() : nullptr,
                                   T, k, K, dtype_enum(few), current_stream()),
                 "tsb_expert_spread");
  return std::make_tuple(many, dot);
}

// (few, dot or a placeholder): many [M, ...] -> few [*, ...]
std::tuple<torch::Tensor, torch::Tensor> fold_impl(torch::Tensor many_, torch::Tensor slot_, std::optional<torch::Tensor> weight_,
                                                   std::optional<torch::Tensor> other_) {
  c10::cuda::CUDAGuard guard(many_.device());
  auto many = many_.contiguous(), slot = slot_.contiguous();
  auto weight = opt_contiguous(weight_), other = opt_contiguous(other_);
  const int64_t lead = slot.dim() - 1, k = slot.size(-1), T = k > 0 ? slot.numel() / k : 0, K = features_of(many, 1);
  std::vector<int64_t> sizes(slot.sizes().begin(), slot.sizes().begin() + lead);
  for (int64_t i = 1; i < many.dim(); i++) sizes.push_back(many.size(i));
  auto few = torch::empty(sizes, many.options());
  auto dot = other.has_value() ? torch::empty(slot.sizes(), many.options().dtype(acc_dtype(many))) : no_tensor(many);
  if (slot.numel() > 0)
    check_status(tsb_expert_fold(many.data_ptr(), slot.data_ptr<int64_t>(), opt_ptr(weight), opt_ptr(other), few.data_ptr(),
                                 other.has_value() ? dot.data_ptr() : nullptr, T, k, K, dtype_enum(many), current_stream()),
                 "tsb_expert_fold");
  else
    few.zero_();  // tokens without choices
  return std::make_tuple(few, dot);
}

std::tuple<torch::Tensor, torch::Tensor> spread(const torch::Tensor &few, const torch::Tensor &slot, const torch::Tensor &indptr,
                                                const std::optional<torch::Tensor> &weight, const std::optional<torch::Tensor> &rows) {
  static auto op = internal_op<std::tuple<torch::Tensor, torch::Tensor>(torch::Tensor, torch::Tensor, torch::Tensor, std::optional<torch::Tensor>,
                                                                        std::optional<torch::Tensor>)>("torch_scatter::_expert_spread");
  return op.call(few, slot, indptr, weight, rows);
}
std::tuple<torch::Tensor, torch::Tensor> fold(const torch::Tensor &many, const torch::Tensor &slot, const std::optional<torch::Tensor> &weight,
                                              const std::optional<torch::Tensor> &other) {
  static auto op = internal_op<std::tuple<torch::Tensor, torch::Tensor>(torch::Tensor, torch::Tensor, std::optional<torch::Tensor>,
                                                                        std::optional<torch::Tensor>)>("torch_scatter::_expert_fold");
  return op.call(many, slot, weight, other);
}

// DISPATCH: rows = spread(src);  grad_src = fold(grad), grad_weight = <src, grad rows>
// COMBINE:  out = fold(rows);    grad_rows = spread(grad), grad_weight = <grad, rows>
template <bool DISPATCH> class ExpertRows : public torch::autograd::Function<ExpertRows<DISPATCH>> {
public:
  static variable_list forward(AutogradContext *ctx, Variable x, Variable slot, Variable indptr, std::optional<Variable> weight) {
    auto out = std::get<0>(DISPATCH ? spread(x, slot, indptr, weight, std::nullopt) : fold(x, slot, weight, std::nullopt));
    const bool weighted = weight.has_value();
    // the data itself is needed for the gradient of the weights alone
    ctx->saved_data["dots"] = weighted && weight.value().requires_grad();
    ctx->save_for_backward({weighted && weight.value().requires_grad() ? x : Variable(), slot, indptr, weighted ? weight.value() : Variable()});
    return {out};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad_outs) {
    auto saved = ctx->get_saved_variables();
    auto x = saved[0], slot = saved[1], indptr = saved[2], weight = saved[3];
    const bool dots = ctx->saved_data["dots"].toBool();
    const auto w = some_if_defined(weight), data = dots ? std::optional<torch::Tensor>(x) : std::nullopt;
    auto r = DISPATCH ? fold(grad_outs[0], slot, w, data) : spread(grad_outs[0], slot, indptr, w, data);
    return first_order({std::get<0>(r), Variable(), Variable(), dots ? std::get<1>(r) : Variable()}, {grad_outs[0], x, weight});
  }
};

void check_plan(const char *name, const torch::Tensor &x, const torch::Tensor &slot, const torch::Tensor &indptr,
                const std::optional<torch::Tensor> &weight) {
  TSB_CHECK_CUDA(x);
  TSB_CHECK_CUDA(slot);
  TSB_CHECK_CUDA(indptr);
  check_float_dtype(x, name);
  check_index_dtype(slot, "slot");
  check_index_dtype(indptr, "indptr");
  TORCH_CHECK(slot.dim() >= 2, name, ": slot must be [..., k] with at least one dimension of tokens");
  TORCH_CHECK(indptr.dim() == 1 && indptr.numel() >= 1, name, ": indptr must be a non-empty 1-D tensor");
  TORCH_CHECK(slot.device() == x.device() && indptr.device() == x.device(), name, ": all tensors must be on the same device");
  if (!weight.has_value()) return;
  TSB_CHECK_CUDA(weight.value());
  TORCH_CHECK(weight.value().device() == x.device(), name, ": all tensors must be on the same device");
  TORCH_CHECK(weight.value().sizes() == slot.sizes(), name, ": weight must have the shape of slot");
  TORCH_CHECK(weight.value().scalar_type() == acc_dtype(x), name, ": weight must be a ", acc_dtype(x), " tensor, got ", weight.value().scalar_type());
}

torch::Tensor expert_dispatch(torch::Tensor src, torch::Tensor slot, torch::Tensor indptr, std::optional<torch::Tensor> weight) {
  check_plan("expert_dispatch", src, slot, indptr, weight);
  const int64_t lead = slot.dim() - 1;
  TORCH_CHECK(src.dim() >= lead, "expert_dispatch: src must begin with slot's dimensions of tokens");
  for (int64_t i = 0; i < lead; i++)
    TORCH_CHECK(src.size(i) == slot.size(i), "expert_dispatch: src must begin with slot's dimensions of tokens");
  if (no_grad_for({src, weight.value_or(torch::Tensor())})) return std::get<0>(spread(src, slot, indptr, weight, std::nullopt));
  return ExpertRows<true>::apply(src, slot, indptr, weight)[0];
}

torch::Tensor expert_combine(torch::Tensor rows, torch::Tensor slot, torch::Tensor indptr, std::optional<torch::Tensor> weight) {
  check_plan("expert_combine", rows, slot, indptr, weight);
  TORCH_CHECK(rows.dim() >= 1 && rows.size(0) == slot.numel(), "expert_combine: rows must have one row for each entry of slot (", std::to_string(slot.numel()), ")");
  if (no_grad_for({rows, weight.value_or(torch::Tensor())})) return std::get<0>(fold(rows, slot, weight, std::nullopt));
  return ExpertRows<false>::apply(rows, slot, indptr, weight)[0];
}

}  // namespace
}  // namespace tsb_ops

TORCH_LIBRARY_FRAGMENT(torch_scatter, m) {
  m.def("expert_topk", &tsb_ops::expert_topk);
  m.def("expert_sort", &tsb_ops::expert_sort);
  m.def("expert_dispatch", &tsb_ops::expert_dispatch);
  m.def("expert_combine", &tsb_ops::expert_combine);
  m.def("_expert_topk_fw(Tensor logits, int k, bool normalize) -> (Tensor, Tensor)");
  m.def("_expert_topk_bw(Tensor grad, Tensor logits, Tensor weight, Tensor index, bool normalize) -> Tensor");
  m.def("_expert_sort(Tensor index, int num_experts) -> (Tensor, Tensor, Tensor)");
  m.def("_expert_spread(Tensor few, Tensor slot, Tensor indptr, Tensor? weight, Tensor? rows) -> (Tensor, Tensor)");
  m.def("_expert_fold(Tensor many, Tensor slot, Tensor? weight, Tensor? other) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(torch_scatter, CUDA, m) {
  m.impl("_expert_topk_fw", &tsb_ops::topk_fw_impl);
  m.impl("_expert_topk_bw", &tsb_ops::topk_bw_impl);
  m.impl("_expert_sort", &tsb_ops::sort_impl);
  m.impl("_expert_spread", &tsb_ops::spread_impl);
  m.impl("_expert_fold", &tsb_ops::fold_impl);
}
