// torch_scatter::scan_csr, scan_csr_state, scan_step: the gated linear recurrence over CSR segments.  Not part of
// upstream's operator set.  Argument checks and autograd here, the data-touching halves are operators of their own (see
// ops_common.h).
#include "ops_common.h"

#include <ATen/MemoryOverlap.h>

namespace tsb_ops {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

struct ScanDims { int64_t B, E, K, N, width; };

ScanDims scan_dims(const torch::Tensor &src, const torch::Tensor &gate, const torch::Tensor &indptr) {
  const int64_t dim = indptr.dim() - 1;
  ScanDims d{1, src.size(dim), 1, indptr.size(-1) - 1, 1};
  for (int64_t i = 0; i < dim; i++) d.B *= src.size(i);
  for (int64_t i = dim + 1; i < src.dim(); i++) {
    d.K *= src.size(i);
    if (gate.size(i) != src.size(i)) d.width *= src.size(i);
  }
  if (d.K == 0) d.width = 1;  // gates that no channel shares
  return d;
}

torch::Tensor state_like(const torch::Tensor &src, const torch::Tensor &indptr) {
  auto sizes = src.sizes().vec();
  sizes[indptr.dim() - 1] = indptr.size(-1) - 1;
  return torch::empty(sizes, src.options().dtype(acc_dtype(src)));
}

torch::Tensor expand_indptr(const torch::Tensor &indptr, const torch::Tensor &src) {
  auto sizes = indptr.sizes().vec();
  for (int64_t i = 0; i < indptr.dim() - 1; i++) sizes[i] = src.size(i);
  return indptr.expand(sizes);
}

// (out, last, h in the accumulation type); the last two are placeholders where they are not wanted
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> scan_fw_impl(torch::Tensor src_, torch::Tensor gate_, torch::Tensor indptr,
                                                                     std::optional<torch::Tensor> state_, bool want_last, bool want_wide) {
  c10::cuda::CUDAGuard guard(src_.device());
  auto src = src_.contiguous(), gate = gate_.contiguous();
  auto state = opt_contiguous(state_);
  const ScanDims d = scan_dims(src, gate, indptr);
  auto out = torch::empty_like(src);
  auto last = want_last ? state_like(src, indptr) : no_tensor(src);
  auto wide = want_wide ? torch::empty(src.sizes(), src.options().dtype(acc_dtype(src))) : no_tensor(src);
  BatchedRows rows = batched_rows(expand_indptr(indptr, src));
  check_status(tsb_scan_csr(src.data_ptr(), gate.data_ptr(), rows.ptr(), opt_ptr(state), out.data_ptr(), want_last ? last.data_ptr() : nullptr,
                            want_wide ? wide.data_ptr() : nullptr, d.B, d.E, d.K, d.N, d.width, rows.batch_stride, dtype_enum(src), dtype_enum(gate), current_stream()),
               "tsb_scan_csr");
  return std::make_tuple(out, last, wide);
}

// (grad_src, grad_gate, grad_state); the last two are placeholders where they are not wanted
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> scan_bw_impl(std::optional<torch::Tensor> grad_out_, std::optional<torch::Tensor> grad_last_,
                                                                     torch::Tensor gate_, torch::Tensor out_, std::optional<torch::Tensor> wide_,
                                                                     torch::Tensor indptr, std::optional<torch::Tensor> state_, bool want_gate,
                                                                     bool want_state) {
  c10::cuda::CUDAGuard guard(out_.device());
  auto gate = gate_.contiguous(), out = out_.contiguous();
  auto wide = opt_contiguous(wide_);
  auto grad_out = opt_contiguous(grad_out_), grad_last = opt_contiguous(grad_last_), state = opt_contiguous(state_);
  const ScanDims d = scan_dims(out, gate, indptr);
  auto grad_src = torch::empty_like(out);
  auto grad_gate = want_gate ? torch::empty_like(gate) : no_tensor(gate);
  if (want_gate && d.K == 0) grad_gate.zero_();  // empty sums: a shared gate exists without channels
  auto grad_state = want_state ? state_like(out, indptr) : no_tensor(out);
  BatchedRows rows = batched_rows(expand_indptr(indptr, out));
  TORCH_CHECK(!want_gate || wide.has_value() || out.scalar_type() == acc_dtype(out), "scan_csr: the gradient of the gate needs h in the accumulation type");
  const void *h = !want_gate ? nullptr : wide.has_value() ? wide.value().data_ptr() : out.data_ptr();
  const size_t ws_bytes = tsb_scan_csr_backward_workspace_bytes(d.B, d.E, d.K, d.N, d.width, dtype_enum(out), dtype_enum(gate));
  auto workspace = torch::empty({(int64_t)ws_bytes}, out.options().dtype(torch::kUInt8));
  check_status(tsb_scan_csr_backward(opt_ptr(grad_out), opt_ptr(grad_last), gate.data_ptr(),
                                     h, rows.ptr(), opt_ptr(state),
                                     grad_src.data_ptr(), want_gate ? grad_gate.data_ptr() : nullptr, want_state ? grad_state.data_ptr() : nullptr,
                                     d.B, d.E, d.K, d.N, d.width, rows.batch_stride, dtype_enum(out), dtype_enum(gate), workspace.data_ptr(), ws_bytes,
                                     current_stream()),
               "tsb_scan_csr_backward");
  return std::make_tuple(grad_src, grad_gate, grad_state);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> scan_fw(const torch::Tensor &src, const torch::Tensor &gate, const torch::Tensor &indptr,
                                                                const std::optional<torch::Tensor> &state, bool want_last, bool want_wide) {
  static auto op = internal_op<std::tuple<torch::Tensor, torch::Tensor, torch::Tensor>(torch::Tensor, torch::Tensor, torch::Tensor,
                                                                                       std::optional<torch::Tensor>, bool, bool)>("torch_scatter::_scan_csr_fw");
  return op.call(src, gate, indptr, state, want_last, want_wide);
}

class ScanCSR : public torch::autograd::Function<ScanCSR> {
public:
  static variable_list forward(AutogradContext *ctx, Variable src, Variable gate, Variable indptr, std::optional<Variable> state, bool want_last,
                               bool want_wide) {
    auto r = scan_fw(src, gate, indptr, state, want_last, want_wide);
    ctx->saved_data["want_gate"] = gate.requires_grad();
    ctx->saved_data["want_state"] = state.has_value() && state.value().requires_grad();
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({gate, std::get<0>(r), indptr, state.has_value() ? state.value() : Variable(), want_wide ? std::get<2>(r) : Variable()});
    if (want_last) return {std::get<0>(r), std::get<1>(r)};
    return {std::get<0>(r)};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad_outs) {
    static auto op = internal_op<std::tuple<torch::Tensor, torch::Tensor, torch::Tensor>(std::optional<torch::Tensor>, std::optional<torch::Tensor>,
                                                                                         torch::Tensor, torch::Tensor, std::optional<torch::Tensor>, torch::Tensor,
                                                                                         std::optional<torch::Tensor>, bool, bool)>("torch_scatter::_scan_csr_bw");
    auto saved = ctx->get_saved_variables();
    auto gate = saved[0], out = saved[1], indptr = saved[2], state = saved[3];
    const bool want_gate = ctx->saved_data["want_gate"].toBool(), want_state = ctx->saved_data["want_state"].toBool();
    const auto grad_last = grad_outs.size() > 1 ? some_if_defined(grad_outs[1]) : std::nullopt;
    auto r = op.call(some_if_defined(grad_outs[0]), grad_last, gate, out, some_if_defined(saved[4]), indptr, some_if_defined(state), want_gate, want_state);
    return first_order({std::get<0>(r), want_gate ? std::get<1>(r) : Variable(), Variable(), want_state ? std::get<2>(r) : Variable(), Variable(), Variable()},
                       {grad_outs[0], grad_last.has_value() ? grad_last.value() : Variable(), gate, out, state});
  }
};

// gate: src's shape, or 1 in trailing dimensions whose channels share a gate (kept as it is); any other broadcast is expanded
torch::Tensor checked_gate(const char *name, const torch::Tensor &src, const torch::Tensor &gate, int64_t dim) {
  TSB_CHECK_CUDA(gate);
  TORCH_CHECK(gate.device() == src.device(), name, ": all tensors must be on the same device");
  TORCH_CHECK(gate.scalar_type() == src.scalar_type() || (gate.scalar_type() == at::ScalarType::Float && src.scalar_type() != at::ScalarType::Double),
              name, ": gate must have src's dtype, or float32 with 16-bit data; got ", gate.scalar_type(), " with ", src.scalar_type());
  TORCH_CHECK(gate.dim() == src.dim(), name, ": gate must have as many dimensions as src");
  bool as_it_is = true, shared = false;
  for (int64_t i = 0; i < src.dim(); i++) {
    TORCH_CHECK(gate.size(i) == src.size(i) || gate.size(i) == 1, name, ": gate does not broadcast against src at dimension ", std::to_string(i));
    if (gate.size(i) == src.size(i)) {
      if (shared && src.size(i) != 1) as_it_is = false;
    } else {
      shared = true;
      if (i <= dim) as_it_is = false;
    }
  }
  return as_it_is ? gate : gate.expand(src.sizes());
}

variable_list scan(const char *name, torch::Tensor src, torch::Tensor gate, torch::Tensor indptr, std::optional<torch::Tensor> state, bool want_last) {
  TSB_CHECK_CUDA(src);
  TSB_CHECK_CUDA(indptr);
  check_float_dtype(src, name);
  check_index_dtype(indptr, "indptr");
  TORCH_CHECK(indptr.device() == src.device(), name, ": all tensors must be on the same device");
  TORCH_CHECK(indptr.dim() >= 1 && indptr.size(-1) >= 1, name, ": indptr must hold at least one offset");
  TORCH_CHECK(src.dim() >= indptr.dim(), name, ": src must have at least as many dimensions as indptr");
  const int64_t dim = indptr.dim() - 1;
  for (int64_t i = 0; i < dim; i++)
    TORCH_CHECK(indptr.size(i) == src.size(i) || indptr.size(i) == 1, name, ": indptr does not broadcast against src at dimension ", std::to_string(i));
  gate = checked_gate(name, src, gate, dim);
  if (state.has_value()) {
    const auto &s = state.value();
    TSB_CHECK_CUDA(s);
    TORCH_CHECK(s.device() == src.device(), name, ": all tensors must be on the same device");
    TORCH_CHECK(s.scalar_type() == acc_dtype(src), name, ": state must be a ", acc_dtype(src), " tensor, got ", s.scalar_type());
    TORCH_CHECK(s.dim() == src.dim(), name, ": state must have as many dimensions as src");
    for (int64_t i = 0; i < src.dim(); i++)
      TORCH_CHECK(s.size(i) == (i == dim ? indptr.size(-1) - 1 : src.size(i)), name, ": state must have src's shape with one row for each segment");
  }
  if (no_grad_for({src, gate, state.value_or(torch::Tensor())})) {
    auto r = scan_fw(src, gate, indptr, state, want_last, false);
    return {std::get<0>(r), std::get<1>(r)};
  }
  // the gradient of the gate needs h as the recurrence held it (see the kernel)
  const bool want_wide = src.scalar_type() != acc_dtype(src) && gate.requires_grad();
  return ScanCSR::apply(src, gate, indptr, state, want_last, want_wide);
}

torch::Tensor scan_csr(torch::Tensor src, torch::Tensor gate, torch::Tensor indptr, std::optional<torch::Tensor> state) {
  return scan("scan_csr", src, gate, indptr, state, false)[0];
}
std::tuple<torch::Tensor, torch::Tensor> scan_csr_state(torch::Tensor src, torch::Tensor gate, torch::Tensor indptr, std::optional<torch::Tensor> state) {
  auto r = scan("scan_csr_state", src, gate, indptr, state, true);
  return std::make_tuple(r[0], r[1]);
}

torch::Tensor scan_step_impl(torch::Tensor src_, torch::Tensor gate_, torch::Tensor state) {
  c10::cuda::CUDAGuard guard(src_.device());
  auto src = src_.contiguous(), gate = gate_.contiguous();
  auto out = torch::empty_like(src);
  const int64_t n = src.size(0), K = n > 0 ? src.numel() / n : 0, gates = n > 0 ? gate.numel() / n : 0;
  if (src.numel() == 0) return out;
  for (const auto &t : {src, gate})  // (the state itself may be one of them: every value is read by the thread that replaces it)
    TORCH_CHECK(at::get_overlap_status(state, t) != at::MemOverlapStatus::Partial, "scan_step: src and gate must not overlap the state in part");
  check_status(tsb_scan_step(src.data_ptr(), gate.data_ptr(), state.data_ptr(), out.data_ptr(), n, K, K / gates, state.stride(0), dtype_enum(src),
                             dtype_enum(gate), current_stream()),
               "tsb_scan_step");
  return out;
}

torch::Tensor scan_step(torch::Tensor src, torch::Tensor gate, torch::Tensor state) {
  TSB_CHECK_CUDA(src);
  TSB_CHECK_CUDA(state);
  check_float_dtype(src, "scan_step");
  TORCH_CHECK(src.dim() >= 1, "scan_step: src must be [n, ...], one token for each state");
  TORCH_CHECK(state.device() == src.device(), "scan_step: all tensors must be on the same device");
  TORCH_CHECK(state.scalar_type() == acc_dtype(src), "scan_step: state must be a ", acc_dtype(src), " tensor, got ", state.scalar_type());
  TORCH_CHECK(state.sizes() == src.sizes(), "scan_step: state must have src's shape");
  gate = checked_gate("scan_step", src, gate, 0);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(src.requires_grad() || gate.requires_grad() || state.requires_grad()),
              "scan_step updates the state in place and has no gradient: call it under torch.no_grad(), or scan_csr_state for training");
  TORCH_CHECK(!has_tangent(src) && !has_tangent(gate) && !has_tangent(state), "scan_step has no forward-mode derivative");
  if (src.numel() > 0) {
    int64_t K = 1;  // inside a state the elements are dense; consecutive states may lie apart
    for (int64_t i = src.dim() - 1; i >= 1; i--) {
      TORCH_CHECK(state.size(i) == 1 || state.stride(i) == K, "scan_step: each state must be contiguous");
      K *= state.size(i);
    }
    TORCH_CHECK(state.size(0) == 1 || state.stride(0) >= K, "scan_step: states must not overlap");
  }
  static auto op = internal_op<torch::Tensor(torch::Tensor, torch::Tensor, torch::Tensor)>("torch_scatter::_scan_step");
  auto out = op.call(src, gate, state);
  if (src.numel() > 0) state.unsafeGetTensorImpl()->bump_version();  // saved copies of the old state are stale now
  return out;
}

}  // namespace
}  // namespace tsb_ops

TORCH_LIBRARY_FRAGMENT(torch_scatter, m) {
  m.def("scan_csr", &tsb_ops::scan_csr);
  m.def("scan_csr_state", &tsb_ops::scan_csr_state);
  m.def("scan_step(Tensor src, Tensor gate, Tensor(a!) state) -> Tensor", &tsb_ops::scan_step);
  m.def("_scan_csr_fw(Tensor src, Tensor gate, Tensor indptr, Tensor? state, bool want_last, bool want_wide) -> (Tensor, Tensor, Tensor)");
  m.def("_scan_csr_bw(Tensor? grad_out, Tensor? grad_last, Tensor gate, Tensor out, Tensor? wide, Tensor indptr, Tensor? state, bool want_gate, "
        "bool want_state) -> (Tensor, Tensor, Tensor)");
  m.def("_scan_step(Tensor src, Tensor gate, Tensor(a!) state) -> Tensor");
}

TORCH_LIBRARY_IMPL(torch_scatter, CUDA, m) {
  m.impl("_scan_csr_fw", &tsb_ops::scan_fw_impl);
  m.impl("_scan_csr_bw", &tsb_ops::scan_bw_impl);
  m.impl("_scan_step", &tsb_ops::scan_step_impl);
}
