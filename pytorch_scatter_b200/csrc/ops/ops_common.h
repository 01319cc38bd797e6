// Host side of the torch_scatter operator set: argument checking, shape flattening, output
// allocation and autograd.  All arithmetic happens behind the C ABI declared in tsb200.h; this
// layer only moves torch tensors' device pointers, sizes and the current CUDA stream across it.
#pragma once

#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/script.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../../include/tsb200.h"

namespace tsb_ops {

// Messages hold numbers as std::to_string: an integer streamed into a message needs the locale facets of the C++ runtime
// that this file was compiled against, which need not be the one that the process has loaded.
// Same wording as the upstream checks (csrc/cuda/utils.cuh:5-7) so callers see familiar errors.
#define TSB_CHECK_CUDA(x) TORCH_CHECK((x).device().is_cuda(), #x " must be CUDA tensor (this build has no CPU path)")
#define TSB_CHECK_INPUT(x) TORCH_CHECK(x, "Input mismatch")

inline int dtype_enum(const torch::Tensor &t) {
  switch (t.scalar_type()) {
    case at::ScalarType::Float: return TSB_F32;
    case at::ScalarType::Double: return TSB_F64;
    case at::ScalarType::Half: return TSB_F16;
    case at::ScalarType::BFloat16: return TSB_BF16;
    case at::ScalarType::Int: return TSB_I32;
    case at::ScalarType::Long: return TSB_I64;
    case at::ScalarType::Byte: return TSB_U8;
    case at::ScalarType::Char: return TSB_I8;
    case at::ScalarType::Short: return TSB_I16;
    default: TORCH_CHECK(false, "torch_scatter (B200 build): unsupported dtype ", t.scalar_type());
  }
}

inline int reduce_enum(const std::string &reduce) {
  if (reduce == "sum" || reduce == "add") return TSB_SUM;
  if (reduce == "mean") return TSB_MEAN;
  if (reduce == "min") return TSB_MIN;
  if (reduce == "max") return TSB_MAX;
  if (reduce == "mul") return TSB_MUL;
  TORCH_CHECK(false, "unknown reduce '", reduce, "'");
}

inline void check_status(int status, const char *what) {
  TORCH_CHECK(status == TSB_OK, what, " failed: ", tsb_status_string(status));
}

inline tsb_stream_t current_stream() {
  return reinterpret_cast<tsb_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

inline void check_index_dtype(const torch::Tensor &index, const char *name) {
  TORCH_CHECK(index.scalar_type() == at::ScalarType::Long, name, " must be an int64 tensor");
}

inline std::vector<int64_t> list2vec(const c10::List<int64_t> &list) {
  std::vector<int64_t> result;
  result.reserve(list.size());
  for (size_t i = 0; i < list.size(); i++) result.push_back(list[i]);
  return result;
}

// A [.., L] int64 tensor whose leading dims were expanded to `B` batches, reduced to what the
// kernels take: a dense base pointer plus the distance between consecutive batches (0 when every
// batch shares one row).  Keeps the backing tensor alive.
struct BatchedRows {
  torch::Tensor holder;
  int64_t batch_stride;
  const int64_t *ptr() const { return holder.data_ptr<int64_t>(); }
};

inline BatchedRows batched_rows(const torch::Tensor &t) {
  const int64_t last = t.dim() - 1;
  bool shared = true;
  for (int64_t i = 0; i < last; i++)
    if (t.size(i) != 1 && t.stride(i) != 0) shared = false;
  BatchedRows r;
  if (shared) {
    torch::Tensor row = t;
    for (int64_t i = 0; i < last; i++) row = row.select(0, 0);
    r.holder = row.contiguous();
    r.batch_stride = 0;
  } else {
    r.holder = t.contiguous();
    r.batch_stride = t.size(last);
  }
  return r;
}

// Every routine that touches tensor DATA is an operator of its own (torch_scatter::_*, CUDA kernels registered in the
// registry files, shape-only "fake" kernels registered from Python in pytorch_scatter_b200/_meta.py).  The drivers
// below look their operator up once and call it through the dispatcher, so the public operators - argument handling
// and autograd written against these drivers - run unchanged on real tensors, and on fake tensors when a tracing
// compiler propagates shapes through them (upstream registers no fake kernels: its operators break the graph).
template <typename Signature> inline c10::TypedOperatorHandle<Signature> internal_op(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
inline torch::Tensor no_tensor(const torch::Tensor &like) { return torch::empty({0}, like.options()); }

// The operators on packed batches have a first derivative only.  A gradient computed under create_graph passes through
// this node, so that differentiating it again raises instead of silently giving nothing.
class FirstOrderOnly : public torch::autograd::Function<FirstOrderOnly> {
public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *, torch::autograd::Variable grad, at::TensorList) {
    return {grad.detach()};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *, torch::autograd::variable_list) {
    TORCH_CHECK(false, "torch_scatter: this operator has no second derivative");
  }
};
// Whether the tensor carries a forward-mode derivative, which these operators do not have.
inline bool has_tangent(const torch::Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
inline torch::autograd::variable_list first_order(torch::autograd::variable_list grads, std::vector<torch::Tensor> from) {
  for (auto &t : from) TORCH_CHECK(!has_tangent(t), "torch_scatter: the gradient of this operator has no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return grads;
  std::vector<torch::Tensor> known;
  for (auto &t : from)
    if (t.defined()) known.push_back(t);
  for (auto &g : grads)
    if (g.defined()) g = FirstOrderOnly::apply(g, at::TensorList(known))[0];
  return grads;
}

// accumulation type of a floating dtype: fp64 for fp64, else fp32
inline at::ScalarType acc_dtype(const torch::Tensor &t) {
  return t.scalar_type() == at::ScalarType::Double ? at::ScalarType::Double : at::ScalarType::Float;
}
inline void check_float_dtype(const torch::Tensor &t, const char *name) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::ScalarType::Float || s == at::ScalarType::Double || s == at::ScalarType::Half || s == at::ScalarType::BFloat16,
              name, " must be a float32, float64, float16 or bfloat16 tensor, got ", s);
}
// No gradient can be asked for: the operator is called without an autograd node around it (2 us of the host's time).
// Forward-mode derivatives go through the node, which refuses them, also under no_grad.
inline bool no_grad_for(std::initializer_list<torch::Tensor> ts) {
  for (auto &t : ts)
    if (has_tangent(t)) return false;
  if (!at::GradMode::is_enabled()) return true;
  for (auto &t : ts)
    if (t.defined() && t.requires_grad()) return false;
  return true;
}
inline const void *opt_ptr(const std::optional<torch::Tensor> &t) { return t.has_value() ? t.value().data_ptr() : nullptr; }
inline std::optional<torch::Tensor> opt_contiguous(const std::optional<torch::Tensor> &t) {
  return t.has_value() ? std::optional<torch::Tensor>(t.value().contiguous()) : std::nullopt;
}
inline std::optional<torch::Tensor> some_if_defined(const torch::Tensor &t) {
  return t.defined() ? std::optional<torch::Tensor>(t) : std::nullopt;
}

// ---- forward/backward drivers shared by the registry files ------------------------------------
std::tuple<torch::Tensor, std::optional<torch::Tensor>>
segment_csr_fw(torch::Tensor src, torch::Tensor indptr, std::optional<torch::Tensor> optional_out,
               const std::string &reduce);
torch::Tensor gather_csr_fw(torch::Tensor src, torch::Tensor indptr, std::optional<torch::Tensor> optional_out,
                            bool divide_by_count, std::optional<int64_t> length);

std::tuple<torch::Tensor, std::optional<torch::Tensor>>
segment_coo_fw(torch::Tensor src, torch::Tensor index, std::optional<torch::Tensor> optional_out,
               std::optional<int64_t> dim_size, const std::string &reduce);
torch::Tensor gather_coo_fw(torch::Tensor src, torch::Tensor index, std::optional<torch::Tensor> optional_out,
                            std::optional<torch::Tensor> count);

// grad_in[.., arg, ..] = grad_out along `dim`, for every MIN/MAX backward.
torch::Tensor arg_backward(const torch::Tensor &grad_out, const torch::Tensor &arg_out,
                           std::vector<int64_t> src_shape, int64_t dim);

}  // namespace tsb_ops
