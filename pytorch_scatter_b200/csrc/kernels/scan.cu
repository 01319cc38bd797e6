// Entry points of the gated linear recurrence (the tile kernel is in scan.cuh) and its single-token form.
#include "scan.cuh"

namespace tsb {
namespace {

using scan::ScanParams;

template <typename T, typename G>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const T *__restrict__ src, const G *__restrict__ gate, acc_t<T> *__restrict__ state,
                                                             T *__restrict__ out, int64_t n, int64_t K, int64_t width, int64_t stride) {
  for (int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x; it < n * K; it += (int64_t)gridDim.x * kThreads) {
    const int64_t i = it / K, c = it - i * K;
    acc_t<T> &s = state[i * stride + c];
    const acc_t<T> h = to_acc<G>(gate[i * (K / width) + c / width]) * s + to_acc<T>(src[it]);
    s = h;
    out[it] = from_acc<T>(h);
  }
}

template <typename F> int with_types(int dtype, int gate_dtype, F f) {
  switch (dtype) {
    case TSB_F32: return f(float(), float());
    case TSB_F64: return f(double(), double());
    case TSB_F16: return gate_dtype == TSB_F32 ? f(__half(), float()) : f(__half(), __half());
    default: return gate_dtype == TSB_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
  }
}

int check(int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int dtype, int gate_dtype) {
  if (B < 0 || E < 0 || K < 0 || N < 0 || width < 1 || K % width != 0) return TSB_ERR_ARG;
  if (dtype != TSB_F32 && dtype != TSB_F64 && dtype != TSB_F16 && dtype != TSB_BF16) return TSB_ERR_DTYPE;
  if (gate_dtype != dtype && !(gate_dtype == TSB_F32 && dtype != TSB_F64)) return TSB_ERR_DTYPE;
  if (N >= scan::kMostSegments) return TSB_ERR_TOO_LARGE;
  return TSB_OK;
}

int launch_tiles(const ScanParams &p, int dtype, int gate_dtype, bool backward, tsb_stream_t stream) {
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case TSB_F32: return scan::launch_f32(p, gate_dtype, backward, st);
    case TSB_F64: return scan::launch_f64(p, gate_dtype, backward, st);
    case TSB_F16: return scan::launch_f16(p, gate_dtype, backward, st);
    default: return scan::launch_bf16(p, gate_dtype, backward, st);
  }
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_scan_csr(const void *src, const void *gate, const int64_t *indptr, const void *state, void *out, void *last,
                            void *wide, int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int64_t indptr_batch_stride, int dtype,
                            int gate_dtype, tsb_stream_t stream) {
  if (const int st = check(B, E, K, N, width, dtype, gate_dtype)) return st;
  if (B == 0 || K == 0 || (E == 0 && (N == 0 || !last))) return TSB_OK;
  if (!indptr || (E > 0 && (!src || !gate || !out))) return TSB_ERR_ARG;
  ScanParams p{};
  if (wide && gate_dtype == dtype) return TSB_ERR_ARG;
  p.src = src; p.gate = gate; p.state = state; p.indptr = indptr; p.out = out; p.last = last; p.wide = wide;
  p.B = B; p.E = E; p.K = K; p.N = N; p.width = width; p.bstride = indptr_batch_stride;
  return launch_tiles(p, dtype, gate_dtype, false, stream);
}

extern "C" size_t tsb_scan_csr_backward_workspace_bytes(int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int dtype, int gate_dtype) {
  if (check(B, E, K, N, width, dtype, gate_dtype) != TSB_OK || width == 1) return 0;
  return (size_t)(B * E * scan::partials_of_row(K, width, dtype_elem_bytes(dtype))) * dtype_acc_bytes(dtype);
}

extern "C" int tsb_scan_csr_backward(const void *grad_out, const void *grad_last, const void *gate, const void *h,
                                     const int64_t *indptr, const void *state, void *grad_src, void *grad_gate, void *grad_state,
                                     int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int64_t indptr_batch_stride,
                                     int dtype, int gate_dtype, void *workspace, size_t workspace_bytes, tsb_stream_t stream) {
  if (const int st = check(B, E, K, N, width, dtype, gate_dtype)) return st;
  if (B == 0 || K == 0 || (E == 0 && (N == 0 || !grad_state))) return TSB_OK;
  if (!indptr || (E > 0 && (!gate || (grad_gate && !h) || !grad_src))) return TSB_ERR_ARG;
  const size_t need = grad_gate && E > 0 ? tsb_scan_csr_backward_workspace_bytes(B, E, K, N, width, dtype, gate_dtype) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return TSB_ERR_WORKSPACE;
  ScanParams p{};
  p.src = grad_out; p.gate = gate; p.state = grad_last; p.fwd = h; p.init = state; p.indptr = indptr;
  p.out = grad_src; p.last = grad_state; p.grad_gate = grad_gate; p.partial = workspace;
  p.B = B; p.E = E; p.K = K; p.N = N; p.width = width; p.bstride = indptr_batch_stride;
  return launch_tiles(p, dtype, gate_dtype, true, stream);
}

extern "C" int tsb_scan_step(const void *src, const void *gate, void *state, void *out, int64_t n, int64_t K, int64_t width,
                             int64_t state_stride, int dtype, int gate_dtype, tsb_stream_t stream) {
  if (const int st = check(1, n, K, 0, width, dtype, gate_dtype)) return st;
  if (n > 1 && state_stride < K) return TSB_ERR_ARG;
  if (n == 0 || K == 0) return TSB_OK;
  if (!src || !gate || !state || !out) return TSB_ERR_ARG;
  return with_types(dtype, gate_dtype, [&](auto t, auto g) -> int {
    using T = decltype(t);
    using G = decltype(g);
    scan_step_kernel<T, G><<<scan::flat_blocks(n * K), kThreads, 0, (cudaStream_t)stream>>>(
        static_cast<const T *>(src), static_cast<const G *>(gate), static_cast<acc_t<T> *>(state), static_cast<T *>(out), n, K, width, state_stride);
    return launch_status();
  });
}
