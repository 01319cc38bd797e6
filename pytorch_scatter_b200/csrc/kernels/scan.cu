// Gated linear recurrence over the rows of CSR segments, forward and backward, and its single-token form.
//
//   h[e] = gate[e] * h[e-1] + src[e] along [indptr[n], indptr[n+1]), h before the first row = state[n] or 0
//   backward: dh[e] = grad_out[e] + gate[e+1] * dh[e+1] (+ grad_last[n] at the last row);
//             grad_src = dh, grad_gate[e] = sum over the channels that share it of dh[e] * h[e-1],
//             grad_state[n] = gate[first] * dh[first]
//
// One thread walks one channel of one segment.
#include <algorithm>

#include "common.cuh"

namespace tsb {
namespace {

struct ScanParams {
  const void *src, *gate, *state;
  const int64_t *indptr;
  void *out, *last;
  // backward
  const void *grad_out, *grad_last, *fwd;
  void *grad_src, *grad_gate, *grad_state, *partial;
  int64_t B, E, K, N, width, bstride;
};

template <typename T, typename G> __global__ void __launch_bounds__(kThreads) scan_walk_kernel(ScanParams p) {
  using A = acc_t<T>;
  const int64_t items = p.B * p.N * p.K, gates = p.K / p.width;
  for (int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x; it < items; it += (int64_t)gridDim.x * kThreads) {
    const int64_t c = it % p.K, n = it / p.K % p.N, b = it / p.K / p.N;
    const int64_t *ip = p.indptr + b * p.bstride;
    const int64_t lo = clamp64(ip[n], 0, p.E), hi = clamp64(ip[n + 1], lo, p.E);
    A h = p.state ? static_cast<const A *>(p.state)[it] : (A)0;
    for (int64_t e = b * p.E + lo; e < b * p.E + hi; ++e) {
      h = to_acc<G>(static_cast<const G *>(p.gate)[e * gates + c / p.width]) * h + to_acc<T>(static_cast<const T *>(p.src)[e * p.K + c]);
      static_cast<T *>(p.out)[e * p.K + c] = from_acc<T>(h);
    }
    if (p.last) static_cast<A *>(p.last)[it] = h;
  }
}

template <typename T, typename G> __global__ void __launch_bounds__(kThreads) scan_walk_backward_kernel(ScanParams p) {
  using A = acc_t<T>;
  const int64_t items = p.B * p.N * p.K, gates = p.K / p.width;
  for (int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x; it < items; it += (int64_t)gridDim.x * kThreads) {
    const int64_t c = it % p.K, n = it / p.K % p.N, b = it / p.K / p.N;
    const int64_t *ip = p.indptr + b * p.bstride;
    const int64_t lo = clamp64(ip[n], 0, p.E), hi = clamp64(ip[n + 1], lo, p.E);
    const A init = p.state ? static_cast<const A *>(p.state)[it] : (A)0;
    A carry = p.grad_last ? static_cast<const A *>(p.grad_last)[it] : (A)0;
    for (int64_t e = b * p.E + hi - 1; e >= b * p.E + lo; --e) {
      const int64_t at = e * p.K + c;
      const A dh = carry + (p.grad_out ? to_acc<T>(static_cast<const T *>(p.grad_out)[at]) : (A)0);
      static_cast<T *>(p.grad_src)[at] = from_acc<T>(dh);
      const A before = e > b * p.E + lo ? to_acc<T>(static_cast<const T *>(p.fwd)[at - p.K]) : init;
      if (p.partial) static_cast<A *>(p.partial)[at] = dh * before;
      else if (p.grad_gate) static_cast<G *>(p.grad_gate)[at] = from_acc<G>(dh * before);
      carry = to_acc<G>(static_cast<const G *>(p.gate)[e * gates + c / p.width]) * dh;
    }
    if (p.grad_state) static_cast<A *>(p.grad_state)[it] = carry;
  }
}

// rows outside every segment: zeros
template <typename T, typename G> __global__ void __launch_bounds__(kThreads) scan_outside_kernel(ScanParams p, T *x, G *y, acc_t<T> *z) {
  const int64_t items = p.B * p.E * p.K;
  for (int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x; it < items; it += (int64_t)gridDim.x * kThreads) {
    const int64_t e = it / p.K % p.E, b = it / p.K / p.E;
    const int64_t *ip = p.indptr + b * p.bstride;
    if (p.N > 0 && e >= ip[0] && e < ip[p.N]) continue;
    if (x) x[it] = from_acc<T>(0);
    if (y) y[it] = from_acc<G>(0);
    if (z) z[it] = 0;
  }
}

template <typename A, typename G> __global__ void __launch_bounds__(kThreads) scan_gate_sum_kernel(const A *__restrict__ part, G *__restrict__ out, int64_t n, int64_t width) {
  for (int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x; it < n; it += (int64_t)gridDim.x * kThreads) {
    A s = 0;
    for (int64_t i = 0; i < width; ++i) s += part[it * width + i];
    out[it] = from_acc<G>(s);
  }
}

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

unsigned flat_blocks(int64_t items) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + kThreads - 1) / kThreads, (int64_t)sm_count() * 64));
}

template <typename F> int with_types(int dtype, int gate_dtype, F f) {
  switch (dtype) {
    case TSB_F32: return gate_dtype == TSB_F32 ? f(float(), float()) : (int)TSB_ERR_DTYPE;
    case TSB_F64: return gate_dtype == TSB_F64 ? f(double(), double()) : (int)TSB_ERR_DTYPE;
    case TSB_F16: return gate_dtype == TSB_F16 ? f(__half(), __half()) : gate_dtype == TSB_F32 ? f(__half(), float()) : (int)TSB_ERR_DTYPE;
    case TSB_BF16:
      return gate_dtype == TSB_BF16 ? f(__nv_bfloat16(), __nv_bfloat16()) : gate_dtype == TSB_F32 ? f(__nv_bfloat16(), float()) : (int)TSB_ERR_DTYPE;
    default: return TSB_ERR_DTYPE;
  }
}

bool bad_shape(int64_t B, int64_t E, int64_t K, int64_t N, int64_t width) {
  return B < 0 || E < 0 || K < 0 || N < 0 || width < 1 || K % width != 0;
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" size_t tsb_scan_csr_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int, int) { return 0; }

extern "C" int tsb_scan_csr(const void *src, const void *gate, const int64_t *indptr, const void *state, void *out, void *last,
                            int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int64_t indptr_batch_stride, int dtype,
                            int gate_dtype, void *, size_t, tsb_stream_t stream) {
  if (bad_shape(B, E, K, N, width)) return TSB_ERR_ARG;
  return with_types(dtype, gate_dtype, [&](auto t, auto g) -> int {
    using T = decltype(t);
    using G = decltype(g);
    if (B == 0 || K == 0 || (E == 0 && (N == 0 || !last))) return TSB_OK;
    if (!indptr || (E > 0 && (!src || !gate || !out))) return TSB_ERR_ARG;
    ScanParams p{};
    p.src = src; p.gate = gate; p.state = state; p.indptr = indptr; p.out = out; p.last = last;
    p.B = B; p.E = E; p.K = K; p.N = N; p.width = width; p.bstride = indptr_batch_stride;
    if (E > 0) scan_outside_kernel<T, G><<<flat_blocks(B * E * K), kThreads, 0, (cudaStream_t)stream>>>(p, static_cast<T *>(out), nullptr, nullptr);
    if (N > 0) scan_walk_kernel<T, G><<<flat_blocks(B * N * K), kThreads, 0, (cudaStream_t)stream>>>(p);
    return launch_status();
  });
}

extern "C" size_t tsb_scan_csr_backward_workspace_bytes(int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int dtype, int) {
  if (bad_shape(B, E, K, N, width) || width == 1) return 0;
  return (size_t)(B * E * K) * dtype_acc_bytes(dtype);
}

extern "C" int tsb_scan_csr_backward(const void *grad_out, const void *grad_last, const void *gate, const void *out,
                                     const int64_t *indptr, const void *state, void *grad_src, void *grad_gate, void *grad_state,
                                     int64_t B, int64_t E, int64_t K, int64_t N, int64_t width, int64_t indptr_batch_stride,
                                     int dtype, int gate_dtype, void *workspace, size_t workspace_bytes, tsb_stream_t stream) {
  if (bad_shape(B, E, K, N, width)) return TSB_ERR_ARG;
  return with_types(dtype, gate_dtype, [&](auto t, auto g) -> int {
    using T = decltype(t);
    using G = decltype(g);
    using A = acc_t<T>;
    if (B == 0 || K == 0 || (E == 0 && (N == 0 || !grad_state))) return TSB_OK;
    if (!indptr || (E > 0 && (!gate || !out || !grad_src))) return TSB_ERR_ARG;
    const bool shared = grad_gate && width > 1 && E > 0;
    if (shared && (!workspace || workspace_bytes < tsb_scan_csr_backward_workspace_bytes(B, E, K, N, width, dtype, gate_dtype)))
      return TSB_ERR_WORKSPACE;
    ScanParams p{};
    p.gate = gate; p.state = state; p.indptr = indptr; p.grad_out = grad_out; p.grad_last = grad_last; p.fwd = out;
    p.grad_src = grad_src; p.grad_gate = grad_gate; p.grad_state = grad_state; p.partial = shared ? workspace : nullptr;
    p.B = B; p.E = E; p.K = K; p.N = N; p.width = width; p.bstride = indptr_batch_stride;
    cudaStream_t st = (cudaStream_t)stream;
    if (E > 0)
      scan_outside_kernel<T, G><<<flat_blocks(B * E * K), kThreads, 0, st>>>(
          p, static_cast<T *>(grad_src), width == 1 ? static_cast<G *>(grad_gate) : nullptr, shared ? static_cast<A *>(workspace) : nullptr);
    if (N > 0) scan_walk_backward_kernel<T, G><<<flat_blocks(B * N * K), kThreads, 0, st>>>(p);
    if (shared)
      scan_gate_sum_kernel<A, G><<<flat_blocks(B * E * (K / width)), kThreads, 0, st>>>(static_cast<const A *>(workspace), static_cast<G *>(grad_gate), B * E * (K / width), width);
    return launch_status();
  });
}

extern "C" int tsb_scan_step(const void *src, const void *gate, void *state, void *out, int64_t n, int64_t K, int64_t width,
                             int64_t state_stride, int dtype, int gate_dtype, tsb_stream_t stream) {
  if (n < 0 || K < 0 || width < 1 || K % width != 0 || (n > 1 && state_stride < K)) return TSB_ERR_ARG;
  return with_types(dtype, gate_dtype, [&](auto t, auto g) -> int {
    using T = decltype(t);
    using G = decltype(g);
    if (n == 0 || K == 0) return TSB_OK;
    if (!src || !gate || !state || !out) return TSB_ERR_ARG;
    scan_step_kernel<T, G><<<flat_blocks(n * K), kThreads, 0, (cudaStream_t)stream>>>(
        static_cast<const T *>(src), static_cast<const G *>(gate), static_cast<acc_t<T> *>(state), static_cast<T *>(out), n, K, width, state_stride);
    return launch_status();
  });
}
