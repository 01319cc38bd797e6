// Entry points of the gated linear recurrence (the tile kernel is in scan.cuh) and its single-token form.
#include "scan.cuh"

namespace tsb {
namespace {

using scan::ScanParams;

// state = gate * state + src in place, one thread for VEC channels of a state.  Bound by HBM where there are enough states:
// src, gate, state twice, out, each moved once.
template <typename T, typename G, int VEC, bool SHARED>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const T *src, const G *gate, acc_t<T> *state, T *out, int64_t n, int64_t K,
                                                             int64_t width, int64_t stride) {
  using A = acc_t<T>;
  const int64_t Kv = K / VEC, items = n * Kv;
  const bool small = items <= 0xffffffffLL;  // 32-bit divisions
  for (int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x; it < items; it += (int64_t)gridDim.x * kThreads) {
    const int64_t i = small ? (int64_t)((unsigned)it / (unsigned)Kv) : it / Kv, c = (it - i * Kv) * VEC;
    const Pack<T, VEC> x = ld_stream<T, VEC>(src + i * K + c);
    Pack<A, VEC> s = ld_pack<A, VEC>(state + i * stride + c);
    Pack<T, VEC> o;
    if constexpr (SHARED) {
      const A g = to_acc<G>(gate[i * (K / width) + (small ? (int64_t)((unsigned)c / (unsigned)width) : c / width)]);
#pragma unroll
      for (int v = 0; v < VEC; ++v) s.v[v] = g * s.v[v] + to_acc<T>(x.v[v]);
    } else {
      const Pack<G, VEC> g = ld_stream<G, VEC>(gate + i * K + c);
#pragma unroll
      for (int v = 0; v < VEC; ++v) s.v[v] = to_acc<G>(g.v[v]) * s.v[v] + to_acc<T>(x.v[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.v[v] = from_acc<T>(s.v[v]);
    st_pack<A, VEC>(state + i * stride + c, s);
    st_stream<T, VEC>(out + i * K + c, o);
  }
}

template <typename T, typename G>
int launch_step(const T *src, const G *gate, acc_t<T> *state, T *out, int64_t n, int64_t K, int64_t width, int64_t stride, cudaStream_t stream) {
  constexpr int VEC = 16 / (int)sizeof(acc_t<T>);  // 16 bytes of the state
  const bool packs = K % VEC == 0 && (n <= 1 || stride % VEC == 0) && (width == 1 || width % VEC == 0) && aligned16(state) &&
                     aligned16(src) && aligned16(out) && (width > 1 || aligned16(gate));
  const auto go = [&](auto v, auto shared) {
    constexpr int V = decltype(v)::value;
    scan_step_kernel<T, G, V, decltype(shared)::value><<<scan::flat_blocks(n * (K / V)), kThreads, 0, stream>>>(src, gate, state, out, n, K, width, stride);
    return launch_status();
  };
  const auto with_vec = [&](auto v) { return width > 1 ? go(v, std::true_type()) : go(v, std::false_type()); };
  return packs ? with_vec(std::integral_constant<int, VEC>()) : with_vec(std::integral_constant<int, 1>());
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
  if (wide && dtype != TSB_F16 && dtype != TSB_BF16) return TSB_ERR_ARG;
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
    return launch_step<T, G>(static_cast<const T *>(src), static_cast<const G *>(gate), static_cast<acc_t<T> *>(state), static_cast<T *>(out), n, K,
                             width, state_stride, (cudaStream_t)stream);
  });
}
