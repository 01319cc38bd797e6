// Rows to the experts and back: spread (one row of few copied to its k places in many) and fold (k rows of many summed
// into one row of few), with weights and, for the weights' gradient, the k dot products alongside.
//
//   spread: many[slot[t,j], :] = few[t, :] (* weight[t,j])          dot[t,j] = <few[t, :], rows[slot[t,j], :]>
//   fold:   few[t, :] = sum_j many[slot[t,j], :] (* weight[t,j])    dot[t,j] = <other[t, :], many[slot[t,j], :]>
//
// Both are bound by HBM: a pass moves T rows of few and T*k rows of many once.  Work is driven by the tokens, because a
// row of few is then read (or written) once; driven by the places, dispatch would read it k times, far apart in time.
#include <algorithm>

#include "common.cuh"

namespace tsb {
namespace {

struct RowsParams {
  const void *few_in;        // spread: the source; fold with dot: `other`
  const void *many_in;       // fold: the source; spread with dot: `rows`
  const int64_t *slot;
  const int64_t *used;       // spread: rows of many from *used on are zeroed
  const void *weight;
  void *few_out, *many_out, *dot;
  int64_t T, k, K, M;
};

// one thread: one pack of one token
template <typename T, int VEC, bool SPREAD>
__global__ void __launch_bounds__(kThreads) rows_kernel(RowsParams p) {
  using A = acc_t<T>;
  const A *__restrict__ weight = static_cast<const A *>(p.weight);
  const int64_t Kv = p.K / VEC, items = p.T * Kv;
  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t it = first; it < items; it += step) {
    const int64_t t = it / Kv, c = (it - t * Kv) * VEC;
    const int64_t *slot = p.slot + t * p.k;
    if constexpr (SPREAD) {
      const Pack<T, VEC> v = ld_stream<T, VEC>(static_cast<const T *>(p.few_in) + t * p.K + c);
      T *many = static_cast<T *>(p.many_out) + c;
      for (int64_t j = 0; j < p.k; ++j) {
        const int64_t to = slot[j];
        if (to < 0 || to >= p.M) continue;
        Pack<T, VEC> o = v;
        if (weight) {
          const A w = weight[t * p.k + j];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o.v[i] = from_acc<T>(to_acc<T>(v.v[i]) * w);
        }
        st_stream<T, VEC>(many + to * p.K, o);
      }
    } else {
      const T *many = static_cast<const T *>(p.many_in) + c;
      A sum[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] = 0;
      for (int64_t j = 0; j < p.k; ++j) {
        const int64_t from = slot[j];
        if (from < 0 || from >= p.M) continue;
        const Pack<T, VEC> v = ld_stream<T, VEC>(many + from * p.K);
        const A w = weight ? weight[t * p.k + j] : (A)1;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += to_acc<T>(v.v[i]) * w;
      }
      Pack<T, VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_acc<T>(sum[i]);
      st_stream<T, VEC>(static_cast<T *>(p.few_out) + t * p.K + c, o);
    }
  }
  if constexpr (SPREAD) {
    const int64_t used = clamp64(*p.used, 0, p.M);
    T *tail = static_cast<T *>(p.many_out) + used * p.K;
    Pack<T, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.v[i] = from_acc<T>((A)0);
    for (int64_t it = first; it < (p.M - used) * Kv; it += step) st_stream<T, VEC>(tail + it * VEC, zero);
  }
}

// one warp: one (token, choice), its dot product
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rows_dot_kernel(RowsParams p) {
  using A = acc_t<T>;
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < p.M; i += step) {
    const int64_t t = i / p.k, at = p.slot[i];
    A sum = 0;
    if (at >= 0 && at < p.M) {
      const T *a = static_cast<const T *>(p.few_in) + t * p.K, *b = static_cast<const T *>(p.many_in) + at * p.K;
      for (int64_t c = (int64_t)lane * VEC; c < p.K; c += 32 * VEC) {
        const Pack<T, VEC> x = ld_pack<T, VEC>(a + c), y = ld_stream<T, VEC>(b + c);
#pragma unroll
        for (int q = 0; q < VEC; ++q) sum += to_acc<T>(x.v[q]) * to_acc<T>(y.v[q]);
      }
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) sum += shfl_xor(sum, m);
    if (lane == 0) static_cast<A *>(p.dot)[i] = sum;
  }
}

template <typename T, int VEC, bool SPREAD> int launch_rows(const RowsParams &p, cudaStream_t stream) {
  const int64_t most = (int64_t)sm_count() * 64;
  const int64_t blocks = std::max<int64_t>(1, std::min(most, (p.T * (p.K / VEC) + kThreads - 1) / kThreads));
  rows_kernel<T, VEC, SPREAD><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
  if (p.dot) {
    const int64_t warps = std::min(most, (p.M + kThreads / 32 - 1) / (kThreads / 32));
    rows_dot_kernel<T, VEC><<<(unsigned)warps, kThreads, 0, stream>>>(p);
  }
  return launch_status();
}

template <bool SPREAD> int rows_entry(const RowsParams &p, int dtype, cudaStream_t stream) {
  if (dtype != TSB_F32 && dtype != TSB_F64 && dtype != TSB_F16 && dtype != TSB_BF16) return TSB_ERR_DTYPE;
  if (p.K == 0) {  // rows without features: empty products
    if (p.dot && cudaMemsetAsync(p.dot, 0, (size_t)p.M * dtype_acc_bytes(dtype), stream) != cudaSuccess) return TSB_ERR_LAUNCH;
    return TSB_OK;
  }
  const bool aligned = aligned16(p.few_in) && aligned16(p.many_in) && aligned16(p.few_out) && aligned16(p.many_out);
  const auto go = [&](auto type) {
    using T = decltype(type);
    constexpr int full = full_vec<T>();
    return aligned && p.K % full == 0 ? launch_rows<T, full, SPREAD>(p, stream) : launch_rows<T, 1, SPREAD>(p, stream);
  };
  switch (dtype) {
    case TSB_F32: return go(float());
    case TSB_F64: return go(double());
    case TSB_F16: return go(__half());
    default: return go(__nv_bfloat16());
  }
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_expert_spread(const void *few, const int64_t *slot, const int64_t *used, const void *weight,
                                 const void *rows, void *many, void *dot, int64_t T, int64_t k, int64_t K, int dtype,
                                 tsb_stream_t stream) {
  if (T < 0 || k < 1 || K < 0 || (K > 0 && (rows != nullptr) != (dot != nullptr))) return TSB_ERR_ARG;
  if (T == 0) return TSB_OK;
  if (!slot || (K > 0 && (!few || !many || !used))) return TSB_ERR_ARG;
  return rows_entry<true>({few, rows, slot, used, weight, nullptr, many, dot, T, k, K, T * k}, dtype, (cudaStream_t)stream);
}

extern "C" int tsb_expert_fold(const void *many, const int64_t *slot, const void *weight, const void *other, void *few,
                               void *dot, int64_t T, int64_t k, int64_t K, int dtype, tsb_stream_t stream) {
  if (T < 0 || k < 1 || K < 0 || (K > 0 && (other != nullptr) != (dot != nullptr))) return TSB_ERR_ARG;
  if (T == 0) return TSB_OK;
  if (!slot || (K > 0 && (!few || !many))) return TSB_ERR_ARG;
  return rows_entry<false>({other, many, slot, nullptr, weight, few, nullptr, dot, T, k, K, T * k}, dtype,
                           (cudaStream_t)stream);
}
