// The router's choice: softmax over E expert logits, the k largest, and the gradient.
//
//   p = softmax(logits[t, :]);  index[t, :] = the k largest logits;  weight[t, j] = p[index[t, j]] (/ their sum)
//
// A warp owns a token and keeps its logits in registers (logits 32 r + lane in register r), so they are read once.
// The order of the logits is that of a 32-bit key (sign-folded bits of the fp32 value): one iteration of the choice is a
// maximum over the lane's registers, one warp reduction of the key and one of the smallest index that holds it.
#include "common.cuh"

namespace tsb {
namespace {

// Ascending in the value, NaN above +inf, -0 = +0.  -inf maps to kNever: such experts are never chosen, and a chosen
// expert's key is set to it, so it cannot be chosen again.
constexpr unsigned kNever = 0;
__device__ __forceinline__ unsigned order_key(float v) {
  if (v != v) return 0xffffffffu;
  const unsigned u = __float_as_uint(v + 0.0f);  // -0 + 0 = +0
  if (u == 0xff800000u) return kNever;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <int R> struct Logits { float v[R]; };

template <typename T, int R> __device__ __forceinline__ Logits<R> load_logits(const T *row, int E, int lane) {
  Logits<R> x;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = r * 32 + lane;
    x.v[r] = e < E ? to_acc<T>(row[e]) : -INFINITY;
  }
  return x;
}

// Largest logit of the row, and the sum of exp(logit - largest).  A row of -inf alone has the sum 0.
template <int R> __device__ __forceinline__ void softmax_stats(const Logits<R> &x, float &top, float &total) {
  float m = x.v[0];
#pragma unroll
  for (int r = 1; r < R; ++r) m = fmaxf(m, x.v[r]);
#pragma unroll
  for (int s = 16; s; s >>= 1) m = fmaxf(m, shfl_xor(m, s));
  const float base = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) sum += expf(x.v[r] - base);
#pragma unroll
  for (int s = 16; s; s >>= 1) sum += shfl_xor(sum, s);
  top = base;
  total = sum;
}

template <typename T, int R>
__global__ void __launch_bounds__(kThreads) topk_kernel(const T *__restrict__ logits, float *__restrict__ weight,
                                                        int64_t *__restrict__ index, int64_t T_, int E, int k,
                                                        int normalize) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < T_; t += step) {
    const Logits<R> x = load_logits<T, R>(logits + t * E, E, lane);
    float top, total;
    softmax_stats<R>(x, top, total);
    unsigned key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = order_key(x.v[r]);

    // lane j of a block of 32 choices keeps the j-th; the sum of the chosen runs along in the order of the choice
    float chosen_sum = 0.0f;
    for (int j0 = 0; j0 < k; j0 += 32) {
      float my_e = 0.0f;
      int my_i = -1;
      const int n = min(32, k - j0);
      for (int j = 0; j < n; ++j) {
        unsigned best = key[0];
        int at = lane;
        float val = x.v[0];
#pragma unroll
        for (int r = 1; r < R; ++r)
          if (key[r] > best) { best = key[r]; at = r * 32 + lane; val = x.v[r]; }
        const unsigned win = __reduce_max_sync(kFullMask, best);
        if (win == kNever) break;  // nothing left: this choice and the rest stay -1 with weight 0
        const int who = (int)__reduce_min_sync(kFullMask, best == win ? (unsigned)at : 0xffffffffu);
        const float p = expf(__shfl_sync(kFullMask, val, who & 31) - top);
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (who == r * 32 + lane) key[r] = kNever;
        chosen_sum += p;
        if (lane == j) { my_e = p; my_i = who; }
      }
      if (lane < n) {
        index[t * k + j0 + lane] = my_i;
        weight[t * k + j0 + lane] = my_e;  // still without its denominator
      }
    }
    const float den = normalize ? chosen_sum : total;
    __syncwarp();
    for (int j = lane; j < k; j += 32) {
      const float w = weight[t * k + j];
      weight[t * k + j] = index[t * k + j] < 0 ? 0.0f : w / den;
    }
  }
}

// normalize: the softmax over the chosen logits alone, grad[i_j] = w_j (g_j - sum w g), zero elsewhere;
// else: grad = -p S, plus w_j g_j at the chosen, with S = sum w g.
template <typename T, int R>
__global__ void __launch_bounds__(kThreads)
topk_backward_kernel(const T *__restrict__ logits, const float *__restrict__ weight, const int64_t *__restrict__ index,
                     const float *__restrict__ grad_weight, T *__restrict__ grad_logits, int64_t T_, int E, int k,
                     int normalize) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < T_; t += step) {
    float s = 0.0f;
    for (int j = lane; j < k; j += 32) s += weight[t * k + j] * grad_weight[t * k + j];
#pragma unroll
    for (int m = 16; m; m >>= 1) s += shfl_xor(s, m);
    Logits<R> g;
    if (normalize) {
#pragma unroll
      for (int r = 0; r < R; ++r) g.v[r] = 0.0f;
    } else {
      g = load_logits<T, R>(logits + t * E, E, lane);
      float top, total;
      softmax_stats<R>(g, top, total);
#pragma unroll
      for (int r = 0; r < R; ++r) g.v[r] = total == 0.0f ? 0.0f : -s * (expf(g.v[r] - top) / total);
    }
    for (int j = 0; j < k; ++j) {
      const int64_t e = index[t * k + j];
      if (e < 0) continue;
      const float w = weight[t * k + j], gw = grad_weight[t * k + j];
      const float d = w * (normalize ? gw - s : gw);
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (e == r * 32 + lane) g.v[r] += d;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = r * 32 + lane;
      if (e < E) grad_logits[t * E + e] = from_acc<T>(g.v[r]);
    }
  }
}

int topk_check(int64_t T, int64_t E, int64_t k, int dtype) {
  if (T < 0 || E < 1 || k < 1 || k > E) return TSB_ERR_ARG;
  if (E > 1024) return TSB_ERR_TOO_LARGE;
  if (dtype != TSB_F32 && dtype != TSB_F16 && dtype != TSB_BF16) return TSB_ERR_DTYPE;
  return TSB_OK;
}

unsigned token_blocks(int64_t T) {
  const int64_t want = (T + kThreads / 32 - 1) / (kThreads / 32), most = (int64_t)sm_count() * 8;
  return (unsigned)(want < most ? want : most);
}

// registers a lane needs for E logits, as a compile-time number
template <typename F> int with_registers(int64_t E, F f) {
  if (E <= 32) return f(std::integral_constant<int, 1>());
  if (E <= 64) return f(std::integral_constant<int, 2>());
  if (E <= 128) return f(std::integral_constant<int, 4>());
  if (E <= 256) return f(std::integral_constant<int, 8>());
  if (E <= 512) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}

template <typename F> int with_float_type(int dtype, F f) {
  if (dtype == TSB_F32) return f(float());
  if (dtype == TSB_F16) return f(__half());
  return f(__nv_bfloat16());
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_expert_topk(const void *logits, float *weight, int64_t *index, int64_t T, int64_t E, int64_t k,
                               int normalize, int dtype, tsb_stream_t stream) {
  if (const int st = topk_check(T, E, k, dtype)) return st;
  if (T == 0) return TSB_OK;
  if (!logits || !weight || !index) return TSB_ERR_ARG;
  return with_float_type(dtype, [&](auto type) {
    using scalar_t = decltype(type);
    return with_registers(E, [&](auto regs) {
      topk_kernel<scalar_t, decltype(regs)::value><<<token_blocks(T), kThreads, 0, (cudaStream_t)stream>>>(
          static_cast<const scalar_t *>(logits), weight, index, T, (int)E, (int)k, normalize);
      return launch_status();
    });
  });
}

extern "C" int tsb_expert_topk_backward(const void *logits, const float *weight, const int64_t *index,
                                        const float *grad_weight, void *grad_logits, int64_t T, int64_t E, int64_t k,
                                        int normalize, int dtype, tsb_stream_t stream) {
  if (const int st = topk_check(T, E, k, dtype)) return st;
  if (T == 0) return TSB_OK;
  if (!logits || !weight || !index || !grad_weight || !grad_logits) return TSB_ERR_ARG;
  return with_float_type(dtype, [&](auto type) {
    using scalar_t = decltype(type);
    return with_registers(E, [&](auto regs) {
      topk_backward_kernel<scalar_t, decltype(regs)::value><<<token_blocks(T), kThreads, 0, (cudaStream_t)stream>>>(
          static_cast<const scalar_t *>(logits), weight, index, grad_weight, static_cast<scalar_t *>(grad_logits), T,
          (int)E, (int)k, normalize);
      return launch_status();
    });
  });
}
