// The router's choice: softmax over E expert logits, the k largest, and the gradient.
//
//   p = softmax(logits[t, :]);  index[t, :] = the k largest logits;  weight[t, j] = p[index[t, j]] (/ their sum)
//
// A warp owns a token and keeps its logits in registers (logit 32 r + lane in register r), so they are read once.  The
// order of the logits is that of a 32-bit key, so that one warp reduction finds a maximum.  Bound by the instructions of
// the choice, not by HBM: of a few hundred logits, most are ruled out first.  The k-th largest of the 32 lane maxima is a
// lower bound of the k-th largest logit; the logits that reach it, rarely more than 2 k, move to one register of the
// warp, and the k rounds of the choice run on that register.  (65536 x 256 fp32, k = 8: 50 us, 87 with every round
// over all registers; the backward, which writes, 25: it waits for its loads of weight, gradient and index.)
#include "common.cuh"

namespace tsb {
namespace {

// Ascending in the value, NaN above +inf, -0 = +0 (adding 0 also makes every NaN the same).  Keys up to that of -inf are
// never chosen; a chosen expert's key is set to 0, so it cannot be chosen again.
constexpr unsigned kNever = 0x007fffffu;
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned u = __float_as_uint(v + 0.0f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

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

// What a lane knows of a choice of up to 32: it holds the rank-th chosen expert (rank -1: none).
struct Choice { unsigned key; int expert, rank; };

// Up to 32 rounds over all registers; returns how many experts were chosen, fewer than n if nothing was left.
template <int R> __device__ __forceinline__ int choose_all(unsigned (&key)[R], int n, int lane, Choice &mine) {
  for (int j = 0; j < n; ++j) {
    unsigned best = key[0];
    int at = lane;
#pragma unroll
    for (int r = 1; r < R; ++r)
      if (key[r] > best) { best = key[r]; at = r * 32 + lane; }
    const unsigned win = __reduce_max_sync(kFullMask, best);
    if (win <= kNever) return j;
    const int who = (int)__reduce_min_sync(kFullMask, best == win ? (unsigned)at : 0xffffffffu);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (who == r * 32 + lane) key[r] = 0;
    if (lane == j) mine = {win, who, j};
  }
  return n;
}

// The same for n <= 32 through the candidates that reach a lower bound of the n-th largest logit; -1 if they are more than
// 32 (many equal logits), with nothing changed.  Candidates lie in the order of the experts, so of equal ones the first
// lane's goes first.
template <int R> __device__ __forceinline__ int choose_few(const unsigned (&key)[R], int n, int lane, uint2 *room, Choice &mine) {
  unsigned top = key[0];
#pragma unroll
  for (int r = 1; r < R; ++r) top = max(top, key[r]);
  unsigned bound = kNever + 1;  // fewer than n lanes hold a logit that may be chosen: all of those are candidates
  for (int j = 0; j < n; ++j) {
    const unsigned win = __reduce_max_sync(kFullMask, top);
    bound = max(win, kNever + 1);
    if (win <= kNever) break;
    if (top == win) top = 0;  // (equal maxima leave together: the bound is then lower than it could be)
  }
  int found = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = key[r] >= bound;
    const unsigned all = __ballot_sync(kFullMask, in);
    const int place = found + __popc(all & ((1u << lane) - 1u));
    if (in && place < 32) room[place] = make_uint2(key[r], r * 32 + lane);
    found += __popc(all);
  }
  __syncwarp();
  if (found > 32) return -1;
  const uint2 own = lane < found ? room[lane] : make_uint2(0, 0);
  mine = {own.x, (int)own.y, -1};
  unsigned left = own.x;
  for (int j = 0; j < n; ++j) {
    const unsigned win = __reduce_max_sync(kFullMask, left);
    if (win <= kNever) return j;
    if (lane == __ffs(__ballot_sync(kFullMask, left == win)) - 1) {
      left = 0;
      mine.rank = j;
    }
  }
  return n;
}

template <typename T, int R>
__global__ void __launch_bounds__(kThreads) topk_kernel(const T *__restrict__ logits, float *__restrict__ weight,
                                                        int64_t *__restrict__ index, int64_t T_, int E, int k,
                                                        int normalize) {
  __shared__ uint2 s_room[R > 2 ? kThreads : 1];
  const int lane = threadIdx.x & 31;
  uint2 *room = R > 2 ? s_room + (threadIdx.x & ~31) : s_room;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < T_; t += step) {
    const Logits<R> x = load_logits<T, R>(logits + t * E, E, lane);
    unsigned key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = order_key(x.v[r]);
    float top = 0.0f, den = 0.0f;
    if (!normalize) softmax_stats<R>(x, top, den);

    // choices 32 at a time, lane j the j-th of them; normalised weights get their denominator at the end
    float chosen = 0.0f;
    for (int j0 = 0; j0 < k; j0 += 32) {
      const int n = min(32, k - j0);
      Choice mine{0, -1, -1};
      int found = -1;
      if constexpr (R > 2)
        if (k <= 32) found = choose_few<R>(key, n, lane, room, mine);
      if (found < 0) {
        mine = {0, -1, -1};
        found = choose_all<R>(key, n, lane, mine);
      }
      const float v = key_value(mine.key);
      if (normalize && j0 == 0) {  // the largest of all
        const unsigned first = __ballot_sync(kFullMask, mine.rank == 0);
        top = __shfl_sync(kFullMask, v, first ? __ffs(first) - 1 : 0);
      }
      const float p = mine.rank < 0 ? 0.0f : expf(v - top);
      if (normalize) {
        float sum = p;
#pragma unroll
        for (int s = 16; s; s >>= 1) sum += shfl_xor(sum, s);
        chosen += sum;
      }
      if (mine.rank >= 0) {
        index[t * k + j0 + mine.rank] = mine.expert;
        weight[t * k + j0 + mine.rank] = k <= 32 ? p / (normalize ? chosen : den) : p;
      }
      if (lane >= found && lane < n) {
        index[t * k + j0 + lane] = -1;
        weight[t * k + j0 + lane] = 0.0f;
      }
    }
    if (k > 32) {
      if (normalize) den = chosen;
      __syncwarp();
      for (int j = lane; j < k; j += 32)
        if (index[t * k + j] >= 0) weight[t * k + j] /= den;
    }
  }
}

// At the chosen: w_j (g_j - S) with S = sum w g; elsewhere 0 if the weights are normalised (a softmax over the chosen
// logits alone), else -p S.  The row is written first, then the k chosen values over it.
template <typename T, int R>
__global__ void __launch_bounds__(kThreads)
topk_backward_kernel(const T *__restrict__ logits, const float *__restrict__ weight, const int64_t *__restrict__ index,
                     const float *__restrict__ grad_weight, T *__restrict__ grad_logits, int64_t T_, int E, int k,
                     int normalize) {
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < T_; t += step) {
    T *row = grad_logits + t * E;
    const float w0 = lane < k ? weight[t * k + lane] : 0.0f, g0 = lane < k ? grad_weight[t * k + lane] : 0.0f;
    const int64_t e0 = lane < k ? index[t * k + lane] : -1;
    float s = e0 < 0 ? 0.0f : w0 * g0;
    for (int j = lane + 32; j < k; j += 32)
      if (index[t * k + j] >= 0) s += weight[t * k + j] * grad_weight[t * k + j];
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
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = r * 32 + lane;
      if (e < E) row[e] = from_acc<T>(g.v[r]);
    }
    __syncwarp();
    if (e0 >= 0 && e0 < E) row[e0] = from_acc<T>(w0 * (g0 - s));
    for (int j = lane + 32; j < k; j += 32) {
      const int64_t e = index[t * k + j];
      if (e >= 0 && e < E) row[e] = from_acc<T>(weight[t * k + j] * (grad_weight[t * k + j] - s));
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
