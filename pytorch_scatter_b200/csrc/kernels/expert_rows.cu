// Rows to the experts and back: spread (one row of few copied to its k places in many) and fold (k rows of many summed
// into one row of few), with weights and, for the weights' gradient, the k dot products alongside.
//
//   spread: many[slot[t,j], :] = few[t, :] (* weight[t,j])          dot[t,j] = <few[t, :], rows[slot[t,j], :]>
//   fold:   few[t, :] = sum_j many[slot[t,j], :] (* weight[t,j])    dot[t,j] = <other[t, :], many[slot[t,j], :]>
//
// Both are bound by HBM: a pass moves T rows of few and T*k rows of many once.  Work is driven by the tokens, because a
// row of few is then read (or written) once; driven by the places, dispatch would read it k times, far apart in time.
// Rows move in 16-byte chunks.  Where the row length is no multiple of 16 bytes, chunks are those of the row that is
// written, and the data comes out of the two aligned chunks of the source row that hold it, shifted into place: twice the
// load instructions, but whole sectors and 16-byte stores instead of single values.
//
// Rows of many that no slot names are zeroed: those behind the last expert's, and those inside whose entries were dropped
// after the sort (a capacity limit).  Up to kOneList entries a few blocks of the spread look all slots up for the rows that
// they guard; beyond that a second kernel first counts the slots, since usually there are as many as rows (3 to 5 us).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <utility>

#include "mbarrier.cuh"

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
  int zero_blocks;           // spread with ZERO: the first blocks zero the rows that no slot names
};

template <typename T> constexpr int chunk_len() { return 16 / (int)sizeof(T); }

// elements [a, b) of a chunk belong to the row
struct Span { int a, b; };

// V elements from p on, wherever p is; those outside the span are 0.  The loads are issued here, so that those of several
// rows are in flight at once, and read() shifts the elements into place.  lo, hi: the ends of the array p points into; a
// chunk whose two aligned halves are not both inside is read element by element.
template <typename T> struct AnyChunk {
  static constexpr int V = chunk_len<T>();
  uint4 x, y;
  const T *p;
  Span s;
  int off;  // -1: element by element
  __device__ __forceinline__ void load(const T *p_, Span s_, const T *lo, const T *hi) {
    p = p_;
    s = s_;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), base = at & ~(uintptr_t)15;
    off = (int)(at & 15);
    const bool inside = base >= reinterpret_cast<uintptr_t>(lo) && base + 32 <= reinterpret_cast<uintptr_t>(hi);
    if (s.a == 0 && s.b == V && (off == 0 || inside)) {
      x = *reinterpret_cast<const uint4 *>(base);
      y = *reinterpret_cast<const uint4 *>(base + (off ? 16 : 0));
    } else {
      off = -1;
    }
  }
  __device__ __forceinline__ Pack<T, V> read() const {
    Pack<T, V> r;
    if (off >= 0) {
      unsigned w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], off & 2 ? 16 : 0);
      return *reinterpret_cast<const Pack<T, V> *>(w);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = i >= s.a && i < s.b ? p[i] : from_acc<T>((acc_t<T>)0);
    return r;
  }
};
// The same, loaded and shifted at once: where occupancy hides the latency, fewer registers and the branches that spare the
// second load and the shifts win (fold of 16384 x 4 x 2047 bf16: 162 us, 217 with all loads first; with dot products it
// is the other way round, 303 and 237).
template <typename T>
__device__ __forceinline__ Pack<T, chunk_len<T>()> load_any(const T *p, Span s, const T *lo, const T *hi) {
  constexpr int V = chunk_len<T>();
  Pack<T, V> r;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), base = at & ~(uintptr_t)15;
  const int off = (int)(at & 15);
  if (s.a == 0 && s.b == V && (off == 0 || (base >= reinterpret_cast<uintptr_t>(lo) && base + 32 <= reinterpret_cast<uintptr_t>(hi)))) {
    const uint4 x = *reinterpret_cast<const uint4 *>(base);
    if (off == 0) return *reinterpret_cast<const Pack<T, V> *>(&x);
    const uint4 y = *reinterpret_cast<const uint4 *>(base + 16);
    unsigned w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    if (off & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (off & 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    return *reinterpret_cast<const Pack<T, V> *>(w);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = i >= s.a && i < s.b ? p[i] : from_acc<T>((acc_t<T>)0);
  return r;
}
template <typename T> struct AlignedChunk {
  static constexpr int V = chunk_len<T>();
  Pack<T, V> v;
  __device__ __forceinline__ void load(const T *p, Span, const T *, const T *) { v = ld_stream<T, V>(p); }
  __device__ __forceinline__ Pack<T, V> read() const { return v; }
};
template <typename T, bool ALIGNED> using Chunk = std::conditional_t<ALIGNED, AlignedChunk<T>, AnyChunk<T>>;

template <typename T> __device__ __forceinline__ void store_span(T *p, const Pack<T, chunk_len<T>()> &v, Span s) {
  constexpr int V = chunk_len<T>();
  if (s.a == 0 && s.b == V) {
    st_stream<T, V>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= s.a && i < s.b) p[i] = v.v[i];
  }
}

// The c-th 16-byte chunk of a row: its first element (negative where the row begins inside the chunk) and its span.
template <typename T, bool ALIGNED> __device__ __forceinline__ int64_t chunk_of(const T *row, int64_t c, int64_t K, Span &s) {
  constexpr int V = chunk_len<T>();
  if constexpr (ALIGNED) {
    s = {0, V};
    return c * V;
  } else {
    const int64_t e0 = c * V - (int64_t)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    s.a = e0 < 0 ? (int)-e0 : 0;
    s.b = K - e0 < V ? (int)(K - e0) : V;
    return e0;
  }
}
template <typename T, bool ALIGNED> __host__ __device__ __forceinline__ int64_t chunks_of(int64_t K) {
  constexpr int V = chunk_len<T>();
  return ALIGNED ? K / V : (K + 2 * V - 2) / V;
}
template <typename T, typename A> __device__ __forceinline__ Pack<T, chunk_len<T>()> scaled(const Pack<T, chunk_len<T>()> &v, A w) {
  Pack<T, chunk_len<T>()> o;
#pragma unroll
  for (int i = 0; i < chunk_len<T>(); ++i) o.v[i] = from_acc<T>(to_acc<T>(v.v[i]) * w);
  return o;
}

// zeros for the rows of many that no token owns
template <typename T, bool ALIGNED> __device__ __forceinline__ void zero_tail(const RowsParams &p, int64_t first, int64_t step) {
  const int64_t used = clamp64(*p.used, 0, p.M);
  T *tail = static_cast<T *>(p.many_out) + used * p.K;
  constexpr int V = ALIGNED ? chunk_len<T>() : 1;
  Pack<T, V> zero;
#pragma unroll
  for (int i = 0; i < V; ++i) zero.v[i] = from_acc<T>((acc_t<T>)0);
  for (int64_t i = first; i < (p.M - used) * p.K / V; i += step) st_stream<T, V>(tail + i * V, zero);
}

// zeros for the rows [lo, hi) of many that no slot names, by a whole CTA
constexpr int64_t kOneList = 4096;  // entries
template <typename T, bool ALIGNED, int WORDS>
__device__ __forceinline__ void zero_unnamed(const RowsParams &p, int64_t lo, int64_t hi, unsigned (&s_named)[WORDS]) {
  constexpr int V = ALIGNED ? chunk_len<T>() : 1;
  Pack<T, V> zero;
#pragma unroll
  for (int i = 0; i < V; ++i) zero.v[i] = from_acc<T>((acc_t<T>)0);
  for (; lo < hi; lo += WORDS * 32) {
    const int n = (int)(hi - lo < WORDS * 32 ? hi - lo : WORDS * 32);
    for (int i = threadIdx.x; i * 32 < n; i += blockDim.x) s_named[i] = 0;
    __syncthreads();
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < p.M; i += blockDim.x) {
      const uint64_t r = (uint64_t)(p.slot[i] - lo);  // (slots below lo are beyond n, too)
      if (r < (uint64_t)n) atomicOr(&s_named[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < n; r += blockDim.x >> 5) {
      if (s_named[r >> 5] >> (r & 31) & 1) continue;
      T *row = static_cast<T *>(p.many_out) + (lo + r) * p.K;
      for (int64_t c = threadIdx.x & 31; c < p.K / V; c += 32) st_stream<T, V>(row + c * V, zero);
    }
    __syncthreads();
  }
}
// The block's part where the first blocks do that; true: the block has nothing else to do.
template <typename T, bool ALIGNED> __device__ __forceinline__ bool zero_part(const RowsParams &p) {
  if ((int)blockIdx.x >= p.zero_blocks) return false;
  __shared__ unsigned s_named[kOneList / 32];
  const int64_t per = (p.M + p.zero_blocks - 1) / p.zero_blocks, lo = blockIdx.x * per;
  zero_unnamed<T, ALIGNED>(p, lo, lo + per < p.M ? lo + per : p.M, s_named);
  return true;
}

// Many entries: next to the spread, which zeroes the rows from *used on.  Every cluster counts the slots; are there fewer than
// rows, its CTAs look them up for parts of the rows.  Launched to start while the spread's last CTAs run (the two write
// different rows, and what this one reads was there before the spread began), and over when the spread is.
constexpr int kHoleThreads = 1024, kHoleCluster = 8, kHoleWords = 2048;
template <typename T, bool ALIGNED> __global__ void __launch_bounds__(kHoleThreads) __cluster_dims__(kHoleCluster) holes_kernel(RowsParams p) {
  namespace cg = cooperative_groups;
  __shared__ unsigned s_named[kHoleWords];
  __shared__ unsigned s_warp[kHoleThreads / 32];
  __shared__ int64_t s_counts[kHoleCluster];
  auto cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  auto all_run = cluster.barrier_arrive();
  const int64_t used = clamp64(*p.used, 0, p.M);
  unsigned named = 0;
#pragma unroll 8
  for (int64_t i = rank * kHoleThreads + (int)threadIdx.x; i < p.M; i += kHoleCluster * kHoleThreads) named += (uint64_t)p.slot[i] < (uint64_t)used;
  named = __reduce_add_sync(kFullMask, named);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = named;
  __syncthreads();
  cluster.barrier_wait(std::move(all_run));
  if (threadIdx.x < kHoleCluster) {
    int64_t sum = 0;
    for (int w = 0; w < kHoleThreads / 32; ++w) sum += s_warp[w];
    *cluster.map_shared_rank(&s_counts[rank], threadIdx.x) = sum;
  }
  cluster.sync();  // (nobody leaves before all others have written to its shared memory)
  int64_t count = 0;
#pragma unroll
  for (int q = 0; q < kHoleCluster; ++q) count += s_counts[q];
  if (count != used) {
    const int64_t per = (used + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * per;
    zero_unnamed<T, ALIGNED>(p, lo, lo + per < used ? lo + per : used, s_named);
  }
  cudaGridDependencySynchronize();  // the spread is over and its rows are there before this kernel is over
}
template <typename T, bool ALIGNED> int launch_holes(const RowsParams &p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(kHoleCluster * std::max<int64_t>(1, std::min<int64_t>(16, p.M / 16384))));
  cfg.blockDim = dim3(kHoleThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, holes_kernel<T, ALIGNED>, p) == cudaSuccess ? TSB_OK : TSB_ERR_LAUNCH;
}

// Without dot products: one thread, one chunk of one token.  The rows of several choices are in flight at once.
// ZERO (in code of its own: with it the kernel takes 64 registers instead of 46): see zero_part.
template <typename T, bool SPREAD, bool ALIGNED, bool ZERO>
__global__ void __launch_bounds__(kThreads) rows_kernel(RowsParams p) {
  using A = acc_t<T>;
  constexpr int V = chunk_len<T>(), J = 4;
  const A *__restrict__ weight = static_cast<const A *>(p.weight);
  const T *few_in = static_cast<const T *>(p.few_in), *many_in = static_cast<const T *>(p.many_in);
  T *few_out = static_cast<T *>(p.few_out), *many_out = static_cast<T *>(p.many_out);
  const int64_t Kc = chunks_of<T, ALIGNED>(p.K), items = p.T * Kc;
  if constexpr (SPREAD && !ZERO) cudaTriggerProgrammaticLaunchCompletion();  // holes_kernel may start
  if constexpr (ZERO)
    if (zero_part<T, ALIGNED>(p)) return;
  const int skip = ZERO ? p.zero_blocks : 0;
  const int64_t step = (int64_t)(gridDim.x - skip) * kThreads, first = (int64_t)(blockIdx.x - skip) * kThreads + threadIdx.x;
  for (int64_t it = first; it < items; it += step) {
    const int64_t t = items <= 0xffffffffLL ? (int64_t)((unsigned)it / (unsigned)Kc) : it / Kc, c = it - t * Kc;
    const int64_t *slot = p.slot + t * p.k;
    Span s;
    if constexpr (SPREAD) {
      if constexpr (ALIGNED) {
        s = {0, V};
        const Pack<T, V> v = ld_stream<T, V>(few_in + t * p.K + c * V);
        for (int64_t j = 0; j < p.k; ++j) {
          const int64_t to = slot[j];
          if (to < 0 || to >= p.M) continue;
          store_span<T>(many_out + to * p.K + c * V, weight ? scaled<T, A>(v, weight[t * p.k + j]) : v, s);
        }
      } else {
        for (int64_t j = 0; j < p.k; ++j) {
          const int64_t to = slot[j];
          if (to < 0 || to >= p.M) continue;
          T *row = many_out + to * p.K;
          const int64_t e0 = chunk_of<T, false>(row, c, p.K, s);
          if (s.b <= s.a) continue;
          const Pack<T, V> v = load_any<T>(few_in + t * p.K + e0, s, few_in, few_in + p.T * p.K);
          store_span<T>(row + e0, weight ? scaled<T, A>(v, weight[t * p.k + j]) : v, s);
        }
      }
    } else {
      T *row = few_out + t * p.K;
      const int64_t e0 = chunk_of<T, ALIGNED>(row, c, p.K, s);
      if (!ALIGNED && s.b <= s.a) continue;
      A sum[V];
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = 0;
      for (int64_t j0 = 0; j0 < p.k; j0 += J) {
        Pack<T, V> v[J];
        bool some[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int64_t from = j0 + j < p.k ? slot[j0 + j] : -1;
          some[j] = from >= 0 && from < p.M;
          if (!some[j]) continue;
          if constexpr (ALIGNED) v[j] = ld_stream<T, V>(many_in + from * p.K + e0);
          else v[j] = load_any<T>(many_in + from * p.K + e0, s, many_in, many_in + p.M * p.K);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (!some[j]) continue;
          const A w = weight ? weight[t * p.k + j0 + j] : (A)1;
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] += to_acc<T>(v[j].v[i]) * w;
        }
      }
      Pack<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = from_acc<T>(sum[i]);
      store_span<T>(row + e0, o, s);
    }
  }
  if constexpr (SPREAD && !ZERO) zero_tail<T, ALIGNED>(p, first, step);
}

// With dot products: G threads (lanes of a warp, or the CTA) walk one token's chunks, J choices at a time.  WRITE: also
// spread or fold; a fold needs all choices of a chunk at once, so it has J >= k.  Unaligned chunks take
// twice the registers, so fewer choices are in flight.
template <typename T, bool SPREAD, bool ALIGNED, bool WRITE, bool ZERO, int J, int G>
__global__ void __launch_bounds__(kThreads) rows_dot_kernel(RowsParams p) {
  using A = acc_t<T>;
  constexpr int V = chunk_len<T>(), kGroups = kThreads / G, kWarps = kThreads / 32;
  __shared__ A s_part[G > 32 ? kWarps * J : 1];
  const A *__restrict__ weight = static_cast<const A *>(p.weight);
  const T *few_in = static_cast<const T *>(p.few_in), *many_in = static_cast<const T *>(p.many_in);
  T *few_out = static_cast<T *>(p.few_out), *many_out = static_cast<T *>(p.many_out);
  A *dot = static_cast<A *>(p.dot);
  const int64_t Kc = chunks_of<T, ALIGNED>(p.K);
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  if constexpr (SPREAD && !ZERO) cudaTriggerProgrammaticLaunchCompletion();
  if constexpr (ZERO)
    if (zero_part<T, ALIGNED>(p)) return;
  const int skip = ZERO ? p.zero_blocks : 0;
  // whole warps stay together: the last round of tokens may hold groups without one
  for (int64_t t0 = (int64_t)(blockIdx.x - skip) * kGroups; t0 < p.T; t0 += (int64_t)(gridDim.x - skip) * kGroups) {
    const int64_t t = t0 + group;
    const bool live = t < p.T;
    for (int64_t j0 = 0; j0 < p.k; j0 += J) {
      int64_t at[J];
      A w[J], sum[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int64_t i = live && j0 + j < p.k ? p.slot[t * p.k + j0 + j] : -1;
        at[j] = i < p.M ? i : -1;
        w[j] = weight && at[j] >= 0 ? weight[t * p.k + j0 + j] : (A)1;
        sum[j] = 0;
      }
      if (live) {
        const T *few = few_in + t * p.K;
        for (int64_t c = lane; c < Kc; c += G) {
          // the chunks of the row that is written; with many rows written and no alignment, those of each choice's row
          constexpr bool kEach = SPREAD && !ALIGNED;
          Chunk<T, ALIGNED> x[kEach ? J : 1], y[J];
          Span s[kEach ? J : 1];
          int64_t e0[kEach ? J : 1];
          if constexpr (!kEach) {
            e0[0] = chunk_of<T, ALIGNED>(SPREAD || !WRITE ? few : few_out + t * p.K, c, p.K, s[0]);
            if (!ALIGNED && s[0].b <= s[0].a) continue;
            x[0].load(few + e0[0], s[0], few_in, few_in + p.T * p.K);
          }
#pragma unroll
          for (int j = 0; j < J; ++j) {
            if (at[j] < 0) continue;
            if constexpr (kEach) {
              e0[j] = chunk_of<T, false>(many_out + at[j] * p.K, c, p.K, s[j]);
              if (s[j].b <= s[j].a) continue;
              x[j].load(few + e0[j], s[j], few_in, few_in + p.T * p.K);
            }
            y[j].load(many_in + at[j] * p.K + e0[kEach ? j : 0], s[kEach ? j : 0], many_in, many_in + p.M * p.K);
          }
          A fold[V];
#pragma unroll
          for (int i = 0; i < V; ++i) fold[i] = 0;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const Span sj = s[kEach ? j : 0];
            if (at[j] < 0 || (!ALIGNED && sj.b <= sj.a)) continue;
            const Pack<T, V> xv = x[kEach ? j : 0].read(), yv = y[j].read();
            if constexpr (SPREAD && WRITE) store_span<T>(many_out + at[j] * p.K + e0[kEach ? j : 0], weight ? scaled<T, A>(xv, w[j]) : xv, sj);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const A a = to_acc<T>(yv.v[i]);
              sum[j] += to_acc<T>(xv.v[i]) * a;
              if (!SPREAD && WRITE) fold[i] += a * w[j];
            }
          }
          if constexpr (!SPREAD && WRITE) {
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = from_acc<T>(fold[i]);
            store_span<T>(few_out + t * p.K + e0[0], o, s[0]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int m = (G < 32 ? G : 32) / 2; m; m >>= 1) sum[j] += shfl_xor(sum[j], m);
      }
      if constexpr (G > 32) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
          for (int j = 0; j < J; ++j) s_part[(threadIdx.x >> 5) * J + j] = sum[j];
        }
        __syncthreads();
        if (threadIdx.x < J && j0 + threadIdx.x < p.k) {
          A all = 0;
          for (int i = 0; i < kWarps; ++i) all += s_part[i * J + threadIdx.x];
          dot[t * p.k + j0 + threadIdx.x] = all;
        }
        __syncthreads();
      } else if (live) {
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (lane == j % G && j0 + j < p.k) dot[t * p.k + j0 + j] = sum[j];
      }
    }
  }
  if constexpr (SPREAD && !ZERO) zero_tail<T, ALIGNED>(p, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)gridDim.x * kThreads);
}

// Folds, and spreads with dot products, of long aligned rows of many tokens.  Every warp runs a pipeline of its own: bulk
// copies bring pieces of its tokens' rows into a ring in shared memory, two steps and more ahead of the step that is
// worked on, so the bytes in flight depend neither on registers nor on occupancy.  Lane j carries the j-th choice.
// (Combine of 32768 x 2 x 4096 bf16: 139 us against 170 with the rows in flight in registers; with the products, backward,
// 234 against 256 without holes_kernel, 236 with it.  A plain spread has nothing to wait for but one load and stays with
// rows_kernel, 205 us against 225, 209 with holes_kernel.)
constexpr int kBulkWarps = 8, kBulkMostStages = 8, kBulkChunks = 2, kBulkMostDots = 8;
constexpr int kBulkWarpBytes = 27 * 512;  // three steps of 9 pieces of 512 bytes; two CTAs fit an SM
constexpr int kBulkSmem = kBulkWarps * kBulkWarpBytes;

struct BulkShape { int piece, stages, rows; };  // bytes of a row in a step, steps in the ring, rows of a step

template <typename T, bool SPREAD, bool DOT>
__global__ void __launch_bounds__(kBulkWarps * 32, 2) rows_bulk_kernel(RowsParams p, BulkShape shape) {
  using A = acc_t<T>;
  constexpr int V = chunk_len<T>(), U = kBulkChunks;
  extern __shared__ __align__(128) char s_ring[];
  __shared__ __align__(8) uint64_t s_bar[kBulkWarps][kBulkMostStages];
  if constexpr (SPREAD) cudaTriggerProgrammaticLaunchCompletion();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = (int)p.k;
  const unsigned ring = smem_at(s_ring) + warp * kBulkWarpBytes, bar = smem_at(&s_bar[warp][0]);
  const char *ring_p = s_ring + warp * kBulkWarpBytes;
  if (lane < shape.stages) mbar_init(bar + lane * 8);
  mbar_init_done();
  __syncwarp();

  const A *weight = static_cast<const A *>(p.weight);
  const int64_t row_bytes = p.K * (int64_t)sizeof(T);
  const int pieces = (int)((row_bytes + shape.piece - 1) / shape.piece), step_bytes = shape.rows * shape.piece;
  const int64_t warps = (int64_t)gridDim.x * kBulkWarps, first = (int64_t)blockIdx.x * kBulkWarps + warp;
  const char *few_in = static_cast<const char *>(p.few_in), *many_in = static_cast<const char *>(p.many_in);
  char *few_out = static_cast<char *>(p.few_out), *many_out = static_cast<char *>(p.many_out);
  const auto slot_of = [&](int64_t t) -> int64_t {
    if (t >= p.T || lane >= k) return -1;
    const int64_t s = p.slot[t * k + lane];
    return s < p.M ? s : -1;
  };

  // the step that is issued next, its token's slots, and the slots of the token behind it
  int64_t it = first, islot = slot_of(first), inext = slot_of(first + warps);
  int ipiece = 0, istage = 0;
  const auto issue = [&]() {
    if (it < p.T) {
      const int64_t off = (int64_t)ipiece * shape.piece;
      const unsigned len = (unsigned)(row_bytes - off < shape.piece ? row_bytes - off : shape.piece);
      const unsigned b = bar + istage * 8, to = ring + istage * step_bytes;
      const int rows = __popc(__ballot_sync(kFullMask, islot >= 0)) + (DOT ? 1 : 0);
      if (lane == 0) mbar_expect(b, rows * len);
      __syncwarp();
      if (DOT && lane == 0) bulk_load(to, few_in + it * row_bytes + off, len, b);
      if (islot >= 0) bulk_load(to + (lane + (DOT ? 1 : 0)) * shape.piece, many_in + islot * row_bytes + off, len, b);
      if (++ipiece == pieces) {
        ipiece = 0;
        it += warps;
        islot = inext;
        inext = slot_of(it + warps);
      }
    }
    istage = istage + 1 == shape.stages ? 0 : istage + 1;
  };
  for (int i = 0; i < shape.stages - 1; ++i) issue();

  int stage = 0;
  unsigned phase = 0;
  for (int64_t t = first; t < p.T; t += warps) {
    const int64_t my_slot = slot_of(t);
    const A my_weight = weight && lane < k ? weight[t * k + lane] : (A)1;
    const unsigned valid = __ballot_sync(kFullMask, my_slot >= 0);
    A d[kBulkMostDots];
#pragma unroll
    for (int j = 0; j < kBulkMostDots; ++j) d[j] = 0;
    for (int q = 0; q < pieces; ++q) {
      const int64_t off = (int64_t)q * shape.piece;
      const int len = (int)(row_bytes - off < shape.piece ? row_bytes - off : shape.piece);
      const A lost = mbar_wait(bar + stage * 8, phase) ? (A)0 : (A)NAN;
      const char *at = ring_p + stage * step_bytes;
      for (int c0 = lane * 16; c0 - lane * 16 < len; c0 += 32 * 16 * U) {
        Pack<T, V> few[U];
        A sum[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * 512;
          if (DOT && c < len) few[u] = *reinterpret_cast<const Pack<T, V> *>(at + c);
#pragma unroll
          for (int i = 0; i < V; ++i) sum[u][i] = lost;
        }
        const auto choice = [&](int j, A &dj) {
          if (!(valid >> j & 1)) return;
          const A w = __shfl_sync(kFullMask, my_weight, j);
          const char *row = at + (j + (DOT ? 1 : 0)) * shape.piece;
          const int64_t to = SPREAD ? __shfl_sync(kFullMask, my_slot, j) * row_bytes + off : 0;
          dj += lost;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * 512;
            if (c >= len) continue;
            const Pack<T, V> m = *reinterpret_cast<const Pack<T, V> *>(row + c);
            if constexpr (SPREAD) st_stream<T, V>(reinterpret_cast<T *>(many_out + to + c), weight ? scaled<T, A>(few[u], w) : few[u]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const A a = to_acc<T>(m.v[i]);
              if (DOT) dj += to_acc<T>(few[u].v[i]) * a;
              if (!SPREAD) sum[u][i] += a * w;
            }
          }
        };
        if constexpr (DOT) {
#pragma unroll
          for (int j = 0; j < kBulkMostDots; ++j) choice(j, d[j]);
        } else {
          for (int j = 0; j < k; ++j) choice(j, d[0]);
        }
        if constexpr (!SPREAD) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + u * 512;
            if (c >= len) continue;
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = from_acc<T>(sum[u][i]);
            st_stream<T, V>(reinterpret_cast<T *>(few_out + t * row_bytes + off + c), o);
          }
        }
      }
      __syncwarp();  // all lanes have read the step: its place may be filled again
      issue();
      if (++stage == shape.stages) { stage = 0; phase ^= 1; }
    }
    if constexpr (DOT) {
      A mine = 0;
#pragma unroll
      for (int j = 0; j < kBulkMostDots; ++j) {
#pragma unroll
        for (int s = 16; s; s >>= 1) d[j] += shfl_xor(d[j], s);
        if (lane == j) mine = d[j];
      }
      if (lane < k) static_cast<A *>(p.dot)[t * k + lane] = mine;
    }
  }
  if constexpr (SPREAD) zero_tail<T, true>(p, (int64_t)blockIdx.x * kBulkWarps * 32 + threadIdx.x, (int64_t)gridDim.x * kBulkWarps * 32);
}

// Whether the pipeline takes the problem: enough tokens for every warp to have some, rows of 512 bytes and more, a lane
// for each choice (and a register for its product), and at least three steps in the ring.
template <typename T, bool DOT> bool bulk_shape(const RowsParams &p, BulkShape &s) {
  const int64_t row_bytes = p.K * (int64_t)sizeof(T);
  if (p.k > (DOT ? kBulkMostDots : 32) || row_bytes < 512 || row_bytes > 1 << 30 || p.T < (int64_t)sm_count() * kBulkWarps * 2) return false;
  s.rows = (int)p.k + (DOT ? 1 : 0);
  s.piece = 4096;
  while (s.piece > 512 && (s.piece > row_bytes || s.rows * s.piece * 3 > kBulkWarpBytes)) s.piece /= 2;
  s.stages = std::min(kBulkMostStages, kBulkWarpBytes / (s.rows * s.piece));
  return s.stages >= 3;
}

template <typename T, bool SPREAD, bool DOT> int launch_bulk(const RowsParams &p, const BulkShape &shape, cudaStream_t stream) {
  static std::atomic<bool> allowed[64];  // per device; setting the attribute twice is harmless
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TSB_ERR_LAUNCH;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(rows_bulk_kernel<T, SPREAD, DOT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBulkSmem) != cudaSuccess) return TSB_ERR_LAUNCH;
    allowed[dev] = true;
  }
  rows_bulk_kernel<T, SPREAD, DOT><<<(unsigned)sm_count() * 2, kBulkWarps * 32, kBulkSmem, stream>>>(p, shape);
  return launch_status();
}

template <typename T, bool SPREAD, bool ALIGNED, bool WRITE, bool ZERO> int launch_dot(const RowsParams &p, cudaStream_t stream) {
  const auto go = [&](auto jn, auto gn) {
    constexpr int J = decltype(jn)::value, G = decltype(gn)::value;
    const int64_t want = (p.T + kThreads / G - 1) / (kThreads / G);
    const int64_t blocks = std::min<int64_t>(want, (int64_t)sm_count() * 32);
    rows_dot_kernel<T, SPREAD, ALIGNED, WRITE, ZERO, J, G><<<(unsigned)blocks + p.zero_blocks, kThreads, 0, stream>>>(p);
    return launch_status();
  };
  const auto with_j = [&](auto gn) {
    if constexpr (SPREAD && !ALIGNED) {
      return go(std::integral_constant<int, 2>(), gn);
    } else {
      if (p.k <= 2) return go(std::integral_constant<int, 2>(), gn);
      if constexpr (ALIGNED && WRITE)
        if (p.k > 4) return go(std::integral_constant<int, 8>(), gn);
      return go(std::integral_constant<int, 4>(), gn);
    }
  };
  // Threads of a token: what its chunks keep busy, and a whole CTA where the tokens alone would not fill the GPU.
  const int64_t Kc = chunks_of<T, ALIGNED>(p.K);
  if (Kc <= 8) return with_j(std::integral_constant<int, 8>());
  if (Kc <= 32 || p.T >= (int64_t)sm_count() * 16) return with_j(std::integral_constant<int, 32>());
  return with_j(std::integral_constant<int, kThreads>());
}

template <typename T, bool SPREAD, bool ALIGNED, bool ZERO> int launch_moves(const RowsParams &p, cudaStream_t stream) {
  if (p.dot && (SPREAD || p.k <= (ALIGNED ? 8 : 4))) return launch_dot<T, SPREAD, ALIGNED, true, ZERO>(p, stream);
  const int64_t items = p.T * chunks_of<T, ALIGNED>(p.K);
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((int64_t)sm_count() * 64, (items + kThreads - 1) / kThreads));
  rows_kernel<T, SPREAD, ALIGNED, ZERO><<<(unsigned)blocks + p.zero_blocks, kThreads, 0, stream>>>(p);
  if constexpr (!SPREAD)
    if (p.dot) return launch_dot<T, SPREAD, ALIGNED, false, false>(p, stream);
  return launch_status();
}

template <typename T, bool SPREAD, bool ALIGNED> int launch_rows(RowsParams p, cudaStream_t stream) {
  BulkShape shape;
  if constexpr (!SPREAD) {
    if constexpr (ALIGNED) {
      if (p.dot && bulk_shape<T, true>(p, shape)) return launch_bulk<T, false, true>(p, shape, stream);
      if (!p.dot && bulk_shape<T, false>(p, shape)) return launch_bulk<T, false, false>(p, shape, stream);
    }
    return launch_moves<T, false, ALIGNED, false>(p, stream);
  } else {
    const bool bulk = ALIGNED && p.dot && bulk_shape<T, true>(p, shape);
    if (!bulk && p.M <= kOneList) {
      p.zero_blocks = (int)std::min<int64_t>(128, (p.M + 63) / 64);
      return launch_moves<T, true, ALIGNED, true>(p, stream);
    }
    int st;
    if constexpr (ALIGNED) st = bulk ? launch_bulk<T, true, true>(p, shape, stream) : launch_moves<T, true, true, false>(p, stream);
    else st = launch_moves<T, true, false, false>(p, stream);
    return st == TSB_OK ? launch_holes<T, ALIGNED>(p, stream) : st;
  }
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
    return aligned && p.K % chunk_len<T>() == 0 ? launch_rows<T, SPREAD, true>(p, stream) : launch_rows<T, SPREAD, false>(p, stream);
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
  return rows_entry<true>({few, rows, slot, used, weight, nullptr, many, dot, T, k, K, T * k, 0}, dtype, (cudaStream_t)stream);
}

extern "C" int tsb_expert_fold(const void *many, const int64_t *slot, const void *weight, const void *other, void *few,
                               void *dot, int64_t T, int64_t k, int64_t K, int dtype, tsb_stream_t stream) {
  if (T < 0 || k < 1 || K < 0 || (K > 0 && (other != nullptr) != (dot != nullptr))) return TSB_ERR_ARG;
  if (T == 0) return TSB_OK;
  if (!slot || (K > 0 && (!few || !many))) return TSB_ERR_ARG;
  return rows_entry<false>({other, many, slot, nullptr, weight, few, nullptr, dot, T, k, K, T * k, 0}, dtype,
                           (cudaStream_t)stream);
}
