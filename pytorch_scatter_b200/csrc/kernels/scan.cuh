// Gated linear recurrence over the rows of CSR segments, forward and backward: the tile kernel.
//
//   forward:   h[e] = gate[e] * h[e-1] + src[e]; before a segment's first row h = state[n] or 0
//   backward:  walks the rows from the end with q[e] = gate[e] * dh[e], what row e hands to the row before it:
//              dh[e] = grad_out[e] + q[e+1]; behind a segment's last row q = grad_last[n] or 0
//              grad_src = dh, grad_gate[e] = dh[e] * h[e-1] (summed over the channels that share the gate),
//              grad_state[n] = q[first row]
//
// Both are affine maps of the running value, value' = A * value + B, and maps compose: rows are cut into tiles of L rows,
// and every input is read from HBM once.  A thread owns VEC channels (16 bytes) of R consecutive rows of a tile, which it
// copies to its own slots of shared memory one tile ahead (cp.async; nobody else reads them, so the data needs no
// barrier; the chunks of rows that begin off a 16-byte boundary are shared by a row's lanes, see Ragged).  (1) It composes
// its rows' maps and leaves the result in shared memory.  (2) Turned over, a thread takes VEC consecutive maps of one
// channel, composes them and scans over the lanes that share the channel; the CTAs of a cluster hold neighbouring tiles of
// the same channels and exchange their totals through distributed shared memory; then the value that reaches each
// thread's rows is known.  (3) Each thread walks its rows again from that value and writes the outputs.  The cluster moves
// on by its CTAs' tiles, carrying the value along in registers, so that one launch covers any length without waiting on
// anything but its own cluster.  The composition has a fixed shape: results do not vary from run to run.
//
// 65536 x 2048 bf16 in 37 segments: forward 180 us, 4.5 TB/s, with h kept in 32 bits for a backward 299 us, 4.5 TB/s,
// backward 323 us, 5.0 TB/s; bound by the latency of a tile's chain of steps with eight warps on an SM.
//
// A segment's first row (backward: its last) does not take the value from the row before: such a map is marked `reset`
// and drops what comes in, so infinities and NaN of one segment never reach the next.  Tiles that no segment border
// touches run a copy of the code without these checks.
#pragma once

#include <algorithm>
#include <atomic>

#include "mbarrier.cuh"

namespace tsb {
namespace scan {

constexpr int kScanThreads = 128;           // threads that carry channels; a fifth warp looks for segment borders
constexpr int kStages = 2;
constexpr int kMarkStages = 3;
constexpr int kMostCluster = 8;

struct ScanParams {
  const void *src, *gate, *state;  // backward: src = grad_out (may be null), state = grad_last
  const void *fwd, *init;          // backward: the forward's h in the accumulation type, and its state
  const int64_t *indptr;
  void *out, *last;                // backward: grad_src, grad_state
  void *grad_gate, *partial;       // backward
  void *wide;                      // forward: h in the accumulation type as well, or null
  int64_t B, E, K, N, width, bstride;
  int64_t parts, tiles_k;
  int lx_log2, cluster, lanes_log2;  // lanes_log2: lanes of one row whose gate products are summed by shuffles
};

// row marks: the row's segment and flags
constexpr int kStart = 1, kEnd = 2, kDead = 4, kPad = 8, kMarkBits = 4;
constexpr int64_t kMostSegments = (int64_t)1 << 27;

// A copy of VEC values to the thread's own slot.  One 2-byte value travels in the 4-byte word that holds it (cp.async has
// no smaller form), unless that word reaches over the array's ends (`edge`: it may); `half` says which half it is.
template <typename T, int VEC> struct Slot {
  static constexpr bool kWord = sizeof(T) * VEC == 2;
  static constexpr int kBytes = kWord ? 4 : (int)sizeof(T) * VEC;
  static __device__ __forceinline__ int half(const T *p) { return kWord ? (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 1 : 0; }
  static __device__ __forceinline__ void copy(char *slot, const T *p, bool edge, const T *lo, const T *hi) {
    if constexpr (kWord) {
      const uintptr_t word = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3;
      if (!edge || (word >= reinterpret_cast<uintptr_t>(lo) && word + 4 <= reinterpret_cast<uintptr_t>(hi))) {
        const unsigned dst = (unsigned)__cvta_generic_to_shared(slot);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(word) : "memory");
      } else {
        reinterpret_cast<T *>(slot)[half(p)] = *p;
      }
    } else {
      async_copy_pack<T, VEC>(reinterpret_cast<Pack<T, VEC> *>(slot), p);
    }
  }
  static __device__ __forceinline__ Pack<T, VEC> get(const char *slot, int half) {
    if constexpr (kWord) {
      Pack<T, VEC> r;
      r.v[0] = reinterpret_cast<const T *>(slot)[half];
      return r;
    } else {
      return *reinterpret_cast<const Pack<T, VEC> *>(slot);
    }
  }
};

// Rows that begin anywhere (60000 x 333 fp16 in 3001 segments, forward / backward: 131 / 215 us; one channel to a thread
// instead: 191 / 369, the latter with h in 16 bits): the lanes of a row share its aligned 16-byte chunks, n of them to a lane and one more, and a
// lane shifts its values out of its own and the next one (the lanes of a row are lanes of one warp).
template <typename X, int VEC> struct Ragged {
  static constexpr int n = (int)sizeof(X) * VEC / 16;
  static __device__ __forceinline__ void copy_chunk(char *dst, uintptr_t src, bool edge, const X *lo, const X *hi) {
    if (!edge || (src >= reinterpret_cast<uintptr_t>(lo) && src + 16 <= reinterpret_cast<uintptr_t>(hi))) {
      const unsigned to = (unsigned)__cvta_generic_to_shared(dst);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
    } else {  // over the array's ends
      const X *p = reinterpret_cast<const X *>(src);
#pragma unroll
      for (int i = 0; i < 16 / (int)sizeof(X); ++i)
        if (p + i >= lo && p + i < hi) reinterpret_cast<X *>(dst)[i] = p[i];
    }
  }
  // p: the row's first value of the tile, of `bytes` that belong to the row
  static __device__ __forceinline__ void copy(char *row, const X *p, int col, int lx, int bytes, bool edge, const X *lo, const X *hi) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), base = at & ~(uintptr_t)15;
    const int end = (int)(at & 15) + bytes;
#pragma unroll
    for (int i = 0; i < n; ++i)
      if ((col * n + i) * 16 < end) copy_chunk(row + (col * n + i) * 16, base + (col * n + i) * 16, edge, lo, hi);
    if (col == lx - 1 && lx * n * 16 < end) copy_chunk(row + lx * n * 16, base + lx * n * 16, edge, lo, hi);
  }
  // off: bytes between the aligned chunk and the row's first value
  static __device__ __forceinline__ Pack<X, VEC> get(const char *row, int col, int off) {
    unsigned w[4 * n + 4];
#pragma unroll
    for (int i = 0; i <= n; ++i) {
      const uint4 q = *reinterpret_cast<const uint4 *>(row + (col * n + i) * 16);
      w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
    }
#pragma unroll
    for (int i = 0; i < 4 * n + 2; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
    if constexpr (sizeof(X) <= 4) {
#pragma unroll
      for (int i = 0; i < 4 * n + 1; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
    }
    if constexpr (sizeof(X) <= 2) {
#pragma unroll
      for (int i = 0; i < 4 * n; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], off & 2 ? 16 : 0);
    }
    Pack<X, VEC> r;
    unsigned *out = reinterpret_cast<unsigned *>(&r);
#pragma unroll
    for (int i = 0; i < 4 * n; ++i) out[i] = w[i];
    return r;
  }
  // The way back, all lanes of a row together (`lanes`): a lane writes its aligned chunks, whose first values are the last
  // of the lane before.  p: the row's first value of the tile.  The row's ends are written value by value.
  static __device__ __forceinline__ void store(X *p, const Pack<X, VEC> &v, int col, int lx, int bytes, unsigned lanes) {
    constexpr int V = 16 / (int)sizeof(X);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const int off = (int)(at & 15), end = off + bytes;
    X *base = reinterpret_cast<X *>(at & ~(uintptr_t)15);
    const unsigned *own = reinterpret_cast<const unsigned *>(&v);
    unsigned w[4 * n + 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(lanes, own[4 * n - 4 + i], 1);
#pragma unroll
    for (int i = 0; i < 4 * n; ++i) w[4 + i] = own[i];
    // skip 16 - off bytes of these; with off = 0 that is all of the neighbour's
    if (off == 0) {
#pragma unroll
      for (int i = 0; i < 4 * n; ++i) w[i] = w[i + 4];
    } else {
      const int skip = 16 - off;
#pragma unroll
      for (int i = 0; i < 4 * n + 2; ++i) w[i] = skip & 8 ? w[i + 2] : w[i];
      if constexpr (sizeof(X) <= 4) {
#pragma unroll
        for (int i = 0; i < 4 * n + 1; ++i) w[i] = skip & 4 ? w[i + 1] : w[i];
      }
      if constexpr (sizeof(X) <= 2) {
#pragma unroll
        for (int i = 0; i < 4 * n; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], skip & 2 ? 16 : 0);
      }
    }
#pragma unroll
    for (int c = 0; c < n; ++c) {
      const int first = (col * n + c) * 16;
      const X *x = reinterpret_cast<const X *>(&w[4 * c]);
      if (first >= off && first + 16 <= end) {
        __stcs(reinterpret_cast<uint4 *>(base + first / (int)sizeof(X)), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int b = first + i * (int)sizeof(X);
          if (b >= off && b < end) base[b / (int)sizeof(X)] = x[i];
        }
      }
    }
    if (col == lx - 1 && off > 0) {  // what reaches into the chunk behind the last lane's
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int b = off + (col * VEC + i) * (int)sizeof(X);
        if (b >= lx * n * 16 && b < end) base[b / (int)sizeof(X)] = v.v[i];
      }
    }
  }
};

template <typename A, int VEC> __device__ __forceinline__ void load_acc(A (&v)[VEC], const void *base, int64_t at, int nv) {
  const A *p = static_cast<const A *>(base);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = p && i < nv ? p[at + i] : (A)0;
}
template <typename A, int VEC> __device__ __forceinline__ void store_acc(const A (&v)[VEC], void *base, int64_t at, int nv) {
  A *p = static_cast<A *>(base);
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < nv) p[at + i] = v[i];
}

// VEC values of one thread to and from shared memory, 16 bytes at a time where there are as many
template <typename A, int VEC> __device__ __forceinline__ void put(A *p, const A (&v)[VEC]) {
  constexpr int n = VEC * sizeof(A) >= 16 ? 16 / (int)sizeof(A) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += n) {
    Pack<A, n> q;
#pragma unroll
    for (int j = 0; j < n; ++j) q.v[j] = v[i + j];
    *reinterpret_cast<Pack<A, n> *>(p + i) = q;
  }
}
// to global memory, which is 16-byte aligned where there are as many
template <typename A, int VEC> __device__ __forceinline__ void store_wide(A *p, const A (&v)[VEC]) {
  constexpr int n = VEC * sizeof(A) >= 16 ? 16 / (int)sizeof(A) : 1;
#pragma unroll
  for (int i = 0; i < VEC; i += n) {
    Pack<A, n> q;
#pragma unroll
    for (int j = 0; j < n; ++j) q.v[j] = v[i + j];
    st_stream<A, n>(p + i, q);
  }
}
template <typename A, int VEC> __device__ __forceinline__ void take(A (&v)[VEC], const A *p) {
  constexpr int n = VEC * sizeof(A) >= 16 ? 16 / (int)sizeof(A) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += n) {
    const Pack<A, n> q = *reinterpret_cast<const Pack<A, n> *>(p + i);
#pragma unroll
    for (int j = 0; j < n; ++j) v[i + j] = q.v[j];
  }
}

// A pack in the accumulation type: a bf16 value is the upper half of the fp32 value, so two come out of a word with a
// shift and a mask.
template <typename T, int VEC, typename A> __device__ __forceinline__ void widen(A (&v)[VEC], const Pack<T, VEC> &q) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const unsigned w = *reinterpret_cast<const unsigned *>(&q.v[i]);
      v[i] = __uint_as_float(w << 16);
      v[i + 1] = __uint_as_float(w & 0xffff0000u);
    }
  } else if constexpr (std::is_same<T, __half>::value && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&q.v[i]));
      v[i] = f.x;
      v[i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_acc<T>(q.v[i]);
  }
}

// a * b + c, a * b and a + b over VEC channels, two fp32 channels in one instruction
template <typename A, int VEC, typename F2, typename F1> __device__ __forceinline__ void pairwise(A (&d)[VEC], F2 two, F1 one) {
  if constexpr (std::is_same<A, float>::value && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 r = two(i);
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) d[i] = one(i);
  }
}
template <typename A, int VEC> __device__ __forceinline__ void fma_all(A (&d)[VEC], const A (&a)[VEC], const A (&b)[VEC], const A (&c)[VEC]) {
  pairwise<A, VEC>(d, [&](int i) { return __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1])); },
                   [&](int i) { return a[i] * b[i] + c[i]; });
}
template <typename A, int VEC> __device__ __forceinline__ void mul_all(A (&d)[VEC], const A (&a)[VEC], const A (&b)[VEC]) {
  pairwise<A, VEC>(d, [&](int i) { return __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1])); },
                   [&](int i) { return a[i] * b[i]; });
}
template <typename A, int VEC> __device__ __forceinline__ void add_all(A (&d)[VEC], const A (&a)[VEC], const A (&b)[VEC]) {
  pairwise<A, VEC>(d, [&](int i) { return __fadd2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1])); },
                   [&](int i) { return a[i] + b[i]; });
}

// Round to the output's type, once; pairs of 16-bit values in one instruction.
template <typename T, int VEC, typename A> __device__ __forceinline__ void round_pack(Pack<T, VEC> &o, const A (&v)[VEC]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) *reinterpret_cast<__nv_bfloat162 *>(&o.v[i]) = __floats2bfloat162_rn(v[i], v[i + 1]);
  } else if constexpr (std::is_same<T, __half>::value && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) *reinterpret_cast<__half2 *>(&o.v[i]) = __floats2half2_rn(v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = from_acc<T>(v[i]);
  }
}

// A product of gates, brought back into the range of numbers.  It may overflow where the recurrence itself stays at zero:
// kept finite, so that A * 0 + B = B.  One that underflows keeps the smallest magnitude unless a gate is 0 (`zero`): an
// infinite value that comes in stays infinite, as it does row by row, and only a gate of 0 makes it NaN.  (A finite value
// times the smallest magnitude is off by less than one step of the product of the two.)  NaN stays NaN.
__device__ __forceinline__ float in_range(float a, bool zero) {
  const float least = zero ? 0.0f : __int_as_float(1);
  float r;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(std::numeric_limits<float>::max()));
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(least));
  return r;
}
__device__ __forceinline__ double in_range(double a, bool zero) {
  constexpr double most = std::numeric_limits<double>::max();
  a = a > most ? most : a < -most ? -most : a;
  return a == 0 && !zero ? copysign(std::numeric_limits<double>::denorm_min(), a) : a;
}

// The least magnitude of the gates of N channels, row after row: was one of a channel's gates 0?  16-bit gates two to an
// instruction.
template <typename G, int N> struct Least {
  static constexpr bool kPairs = sizeof(G) == 2 && N % 2 == 0;
  using W = std::conditional_t<kPairs, std::conditional_t<std::is_same<G, __half>::value, __half2, __nv_bfloat162>, acc_t<G>>;
  static constexpr int n = kPairs ? N / 2 : N;
  W w[n];
  __device__ __forceinline__ Least() {
    Pack<G, N> ones;
#pragma unroll
    for (int i = 0; i < N; ++i) ones.v[i] = from_acc<G>(1);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      if constexpr (kPairs) w[i] = *reinterpret_cast<const W *>(&ones.v[2 * i]);
      else w[i] = 1;
    }
  }
  __device__ __forceinline__ void add(const Pack<G, N> &g) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      if constexpr (kPairs) w[i] = __hmin2(w[i], __habs2(*reinterpret_cast<const W *>(&g.v[2 * i])));
      else w[i] = fmin(w[i], fabs(to_acc<G>(g.v[i])));
    }
  }
  __device__ __forceinline__ bool zero(int i) const {
    if constexpr (kPairs) return to_acc<G>(i & 1 ? w[i / 2].y : w[i / 2].x) == 0;
    else return w[i] == 0;
  }
};

// A map that drops what comes in travels between CTAs with this A, which no product of gates can be.
template <typename A> __device__ __forceinline__ A reset_mark() {
  if constexpr (sizeof(A) == 8) return __longlong_as_double(0x7ff8c0dec0dec0deLL);
  else return __int_as_float(0x7fc0c0de);
}
__device__ __forceinline__ bool is_reset_mark(float a) { return __float_as_int(a) == 0x7fc0c0de; }
__device__ __forceinline__ bool is_reset_mark(double a) { return __double_as_longlong(a) == 0x7ff8c0dec0dec0deLL; }

// first index in [lo, hi) with indptr[index] > row (UPPER) or >= row; hi if there is none
template <bool UPPER> __device__ __forceinline__ int64_t bound(const int64_t *indptr, int64_t lo, int64_t hi, int64_t row) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    const int64_t v = indptr[mid];
    if (UPPER ? v > row : v >= row) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Where part q of the rows begins: the first segment boundary behind its even share, so that no part takes a value from
// another one.
__device__ __forceinline__ int64_t part_begin(const ScanParams &p, const int64_t *indptr, int64_t q) {
  if (q == 0) return 0;
  if (q == p.parts) return p.E;
  const int64_t even = p.E / p.parts * q;
  const int64_t s = bound<false>(indptr, 0, p.N + 1, even);
  return s <= p.N ? clamp64(indptr[s], 0, p.E) : even;
}

// ---- exchange between the CTAs of a cluster: values stored into a neighbour's shared memory complete bytes of a barrier
// there, so a CTA waits for what it needs and for nothing else (a cluster-wide barrier would also wait for the outputs'
// stores to drain: 1.2 of 7.9 cycles between two instructions of a warp went there)
__device__ __forceinline__ unsigned remote_at(unsigned addr, int rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void send(unsigned addr, unsigned bar, float a, float b) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(addr), "f"(a), "f"(b), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(unsigned addr, unsigned bar, double a, double b) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];" ::"r"(addr), "d"(a), "d"(b), "r"(bar) : "memory");
}
template <typename T, typename G, int VEC, bool SHARED, bool BWD, bool RAGGED> struct ScanShape {
  using A = acc_t<T>;
  static constexpr int kGateVec = SHARED ? 1 : VEC;
  // The backward multiplies dh by the h before it as the recurrence held it, not by the rounded output, whose rounding
  // the gradient would carry besides its own (relative error against 64 bits 2.3e-3 instead of 1.7e-3 in bf16, 2.9e-4
  // instead of 2.1e-4 in fp16).  With 16-bit data the forward writes h a second time for it, in 32 bits.
  using SrcSlot = Slot<T, VEC>;
  using GateSlot = Slot<G, kGateVec>;
  using FwdSlot = Slot<A, VEC>;
  static constexpr int kRowBytes = SrcSlot::kBytes + (BWD ? FwdSlot::kBytes : 0) + GateSlot::kBytes;
  // Rows of a thread: 42 KB for each of the two stages at most, so that two CTAs fit an SM.  What a tile costs besides its
  // rows, step (2), is then a small part (65536 x 4096 bf16: 291 us with 10 rows and 2 stages, 302 with 7 rows and 3
  // stages, 391 with 5 rows, 2 stages and four CTAs).
  static constexpr int kRows = (RAGGED ? 296 : 336) / kRowBytes < 16 ? (RAGGED ? 296 : 336) / kRowBytes : 16;
  static constexpr int kCtas = kRowBytes <= 16 ? 4 : 2;  // of an SM, by the registers
  // of the two stages; ragged rows have one more chunk in each array
  static __host__ __device__ int stage_bytes(int lx) {
    return kScanThreads * kRows * kRowBytes + (RAGGED ? kScanThreads / lx * kRows * 16 * (BWD ? 3 : 2) : 0);
  }
  static constexpr int kMaps = kScanThreads * VEC + 128;      // [ty][C], see `skew`
  static constexpr int kMapBytes = 2 * kMaps * (int)sizeof(A);
  static size_t bytes(int lx, int cluster) {
    const size_t C = (size_t)lx * VEC, L = (size_t)(kScanThreads / lx) * kRows;
    return (size_t)kStages * stage_bytes(lx) + kMapBytes + (cluster > 1 ? sizeof(A) * C * 4 * cluster : 0) + sizeof(int) * kMarkStages * L;
  }
};

template <typename T, typename G, int VEC, bool SHARED, bool BWD, bool RAGGED>
__global__ void __launch_bounds__(kScanThreads + 32, ScanShape<T, G, VEC, SHARED, BWD, RAGGED>::kCtas) scan_kernel(ScanParams p) {
  using S = ScanShape<T, G, VEC, SHARED, BWD, RAGGED>;
  using SrcSlot = typename S::SrcSlot;
  using GateSlot = typename S::GateSlot;
  using FwdSlot = typename S::FwdSlot;
  using A = acc_t<T>;
  constexpr int R = S::kRows;
  // A ragged row is a few hundred instructions: unrolled, the loops over a thread's rows do not fit the instruction cache
  // (60000 x 333 fp16 in 3001 segments: 243 us, most of it waiting for instructions, against 131).
  constexpr int kUnroll = RAGGED ? 1 : R;


  const int tid = threadIdx.x;
  const int lx = 1 << p.lx_log2, C = lx * VEC, L = (kScanThreads >> p.lx_log2) * R;
  const int col = tid & (lx - 1), ty = tid >> p.lx_log2;
  // shared memory from a thread's row to its next one, and of a ragged row (one more chunk than its lanes hold)
  const int ragged_row = RAGGED ? (kScanThreads >> p.lx_log2) * 16 : 0;
  const int kSrcRow = kScanThreads * SrcSlot::kBytes + ragged_row, kGateRow = kScanThreads * GateSlot::kBytes + ragged_row,
            kFwdRow = kScanThreads * FwdSlot::kBytes + ragged_row;
  const int cs = p.cluster, rank = (int)(blockIdx.x % cs);
  int64_t id = blockIdx.x / cs;
  const int64_t kt = id % p.tiles_k;
  id /= p.tiles_k;
  const int64_t part = id % p.parts, b = id / p.parts;

  const int64_t *indptr = p.indptr + b * p.bstride;
  const int64_t lo = part_begin(p, indptr, part), hi = part_begin(p, indptr, part + 1);
  const int64_t len = hi - lo;
  if (len <= 0) return;  // the same for the whole cluster
  const int64_t step = (int64_t)cs * L;

  extern __shared__ __align__(128) char smem[];
  A *s_a = reinterpret_cast<A *>(smem + (size_t)kStages * S::stage_bytes(lx));  // maps of the threads [ty][C]; then the values
  A *s_b = s_a + S::kMaps;                                         // that reach them, in place of A
  A *s_total = s_b + S::kMaps;                           // maps of the cluster's CTAs [2][cs][C][A, B]
  int *s_marks = reinterpret_cast<int *>(s_total + (cs > 1 ? 4 * cs * C : 0));  // [stage][L]
  __shared__ int s_reset[kScanThreads];
  __shared__ int s_marked[kMarkStages];                                      // does a segment border touch the tile?
  __shared__ __align__(8) uint64_t s_bar[2];

  if (cs > 1) {
    if (tid < 2) {
      mbar_init(smem_at(&s_bar[tid]));
      mbar_init_done();
    }
    cluster_barrier();  // all CTAs run, with their barriers ready, before anyone writes to their shared memory
  }

  const auto row_of = [&](int64_t pos) { return BWD ? hi - 1 - pos : lo + pos; };

  // ---- the fifth warp: where segments begin and end, one tile ahead of the others
  if (tid >= kScanThreads) {
    const int lane = tid - kScanThreads;
    const auto border = [&](int64_t s) { return clamp64(indptr[s], 0, p.E); };  // (offsets beyond the rows end at them)
    const int64_t first = border(0), behind = border(p.N);
    int64_t cursor = BWD ? p.N + 1 : 0;  // bound of the row looked up last
    const auto look = [&](int64_t tile, int stage) {
      // the segment of the tile's first row on the way: does it hold the whole tile, without beginning or ending in it?
      const int64_t from = row_of(tile < len ? tile : len - 1), to = row_of(tile + L <= len ? tile + L - 1 : len - 1);
      const int64_t u = BWD ? bound<true>(indptr, 0, cursor, from) : bound<true>(indptr, cursor, p.N + 1, from);
      cursor = u;
      const int64_t low = BWD ? to : from, high = BWD ? from : to;
      const bool plain = tile + L <= len && u >= 1 && u <= p.N && border(u - 1) < low && border(u) > high + 1;
      if (!plain) {
        int *mark = s_marks + stage * L;
        for (int j = lane; j < L; j += 32) {
          const int64_t t = row_of(tile + j);
          mark[j] = tile + j >= len ? kPad : t < first || t >= behind ? kDead : 0;
        }
        __syncwarp();
        // borders from the first row's segment on, 32 at a time, until one is beyond the tile
        for (int64_t s0 = BWD ? u : u - 1;;) {
          const int64_t s = BWD ? s0 - lane : s0 + lane;
          bool beyond = s < 0 || s > p.N;
          int64_t at = -1;
          if (!beyond) {
            at = border(s);
            beyond = BWD ? at < low : at > high + 1;
            if (at >= low && at <= high && s < p.N && border(s + 1) > at)
              atomicOr(&mark[BWD ? high - at : at - low], (int)s << kMarkBits | kStart);
            if (at > low && at <= high + 1 && s > 0 && border(s - 1) < at)
              atomicOr(&mark[BWD ? high - (at - 1) : at - 1 - low], (int)(s - 1) << kMarkBits | kEnd);
          }
          if (__any_sync(kFullMask, beyond && (BWD ? s <= p.N : s >= 0))) break;
          // a run of empty segments at one row: on to its last border, the only other one that matters
          const long long at0 = __shfl_sync(kFullMask, (long long)at, 0), at31 = __shfl_sync(kFullMask, (long long)at, 31);
          s0 += BWD ? -32 : 32;
          if (at0 == at31) {
            const int64_t end = BWD ? bound<false>(indptr, 0, s0 + 1, at0) : bound<true>(indptr, s0, p.N + 1, at0) - 1;
            s0 = BWD ? (end < s0 ? end : s0) : (end > s0 ? end : s0);
          }
        }
      }
      if (lane == 0) s_marked[stage] = !plain;
    };
    int64_t tile = (int64_t)rank * L;
    int stage = 0;
    look(tile, 0);
    __syncthreads();
    for (int64_t done = 0; done < len; done += step) {
      tile += step;
      stage = stage == kMarkStages - 1 ? 0 : stage + 1;
      if (done + step < len) look(tile, stage);  // of the three sets of marks, the others may still read two
      __syncthreads();                           // (1) of the tile before is done
      __syncthreads();                           // (2)
    }
    return;
  }

  const int64_t c0 = kt * C + (int64_t)col * VEC;   // this thread's first channel
  const bool live = c0 < p.K;
  const int nv = RAGGED ? (int)(p.K - c0 < VEC ? p.K - c0 : VEC) : VEC;  // channels of this thread that there are
  const int tile_c = (int)(p.K - kt * C < C ? p.K - kt * C : C);           // and of the tile
  const int64_t gates = p.K / p.width, g0 = SHARED ? c0 / p.width : c0;
  const int64_t dk = BWD ? -p.K : p.K, dgates = BWD ? -gates : gates;  // from a row to the next one on the way
  const int64_t srow = b * p.N;                     // first row of this batch in the state arrays
  const bool have_src = !BWD || p.src, want_gate = BWD && p.grad_gate;
  const T *src_lo = static_cast<const T *>(p.src), *src_hi = src_lo + p.B * p.E * p.K;
  const A *fwd_lo = static_cast<const A *>(p.fwd), *fwd_hi = fwd_lo + p.B * p.E * p.K;
  const G *gate_lo = static_cast<const G *>(p.gate), *gate_hi = gate_lo + p.B * p.E * gates;

  // this thread's slots [stage][row][thread], and its pointers to the next tile to load and to the tile at work
  char *s_src = smem + (RAGGED ? ty * (lx * SrcSlot::kBytes + 16) : tid * SrcSlot::kBytes);
  char *s_fwd = smem + kStages * R * kSrcRow + (RAGGED ? ty * (lx * FwdSlot::kBytes + 16) : tid * FwdSlot::kBytes);
  char *s_gate = smem + kStages * R * (kSrcRow + (BWD ? kFwdRow : 0)) + (RAGGED ? ty * (lx * GateSlot::kBytes + 16) : tid * GateSlot::kBytes);
  int64_t ahead = (int64_t)rank * L + ty * R;       // position of the thread's next rows to load
  const int64_t at = b * p.E + row_of(ahead);
  const T *lsrc = src_lo + (have_src ? at * p.K + c0 : 0);
  const A *lfwd = fwd_lo + (BWD ? (at - 1) * p.K + c0 : 0);  // h of the row before
  const G *lgate = gate_lo + at * gates + g0;
  T *os = static_cast<T *>(p.out) + at * p.K + c0;
  A *ow = static_cast<A *>(p.wide) + (!BWD && p.wide ? at * p.K + c0 : 0);
  G *og = static_cast<G *>(p.grad_gate) + (want_gate ? at * gates + g0 : 0);
  // sums of a shared gate's products: all of them, or what this tile's lanes hold
  const int sum_lanes = SHARED ? 1 << p.lanes_log2 : 1;
  const int64_t sums = SHARED ? p.K / ((int64_t)VEC * sum_lanes) : 0, dsums = BWD ? -sums : sums;
  const bool part_sums = SHARED && sums != gates;
  A *op = static_cast<A *>(p.partial) + (part_sums && want_gate ? at * sums + c0 / ((int64_t)VEC * sum_lanes) : 0);
  const int64_t tile_k = step * dk, tile_gates = step * dgates;
  // Where a row's values are: the half of its word (2-byte slots), or the bytes between the aligned chunk and the row's
  // first value (ragged rows).  From row to row and from tile to tile this moves by the row length.
  const int kcol = RAGGED ? col * VEC : 0;
  const auto where = [&](auto *q, int slot_half) { return RAGGED ? (int)(reinterpret_cast<uintptr_t>(q - kcol) & 15) : slot_half; };
  const auto moved = [&](int from, int64_t rows, int64_t row_len, int size) {
    return RAGGED ? (int)(from + rows * row_len * size) & 15 : (int)(from + rows * row_len) & 1;
  };
  int xat = where(lsrc, SrcSlot::half(lsrc)), fat = where(lfwd, FwdSlot::half(lfwd)), gat = where(lgate, GateSlot::half(lgate));

  const int64_t margin = RAGGED ? 1 + 16 / (p.K * (int64_t)(sizeof(T) < sizeof(G) ? sizeof(T) : sizeof(G))) : 0;  // rows in 16 bytes
  const auto load_rows = [&](int stage) {
    const int64_t left = len - ahead;
    if (RAGGED) __syncwarp();  // the lanes of a row have read each other's chunks of this stage
    if ((live || (RAGGED && (col - 1) * VEC < tile_c)) && left > 0) {  // (a ragged row may end in the chunk of the lane behind)
      const T *xs = lsrc;
      const A *fs = lfwd;
      const G *gs = lgate;
      char *xd = s_src + stage * (R * kSrcRow), *fd = s_fwd + stage * (R * kFwdRow), *gd = s_gate + stage * (R * kGateRow);
      const int n = left < R ? (int)left : R;
      // only the first and the last rows of the whole array hold words or chunks that reach over its ends
      const int64_t row = b * p.E + row_of(ahead);
      const bool edge = BWD ? row <= R + margin || row >= p.B * p.E - 1 - margin : row <= margin || row + R >= p.B * p.E - margin;
#pragma unroll kUnroll
      for (int r = 0; r < R; ++r) {
        if (r < n) {
          if constexpr (RAGGED) {
            if (have_src) Ragged<T, VEC>::copy(xd + r * kSrcRow, xs - kcol, col, lx, tile_c * (int)sizeof(T), edge, src_lo, src_hi);
            Ragged<G, VEC>::copy(gd + r * kGateRow, gs - kcol, col, lx, tile_c * (int)sizeof(G), edge, gate_lo, gate_hi);
            if (BWD && want_gate && fs - kcol >= fwd_lo) Ragged<A, VEC>::copy(fd + r * kFwdRow, fs - kcol, col, lx, tile_c * (int)sizeof(A), edge, fwd_lo, fwd_hi);
          } else {
          if (have_src) SrcSlot::copy(xd + r * kSrcRow, xs, edge, src_lo, src_hi);
          GateSlot::copy(gd + r * kGateRow, gs, edge, gate_lo, gate_hi);
          if (BWD && want_gate && fs >= fwd_lo) FwdSlot::copy(fd + r * kFwdRow, fs, edge, fwd_lo, fwd_hi);  // (row 0 has none before it)
          }
        }
        xs += dk;
        fs += dk;
        gs += dgates;
      }
    }
    async_commit();
    ahead += step;
    lsrc += tile_k;
    lfwd += tile_k;
    lgate += tile_gates;
  };

  // (2) runs with the roles turned over: channel fc, the fh-th of H lanes that share it
  const int hbits = 31 - __clz(kScanThreads) - p.lx_log2 - (31 - __clz(VEC)), H = 1 << hbits;
  const int fc = tid >> hbits, fh = tid & (H - 1);
  // the H lanes of a channel read maps VEC * C apart, all in one bank: each VEC rows of maps start some words further on
  const int skew = H > 8 ? 4 : 32 >> hbits;
  A carry = 0;  // the value that reaches the cluster's tiles in channel fc
  const int own_map = tid * VEC + (H > 1 ? ty / VEC * skew : 0), first_map = fh * VEC * C + fc + (H > 1 ? fh * skew : 0);
  unsigned phases = 0;  // parity to wait for, one bit for each of the two barriers

  const auto tile_work = [&](int stage, int par, int set) {
    // does a border touch the tile, and this warp's rows?
    const bool marked = s_marked[set];
    const int *mark = s_marks + set * L + ty * R;
    bool mine = false;
    if (marked) {
      int any = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) any |= mark[r];
      mine = __any_sync(kFullMask, any != 0);
    }
    const char *xs = s_src + stage * (R * kSrcRow), *gs = s_gate + stage * (R * kGateRow);
    [[maybe_unused]] const char *fs = s_fwd + stage * (R * kFwdRow);
    const unsigned rowmask = lx == 32 ? kFullMask : ((1u << lx) - 1u) << ((tid & 31) & ~(lx - 1));  // the lanes of this row
    const auto store_row = [&](auto *to, const auto &q) {
      using X = std::remove_pointer_t<decltype(to)>;
      if constexpr (RAGGED) Ragged<X, VEC>::store(to - kcol, q, col, lx, tile_c * (int)sizeof(X), rowmask);
      else if (live) st_stream<X, VEC>(to, q);
    };
    const auto read_gates = [&](int r) {
      if constexpr (RAGGED) return Ragged<G, VEC>::get(gs + r * kGateRow, col, moved(gat, r, dgates, sizeof(G)));
      else return GateSlot::get(gs + r * kGateRow, moved(gat, r, dgates, 1));
    };
    const auto read_row = [&](A (&x)[VEC], A (&g)[VEC], int r) {
      if constexpr (RAGGED) widen<T, VEC>(x, Ragged<T, VEC>::get(xs + r * kSrcRow, col, moved(xat, r, dk, sizeof(T))));
      else widen<T, VEC>(x, SrcSlot::get(xs + r * kSrcRow, moved(xat, r, dk, 1)));
      const Pack<G, S::kGateVec> q = read_gates(r);
      if constexpr (SHARED) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) g[v] = to_acc<G>(q.v[0]);
      } else {
        widen<G, VEC>(g, q);
      }
    };

    // ---- (1) the map of this thread's rows
    const auto map_rows = [&](auto has_marks) {
      constexpr bool MARKED = decltype(has_marks)::value;
      A ma[VEC], mb[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) { ma[v] = 1; mb[v] = 0; }
      int reset = 0;
#pragma unroll kUnroll
      for (int r = 0; r < R; ++r) {
        if constexpr (MARKED) {
          const int m = mark[r];
          if (m & kPad) continue;
          if (m & (kDead | (BWD ? kEnd : kStart))) {
            reset = 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) mb[v] = 0;
            if (m & kDead) continue;
            if (live) load_acc<A, VEC>(mb, p.state, (srow + (m >> kMarkBits)) * p.K + c0, nv);
          }
        }
        A x[VEC], g[VEC];
        read_row(x, g, r);
        if constexpr (BWD) {
          if (have_src) add_all(mb, mb, x);
          mul_all(mb, g, mb);
        } else {
          fma_all(mb, g, mb, x);
        }
        if constexpr (SHARED) ma[0] *= g[0];
        else mul_all(ma, ma, g);
      }
      bool gates = true;  // no product is 0
#pragma unroll
      for (int v = 0; v < S::kGateVec; ++v) {
        ma[v] = in_range(ma[v], true);
        gates = gates && (ma[v] != 0 || (RAGGED && v >= nv));
      }
      if constexpr (SHARED) {
#pragma unroll
        for (int v = 1; v < VEC; ++v) ma[v] = ma[0];
      }
      put(s_a + own_map, ma);
      put(s_b + own_map, mb);
      if (marked && col == 0) s_reset[ty] = reset;
      return gates || !live;
    };
    if (!(mine ? map_rows(std::true_type()) : map_rows(std::false_type()))) {
      // Was a gate of the thread's rows 0, or are they small?  (65536 x 2048 bf16 with one gate in a hundred 0, so that all
      // warps come here: 211 us, 178 without; with the loop unrolled 205, but 2% more for all that do not come here.)
      Least<G, S::kGateVec> least;
#pragma unroll(RAGGED ? 1 : 2)
      for (int r = 0; r < R; ++r)
        if (!mine || !(mark[r] & (kPad | kDead))) least.add(read_gates(r));
      A ma[VEC];
      take(ma, s_a + own_map);
#pragma unroll
      for (int v = 0; v < VEC; ++v) ma[v] = in_range(ma[v], least.zero(SHARED ? 0 : v));
      put(s_a + own_map, ma);
    }
    __syncthreads();

    // ---- (2) scan of the maps over the tile and the cluster
    A fa[VEC], fb[VEC];
    unsigned fr = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      fa[j] = s_a[first_map + j * C];
      fb[j] = s_b[first_map + j * C];
      if (marked) fr |= (unsigned)s_reset[fh * VEC + j] << j;
    }
    A ta = fa[0], tb = fb[0];
    int tr = fr & 1;
    bool zero = ta == 0;
#pragma unroll
    for (int j = 1; j < VEC; ++j) {
      const bool rs = marked && (fr >> j & 1);
      tb = rs ? fb[j] : fa[j] * tb + fb[j];
      ta *= fa[j];
      zero = zero || fa[j] == 0;
      tr |= rs;
    }
    ta = in_range(ta, zero);
    for (int d = 1; d < H; d <<= 1) {
      const A pa = __shfl_up_sync(kFullMask, ta, d, H), pb = __shfl_up_sync(kFullMask, tb, d, H);
      const int pr = marked ? __shfl_up_sync(kFullMask, tr, d, H) : 0;
      if (fh >= d) {
        if (!tr) tb = ta * pb + tb;
        ta = in_range(ta * pa, ta == 0 || pa == 0);
        tr |= pr;
      }
    }
    // map of the lanes before this one
    const A ea = __shfl_up_sync(kFullMask, ta, 1, H), eb = __shfl_up_sync(kFullMask, tb, 1, H);
    const int er = marked ? __shfl_up_sync(kFullMask, tr, 1, H) : 0;
    // map of the whole tile
    const A wa = __shfl_sync(kFullMask, ta, H - 1, H), wb = __shfl_sync(kFullMask, tb, H - 1, H);
    const int wr = marked ? __shfl_sync(kFullMask, tr, H - 1, H) : 0;
    A h = carry;
    if (cs > 1) {
      const unsigned bar = smem_at(&s_bar[par]);
      if (tid == 0) mbar_expect(bar, (unsigned)(cs * C * 2 * (int)sizeof(A)));
      const unsigned mine = smem_at(s_total + ((par * cs + rank) * C + fc) * 2);
      for (int q = fh; q < cs; q += H) send(remote_at(mine, q), remote_at(bar, q), wr ? reset_mark<A>() : wa, wb);
      if (!mbar_wait(bar, phases >> par & 1)) carry = (A)NAN;
      phases ^= 1u << par;
      A all = carry;
      for (int q = 0; q < cs; ++q) {
        if (q == rank) h = all;
        const A *m = s_total + ((par * cs + q) * C + fc) * 2;
        const A a = m[0], bb = m[1];
        all = is_reset_mark(a) ? bb : a * all + bb;
      }
      carry = all;
    } else {
      carry = wr ? wb : wa * carry + wb;
    }
    if (fh > 0) h = er ? eb : ea * h + eb;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      s_a[first_map + j * C] = h;
      h = marked && (fr >> j & 1) ? fb[j] : fa[j] * h + fb[j];
    }
    __syncthreads();

    // ---- (3) the rows, from the value that reaches them
    const auto write_rows = [&](auto has_marks) {
    constexpr bool MARKED = decltype(has_marks)::value;
    A v_[VEC];
    take(v_, s_a + own_map);
    T *orow = os;
    A *wrow = ow;
    G *grow = og;
    A *prow = op;
#pragma unroll kUnroll
    for (int r = 0; r < R; ++r, orow += dk, wrow += dk, grow += dgates, prow += dsums) {
      int m = 0;
      if constexpr (MARKED) {
        m = mark[r];
        if (m & kPad) continue;
        if (m & (BWD ? kEnd : kStart)) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) v_[v] = 0;
          if (live) load_acc<A, VEC>(v_, p.state, (srow + (m >> kMarkBits)) * p.K + c0, nv);
        }
      }
      const bool dead = MARKED && (m & kDead);
      A x[VEC], g[VEC];
      read_row(x, g, r);
      Pack<T, VEC> o;
      if constexpr (!BWD) {
        fma_all(v_, g, v_, x);
        if (dead) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) v_[v] = 0;
        }
        round_pack(o, v_);
        store_row(orow, o);
        if constexpr (!std::is_same<A, T>::value)
          if (p.wide) {
            if constexpr (RAGGED) {
              Pack<A, VEC> w;
              round_pack(w, v_);
              store_row(wrow, w);
            } else if (live) {
              store_wide(wrow, v_);
            }
          }
        if (MARKED && live && (m & kEnd) && p.last) store_acc<A, VEC>(v_, p.last, (srow + (m >> kMarkBits)) * p.K + c0, nv);
      } else {
        A dh[VEC], dg[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) dh[v] = v_[v];
        if (have_src) add_all(dh, v_, x);
        if (dead) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) dh[v] = 0;
        }
        round_pack(o, dh);
        store_row(orow, o);
        if (want_gate) {
          A before[VEC];
          if constexpr (RAGGED) widen<A, VEC>(before, Ragged<A, VEC>::get(fs + r * kFwdRow, col, moved(fat, r, dk, sizeof(A))));
          else widen<A, VEC>(before, FwdSlot::get(fs + r * kFwdRow, moved(fat, r, dk, 1)));
          if (MARKED && (m & (kStart | kDead))) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) before[v] = 0;
            if (live && (m & kStart)) load_acc<A, VEC>(before, p.init, (srow + (m >> kMarkBits)) * p.K + c0, nv);
          }
          mul_all(dg, dh, before);
          if constexpr (!SHARED) {
            Pack<G, VEC> q;
            round_pack(q, dg);
            store_row(grow, q);
          } else {
            // sum of the thread's channels, then of the neighbouring lanes that hold the same gate; the lanes of a row
            // are here together: rows are skipped (kPad) by whole rows
            A sum = dg[0];
#pragma unroll
            for (int v = 1; v < VEC; ++v) sum += dg[v];
            for (int d = 1; d < sum_lanes; d <<= 1) sum += __shfl_xor_sync(rowmask, sum, d);
            if (live && (col & (sum_lanes - 1)) == 0) {
              if (part_sums) *prow = sum;
              else *grow = from_acc<G>(sum);
            }
          }
        }
        mul_all(v_, g, dh);
        if (dead) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) v_[v] = 0;
        }
        if (MARKED && live && (m & kStart) && p.last) store_acc<A, VEC>(v_, p.last, (srow + (m >> kMarkBits)) * p.K + c0, nv);
      }
    }
    };
    if (mine) write_rows(std::true_type());
    else write_rows(std::false_type());
  };

  int stage = 0, ahead_stage = kStages - 1, par = 0, set = 0;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_rows(i);
  __syncthreads();  // the first tile's borders are known
  for (int64_t done = 0; done < len; done += step) {
    load_rows(ahead_stage);
    async_wait_all_but<kStages - 1>();
    if (RAGGED) __syncwarp();  // the chunks that the other lanes of a row copied are there
    tile_work(stage, par, set);
    os += tile_k;
    ow += tile_k;
    og += tile_gates;
    op += step * dsums;
    xat = moved(xat, step, dk, RAGGED ? sizeof(T) : 1);
    fat = moved(fat, step, dk, RAGGED ? sizeof(A) : 1);
    gat = moved(gat, step, dgates, RAGGED ? sizeof(G) : 1);
    stage = stage == kStages - 1 ? 0 : stage + 1;
    ahead_stage = ahead_stage == kStages - 1 ? 0 : ahead_stage + 1;
    set = set == kMarkStages - 1 ? 0 : set + 1;
    par ^= 1;
  }
}

// The sums of the partial products of a shared gate, in order.
template <typename A, typename G>
__global__ void __launch_bounds__(kThreads) gate_sum_kernel(const A *__restrict__ part, G *__restrict__ out, int64_t n, int64_t per) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    A s = part[i * per];
    for (int64_t j = 1; j < per; ++j) s += part[i * per + j];
    out[i] = from_acc<G>(s);
  }
}

// Segments without rows hand their start through.
template <typename A>
__global__ void __launch_bounds__(kThreads) empty_segments_kernel(const int64_t *__restrict__ indptr, const A *__restrict__ from,
                                                                  A *__restrict__ to, int64_t B, int64_t E, int64_t N, int64_t K, int64_t bstride) {
  const int lane = threadIdx.x & 31;
  for (int64_t s = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); s < B * N; s += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t *ip = indptr + s / N * bstride + s % N;
    if (clamp64(ip[1], 0, E) > clamp64(ip[0], 0, E)) continue;
    for (int64_t c = lane; c < K; c += 32) to[s * K + c] = from ? from[s * K + c] : (A)0;
  }
}

inline unsigned flat_blocks(int64_t items, int per = kThreads) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + per - 1) / per, (int64_t)sm_count() * 32));
}

// At least four channels: the lanes that share one in step (2) have to be lanes of one warp.
inline int least_lanes(int vec) { return vec >= 4 ? 0 : vec == 2 ? 1 : 2; }
// lanes that hold a row's channels of a tile, at most
inline int lanes_of_row(int64_t K, int vec, size_t elem) {
  const int wide = vec * elem >= 16 ? 3 : 5;  // 128 bytes of a row, or a whole warp of single values
  return std::min(wide, std::max(ilog2_ceil((K + vec - 1) / vec), least_lanes(vec)));
}
// lanes of a row whose gate products a row's shuffles sum: the neighbours that hold the same gate
inline int lanes_of_gate(int64_t width, int vec, int lx_log2) {
  int l = 0;
  while (l < lx_log2 && width / vec % ((int64_t)2 << l) == 0) ++l;
  return l;
}

template <typename T, typename G, int VEC, bool SHARED, bool BWD, bool RAGGED> int launch_tiles(ScanParams p, cudaStream_t stream) {
  using S = ScanShape<T, G, VEC, SHARED, BWD, RAGGED>;
  auto kernel = scan_kernel<T, G, VEC, SHARED, BWD, RAGGED>;
  static std::atomic<int> resident[64][8];  // CTAs of an SM by the lanes of a row; also: the attributes are set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TSB_ERR_LAUNCH;
  const auto ctas_of_sm = [&](int lx_log2) -> int {
    int n = resident[dev][lx_log2].load();
    if (n == 0) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kScanThreads + 32, S::bytes(1 << lx_log2, kMostCluster)) != cudaSuccess || n < 1)
        return 0;
      resident[dev][lx_log2].store(n);
    }
    return n;
  };
  // Work is spread over as many CTAs as the GPU holds.  Rows are cut into parts at segment borders where there are
  // segments enough (six to a part make parts of similar length), and over a cluster for the rest, since
  // its CTAs wait for each other at every tile: 37 segments over 65536 x 2048 bf16 took 199 us with a cluster of 8 and
  // one part, 174 with 2 and 4, 179 with 1 and 9.  Where that leaves half the GPU empty a tile gets fewer channels (down
  // to 32 bytes of a row) and more rows: one segment of 65536 x 1024 takes 139 us at 128 bytes of a row, 98 at 64 and 141
  // at 32, which no longer fit at once.
  int64_t ctas = 0;
  p.lx_log2 = lanes_of_row(p.K, VEC, sizeof(T));
  for (;;) {
    const int64_t C = (int64_t)VEC << p.lx_log2, L = (int64_t)(kScanThreads >> p.lx_log2) * S::kRows;
    p.tiles_k = (p.K + C - 1) / C;
    const int64_t tiles = (p.E + L - 1) / L, want = (int64_t)sm_count() * ctas_of_sm(p.lx_log2);
    if (want == 0) return TSB_ERR_LAUNCH;
    ctas = p.tiles_k * p.B;
    const int64_t even_parts = std::max<int64_t>(1, p.N / 6);
    p.cluster = 1;
    while (p.cluster < kMostCluster && ctas * p.cluster * even_parts < want && p.cluster * 2 <= tiles) p.cluster *= 2;
    ctas *= p.cluster;
    p.parts = std::max<int64_t>(1, std::min<int64_t>({want / ctas, p.N, tiles / p.cluster}));
    ctas *= p.parts;
    if (ctas * 2 > want || p.lx_log2 <= least_lanes(VEC) || C * (int64_t)sizeof(T) <= 32 || tiles < 2 * p.cluster * p.parts) break;
    --p.lx_log2;
  }
  const int lx = 1 << p.lx_log2;
  p.lanes_log2 = SHARED ? lanes_of_gate(p.width, VEC, p.lx_log2) : 0;
  if (ctas > 2147483647LL) return TSB_ERR_TOO_LARGE;
  const size_t bytes = S::bytes(lx, p.cluster);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kScanThreads + 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return TSB_ERR_LAUNCH;
  if constexpr (SHARED && BWD) {
    const int64_t per = VEC << p.lanes_log2;
    if (p.grad_gate && per != p.width) {
      const int64_t n = p.B * p.E * (p.K / p.width);
      gate_sum_kernel<acc_t<T>, G><<<flat_blocks(n), kThreads, 0, stream>>>(static_cast<const acc_t<T> *>(p.partial), static_cast<G *>(p.grad_gate), n, p.width / per);
    }
  }
  return launch_status();
}

// Partial products of shared gates in a row, for whichever pack width the addresses will allow.
inline int64_t partials_of_row(int64_t K, int64_t width, size_t elem) {
  int64_t most = 0;
  for (const int vec : {(int)(16 / elem), 2, 1}) {
    if (K % vec != 0 || width % vec != 0) continue;
    // (a launch may take fewer lanes for a row than there could be)
    const int lanes = std::min(lanes_of_gate(width, vec, lanes_of_row(K, vec, elem)), least_lanes(vec));
    const int64_t per = (int64_t)vec << lanes;
    if (per != width) most = std::max(most, K / per);
  }
  return most;
}

template <typename T, typename G, bool BWD> int launch(const ScanParams &p, cudaStream_t stream) {
  using A = acc_t<T>;
  const void *all[] = {p.src, p.width == 1 ? p.gate : nullptr, p.fwd, p.out, p.wide, p.width == 1 ? p.grad_gate : nullptr};
  bool a16 = true, a4 = true;
  for (const void *q : all) {
    a16 = a16 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    a4 = a4 && (reinterpret_cast<uintptr_t>(q) & 3) == 0;
  }
  if (sizeof(G) > sizeof(T) && p.width == 1) a16 = a16 && aligned32(p.gate) && aligned32(p.grad_gate);  // packs of 32 bytes
  if (p.last && p.N > 0) {
    empty_segments_kernel<A><<<flat_blocks(p.B * p.N, kThreads / 32), kThreads, 0, stream>>>(p.indptr, static_cast<const A *>(p.state), static_cast<A *>(p.last),
                                                                                             p.B, p.E, p.N, p.K, p.bstride);
  }
  if (p.E == 0) return launch_status();
  constexpr int full = full_vec<T>();
  // A gate of its own for every channel: 16 bytes of channels to a thread wherever the rows begin.  Shared gates: as many
  // channels as 16 or 4 bytes hold if that divides the channels that share a gate, else one.
  if (p.width == 1)
    return a16 && p.K % full == 0 ? launch_tiles<T, G, full, false, BWD, false>(p, stream) : launch_tiles<T, G, full, false, BWD, true>(p, stream);
  if (a16 && p.width % full == 0) return launch_tiles<T, G, full, true, BWD, false>(p, stream);
  if constexpr (sizeof(T) == 2)  // (two channels of the h that the backward reads are 8 bytes)
    if (a4 && (reinterpret_cast<uintptr_t>(p.fwd) & 7) == 0 && p.width % 2 == 0) return launch_tiles<T, G, 2, true, BWD, false>(p, stream);
  return launch_tiles<T, G, 1, true, BWD, false>(p, stream);
}

// one translation unit for each data type
int launch_f32(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);
int launch_f64(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);
int launch_f16(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);
int launch_bf16(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);

}  // namespace scan
}  // namespace tsb
