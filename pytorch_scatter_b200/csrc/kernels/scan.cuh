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
// copies to its own slots of shared memory two tiles ahead (cp.async; nobody else reads them, so the data needs no
// barrier).  (1) It composes its rows' maps and leaves the result in shared memory.  (2) Turned over, a thread takes VEC
// consecutive maps of one channel, composes them and scans over the lanes that share the channel; the CTAs of a cluster
// hold neighbouring tiles of the same channels and exchange their totals through distributed shared memory; then the
// value that reaches each thread's rows is known.  (3) Each thread walks its rows again from that value and writes the
// outputs.  The cluster moves on by its CTAs' tiles, carrying the value along in registers, so that one launch covers any
// length without waiting on anything but its own cluster.  The composition has a fixed shape: results do not vary from
// run to run.
//
// A segment's first row (backward: its last) does not take the value from the row before: such a map is marked `reset`
// and drops what comes in, so infinities and NaN of one segment never reach the next.  Tiles that no segment border
// touches run a copy of the code without these checks.
#pragma once

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace tsb {
namespace scan {

constexpr int kScanThreads = 128;           // threads that carry channels; a fifth warp looks for segment borders
constexpr int kStages = 3;
constexpr int kMostCluster = 8;

struct ScanParams {
  const void *src, *gate, *state;  // backward: src = grad_out (may be null), state = grad_last
  const void *fwd, *init;          // backward: the forward's out and state
  const int64_t *indptr;
  void *out, *last;                // backward: grad_src, grad_state
  void *grad_gate, *partial;       // backward
  int64_t B, E, K, N, width, bstride;
  int64_t parts, tiles_k;
  int lx_log2, cluster, lanes_log2;  // lanes_log2: lanes of one row whose gate products are summed by shuffles
};

// row marks: the row's segment and flags
constexpr int kStart = 1, kEnd = 2, kDead = 4, kPad = 8, kMarkBits = 4;
constexpr int64_t kMostSegments = (int64_t)1 << 27;

// A copy of VEC values to the thread's own slot.  One 2-byte value travels in the 4-byte word that holds it (cp.async has
// no smaller form), unless that word reaches over the array's ends; `half` says which half it is.
template <typename T, int VEC> struct Slot {
  static constexpr bool kWord = sizeof(T) * VEC == 2;
  static constexpr int kBytes = kWord ? 4 : (int)sizeof(T) * VEC;
  static __device__ __forceinline__ int half(const T *p) { return kWord ? (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 1 : 0; }
  static __device__ __forceinline__ void copy(char *slot, const T *p, const T *lo, const T *hi) {
    if constexpr (kWord) {
      const uintptr_t word = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3;
      if (word >= reinterpret_cast<uintptr_t>(lo) && word + 4 <= reinterpret_cast<uintptr_t>(hi)) {
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

template <typename A, int VEC> __device__ __forceinline__ void load_acc(A (&v)[VEC], const void *base, int64_t at) {
  const A *p = static_cast<const A *>(base);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = p ? p[at + i] : (A)0;
}
template <typename A, int VEC> __device__ __forceinline__ void store_acc(const A (&v)[VEC], void *base, int64_t at) {
  A *p = static_cast<A *>(base);
#pragma unroll
  for (int i = 0; i < VEC; ++i) p[at + i] = v[i];
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
template <typename A, int VEC> __device__ __forceinline__ void take(A (&v)[VEC], const A *p) {
  constexpr int n = VEC * sizeof(A) >= 16 ? 16 / (int)sizeof(A) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += n) {
    const Pack<A, n> q = *reinterpret_cast<const Pack<A, n> *>(p + i);
#pragma unroll
    for (int j = 0; j < n; ++j) v[i + j] = q.v[j];
  }
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

// A * h + B.  The product of a tile's gates may overflow where the recurrence itself stays at zero.
template <typename A> __device__ __forceinline__ A apply_map(A a, A b, A h) { return h == (A)0 ? b : a * h + b; }

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
__device__ __forceinline__ unsigned smem_at(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned remote_at(unsigned addr, int rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void mbar_init(unsigned bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// false if the bytes did not come within the limit (they always do: the CTAs of a cluster run together)
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity) {
  for (int i = 0; i < (1 << 22); ++i) {
    unsigned ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
  }
  return false;
}
__device__ __forceinline__ void send(unsigned addr, unsigned bar, float a, float b) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(addr), "f"(a), "f"(b), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(unsigned addr, unsigned bar, double a, double b) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];" ::"r"(addr), "d"(a), "d"(b), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(unsigned addr, unsigned bar, int v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(v), "r"(bar) : "memory");
}

template <typename T, typename G, int VEC, bool SHARED, bool BWD> struct ScanShape {
  using A = acc_t<T>;
  static constexpr int kGateVec = SHARED ? 1 : VEC;
  using SrcSlot = Slot<T, VEC>;
  using GateSlot = Slot<G, kGateVec>;
  static constexpr int kRowBytes = SrcSlot::kBytes * (BWD ? 2 : 1) + GateSlot::kBytes;
  // rows of a thread: 28 KB for each of the three stages at most, so that two CTAs and more fit an SM
  static constexpr int kRows = 224 / kRowBytes < 16 ? 224 / kRowBytes : 16;
  static constexpr int kStageBytes = kScanThreads * kRows * kRowBytes;
  static constexpr int kMapBytes = 2 * kScanThreads * VEC * (int)sizeof(A);  // [A, B][ty][C]
  static size_t bytes(int lx, int cluster) {
    const size_t C = (size_t)lx * VEC, L = (size_t)(kScanThreads / lx) * kRows;
    return (size_t)kStages * kStageBytes + kMapBytes + (cluster > 1 ? sizeof(A) * C * 4 * cluster : 0) + sizeof(int) * kStages * L;
  }
};

template <typename T, typename G, int VEC, bool SHARED, bool BWD>
__global__ void __launch_bounds__(kScanThreads + 32) scan_kernel(ScanParams p) {
  using S = ScanShape<T, G, VEC, SHARED, BWD>;
  using SrcSlot = typename S::SrcSlot;
  using GateSlot = typename S::GateSlot;
  using A = acc_t<T>;
  constexpr int R = S::kRows;
  constexpr int kSrcRow = kScanThreads * SrcSlot::kBytes, kGateRow = kScanThreads * GateSlot::kBytes;

  const int tid = threadIdx.x;
  const int lx = 1 << p.lx_log2, C = lx * VEC, L = (kScanThreads >> p.lx_log2) * R;
  const int col = tid & (lx - 1), ty = tid >> p.lx_log2;
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
  A *s_a = reinterpret_cast<A *>(smem + (size_t)kStages * S::kStageBytes);  // maps of the threads [ty][C]; then the values
  A *s_b = s_a + kScanThreads * VEC;                               // that reach them, in place of A
  A *s_total = s_b + kScanThreads * VEC;                           // maps of the cluster's CTAs [2][cs][C][A, B]
  int *s_marks = reinterpret_cast<int *>(s_total + (cs > 1 ? 4 * cs * C : 0));  // [stage][L]
  __shared__ int s_reset[kScanThreads], s_total_reset[2][kMostCluster];
  __shared__ int s_marked[kStages];                                      // does a segment border touch the tile?
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
    int64_t cursor = BWD ? p.N + 1 : 0;  // bound of the last row looked up
    const auto look = [&](int64_t tile, int stage) {
      // lane 0 of each search sees the first and the last row of the tile; the same border means none in between
      const int64_t last = tile + L - 1 < len ? tile + L - 1 : len - 1;
      const int64_t from = row_of(tile < len ? tile : len - 1), to = row_of(last);
      const int64_t u = BWD ? bound<true>(indptr, 0, cursor, from) : bound<true>(indptr, cursor, p.N + 1, from);
      const bool inside = u >= 1 && u <= p.N;
      const bool whole = tile + L <= len;
      const bool marked = !(inside && whole && (BWD ? from + 1 < indptr[u] && to > indptr[u - 1] : from > indptr[u - 1] && to + 1 < indptr[u]));
      cursor = u;
      if (marked) {
        for (int j = lane; j < L; j += 32) {
          const int64_t t = row_of(tile + j < len ? tile + j : len - 1);
          const int64_t w = BWD ? bound<true>(indptr, 0, u, t) : bound<true>(indptr, u, p.N + 1, t);
          int flags;
          if (tile + j >= len) flags = kPad;
          else if (w < 1 || w > p.N) flags = kDead;
          else flags = (int)(w - 1) << kMarkBits | (indptr[w - 1] == t ? kStart : 0) | (indptr[w] == t + 1 ? kEnd : 0);
          s_marks[stage * L + j] = flags;
        }
      }
      if (lane == 0) s_marked[stage] = marked;
    };
    int64_t tile = (int64_t)rank * L;
    int stage = 0;
    look(tile, 0);
    __syncthreads();
    for (int64_t done = 0; done < len; done += step) {
      tile += step;
      stage = stage == kStages - 1 ? 0 : stage + 1;
      if (done + step < len) look(tile, stage);  // of the three stages, the others may still read two
      __syncthreads();                           // (1) of the tile before is done
      __syncthreads();                           // (2)
    }
    return;
  }

  const int64_t c0 = kt * C + (int64_t)col * VEC;   // this thread's first channel
  const bool live = c0 < p.K;
  const int64_t gates = p.K / p.width, g0 = SHARED ? c0 / p.width : c0;
  const int64_t dk = BWD ? -p.K : p.K, dgates = BWD ? -gates : gates;  // from a row to the next one on the way
  const int64_t srow = b * p.N;                     // first row of this batch in the state arrays
  const bool have_src = !BWD || p.src, want_gate = BWD && p.grad_gate;
  const T *src_lo = static_cast<const T *>(p.src), *src_hi = src_lo + p.B * p.E * p.K;
  const T *fwd_lo = static_cast<const T *>(p.fwd), *fwd_hi = fwd_lo + p.B * p.E * p.K;
  const G *gate_lo = static_cast<const G *>(p.gate), *gate_hi = gate_lo + p.B * p.E * gates;

  // this thread's slots [stage][row][thread], and its pointers to the next tile to load and to the tile at work
  char *s_src = smem + tid * SrcSlot::kBytes;
  char *s_fwd = s_src + kStages * R * kSrcRow;
  char *s_gate = smem + kStages * R * kSrcRow * (BWD ? 2 : 1) + tid * GateSlot::kBytes;
  int64_t tile = (int64_t)rank * L;                 // position of the CTA's tile
  int64_t ahead = tile + ty * R;                    // position of the thread's next rows to load
  const int64_t at = b * p.E + row_of(ahead);
  const T *lsrc = src_lo + (have_src ? at * p.K + c0 : 0), *lfwd = fwd_lo + (BWD ? (at - 1) * p.K + c0 : 0);  // fwd: h of the row before
  const G *lgate = gate_lo + at * gates + g0;
  T *os = static_cast<T *>(p.out) + at * p.K + c0;
  G *og = static_cast<G *>(p.grad_gate) + (want_gate ? at * gates + g0 : 0);
  const int64_t tile_k = step * dk, tile_gates = step * dgates;
  // which half of its word a row's value is in (2-byte slots only)
  const int kodd = (int)(p.K & 1), godd = (int)(gates & 1);
  int xhalf = SrcSlot::half(lsrc), fhalf = SrcSlot::half(lfwd), ghalf = GateSlot::half(lgate);
  const int xturn = (int)(tile_k & 1), gturn = (int)(tile_gates & 1);

  const auto load_rows = [&](int stage) {
    const int64_t left = len - ahead;
    if (live && left > 0) {
      const T *xs = lsrc, *fs = lfwd;
      const G *gs = lgate;
      char *xd = s_src + stage * (R * kSrcRow), *fd = s_fwd + stage * (R * kSrcRow), *gd = s_gate + stage * (R * kGateRow);
      const int n = left < R ? (int)left : R;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < n) {
          if (have_src) SrcSlot::copy(xd + r * kSrcRow, xs, src_lo, src_hi);
          GateSlot::copy(gd + r * kGateRow, gs, gate_lo, gate_hi);
          if (BWD && want_gate && fs >= fwd_lo) SrcSlot::copy(fd + r * kSrcRow, fs, fwd_lo, fwd_hi);  // (row 0 has none before it)
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
  A carry = 0;  // the value that reaches the cluster's tiles in channel fc
  unsigned phases = 0;  // parity to wait for, one bit for each of the two barriers

  const auto tile_work = [&](auto has_marks, int stage, int par) {
    constexpr bool MARKED = decltype(has_marks)::value;
    const int *mark = s_marks + stage * L + ty * R;
    const char *xs = s_src + stage * (R * kSrcRow), *fs = s_fwd + stage * (R * kSrcRow), *gs = s_gate + stage * (R * kGateRow);
    // ---- (1) the map of this thread's rows
    {
      A ma[VEC], mb[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) { ma[v] = 1; mb[v] = 0; }
      int reset = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (MARKED) {
          const int m = mark[r];
          if (m & kPad) continue;
          if (m & (kDead | (BWD ? kEnd : kStart))) {
            reset = 1;
#pragma unroll
            for (int v = 0; v < VEC; ++v) mb[v] = 0;
            if (m & kDead) continue;
            if (live) load_acc<A, VEC>(mb, p.state, (srow + (m >> kMarkBits)) * p.K + c0);
          }
        }
        const Pack<T, VEC> x = SrcSlot::get(xs + r * kSrcRow, (xhalf + r * kodd) & 1);
        const Pack<G, S::kGateVec> g = GateSlot::get(gs + r * kGateRow, (ghalf + r * godd) & 1);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const A gv = to_acc<G>(g.v[SHARED ? 0 : v]);
          if constexpr (BWD) mb[v] = gv * (have_src ? mb[v] + to_acc<T>(x.v[v]) : mb[v]);
          else mb[v] = gv * mb[v] + to_acc<T>(x.v[v]);
          if (!SHARED || v == 0) ma[v] *= gv;
        }
      }
      A *pa = s_a + tid * VEC, *pb = s_b + tid * VEC;
      if constexpr (SHARED) {
#pragma unroll
        for (int v = 1; v < VEC; ++v) ma[v] = ma[0];
      }
      put(pa, ma);
      put(pb, mb);
      if (MARKED && col == 0) s_reset[ty] = reset;
    }
    __syncthreads();

    // ---- (2) scan of the maps over the tile and the cluster
    A fa[VEC], fb[VEC];
    unsigned fr = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int at = (fh * VEC + j) * C + fc;
      fa[j] = s_a[at];
      fb[j] = s_b[at];
      if (MARKED) fr |= (unsigned)s_reset[fh * VEC + j] << j;
    }
    A ta = fa[0], tb = fb[0];
    int tr = fr & 1;
#pragma unroll
    for (int j = 1; j < VEC; ++j) {
      const bool rs = MARKED && (fr >> j & 1);
      tb = rs ? fb[j] : apply_map(fa[j], fb[j], tb);
      ta *= fa[j];
      tr |= rs;
    }
    for (int d = 1; d < H; d <<= 1) {
      const A pa = __shfl_up_sync(kFullMask, ta, d, H), pb = __shfl_up_sync(kFullMask, tb, d, H);
      const int pr = MARKED ? __shfl_up_sync(kFullMask, tr, d, H) : 0;
      if (fh >= d) {
        if (!MARKED || !tr) tb = apply_map(ta, tb, pb);
        ta *= pa;
        tr |= pr;
      }
    }
    // map of the lanes before this one
    const A ea = __shfl_up_sync(kFullMask, ta, 1, H), eb = __shfl_up_sync(kFullMask, tb, 1, H);
    const int er = MARKED ? __shfl_up_sync(kFullMask, tr, 1, H) : 0;
    // map of the whole tile
    const A wa = __shfl_sync(kFullMask, ta, H - 1, H), wb = __shfl_sync(kFullMask, tb, H - 1, H);
    const int wr = MARKED ? __shfl_sync(kFullMask, tr, H - 1, H) : 0;
    A h = carry;
    if (cs > 1) {
      const unsigned bar = smem_at(&s_bar[par]);
      if (tid == 0) mbar_expect(bar, (unsigned)(cs * (C * 2 * (int)sizeof(A) + 4)));
      const unsigned mine = smem_at(s_total + ((par * cs + rank) * C + fc) * 2);
      for (int q = fh; q < cs; q += H) send(remote_at(mine, q), remote_at(bar, q), wa, wb);
      if (tid < cs) send(remote_at(smem_at(&s_total_reset[par][rank]), tid), remote_at(bar, tid), wr);
      if (!mbar_wait(bar, phases >> par & 1)) carry = (A)NAN;
      phases ^= 1u << par;
      A all = carry;
      for (int q = 0; q < cs; ++q) {
        if (q == rank) h = all;
        const A *m = s_total + ((par * cs + q) * C + fc) * 2;
        const A a = m[0], bb = m[1];
        all = s_total_reset[par][q] ? bb : apply_map(a, bb, all);
      }
      carry = all;
    } else {
      carry = wr ? wb : apply_map(wa, wb, carry);
    }
    if (fh > 0) h = er ? eb : apply_map(ea, eb, h);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      s_a[(fh * VEC + j) * C + fc] = h;
      h = MARKED && (fr >> j & 1) ? fb[j] : apply_map(fa[j], fb[j], h);
    }
    __syncthreads();

    // ---- (3) the rows, from the value that reaches them
    A v_[VEC];
    take(v_, s_a + tid * VEC);
    T *orow = os;
    G *grow = og;
#pragma unroll
    for (int r = 0; r < R; ++r, orow += dk, grow += dgates) {
      int m = 0;
      if constexpr (MARKED) {
        m = mark[r];
        if (m & kPad) continue;
        if (m & (BWD ? kEnd : kStart)) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) v_[v] = 0;
          if (live) load_acc<A, VEC>(v_, p.state, (srow + (m >> kMarkBits)) * p.K + c0);
        }
      }
      const bool dead = MARKED && (m & kDead);
      const Pack<T, VEC> x = SrcSlot::get(xs + r * kSrcRow, (xhalf + r * kodd) & 1);
      const Pack<G, S::kGateVec> g = GateSlot::get(gs + r * kGateRow, (ghalf + r * godd) & 1);
      Pack<T, VEC> o;
      if constexpr (!BWD) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          v_[v] = to_acc<G>(g.v[SHARED ? 0 : v]) * v_[v] + to_acc<T>(x.v[v]);
          if (dead) v_[v] = 0;
        }
        round_pack(o, v_);
        if (live) {
          st_stream<T, VEC>(orow, o);
          if (MARKED && (m & kEnd) && p.last) store_acc<A, VEC>(v_, p.last, (srow + (m >> kMarkBits)) * p.K + c0);
        }
      } else {
        A dh[VEC], dg[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          dh[v] = have_src ? v_[v] + to_acc<T>(x.v[v]) : v_[v];
          if (dead) dh[v] = 0;
        }
        round_pack(o, dh);
        if (live) st_stream<T, VEC>(orow, o);
        if (want_gate) {
          const Pack<T, VEC> f = SrcSlot::get(fs + r * kSrcRow, (fhalf + r * kodd) & 1);
          if (MARKED && (m & kStart)) {
            A before[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) before[v] = 0;
            if (live) load_acc<A, VEC>(before, p.init, (srow + (m >> kMarkBits)) * p.K + c0);
#pragma unroll
            for (int v = 0; v < VEC; ++v) dg[v] = dh[v] * before[v];
          } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) dg[v] = dead ? (A)0 : dh[v] * to_acc<T>(f.v[v]);
          }
          if constexpr (!SHARED) {
            Pack<G, VEC> q;
            round_pack(q, dg);
            if (live) st_stream<G, VEC>(grow, q);
          } else {
            // sum of the thread's channels, then of the neighbouring lanes that hold the same gate; the lanes of a row
            // are here together: rows are skipped (kPad) by whole rows
            A sum = dg[0];
#pragma unroll
            for (int v = 1; v < VEC; ++v) sum += dg[v];
            const unsigned rowmask = lx == 32 ? kFullMask : ((1u << lx) - 1u) << ((tid & 31) & ~(lx - 1));
            for (int d = 1; d < (1 << p.lanes_log2); d <<= 1) sum += __shfl_xor_sync(rowmask, sum, d);
            if (live && (col & ((1 << p.lanes_log2) - 1)) == 0) {
              const int64_t per = VEC << p.lanes_log2;
              if (per == p.width) *grow = from_acc<G>(sum);
              else static_cast<A *>(p.partial)[(b * p.E + row_of(tile + ty * R + r)) * (p.K / per) + c0 / per] = sum;
            }
          }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) v_[v] = dead ? (A)0 : to_acc<G>(g.v[SHARED ? 0 : v]) * dh[v];
        if (MARKED && live && (m & kStart) && p.last) store_acc<A, VEC>(v_, p.last, (srow + (m >> kMarkBits)) * p.K + c0);
      }
    }
  };

  int stage = 0, ahead_stage = kStages - 1, par = 0;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_rows(i);
  __syncthreads();  // the first tile's borders are known
  for (int64_t done = 0; done < len; done += step) {
    load_rows(ahead_stage);
    const bool marked = s_marked[stage];
    async_wait_all_but<kStages - 1>();
    if (marked) tile_work(std::true_type(), stage, par);
    else tile_work(std::false_type(), stage, par);
    tile += step;
    os += tile_k;
    og += tile_gates;
    xhalf ^= xturn;
    fhalf ^= xturn;
    ghalf ^= gturn;
    stage = stage == kStages - 1 ? 0 : stage + 1;
    ahead_stage = ahead_stage == kStages - 1 ? 0 : ahead_stage + 1;
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

// lanes that hold a row's channels of a tile
inline int lanes_of_row(int64_t K, int vec, size_t elem) {
  const int wide = vec * elem >= 16 ? 3 : 5;  // 128 bytes of a row, or a whole warp of single values
  // at least four channels: the lanes that share one in step (2) are lanes of one warp
  return std::min(wide, std::max(ilog2_ceil((K + vec - 1) / vec), vec >= 4 ? 0 : vec == 2 ? 1 : 2));
}
// lanes of a row whose gate products a row's shuffles sum: the neighbours that hold the same gate
inline int lanes_of_gate(int64_t width, int vec, int lx_log2) {
  int l = 0;
  while (l < lx_log2 && width / vec % ((int64_t)2 << l) == 0) ++l;
  return l;
}

template <typename T, typename G, int VEC, bool SHARED, bool BWD> int launch_tiles(ScanParams p, cudaStream_t stream) {
  using S = ScanShape<T, G, VEC, SHARED, BWD>;
  auto kernel = scan_kernel<T, G, VEC, SHARED, BWD>;
  p.lx_log2 = lanes_of_row(p.K, VEC, sizeof(T));
  p.lanes_log2 = SHARED ? lanes_of_gate(p.width, VEC, p.lx_log2) : 0;
  const int lx = 1 << p.lx_log2;
  const int64_t L = (int64_t)(kScanThreads >> p.lx_log2) * S::kRows, C = (int64_t)lx * VEC;
  p.tiles_k = (p.K + C - 1) / C;
  const int64_t tiles = (p.E + L - 1) / L, want = (int64_t)sm_count() * 2;
  int64_t ctas = p.tiles_k * p.B;
  p.cluster = 1;
  while (p.cluster < kMostCluster && ctas * p.cluster < want && p.cluster * 2 <= tiles) p.cluster *= 2;
  ctas *= p.cluster;
  p.parts = std::max<int64_t>(1, std::min<int64_t>({want / ctas, p.N, tiles / p.cluster}));
  if (ctas * p.parts > 2147483647LL) return TSB_ERR_TOO_LARGE;
  const size_t bytes = S::bytes(lx, p.cluster);
  static std::atomic<int> allowed[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TSB_ERR_LAUNCH;
  if (allowed[dev].load() == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) return TSB_ERR_LAUNCH;
    allowed[dev].store(1);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(ctas * p.parts));
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

// The pack width: as many of a row's channels as 16 bytes hold, or 4 bytes, or one, by what the row length, the sharing
// of the gate and the addresses allow.
template <typename T> int pack_width(int64_t K, int64_t width, bool aligned16_all, bool aligned4_all) {
  constexpr int full = full_vec<T>();
  if (aligned16_all && K % full == 0 && (width == 1 || width % full == 0)) return full;
  if (sizeof(T) == 2 && aligned4_all && K % 2 == 0 && (width == 1 || width % 2 == 0)) return 2;
  return 1;
}

// Partial products of shared gates in a row, for whichever pack width the addresses will allow.
inline int64_t partials_of_row(int64_t K, int64_t width, size_t elem) {
  int64_t most = 0;
  for (const int vec : {(int)(16 / elem), 2, 1}) {
    if (K % vec != 0 || width % vec != 0) continue;
    const int64_t per = (int64_t)vec << lanes_of_gate(width, vec, lanes_of_row(K, vec, elem));
    if (per != width) most = std::max(most, K / per);
  }
  return most;
}

template <typename T, typename G, bool BWD> int launch(const ScanParams &p, cudaStream_t stream) {
  using A = acc_t<T>;
  const void *all[] = {p.src, p.width == 1 ? p.gate : nullptr, p.fwd, p.out, p.width == 1 ? p.grad_gate : nullptr};
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
  const int vec = pack_width<T>(p.K, p.width, a16, a4);
  const auto go = [&](auto v) {
    constexpr int VEC = decltype(v)::value;
    return p.width > 1 ? launch_tiles<T, G, VEC, true, BWD>(p, stream) : launch_tiles<T, G, VEC, false, BWD>(p, stream);
  };
  constexpr int full = full_vec<T>();
  if (vec == full) return go(std::integral_constant<int, full>());
  if constexpr (sizeof(T) == 2)
    if (vec == 2) return go(std::integral_constant<int, 2>());
  return go(std::integral_constant<int, 1>());
}

// one translation unit for each data type
int launch_f32(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);
int launch_f64(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);
int launch_f16(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);
int launch_bf16(const ScanParams &p, int gate_dtype, bool backward, cudaStream_t stream);

}  // namespace scan
}  // namespace tsb
