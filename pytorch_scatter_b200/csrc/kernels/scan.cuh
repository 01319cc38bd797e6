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
// copies to its own slots of shared memory kStages tiles ahead (cp.async; nobody else reads them, so the data needs no
// barrier).  (1) It composes its rows' maps; (2) the maps are scanned over the threads of a warp by shuffles, over the
// warps through shared memory and over the CTAs of a cluster, which hold neighbouring tiles of the same channels, through
// distributed shared memory; (3) it walks its rows again from the value that reaches them and writes the outputs.  The
// cluster then moves on by its CTAs' tiles, carrying the value along, so that one launch covers any length without
// waiting on anything but its own cluster.  The composition has a fixed shape: results do not vary from run to run.
//
// A segment's first row (backward: its last) does not take the value from the row before: such a map is marked `reset`
// and drops what comes in, so infinities and NaN of one segment never reach the next.
#pragma once

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace tsb {
namespace scan {

constexpr int kScanThreads = 128;
constexpr int kScanWarps = kScanThreads / 32;
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

// row flags
constexpr int kStart = 1, kEnd = 2, kDead = 4, kPad = 8;
struct Mark { int seg, flags; };

// A copy of VEC values to the thread's own slot.  One 2-byte value travels in the 4-byte word that holds it (cp.async has
// no smaller form), unless that word reaches over the array's ends.
template <typename T, int VEC> struct Slot {
  static constexpr bool kWord = sizeof(T) * VEC == 2;
  static constexpr int kBytes = kWord ? 4 : (int)sizeof(T) * VEC;
  static __device__ __forceinline__ void copy(char *slot, const T *p, const T *lo, const T *hi) {
    if constexpr (kWord) {
      const uintptr_t word = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3;
      const bool high = reinterpret_cast<uintptr_t>(p) & 2;
      if (word >= reinterpret_cast<uintptr_t>(lo) && word + 4 <= reinterpret_cast<uintptr_t>(hi)) {
        const unsigned dst = (unsigned)__cvta_generic_to_shared(slot);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(word) : "memory");
      } else {
        reinterpret_cast<T *>(slot)[high] = *p;
      }
    } else {
      async_copy_pack<T, VEC>(reinterpret_cast<Pack<T, VEC> *>(slot), p);
    }
  }
  static __device__ __forceinline__ Pack<T, VEC> get(const char *slot, const T *p) {
    if constexpr (kWord) {
      Pack<T, VEC> r;
      r.v[0] = reinterpret_cast<const T *>(slot)[(reinterpret_cast<uintptr_t>(p) >> 1) & 1];
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

// A * h + B.  The product of a tile's gates may overflow where the recurrence itself stays at zero.
template <typename A> __device__ __forceinline__ A apply_map(A a, A b, A h) { return h == (A)0 ? b : a * h + b; }

template <typename A> __device__ __forceinline__ A shfl_up(A v, int d) { return __shfl_up_sync(kFullMask, v, d); }

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

template <typename T, typename G, int VEC, bool SHARED, bool BWD> struct ScanShape {
  using A = acc_t<T>;
  static constexpr int kGateVec = SHARED ? 1 : VEC;
  using SrcSlot = Slot<T, VEC>;
  using GateSlot = Slot<G, kGateVec>;
  static constexpr int kRowBytes = SrcSlot::kBytes * (BWD ? 2 : 1) + GateSlot::kBytes;
  // rows of a thread: 256 bytes of a stage at most, so that two CTAs and more fit an SM
  static constexpr int kRows = kRowBytes * 16 <= 256 ? 16 : kRowBytes * 8 <= 256 ? 8 : 4;
  static constexpr int kStageBytes = kScanThreads * kRows * kRowBytes;
  static size_t bytes(int lx, int cluster) {
    const size_t C = (size_t)lx * VEC, L = (size_t)(kScanThreads / lx) * kRows;
    return (size_t)kStages * kStageBytes + sizeof(A) * C * (4 * kScanWarps + 2 + (cluster > 1 ? 4 * cluster : 0)) +
           sizeof(Mark) * 2 * L;
  }
};

template <typename T, typename G, int VEC, bool SHARED, bool BWD>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(ScanParams p) {
  using S = ScanShape<T, G, VEC, SHARED, BWD>;
  using A = acc_t<T>;
  constexpr int R = S::kRows;
  namespace cg = cooperative_groups;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
  const int64_t rounds = (len + (int64_t)cs * L - 1) / ((int64_t)cs * L);

  const int64_t c0 = kt * C + (int64_t)col * VEC;   // this thread's first channel
  const bool live = c0 < p.K;
  const int64_t gates = p.K / p.width, g0 = SHARED ? c0 / p.width : c0;
  const T *src = static_cast<const T *>(p.src) + (p.src ? b * p.E * p.K + c0 : 0);
  const T *fwd = static_cast<const T *>(p.fwd) + (BWD ? b * p.E * p.K + c0 : 0);
  const G *gate = static_cast<const G *>(p.gate) + b * p.E * gates + g0;
  T *out = static_cast<T *>(p.out) + b * p.E * p.K + c0;
  const int64_t srow = b * p.N;                     // first row of this batch in the state arrays

  extern __shared__ __align__(128) char smem[];
  char *s_src = smem;                                              // [stage][row][thread]
  char *s_fwd = s_src + kStages * R * kScanThreads * S::SrcSlot::kBytes;
  char *s_gate = s_fwd + (BWD ? kStages * R * kScanThreads * S::SrcSlot::kBytes : 0);
  A *s_maps = reinterpret_cast<A *>(smem + (size_t)kStages * S::kStageBytes);  // maps of the warps [2][A, B][warp][C]
  A *s_in = s_maps + 4 * kScanWarps * C;                                 // value that reaches this CTA's tile [C]
  A *s_carry = s_in + C;                                           // value that reaches the cluster's tiles [C]
  A *s_ca = s_carry + C;                                           // maps of the cluster's CTAs [2][cs][C]
  A *s_cb = s_ca + (cs > 1 ? 2 * cs * C : 0);
  Mark *s_mark = reinterpret_cast<Mark *>(s_cb + (cs > 1 ? 2 * cs * C : 0));  // [2][L]
  __shared__ int s_resets[2][kScanWarps], s_creset[2][kMostCluster];
  __shared__ int64_t s_found[2][2];                                // [parity]: bound of the tile's last row, next border

  for (int c = tid; c < C; c += kScanThreads) s_carry[c] = 0;
  if (cs > 1) cg::this_cluster().sync();  // all CTAs run before anyone writes to their shared memory

  const auto row_of = [&](int64_t pos) { return BWD ? hi - 1 - pos : lo + pos; };
  const auto slot = [&](char *base, int bytes, int stage, int r) { return base + (size_t)((stage * R + r) * kScanThreads + tid) * bytes; };
  const auto first_pos = [&](int64_t i) { return (i * cs + rank) * (int64_t)L; };

  const T *src_lo = static_cast<const T *>(p.src), *src_hi = src_lo + p.B * p.E * p.K;
  const T *fwd_lo = static_cast<const T *>(p.fwd), *fwd_hi = fwd_lo + p.B * p.E * p.K;
  const G *gate_lo = static_cast<const G *>(p.gate), *gate_hi = gate_lo + p.B * p.E * gates;

  const auto load_tile = [&](int64_t i) {
    if (i < rounds && live) {
      const int64_t pos = first_pos(i) + (int64_t)ty * R;
      const int stage = (int)(i % kStages);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (pos + r >= len) break;
        const int64_t t = row_of(pos + r);
        if (!BWD || p.src) S::SrcSlot::copy(slot(s_src, S::SrcSlot::kBytes, stage, r), src + t * p.K, src_lo, src_hi);
        S::GateSlot::copy(slot(s_gate, S::GateSlot::kBytes, stage, r), gate + t * gates, gate_lo, gate_hi);
        if (BWD && p.grad_gate && t > 0) S::SrcSlot::copy(slot(s_fwd, S::SrcSlot::kBytes, stage, r), fwd + (t - 1) * p.K, fwd_lo, fwd_hi);
      }
    }
    async_commit();
  };

  for (int i = 0; i < kStages - 1; ++i) load_tile(i);

  // the row that was looked up last: its bound, the next border on the way (none: never met), whether it is outside
  int64_t cursor = BWD ? p.N + 1 : 0, border = BWD ? (int64_t)1 << 62 : -1;
  bool outside = false;

  for (int64_t i = 0; i < rounds; ++i) {
    load_tile(i + kStages - 1);
    const int par = (int)(i & 1), stage = (int)(i % kStages);
    const int64_t tile = first_pos(i);
    // borders touch this tile: a boundary at its rows or right behind its last one
    const int64_t edge = BWD ? row_of(tile + L - 1) : row_of(tile) + L;
    const bool marked = outside || tile + L > len || (BWD ? border >= edge : border <= edge);
    // what the slowest warp may still read of the tile before is kept: these alternate
    Mark *mark = s_mark + par * L;
    A *s_wa = s_maps + par * 2 * kScanWarps * C, *s_wb = s_wa + kScanWarps * C;
    int *s_wreset = s_resets[par];
    if (marked) {
      for (int j = tid; j < L; j += kScanThreads) {
        const int64_t pos = tile + j < len ? tile + j : len - 1;
        const int64_t t = row_of(pos);
        const int64_t u = BWD ? bound<true>(indptr, 0, cursor, t) : bound<true>(indptr, cursor, p.N + 1, t);
        Mark m{(int)(u - 1), 0};
        if (tile + j >= len) m.flags = kPad;
        else if (u < 1 || u > p.N) m.flags = kDead;
        else m.flags = (indptr[u - 1] == t ? kStart : 0) | (indptr[u] == t + 1 ? kEnd : 0);
        mark[j] = m;
        if (j == L - 1) {
          s_found[par][0] = u;
          s_found[par][1] = BWD ? (u > 0 ? indptr[u - 1] : -1) : (u <= p.N ? indptr[u] : (int64_t)1 << 62);
        }
      }
    }
    async_wait_all_but<kStages - 1>();
    if (marked) {
      __syncthreads();
      cursor = s_found[par][0];
      border = s_found[par][1];
      outside = cursor < 1 || cursor > p.N;
    }

    // ---- (1) the map of this thread's rows
    A ma[VEC], mb[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { ma[v] = 1; mb[v] = 0; }
    int reset = 0;
    const int64_t pos0 = tile + (int64_t)ty * R;
    const auto get_src = [&](int r, int64_t t) { return S::SrcSlot::get(slot(s_src, S::SrcSlot::kBytes, stage, r), src + t * p.K); };
    const auto get_gate = [&](int r, int64_t t) { return S::GateSlot::get(slot(s_gate, S::GateSlot::kBytes, stage, r), gate + t * gates); };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t t = row_of(pos0 + r);
      if (marked) {
        const Mark m = mark[ty * R + r];
        if (m.flags & kPad) continue;
        if (m.flags & kDead) {
          reset = 1;
#pragma unroll
          for (int v = 0; v < VEC; ++v) mb[v] = 0;
          continue;
        }
        if (m.flags & (BWD ? kEnd : kStart)) {
          reset = 1;
          if (live) load_acc<A, VEC>(mb, p.state, (srow + m.seg) * p.K + c0);
        }
      }
      const Pack<T, VEC> x = get_src(r, t);
      const Pack<G, S::kGateVec> g = get_gate(r, t);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const A gv = to_acc<G>(g.v[SHARED ? 0 : v]);
        const A xv = !BWD || p.src ? to_acc<T>(x.v[v]) : (A)0;
        mb[v] = BWD ? gv * (mb[v] + xv) : gv * mb[v] + xv;
        ma[v] *= gv;
      }
    }

    // ---- (2) scan of the maps over the warp, then over the warps and the cluster
    A ea[VEC], eb[VEC];  // map of the lanes before this one
    int ereset;
    {
      int ir = reset;
      for (int d = lx; d < 32; d <<= 1) {
        const int pr = __shfl_up_sync(kFullMask, ir, d);
        const bool take = lane >= d;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const A pa = shfl_up(ma[v], d), pb = shfl_up(mb[v], d);
          if (take && !ir) {
            mb[v] = apply_map(ma[v], mb[v], pb);
            ma[v] *= pa;
          }
        }
        if (take) ir |= pr;
      }
      reset = ir;
      ereset = __shfl_up_sync(kFullMask, ir, lx);
      const bool head = lane < lx || lx == 32;
      if (head) ereset = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        ea[v] = shfl_up(ma[v], lx);
        eb[v] = shfl_up(mb[v], lx);
        if (head) { ea[v] = 1; eb[v] = 0; }
      }
    }
    if (lane >= 32 - lx) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s_wa[warp * C + col * VEC + v] = ma[v];
        s_wb[warp * C + col * VEC + v] = mb[v];
      }
      if (lane == 31) s_wreset[warp] = reset;
    }
    __syncthreads();

    if (cs > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      int any = 0;
#pragma unroll
      for (int w = 0; w < kScanWarps; ++w) any |= s_wreset[w];
      for (int c = tid; c < C; c += kScanThreads) {
        A a = 1, bb = 0;
#pragma unroll
        for (int w = 0; w < kScanWarps; ++w) {
          const A wa = s_wa[w * C + c], wb = s_wb[w * C + c];
          bb = s_wreset[w] ? wb : apply_map(wa, wb, bb);
          a *= wa;
        }
        for (int q = 0; q < cs; ++q) {
          cluster.map_shared_rank(s_ca, q)[(par * cs + rank) * C + c] = a;
          cluster.map_shared_rank(s_cb, q)[(par * cs + rank) * C + c] = bb;
        }
      }
      if (tid < cs) cluster.map_shared_rank(&s_creset[0][0], tid)[par * kMostCluster + rank] = any;
      cluster.sync();
      for (int c = tid; c < C; c += kScanThreads) {
        A h = s_carry[c];
        for (int q = 0; q < cs; ++q) {
          if (q == rank) s_in[c] = h;
          const A a = s_ca[(par * cs + q) * C + c], bb = s_cb[(par * cs + q) * C + c];
          h = s_creset[par][q] ? bb : apply_map(a, bb, h);
        }
        s_carry[c] = h;
      }
    } else {
      for (int c = tid; c < C; c += kScanThreads) {
        A h = s_carry[c];
        s_in[c] = h;
#pragma unroll
        for (int w = 0; w < kScanWarps; ++w) {
          const A a = s_wa[w * C + c], bb = s_wb[w * C + c];
          h = s_wreset[w] ? bb : apply_map(a, bb, h);
        }
        s_carry[c] = h;
      }
    }
    __syncthreads();

    // ---- (3) the value that reaches this thread's rows, and the rows
    A h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = s_in[col * VEC + v];
    for (int w = 0; w < warp; ++w) {
      const int wr = s_wreset[w];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const A a = s_wa[w * C + col * VEC + v], bb = s_wb[w * C + col * VEC + v];
        h[v] = wr ? bb : apply_map(a, bb, h[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = ereset ? eb[v] : apply_map(ea[v], eb[v], h[v]);

#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t t = row_of(pos0 + r);
      Mark m{0, 0};
      if (marked) {
        m = mark[ty * R + r];
        if (m.flags & kPad) continue;
        if (m.flags & (BWD ? kEnd : kStart)) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) h[v] = 0;
          if (live) load_acc<A, VEC>(h, p.state, (srow + m.seg) * p.K + c0);
        }
      }
      const bool dead = marked && (m.flags & kDead);
      const Pack<T, VEC> x = get_src(r, t);
      const Pack<G, S::kGateVec> g = get_gate(r, t);
      Pack<T, VEC> o;
      if constexpr (!BWD) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          h[v] = dead ? (A)0 : to_acc<G>(g.v[SHARED ? 0 : v]) * h[v] + to_acc<T>(x.v[v]);
          o.v[v] = from_acc<T>(h[v]);
        }
        if (live) {
          st_stream<T, VEC>(out + t * p.K, o);
          if (marked && (m.flags & kEnd) && p.last) store_acc<A, VEC>(h, p.last, (srow + m.seg) * p.K + c0);
        }
      } else {
        A before[VEC], dg[VEC];
        if (p.grad_gate) {
          const Pack<T, VEC> f = S::SrcSlot::get(slot(s_fwd, S::SrcSlot::kBytes, stage, r), fwd + (t - 1) * p.K);
#pragma unroll
          for (int v = 0; v < VEC; ++v) before[v] = to_acc<T>(f.v[v]);
          if (marked && (m.flags & kStart)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) before[v] = 0;
            if (live) load_acc<A, VEC>(before, p.init, (srow + m.seg) * p.K + c0);
          }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const A dh = dead ? (A)0 : h[v] + (p.src ? to_acc<T>(x.v[v]) : (A)0);
          o.v[v] = from_acc<T>(dh);
          dg[v] = p.grad_gate && !dead ? dh * before[v] : (A)0;
          h[v] = dead ? (A)0 : to_acc<G>(g.v[SHARED ? 0 : v]) * dh;
        }
        if (live) {
          st_stream<T, VEC>(out + t * p.K, o);
          if (marked && (m.flags & kStart) && p.last) store_acc<A, VEC>(h, p.last, (srow + m.seg) * p.K + c0);
        }
        if (p.grad_gate) {
          if constexpr (!SHARED) {
            Pack<G, VEC> og;
#pragma unroll
            for (int v = 0; v < VEC; ++v) og.v[v] = from_acc<G>(dg[v]);
            if (live) st_stream<G, VEC>(static_cast<G *>(p.grad_gate) + (b * p.E + t) * gates + c0, og);
          } else {
            // sum of the thread's channels, then of the neighbouring lanes that hold the same gate; the lanes of a row
            // are in the same iteration together: rows are skipped (kPad) by whole rows
            A sum = dg[0];
#pragma unroll
            for (int v = 1; v < VEC; ++v) sum += dg[v];
            const unsigned rowmask = (lx == 32 ? kFullMask : ((1u << lx) - 1u) << (lane & ~(lx - 1)));
            for (int d = 1; d < (1 << p.lanes_log2); d <<= 1) sum += __shfl_xor_sync(rowmask, sum, d);
            if (live && (col & ((1 << p.lanes_log2) - 1)) == 0) {
              const int64_t per = VEC << p.lanes_log2;
              if (per == p.width) static_cast<G *>(p.grad_gate)[(b * p.E + t) * gates + g0] = from_acc<G>(sum);
              else static_cast<A *>(p.partial)[(b * p.E + t) * (p.K / per) + c0 / per] = sum;
            }
          }
        }
      }
    }
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
  return std::min(wide, ilog2_ceil((K + vec - 1) / vec));
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
  const int64_t tiles = (p.E + L - 1) / L, want = (int64_t)sm_count() * 3;
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
  cfg.blockDim = dim3(kScanThreads);
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
