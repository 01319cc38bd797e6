// Tokens sorted by expert: a stable counting sort of n entries over E experts.
//
// Every block owns a contiguous range of entries, every warp of it a contiguous part of that.  (1) Each block counts its
// entries per expert.  (2) Each block adds up the counts of all blocks, which gives the first place of every expert and
// its own first place inside it, counts again per warp, and hands out places in entry order, the rank inside 32 entries
// coming from a match of the expert ids.  Up to kOneBlock entries one block does without (1).  Nothing depends on the
// order in which blocks run, and no float is involved.
//
// 2,097,152 entries over 256 experts take 37 us; the 24 bytes of each entry, read and written once, would take 8.  The
// placing kernel is the larger part: its warps wait for shared memory (the counting atomics, the matches' counters) twice as
// long as for the index and the counts of all blocks.  Below some 100,000 entries the two launches and the latency of the
// counts bound it (8192 entries: 12 us).
#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace tsb {
namespace {

constexpr int kSortThreads = 1024;
constexpr int64_t kOneBlock = 8192;          // entries
constexpr int64_t kSortMostExperts = 4096;
constexpr int kCountInts = 48 * 1024;        // shared memory for the counts of the warps
constexpr int kBatch = 8;                    // index loads in flight of a warp, 32 entries each

// experts 0 .. E-1, and one more bucket E for entries that name none
__device__ __forceinline__ int bucket_of(int64_t e, int E) { return e >= 0 && e < E ? (int)e : E; }

// The entries of a warp, 32 at a time and in order: f(first entry of the 32, bucket of this lane's, -1 behind the end)
template <typename F> __device__ __forceinline__ void each_entry(const int64_t *__restrict__ index, int64_t lo, int64_t hi, int E, F f) {
  const int lane = threadIdx.x & 31;
  for (int64_t i0 = lo; i0 < hi; i0 += 32 * kBatch) {
    int64_t e[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t i = i0 + b * 32 + lane;
      e[b] = i < hi ? index[i] : 0;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t i = i0 + b * 32;
      if (i >= hi) break;
      f(i, i + lane < hi ? bucket_of(e[b], E) : -1);
    }
  }
}

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const int64_t *__restrict__ index, int *__restrict__ counts, int64_t n, int E, int64_t per_block) {
  extern __shared__ int s_count[];
  for (int e = threadIdx.x; e <= E; e += blockDim.x) s_count[e] = 0;
  __syncthreads();
  const int64_t lo = min(blockIdx.x * per_block, n), hi = min(lo + per_block, n);
  const int64_t part = (hi - lo + blockDim.x / 32 - 1) / (blockDim.x / 32), wlo = lo + (threadIdx.x >> 5) * part;
  each_entry(index, min(wlo, hi), min(wlo + part, hi), E, [&](int64_t, int e) {
    if (e >= 0) atomicAdd(&s_count[e], 1);
  });
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) counts[(int64_t)blockIdx.x * (E + 1) + e] = s_count[e];
}

// shared: [E+1] first places, [warps][E+1] counts of the warps, later their next places
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const int64_t *__restrict__ index, const int *__restrict__ counts, int64_t *__restrict__ slot,
                  int64_t *__restrict__ order, int64_t *__restrict__ indptr, int64_t n, int E, int64_t per_block, int warps) {
  extern __shared__ int s_all[];
  __shared__ int s_sum[32];
  int *s_first = s_all, *s_warp = s_all + (E + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = gridDim.x;
  // the first `warps` warps carry entries; the experts are spread over all threads
  int *mine = s_warp + warp * (E + 1);
  for (int i = threadIdx.x; i < warps * (E + 1); i += blockDim.x) s_warp[i] = 0;
  __syncthreads();
  const int64_t lo = min(blockIdx.x * per_block, n), hi = min(lo + per_block, n);
  const int64_t part = (hi - lo + warps - 1) / warps, wlo = warp < warps ? min(lo + warp * part, hi) : hi, whi = min(wlo + part, hi);
  each_entry(index, wlo, whi, E, [&](int64_t, int e) {
    if (e >= 0) atomicAdd(&mine[e], 1);
  });

  // entries of each expert before this block and in all blocks
  constexpr int kMine = (kSortMostExperts + kSortThreads) / kSortThreads;  // experts of a thread
  int before[kMine] = {}, total[kMine] = {};
  if (counts) {
    // several threads share an expert's column where there are more threads than experts
    const int groups = max(1, (int)blockDim.x / (E + 1));
    if (groups > 1) {
      int *s_part = s_first;  // [E+1] x (before, all) by atomics: integers, any order gives the same sums
      __shared__ int s_before[kSortThreads];
      for (int e = threadIdx.x; e <= E; e += blockDim.x) s_part[e] = s_before[e] = 0;
      __syncthreads();
      const int e = threadIdx.x % (E + 1), g = threadIdx.x / (E + 1);
      if (g < groups) {
        int all = 0, bef = 0;
#pragma unroll 8
        for (int b = g; b < blocks; b += groups) {
          const int c = counts[(int64_t)b * (E + 1) + e];
          all += c;
          bef += b < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(&s_part[e], all);
        atomicAdd(&s_before[e], bef);
      }
      __syncthreads();
      if (threadIdx.x <= E) {
        total[0] = s_part[threadIdx.x];
        before[0] = s_before[threadIdx.x];
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int q = 0; q < kMine; ++q) {
        const int e = q * blockDim.x + threadIdx.x;
        if (e > E) break;
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) {
          const int c = counts[(int64_t)b * (E + 1) + e];
          total[q] += c;
          before[q] += b < (int)blockIdx.x ? c : 0;
        }
      }
    }
    __syncthreads();
  } else {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int e = q * blockDim.x + threadIdx.x;
      if (e > E) break;
      for (int w = 0; w < warps; ++w) total[q] += s_warp[w * (E + 1) + e];
    }
  }

  // first place of each expert: prefix sums of the totals, a row of threads after the other
  int run = 0;
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    if (q * (int)blockDim.x > E) break;
    int incl = total[q];
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(kFullMask, incl, d);
      if (lane >= d) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int add = run;
    for (int w = 0; w < (int)blockDim.x >> 5; ++w) {
      if (w < warp) add += s_sum[w];
      run += s_sum[w];
    }
    const int e = q * blockDim.x + threadIdx.x;
    if (e <= E) {
      int place = add + incl - total[q];
      if (blockIdx.x == 0) indptr[e] = place;
      place += before[q];
      for (int w = 0; w < warps; ++w) {
        const int c = s_warp[w * (E + 1) + e];
        s_warp[w * (E + 1) + e] = place;
        place += c;
      }
    }
    __syncthreads();
  }

  each_entry(index, wlo, whi, E, [&](int64_t i, int e) {
    const unsigned peers = __match_any_sync(kFullMask, e);
    int place = 0;
    if (e >= 0) place = mine[e] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0) {
      if ((peers >> lane) == 1u) mine[e] = place + 1;  // the last of the peers
      slot[i + lane] = e < E ? place : -1;
      order[place] = i + lane;
    }
    __syncwarp();
  });
}

// blocks and the entries of each: one block for few entries, else a multiple of what keeps every SM busy
int64_t sort_blocks(int64_t n) { return n <= kOneBlock ? 1 : std::min<int64_t>(148, (n + 2047) / 2048); }

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" size_t tsb_expert_sort_workspace_bytes(int64_t n, int64_t E) {
  if (n < 0 || E < 0 || n <= kOneBlock) return 0;
  const size_t bytes = sizeof(int) * (size_t)(E + 1) * (size_t)sort_blocks(n);
  return (bytes + 255) / 256 * 256;
}

extern "C" int tsb_expert_sort(const int64_t *index, int64_t *slot, int64_t *order, int64_t *indptr, int64_t n, int64_t E,
                               void *workspace, size_t workspace_bytes, tsb_stream_t stream) {
  if (n < 0 || E < 1 || !indptr) return TSB_ERR_ARG;
  if (n >= 2147483647LL || E > kSortMostExperts) return TSB_ERR_TOO_LARGE;
  cudaStream_t st = (cudaStream_t)stream;
  if (n == 0) return cudaMemsetAsync(indptr, 0, sizeof(int64_t) * (E + 1), st) == cudaSuccess ? TSB_OK : TSB_ERR_LAUNCH;
  if (!index || !slot || !order) return TSB_ERR_ARG;
  if (n > kOneBlock && (!workspace || workspace_bytes < tsb_expert_sort_workspace_bytes(n, E))) return TSB_ERR_WORKSPACE;
  static std::atomic<bool> allowed[64];  // per device; setting the attribute twice is harmless
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TSB_ERR_LAUNCH;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kCountInts + (int)kSortMostExperts + 1) * (int)sizeof(int)) != cudaSuccess)
      return TSB_ERR_LAUNCH;
    allowed[dev] = true;
  }
  const int64_t blocks = sort_blocks(n), per_block = (n + blocks - 1) / blocks;
  // warps: one for each 32 entries, as many as their counts leave room for (11 with 4096 experts)
  const int64_t warps = std::max<int64_t>(1, std::min<int64_t>({32, (per_block + 31) / 32, (int64_t)kCountInts / (E + 1)}));
  int *counts = blocks > 1 ? static_cast<int *>(workspace) : nullptr;
  const size_t one = sizeof(int) * (E + 1);
  if (counts) sort_count_kernel<<<(unsigned)blocks, kSortThreads, one, st>>>(index, counts, n, (int)E, per_block);
  const int64_t threads = std::max<int64_t>(warps * 32, std::min<int64_t>(kSortThreads, (E + 32) / 32 * 32));
  sort_place_kernel<<<(unsigned)blocks, (unsigned)threads, one * (warps + 1), st>>>(index, counts, slot, order, indptr, n, (int)E, per_block, (int)warps);
  return launch_status();
}
