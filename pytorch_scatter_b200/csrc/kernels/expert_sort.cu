// Tokens sorted by expert: a stable counting sort of n entries over E experts.
//
// Every block owns a contiguous chunk of entries, every warp of it a contiguous part of the chunk.  (1) each block counts
// its entries per expert; (2) one block turns the counts, expert by expert and block by block inside an expert, into the
// first place of each (expert, block); (3) each block counts again per warp and hands out places in entry order, the
// rank inside 32 entries coming from a match of the expert ids.  Nothing depends on the order in which blocks run.
#include "common.cuh"

namespace tsb {
namespace {

constexpr int kSortWarps = 8;
constexpr int kSortPerWarp = 512;                         // entries of a warp
constexpr int kSortChunk = kSortWarps * kSortPerWarp;     // entries of a block
constexpr int64_t kSortMostExperts = 4096;

// experts 0 .. E-1, and one more bucket E for entries that name none
__device__ __forceinline__ int bucket_of(int64_t e, int E) { return e >= 0 && e < E ? (int)e : E; }

__global__ void __launch_bounds__(kSortWarps * 32) sort_count_kernel(const int64_t *__restrict__ index, int *__restrict__ counts,
                                                                     int64_t n, int E, int blocks) {
  extern __shared__ int s_count[];
  for (int e = threadIdx.x; e <= E; e += blockDim.x) s_count[e] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * kSortChunk;
  for (int i = threadIdx.x; i < kSortChunk; i += blockDim.x)
    if (lo + i < n) atomicAdd(&s_count[bucket_of(index[lo + i], E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) counts[(int64_t)e * blocks + blockIdx.x] = s_count[e];
}

// counts [E+1][blocks] -> exclusive prefix sums in place; indptr
__global__ void __launch_bounds__(1024) sort_prefix_kernel(int *__restrict__ counts, int64_t *__restrict__ indptr, int E, int blocks) {
  __shared__ int s_warp[32];
  const int64_t total = (int64_t)(E + 1) * blocks;
  const int64_t per = (total + 1023) / 1024;
  const int64_t lo = min((int64_t)threadIdx.x * per, total), hi = min(lo + per, total);
  int sum = 0;
  for (int64_t i = lo; i < hi; ++i) sum += counts[i];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = sum;
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(kFullMask, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int run = incl - sum;
  for (int w = 0; w < warp; ++w) run += s_warp[w];
  for (int64_t i = lo; i < hi; ++i) {
    const int c = counts[i];
    counts[i] = run;
    if (i % blocks == 0) indptr[i / blocks] = run;
    run += c;
  }
}

__global__ void __launch_bounds__(kSortWarps * 32)
sort_place_kernel(const int64_t *__restrict__ index, const int *__restrict__ first, int64_t *__restrict__ slot,
                  int64_t *__restrict__ order, int64_t n, int E, int blocks) {
  extern __shared__ int s_place[];  // [warps][E+1]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < kSortWarps * (E + 1); e += blockDim.x) s_place[e] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * kSortChunk + warp * kSortPerWarp;
  int *mine = s_place + warp * (E + 1);
  for (int i = lane; i < kSortPerWarp; i += 32)
    if (lo + i < n) atomicAdd(&mine[bucket_of(index[lo + i], E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    int run = first[(int64_t)e * blocks + blockIdx.x];
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = s_place[w * (E + 1) + e];
      s_place[w * (E + 1) + e] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int i = lane; i < kSortPerWarp; i += 32) {
    const bool in = lo + i < n;
    const unsigned active = __ballot_sync(kFullMask, in);
    if (in) {
      const int e = bucket_of(index[lo + i], E);
      const unsigned peers = __match_any_sync(active, e);
      const int place = mine[e] + __popc(peers & ((1u << lane) - 1u));
      __syncwarp(active);
      if ((peers >> lane) == 1u) mine[e] = place + 1;  // the last of the peers
      slot[lo + i] = e < E ? place : -1;
      order[place] = lo + i;
    }
    __syncwarp();
  }
}

int64_t sort_blocks(int64_t n) { return (n + kSortChunk - 1) / kSortChunk; }

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" size_t tsb_expert_sort_workspace_bytes(int64_t n, int64_t E) {
  if (n < 0 || E < 0) return 0;
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
  if (!workspace || workspace_bytes < tsb_expert_sort_workspace_bytes(n, E)) return TSB_ERR_WORKSPACE;
  const int blocks = (int)sort_blocks(n);
  int *counts = static_cast<int *>(workspace);
  const size_t one = sizeof(int) * (E + 1), all = one * kSortWarps;
  if (all > 48 * 1024 &&
      cudaFuncSetAttribute(sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)all) != cudaSuccess)
    return TSB_ERR_LAUNCH;
  sort_count_kernel<<<blocks, kSortWarps * 32, one, st>>>(index, counts, n, (int)E, blocks);
  sort_prefix_kernel<<<1, 1024, 0, st>>>(counts, indptr, (int)E, blocks);
  sort_place_kernel<<<blocks, kSortWarps * 32, all, st>>>(index, counts, slot, order, n, (int)E, blocks);
  return launch_status();
}
