// The plan of a ragged product: a stable counting sort of the router's assignments by expert.
#include <algorithm>

#include "common.h"

namespace pulsar {

namespace {

constexpr int kGroupMaxE = 1024, kGroupThreads = 1024, kGroupWaves = kGroupThreads / 64;
// Assignments up to which one workgroup sorts alone: 1024 take it 4.3 us, 4096 8.9; counting and
// placing in two launches takes 6.8 at 4096 and 7.0 at 65536.
constexpr int64_t kGroupOneBlock = 2048;
constexpr int kGroupBlocks = 256;

// Assignments per workgroup, a multiple of its threads: 1024 until the launch has 256.
__host__ __device__ inline int64_t group_chunk(int64_t M) {
  const int64_t c = (M + kGroupBlocks - 1) / kGroupBlocks;
  return (c + kGroupThreads - 1) / kGroupThreads * kGroupThreads;
}

// The expert of an id, -1 for ids that name none.
__device__ __forceinline__ int group_expert(int64_t id, int E) {
  return id >= 0 && id < E ? (int)id : -1;
}

// counts[block][e]: the block's assignments of each expert.
__global__ void __launch_bounds__(kGroupThreads) group_count_kernel(const int64_t* ids, int* counts,
                                                                    int64_t M, int E) {
  __shared__ int hist[kGroupMaxE];
  const int tid = threadIdx.x;
  if (tid < E) hist[tid] = 0;
  __syncthreads();
  const int64_t chunk = group_chunk(M), i0 = blockIdx.x * chunk, i1 = min(M, i0 + chunk);
  for (int64_t i = i0 + tid; i < i1; i += kGroupThreads) {
    const int e = group_expert(ids[i], E);
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  if (tid < E) counts[(int64_t)blockIdx.x * E + tid] = hist[tid];
}

// Slots, rows and offsets. Every workgroup sums the counts of all of them (integers: any order
// gives the same), which yields each expert's start and how many of its assignments lie before
// the workgroup's own; it then ranks its assignments round by round of 1024, 64 at a time
// within a wave by comparing expert bits across lanes. ONE: a single workgroup counts itself.
// 4 assignments take 3.2 us, 65536 of 16 experts 2.6 us of counting and 5.1 here: launches and
// barriers, the 1 MB moved is 0.2 us.
template <bool ONE>
__global__ void __launch_bounds__(kGroupThreads) group_place_kernel(
    const int64_t* ids, const int* counts, int* offsets, int* rows, int* slots, int64_t M, int E,
    int K) {
  __shared__ int total[kGroupMaxE], next[kGroupMaxE], wave_sums[kGroupWaves];
  extern __shared__ int seen[];  // [waves][E]: a round's assignments of each wave, then their starts
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (tid < E) total[tid] = next[tid] = 0;
  __syncthreads();
  const int64_t chunk = ONE ? M : group_chunk(M);
  const int64_t i0 = blockIdx.x * chunk, i1 = min(M, i0 + chunk);
  if constexpr (ONE) {
    for (int64_t i = tid; i < M; i += kGroupThreads) {
      const int e = group_expert(ids[i], E);
      if (e >= 0) atomicAdd(&total[e], 1);
    }
  } else {
    const int n = (int)gridDim.x * E, own = (int)blockIdx.x * E;
    for (int k = tid; k < n; k += kGroupThreads) {
      const int v = counts[k], e = k % E;
      if (v) {
        atomicAdd(&total[e], v);
        if (k < own) atomicAdd(&next[e], v);
      }
    }
  }
  __syncthreads();
  // exclusive scan of the totals: thread e holds expert e
  const int t = tid < E ? total[tid] : 0;
  int incl = t;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(incl, d, 64);
    if (lane >= d) incl += v;
  }
  if (lane == 63) wave_sums[w] = incl;
  __syncthreads();
  int all = 0;
  for (int i = 0; i < kGroupWaves; ++i) {
    if (i == w) incl += all;
    all += wave_sums[i];
  }
  if (tid < E) {
    next[tid] += incl - t;
    if (blockIdx.x == 0) {
      offsets[tid] = incl - t;
      if (tid == E - 1) offsets[E] = all;
    }
  }
  const int bits = 32 - __clz(E);  // of the values 0 .. E
  for (int64_t r = i0; r < i1; r += kGroupThreads) {
    for (int k = tid; k < kGroupWaves * E; k += kGroupThreads) seen[k] = 0;
    __syncthreads();
    const int64_t i = r + tid;
    const int e = i < i1 ? group_expert(ids[i], E) : -1;
    // lanes of the wave with this lane's expert (E stands for none)
    uint64_t same = ~0ull;
    const int key = e < 0 ? E : e;
    for (int b = 0; b < bits; ++b) {
      const uint64_t m = __ballot(key >> b & 1);
      same &= key >> b & 1 ? m : ~m;
    }
    const int rank = (int)__popcll(same & ((1ull << lane) - 1));
    if (e >= 0 && rank == 0) seen[w * E + e] = (int)__popcll(same);
    __syncthreads();
    if (tid < E) {
      int s = next[tid];
      for (int k = 0; k < kGroupWaves; ++k) {
        const int c = seen[k * E + tid];
        seen[k * E + tid] = s;
        s += c;
      }
      next[tid] = s;
    }
    __syncthreads();
    if (i < i1) {
      const int slot = e >= 0 ? seen[w * E + e] + rank : -1;
      slots[i] = slot;
      if (slot >= 0) rows[slot] = (int)(i / K);
      if (i >= all) rows[i] = -1;  // rows of no expert: no assignment is placed there
    }
    __syncthreads();
  }
}

}  // namespace

}  // namespace pulsar

using namespace pulsar;

extern "C" {

int64_t pulsar_moe_group_rows_workspace_bytes(int64_t N, int64_t K, int64_t E) {
  if (N < 0 || K < 1 || E < 1 || E > kGroupMaxE || N > 0x7fffff00 / K) return -1;
  const int64_t M = N * K;
  if (M <= kGroupOneBlock) return 0;
  const int64_t chunk = group_chunk(M);
  return (M + chunk - 1) / chunk * E * 4;
}

int pulsar_moe_group_rows(const int64_t* topk_idx, int32_t* offsets, int32_t* rows, int32_t* slots,
                          int64_t N, int64_t K, int64_t E, void* workspace, hipStream_t stream) {
  const int64_t bytes = pulsar_moe_group_rows_workspace_bytes(N, K, E);
  PULSAR_REQUIRE(bytes >= 0, "moe_group_rows: bad shape (1 <= E <= 1024, K >= 1, N K < 2^31)");
  const int64_t M = N * K;
  PULSAR_REQUIRE(offsets && (M == 0 || (topk_idx && rows && slots)), "moe_group_rows: null pointer");
  PULSAR_REQUIRE(bytes == 0 || workspace, "moe_group_rows: workspace missing");
  const size_t lds = (size_t)kGroupWaves * E * 4;
  if (bytes == 0) {
    group_place_kernel<true><<<1, kGroupThreads, lds, stream>>>(topk_idx, nullptr, offsets, rows,
                                                                slots, M, (int)E, (int)K);
    PULSAR_LAUNCH_CHECK();
    return PULSAR_OK;
  }
  const int64_t chunk = group_chunk(M);
  const unsigned grid = (unsigned)((M + chunk - 1) / chunk);
  int* counts = static_cast<int*>(workspace);
  group_count_kernel<<<grid, kGroupThreads, 0, stream>>>(topk_idx, counts, M, (int)E);
  PULSAR_LAUNCH_CHECK();
  group_place_kernel<false><<<grid, kGroupThreads, lds, stream>>>(topk_idx, counts, offsets, rows,
                                                                  slots, M, (int)E, (int)K);
  PULSAR_LAUNCH_CHECK();
  return PULSAR_OK;
}

}  // extern "C"
