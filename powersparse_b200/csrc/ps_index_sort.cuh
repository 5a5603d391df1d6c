// Stable counting sort of an index array by one thread block cluster, in one launch.
//
// The array is cut into consecutive strips, one a warp, over all blocks of the
// cluster.  A digit pass counts each strip's digits in shared memory (one row of
// counters a warp, so no atomics), turns the counts into the position of each
// strip's first element of each digit (a sum over the warps of the block, over the
// earlier blocks of the cluster through distributed shared memory, and over the
// smaller digits), and walks the strips again to place every element: 32 elements at
// a time, in order, ranked among the lanes of equal digit.  Nothing depends on
// timing, so equal keys keep their order and two runs give the same result.
//
// Why one cluster: at the sizes of a batch (10^4 to 10^5 indices) the passes over the
// data are short and the launches and the counters' round trips through memory between
// them are what costs.  The hardware's cluster barrier orders the passes (it also
// makes their global writes visible to the cluster), without a wait on memory.
#pragma once

#include <cooperative_groups.h>

#include "ps_common.cuh"

namespace psb {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortUnroll = 8;  // loads in flight a lane

struct Strip {
  long long begin, end;
};

// The strip of this warp: 32-element chunks in order, the same number for every warp.
__device__ __forceinline__ Strip warp_strip(long long n, int rank, int blocks) {
  const long long warps = (long long)blocks * kSortWarps;
  const long long len = ((n + warps - 1) / warps + 31) / 32 * 32;
  const long long b = (rank * (long long)kSortWarps + (threadIdx.x >> 5)) * len;
  return {b < n ? b : n, b + len < n ? b + len : n};
}

// row[d] += elements of the strip with digit d (digit(i) < 0: not counted).
template <typename Digit>
__device__ __forceinline__ void count_digits(Strip s, uint32_t* row, Digit&& digit) {
  const int lane = threadIdx.x & 31;
  for (long long base = s.begin; base < s.end; base += 32 * kSortUnroll) {
    int d[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const long long i = base + u * 32 + lane;
      d[u] = i < s.end ? digit(i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const unsigned same = __match_any_sync(0xffffffffu, d[u]);
      if (d[u] >= 0 && lane == __ffs(same) - 1) row[d[u]] += __popc(same);
      __syncwarp();
    }
  }
}

// place(i, p) for every element of the strip: p = row[digit] counted up in order
// (p is not meaningful where digit(i) < 0).
template <typename Digit, typename Place>
__device__ __forceinline__ void place_digits(Strip s, uint32_t* row, Digit&& digit, Place&& place) {
  const int lane = threadIdx.x & 31;
  for (long long base = s.begin; base < s.end; base += 32 * kSortUnroll) {
    int d[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const long long i = base + u * 32 + lane;
      d[u] = i < s.end ? digit(i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const unsigned same = __match_any_sync(0xffffffffu, d[u]);
      const uint32_t first = d[u] >= 0 ? row[d[u]] : 0u;
      __syncwarp();
      if (d[u] >= 0 && lane == __ffs(same) - 1) row[d[u]] = first + __popc(same);
      __syncwarp();
      const long long i = base + u * 32 + lane;
      if (i < s.end) place(i, d[u], first + __popc(same & ((1u << lane) - 1u)));
    }
  }
}

// Exclusive sum over the block's threads; `scratch` holds kSortWarps words.
__device__ __forceinline__ uint32_t block_sum_before(uint32_t v, uint32_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    uint32_t w = lane < kSortWarps ? scratch[lane] : 0u, winc = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, winc, d);
      if (lane >= d) winc += o;
    }
    if (lane < kSortWarps) scratch[lane] = winc - w;
  }
  __syncthreads();
  const uint32_t before = scratch[warp] + inc - v;
  __syncthreads();
  return before;
}

// Shared memory of a pass: kSortWarps rows of `digits` counters, the block's totals and scratch.
inline size_t sort_smem(int digits) { return sizeof(uint32_t) * (size_t(kSortWarps) * digits + digits + kSortWarps); }

struct SortShared {
  uint32_t* rows;     // [kSortWarps][digits]
  uint32_t* total;    // [digits]: this block's count of each digit
  uint32_t* scratch;  // [kSortWarps]
  __device__ SortShared(uint32_t* smem, int digits)
      : rows(smem), total(smem + kSortWarps * digits), scratch(total + digits) {}
};

// One digit pass up to the counters: afterwards sh.rows[w][d] is the position of the
// first element with digit d of warp w's strip.  `widen(count)` is the room that the
// elements of a digit take (at least count); `report(d, begin, count)` is called by
// one thread a digit in every block.  digits <= kSortThreads.
template <typename Digit, typename Widen, typename Report>
__device__ __forceinline__ void digit_positions(SortShared sh, int digits, Strip strip, Digit&& digit, Widen&& widen,
                                                Report&& report) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  for (int i = threadIdx.x; i < kSortWarps * digits; i += kSortThreads) sh.rows[i] = 0;
  __syncthreads();
  count_digits(strip, sh.rows + (threadIdx.x >> 5) * digits, digit);
  __syncthreads();
  const int d = threadIdx.x;
  if (d < digits) {
    uint32_t sum = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = sh.rows[w * digits + d];
      sh.rows[w * digits + d] = sum;
      sum += c;
    }
    sh.total[d] = sum;
  }
  cluster.sync();
  uint32_t count = 0, earlier = 0;
  if (d < digits) {
    for (int b = 0; b < blocks; ++b) {
      const uint32_t c = cluster.map_shared_rank(sh.total, b)[d];
      if (b < rank) earlier += c;
      count += c;
    }
  }
  cluster.sync();  // the totals have been read: a later pass may write them, a block may end
  const uint32_t begin = block_sum_before(d < digits ? widen(count) : 0u, sh.scratch);
  if (d < digits) {
    report(d, begin, count);
    for (int w = 0; w < kSortWarps; ++w) sh.rows[w * digits + d] += begin + earlier;
  }
  __syncthreads();
}

// Blocks of the cluster for n indices: one while a block's warps each have one short
// strip, more as the strips grow (8 is the largest cluster that every sm_100 GPU takes).
inline int sort_blocks(long long n) { return n <= 2048 ? 1 : n <= 8192 ? 4 : 8; }

template <typename... Params, typename... Args>
void launch_cluster(void (*kernel)(Params...), int blocks, size_t smem, cudaStream_t stream, Args&&... args) {
  PSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(kSortThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  PSB_CUDA(cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...));
}

}  // namespace psb
