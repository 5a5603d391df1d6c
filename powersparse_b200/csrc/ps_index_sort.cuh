// Stable counting sort of an index array by one thread block cluster, in one launch.
//
// The array is cut into consecutive strips, one a warp, over all blocks of the
// cluster.  A digit pass counts each strip's digits in shared memory (one row of
// counters a warp, so no atomics), turns the counts into the position of each
// strip's first element of each digit (a sum over the warps of the block, over the
// earlier blocks of the cluster through distributed shared memory, and over the
// smaller digits), and places every element: 32 elements at a time, in order, ranked
// among the lanes of equal digit.  Nothing depends on timing, so equal digits keep
// their order and two runs give the same result.
//
// Why one cluster: at the sizes of a batch (10^4 to 10^5 indices) the passes over the
// data are short, and launches and counters that go through memory between them are
// what costs.  The hardware's cluster barrier orders the passes (it also makes their
// global writes visible to the cluster), without a wait on memory.  A strip of up to
// kKeep * 32 elements stays in registers between counting and placing, its ranks with
// it; a longer one is walked twice.
#pragma once

#include <cooperative_groups.h>

#include <utility>

#include "ps_common.cuh"
#include "ps_rows.cuh"

namespace psb {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 10, kMaxDigits = 1 << kMaxBits;  // one thread a digit
constexpr int kKeep = 8;
constexpr int kSortBlocks = 16;    // the largest cluster there is (above 8 it needs an opt-in)

struct Strip {
  long long begin, end;  // of this warp
  long long length, n;   // of every strip but the last ones, and of all
};

// The strip of this warp: 32-element chunks in order, the same number for every warp.
__device__ __forceinline__ Strip warp_strip(long long n, int rank, int blocks) {
  const long long warps = (long long)blocks * kSortWarps;
  const long long len = ((n + warps - 1) / warps + 31) / 32 * 32;
  const long long b = (rank * (long long)kSortWarps + (threadIdx.x >> 5)) * len;
  return {b < n ? b : n, b + len < n ? b + len : n, len, n};
}

// row[d] of the lanes' digits d (-1: none) before this chunk of 32, plus the number of
// lower lanes of the same digit; row[d] is counted up.  The lanes of equal digit are
// found with a ballot for each of the digit's `bits`: __match_any_sync gives them in
// one call, but an SM answers one in 58 cycles (65536 indices, 64 digits: 15.0k cycles
// of a pass go into the ranks, 8.8k with ballots).
__device__ __forceinline__ uint32_t rank_chunk(uint32_t* row, int d, int bits) {
  const int lane = threadIdx.x & 31;
  unsigned same = __ballot_sync(0xffffffffu, d >= 0);
#pragma unroll
  for (int b = 0; b < kMaxBits; ++b) {
    if (b >= bits) break;
    const bool set = d & (1 << b);
    const unsigned with = __ballot_sync(0xffffffffu, set);
    same &= set ? with : ~with;
  }
  const uint32_t first = d >= 0 ? row[d] : 0u;
  __syncwarp();
  if (d >= 0 && lane == __ffs(same) - 1) row[d] = first + __popc(same);
  __syncwarp();
  return first + __popc(same & ((1u << lane) - 1u));
}

// Exclusive sums of two numbers over the block's threads; `scratch` holds kSortWarps pairs.
__device__ __forceinline__ uint2 warp_sums(uint2 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, v.x, d), y = __shfl_up_sync(0xffffffffu, v.y, d);
    if (lane >= d) {
      v.x += x;
      v.y += y;
    }
  }
  return v;
}
__device__ __forceinline__ uint2 block_sums_before(uint2 v, uint2* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint2 inc = warp_sums(v);
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  static_assert(kSortWarps == 32);
  if (warp == 0) {
    const uint2 w = scratch[lane], all = warp_sums(w);
    scratch[lane] = make_uint2(all.x - w.x, all.y - w.y);
  }
  __syncthreads();
  return make_uint2(scratch[warp].x + inc.x - v.x, scratch[warp].y + inc.y - v.y);
}

// Shared memory of a sort: kSortWarps rows of counters, two sets of block totals (one
// pass writes one while a slower block may still read the other), the digits' bases,
// the digits' first places among the block's staged elements, and scratch; then the
// staged elements.
struct SortShared {
  uint2* scratch;
  uint32_t *rows, *total, *base, *local;
  void* stage;
  __device__ SortShared(void* smem, int digits)
      : scratch(static_cast<uint2*>(smem)),
        rows(reinterpret_cast<uint32_t*>(scratch + kSortWarps)),
        total(rows + kSortWarps * digits),
        base(total + 2 * digits),
        local(base + digits),
        stage(local + digits) {}
};
inline size_t sort_smem(int digits) {
  static_assert((kSortWarps + 4) % 4 == 0, "the staged elements begin at a multiple of 16 bytes");
  return kSortWarps * sizeof(uint2) + sizeof(uint32_t) * (kSortWarps + 4) * size_t(digits);
}
// Bytes of the staged elements of n indices in `blocks` blocks (none where the strips are walked twice).
inline size_t stage_smem(long long n, int blocks, size_t element) {
  const long long strip = ceil_div_ll(ceil_div_ll(n, (long long)blocks * kSortWarps), 32) * 32;
  return strip <= kKeep * 32 ? size_t(strip) * kSortWarps * element : 0;
}

// One pass: place(i, element, p) for every element of the strip, p its position in the
// stable order by digit.  load(i) gives the element i, digit_of(element) its digit (-1:
// the element is not counted, and p means nothing).  widen(count) is the room that the
// elements of a digit take (at least count); report(d, begin, count) is called by one
// thread a digit in every block.  digits <= kMaxDigits.  kStage: elements that are kept
// are put in order in shared memory first and placed from there, so that a warp's
// places lie side by side: for elements that place() moves (8 bytes to scattered places
// leave an SM at one in 2.5 cycles: 50003 of them took 4 us a pass).  kLast: nothing follows that
// needs what the pass places; else it ends with the cluster's barrier, and `parity`
// alternates from pass to pass.
template <typename Element, bool kStage, bool kLast, typename Load, typename DigitOf, typename Widen, typename Report, typename Place>
__device__ __forceinline__ void sort_pass(SortShared sh, int digits, int parity, Strip strip, Load&& load, DigitOf&& digit_of,
                                          Widen&& widen, Report&& report, Place&& place) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int bits = 32 - __clz(digits - 1);
  uint32_t* row = sh.rows + warp * digits;
  for (int d = lane; d < digits; d += 32) row[d] = 0;
  __syncwarp();

  // Every warp's strip is as long, but for the last ones.
  const bool kept = strip.length <= kKeep * 32;
  const long long block_begin = min(strip.n, strip.length * kSortWarps * rank);
  const long long block_end = min(strip.n, block_begin + strip.length * kSortWarps);
  Element e[kKeep];
  uint32_t r[kKeep];
  for (long long base = strip.begin; base < strip.end; base += kKeep * 32) {
#pragma unroll
    for (int u = 0; u < kKeep; ++u) {
      const long long i = base + u * 32 + lane;
      if (i < strip.end) e[u] = load(i);
    }
#pragma unroll
    for (int u = 0; u < kKeep; ++u)
      if (base + u * 32 < strip.end) r[u] = rank_chunk(row, base + u * 32 + lane < strip.end ? digit_of(e[u]) : -1, bits);
  }
  __syncthreads();

  // Counts to positions within the block, a thread a digit.
  const int d = threadIdx.x;
  if (d < digits) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; w += 16) {
      uint32_t c[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) c[k] = sh.rows[(w + k) * digits + d];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        sh.rows[(w + k) * digits + d] = sum;
        sum += c[k];
      }
    }
    sh.total[parity * digits + d] = sum;
  }
  cluster.sync();

  uint32_t count = 0, earlier = 0, own = 0;
  if (d < digits) {
    own = sh.total[parity * digits + d];
    uint32_t c[kSortBlocks];  // all loads before their sum
#pragma unroll
    for (int b = 0; b < kSortBlocks; ++b) c[b] = b < blocks ? cluster.map_shared_rank(sh.total, b)[parity * digits + d] : 0u;
#pragma unroll
    for (int b = 0; b < kSortBlocks; ++b) {
      if (b < rank) earlier += c[b];
      count += c[b];
    }
  }
  // No block may end while another reads its totals: where no barrier follows at once,
  // its two halves stand apart.
  if (kLast) cluster.barrier_arrive();
  const uint2 begin = block_sums_before(make_uint2(d < digits ? widen(count) : 0u, own), sh.scratch);
  const bool staged = kStage && kept;
  if (d < digits) {
    report(d, begin.x, count);
    sh.base[d] = begin.x + earlier - (staged ? begin.y : 0u);
    if (staged) sh.local[d] = begin.y;
  }
  __syncthreads();

  if (staged) {
    auto* stage = static_cast<Element*>(sh.stage);
#pragma unroll
    for (int u = 0; u < kKeep; ++u)
      if (strip.begin + u * 32 + lane < strip.end) {
        const int digit = digit_of(e[u]);
        stage[sh.local[digit] + row[digit] + r[u]] = e[u];
      }
    __syncthreads();
    const int mine = int(block_end - block_begin);
    for (int i = threadIdx.x; i < mine; i += kSortThreads) {
      const Element element = stage[i];
      place(i, element, sh.base[digit_of(element)] + i);
    }
  } else if (kept) {
#pragma unroll
    for (int u = 0; u < kKeep; ++u) {
      const long long i = strip.begin + u * 32 + lane;
      if (i < strip.end) {
        const int digit = digit_of(e[u]);
        place(i, e[u], digit < 0 ? 0u : sh.base[digit] + row[digit] + r[u]);
      }
    }
  } else {
    for (long long base = strip.begin; base < strip.end; base += kKeep * 32) {
#pragma unroll
      for (int u = 0; u < kKeep; ++u) {
        const long long i = base + u * 32 + lane;
        if (i < strip.end) e[u] = load(i);
      }
#pragma unroll
      for (int u = 0; u < kKeep; ++u) {
        if (base + u * 32 >= strip.end) break;
        const long long i = base + u * 32 + lane;
        const int digit = i < strip.end ? digit_of(e[u]) : -1;
        const uint32_t p = rank_chunk(row, digit, bits);
        if (i < strip.end) place(i, e[u], digit < 0 ? 0u : sh.base[digit] + p);
      }
    }
  }
  if (!kLast) cluster.sync();
  else cluster.barrier_wait();
}

// Blocks of the cluster for n indices, more as the strips grow (16384 tokens in two
// passes: 23.7 us with 16, 25.0 with 8; 3000: 19.1 with 4, 19.3 with 8).  (For fewer the
// callers have kernels of their own, by kFewTokens and kFewSlots; wide rows alone come here.)
inline int sort_blocks(long long n) { return n <= 4096 ? 4 : n <= 8192 ? 8 : kSortBlocks; }

// As launch_after, with `clusters` clusters of `blocks` blocks of kSortThreads.
constexpr int kSortSmem = 220 << 10;  // what the most digits and the longest kept strips of 8-byte elements take, and some
template <auto kernel, typename... Args>
void launch_clusters(int blocks, long long clusters, size_t smem, cudaStream_t stream, Args... args) {
  static std::atomic<unsigned long long> prepared{0};  // devices on which the kernel may take its largest shared memory
  int device = 0;
  PSB_CUDA(cudaGetDevice(&device));
  const unsigned long long bit = device < 64 ? 1ULL << device : 0;
  if (!(prepared.load(std::memory_order_relaxed) & bit)) {
    PSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem));
    PSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    prepared.fetch_or(bit, std::memory_order_relaxed);
  }
  if (clusters * blocks > 0x7fffffffLL) throw std::invalid_argument("too many rows for one launch");
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(clusters * blocks));
  config.blockDim = dim3(kSortThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 2;
  PSB_CUDA(cudaLaunchKernelEx(&config, kernel, args...));
}

}  // namespace psb
