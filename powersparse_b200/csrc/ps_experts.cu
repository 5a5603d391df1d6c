// A mixture layer's index operators: the router's softmax and top-k, the tokens'
// rows in the order of their experts, the experts' rows back with their weights, and
// the gradients of all three.
//
// With the slot (t, j) of token t's j-th expert and its row position(t, j) in expert
// order:
//
//   dispatch      rows[position(t, j), :] = x[t, :]
//   combine       out[t, :] = add[t, :] + sum_j w[t, j] * y[position(t, j), :]
//   combine_grad  grad_y[position(t, j), :] = w[t, j] * g[t, :]
//                 grad_w[t, j] = <g[t, :], y[position(t, j), :]>
//
// combine is the SpMM of the matrix with w[t, j] at (t, position(t, j)), the gradient
// of its values is that matrix's SDDMM, and dispatch is the transposed SpMM of ones;
// the matrix is new in every call and has at most top_k elements a row and one a
// column, so every kernel here walks tokens and no sum needs atomics.
#include "ps_index_sort.cuh"
#include "ps_rows.cuh"

namespace psb {
namespace {

// ---- router -----------------------------------------------------------------------
// A warp a token, E / 32 scores a lane in registers.  Scores compare as integers that
// keep the order of the numbers (-0 as +0); of equal scores the lowest index comes
// first.  A score of -inf switches an expert off: it is never chosen.
constexpr int kRouteWarps = 8;

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T, int V>
__device__ __forceinline__ void load_scores(const T* row, int experts, float (&x)[V]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 32 + lane;
    x[v] = e < experts ? to_float(row[e]) : -INFINITY;
  }
}

// Largest score of the row (0 where all are -inf, so that x - max is not NaN), and
// the sum of exp(x - max) over the row.
template <int V>
__device__ __forceinline__ void row_softmax(const float (&x)[V], float& top, float& sum) {
  top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) top = fmaxf(top, x[v]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (top == -INFINITY) top = 0.f;
  sum = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) sum += expf(x[v] - top);
  sum = warp_sum(sum);
}

// The top_k largest of a warp's keys (0: never taken), ranked: take(r, key, index) is
// called by one lane for every rank r that there is; returns their number.
//
// The k-th largest of the 32 lanes' own maxima is a bound that at least k keys reach,
// and rarely many more do: those are gathered in shared memory and each lane ranks one
// of them among all.  Where more than 32 reach it (equal scores), the keys are taken
// one by one instead, as they are for few choices, where that is faster.
constexpr int kTakeOneByOne = 3;

template <int V, typename Take>
__device__ __forceinline__ int top_keys(uint32_t (&key)[V], int top_k, uint2* room, Take&& take) {
  const int lane = threadIdx.x & 31;
  uint32_t best = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) best = max(best, key[v]);
  if (top_k > kTakeOneByOne) {
    uint32_t sorted = best;  // bitonic, largest first
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
      for (int stride = size / 2; stride > 0; stride /= 2) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, sorted, stride);
        const bool larger = ((lane & stride) == 0) == ((lane & size) == 0);
        sorted = larger ? max(sorted, other) : min(sorted, other);
      }
    const uint32_t bound = max(1u, __shfl_sync(0xffffffffu, sorted, top_k - 1));
    int found = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const unsigned reach = __ballot_sync(0xffffffffu, key[v] >= bound);
      const int slot = found + __popc(reach & ((1u << lane) - 1u));
      if (key[v] >= bound && slot < 32) room[slot] = make_uint2(key[v], v * 32 + lane);
      found += __popc(reach);
    }
    if (found <= 32) {
      __syncwarp();
      const uint2 mine = lane < found ? room[lane] : make_uint2(0, 0);
      int rank = 0;  // the slots ascend with the index: of equal keys the lower slot first
      for (int i = 0; i < found; ++i) {
        const uint32_t other = room[i].x;
        rank += other > mine.x || (other == mine.x && i < lane);
      }
      if (lane < found && rank < top_k) take(rank, mine.x, int(mine.y));
      return min(found, top_k);
    }
  }
  for (int j = 0; j < top_k; ++j) {
    const uint32_t largest = __reduce_max_sync(0xffffffffu, best);
    if (largest == 0) return j;
    int at = 0x7fffffff;
#pragma unroll
    for (int v = V - 1; v >= 0; --v)
      if (key[v] == largest) at = v * 32 + lane;
    const int first = __reduce_min_sync(0xffffffffu, at);
    best = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (first == v * 32 + lane) key[v] = 0;
      best = max(best, key[v]);
    }
    if (at == first) take(j, largest, first);
  }
  return top_k;
}

__device__ __forceinline__ float unordered(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) route_tokens(const T* __restrict__ logits, long long stride, int tokens,
                                                                 int experts, int top_k, bool normalize,
                                                                 float* __restrict__ weights, int* __restrict__ chosen) {
  __shared__ uint2 room[kRouteWarps][32];
  __shared__ float taken[kRouteWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = blockIdx.x * (long long)kRouteWarps + warp;
  if (t >= tokens) return;
  float x[V];
  load_scores<T, V>(logits + t * stride, experts, x);
  float top = 0.f, sum = 0.f;
  if (!normalize) row_softmax<V>(x, top, sum);
  bool nan = false;
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    nan = nan || x[v] != x[v];
    key[v] = x[v] > -INFINITY ? ordered(x[v]) : 0u;  // a NaN compares false
  }
  nan = __any_sync(0xffffffffu, nan);
  const int found = top_keys<V>(key, top_k, room[warp], [&](int r, uint32_t k, int e) {
    taken[warp][r] = unordered(k);
    chosen[t * top_k + r] = e;
  });
  __syncwarp();
  if (normalize) top = found > 0 ? taken[warp][0] : 0.f;
  const float e = lane < found ? expf(taken[warp][lane] - top) : 0.f;
  const float total = normalize ? warp_sum(e) : sum;
  if (lane < top_k) {
    weights[t * top_k + lane] = lane >= found ? 0.f : nan ? NAN : e / total;
    if (lane >= found) chosen[t * top_k + lane] = -1;
  }
}

// With p the softmax that the weights are shares of, and G = sum_j g_j w_j:
//   d logits[e] = p[e] * (g of the choice e, or 0) - p[e] * G.
// Shares of all experts: p from the logits, dense.  Shares of the chosen ones
// (normalize): p is the weights, zero elsewhere, and the logits are not read.
template <typename T, int V, bool kNormalize>
__global__ void __launch_bounds__(kRouteWarps * 32) route_grad_tokens(const float* __restrict__ grad, const T* __restrict__ logits,
                                                                      long long stride, const float* __restrict__ weights,
                                                                      const int* __restrict__ chosen, int tokens, int experts,
                                                                      int top_k, T* __restrict__ out, long long out_stride) {
  const int lane = threadIdx.x & 31;
  const long long t = blockIdx.x * (long long)kRouteWarps + (threadIdx.x >> 5);
  if (t >= tokens) return;
  int mine = -1;
  float g = 0.f, w = 0.f;
  if (lane < top_k) {
    mine = chosen[t * top_k + lane];
    if (mine >= 0 && mine < experts) {
      g = grad[t * top_k + lane];
      w = weights[t * top_k + lane];
    } else {
      mine = -1;
    }
  }
  const float inner = warp_sum(g * w);
  float p[V], d[V];
  if (!kNormalize) {
    float top, sum;
    load_scores<T, V>(logits + t * stride, experts, p);
    row_softmax<V>(p, top, sum);
    const float inv = sum > 0.f ? 1.f / sum : sum;  // a NaN stays
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = expf(p[v] - top) * inv;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) d[v] = kNormalize ? 0.f : -p[v] * inner;
  for (int j = 0; j < top_k; ++j) {
    const int e = __shfl_sync(0xffffffffu, mine, j);
    const float gj = __shfl_sync(0xffffffffu, g, j), wj = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e == v * 32 + lane) d[v] += kNormalize ? wj * (gj - inner) : p[v] * gj;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 32 + lane;
    if (e < experts) out[t * out_stride + e] = from_float<T>(d[v]);
  }
}

// ---- order of the slots by expert ---------------------------------------------------
__global__ void __launch_bounds__(kSortThreads) expert_order(const void* __restrict__ chosen, bool wide, long long n, int experts,
                                                             int align, int* __restrict__ position, int* __restrict__ offsets,
                                                             int* __restrict__ counts) {
  extern __shared__ uint32_t smem[];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  let_next_start();
  auto expert = [&](long long i) {
    const long long e = index_at(chosen, wide, i);
    return e >= 0 && e < experts ? int(e) : -1;
  };
  auto widen = [&](uint32_t count) { return (count + uint32_t(align) - 1) / uint32_t(align) * uint32_t(align); };
  sort_pass<int>(
      SortShared(smem, experts), experts, 0, warp_strip(n, rank, blocks), expert, [](int e) { return e; }, widen,
      [&](int e, uint32_t begin, uint32_t count) {
        if (rank != 0) return;
        offsets[e] = int(begin);
        counts[e] = int(count);
        if (e == experts - 1) offsets[experts] = int(begin + widen(count));
      },
      [&](long long i, int e, uint32_t p) { position[i] = e < 0 ? -1 : int(p); });
}

// ---- rows -----------------------------------------------------------------------
// The blocks that write the rows without a token come first: `tail` blocks for the
// rows behind the last expert, then `pad` blocks, kPadBlocks an expert, for the rows
// between an expert's tokens and the next expert.  Then the tokens' blocks:
// 2^lanes_log2 threads a token.
constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;
constexpr int kPadBlocks = 8;
constexpr int kTailBlocks = 512;

struct Blanks {
  const int* offsets;
  const int* counts;
  long long rows;
  int experts, tail, pad;
  __host__ __device__ int blocks() const { return tail + pad; }
};

// Block blockIdx.x < b.blocks() of the rows without a token.  The bounds hold whatever
// the plan's arrays say.
template <int B>
__device__ __forceinline__ void zero_blanks(const Blanks& b, int words, unsigned char* out, long long out_bytes) {
  constexpr int kWarps = kRowThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long begin, end = b.rows;
  int part = blockIdx.x, parts = b.tail;
  if (part < b.tail) {
    begin = b.offsets[b.experts];
  } else {
    const int e = (part - b.tail) / kPadBlocks;
    part = (part - b.tail) % kPadBlocks;
    parts = kPadBlocks;
    begin = (long long)b.offsets[e] + b.counts[e];
    end = min((long long)b.offsets[e + 1], b.rows);
  }
  for (long long r = max(0LL, begin) + part * kWarps + warp; r < end; r += parts * kWarps)
    for (int c = lane; c < words; c += 32) reinterpret_cast<Word<B>*>(out + r * out_bytes)[c] = Word<B>{};
}

// A token's row to the rows of its choices, by `lanes` threads.
template <int B>
__device__ __forceinline__ void copy_row(const unsigned char* x, const int* position, int top_k, long long rows, int words,
                                         unsigned char* out, long long out_bytes, int lanes) {
  const auto* src = reinterpret_cast<const Word<B>*>(x);
  for (int c = threadIdx.x & (lanes - 1); c < words; c += lanes * kRowUnroll) {
    Word<B> v[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u)
      if (c + u * lanes < words) v[u] = __ldg(src + c + u * lanes);
    for (int j = 0; j < top_k; ++j) {
      const int p = position[j];
      if (p < 0 || p >= rows) continue;
      auto* dst = reinterpret_cast<Word<B>*>(out + p * out_bytes);
#pragma unroll
      for (int u = 0; u < kRowUnroll; ++u)
        if (c + u * lanes < words) dst[c + u * lanes] = v[u];
    }
  }
}

// Few slots: one launch in which every block counts all of them for itself, instead
// of a sort and a copy that waits for it.
constexpr int kFewSlots = 2048;

template <int B>
__global__ void __launch_bounds__(kRowThreads) dispatch_few(const unsigned char* __restrict__ x, long long x_bytes,
                                                            const void* __restrict__ chosen, bool wide, int n, int align,
                                                            int* __restrict__ position, int* __restrict__ offsets,
                                                            int* __restrict__ counts, Blanks blanks, int tokens, int top_k, int words,
                                                            unsigned char* __restrict__ out, long long out_bytes, int lanes_log2) {
  __shared__ int expert[kFewSlots], count[kMaxExperts], begin[kMaxExperts + 1], place[kRowThreads / 32 * kMaxTopK];
  __shared__ int warp_total[kRowThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, experts = blanks.experts;
  for (int e = threadIdx.x; e < experts; e += kRowThreads) count[e] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < n; s += kRowThreads) {
    const long long e = index_at(chosen, wide, s);
    expert[s] = e >= 0 && e < experts ? int(e) : -1;
    if (expert[s] >= 0) atomicAdd(count + expert[s], 1);
  }
  __syncthreads();
  constexpr int kEach = kMaxExperts / kRowThreads;
  int room[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x * kEach + i;
    room[i] = e < experts ? (count[e] + align - 1) / align * align : 0;
    sum += room[i];
  }
  int before = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += o;
  }
  if (lane == 31) warp_total[warp] = before;
  __syncthreads();
  before -= sum;
  for (int w = 0; w < warp; ++w) before += warp_total[w];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = threadIdx.x * kEach + i;
    if (e <= experts) begin[e] = before;
    before += room[i];
  }
  if (experts == kMaxExperts && threadIdx.x == kRowThreads - 1) begin[experts] = before;
  __syncthreads();
  if (blockIdx.x == gridDim.x - 1) {
    for (int e = threadIdx.x; e <= experts; e += kRowThreads) {
      offsets[e] = begin[e];
      if (e < experts) counts[e] = count[e];
    }
  }
  if (int(blockIdx.x) < blanks.blocks()) {
    blanks.offsets = begin;
    blanks.counts = count;
    return zero_blanks<B>(blanks, words, out, out_bytes);
  }
  const int lanes = 1 << lanes_log2;  // 32 at least
  const int each = kRowThreads >> lanes_log2, first = (blockIdx.x - blanks.blocks()) * each;
  for (int s = warp; s < each * top_k; s += kRowThreads / 32) {
    const int slot = first * top_k + s;
    if (slot >= n) break;
    const int e = expert[slot];
    int earlier = 0;
    for (int i = lane; i < slot; i += 32) earlier += expert[i] == e;
    earlier = __reduce_add_sync(0xffffffffu, earlier);
    if (lane == 0) position[slot] = place[s] = e < 0 ? -1 : begin[e] + earlier;
  }
  __syncthreads();
  const int own = threadIdx.x >> lanes_log2, t = first + own;
  if (t < tokens) copy_row<B>(x + t * x_bytes, place + own * top_k, top_k, blanks.rows, words, out, out_bytes, lanes);
}

template <int B>
__global__ void __launch_bounds__(kRowThreads) dispatch_rows_kernel(const unsigned char* __restrict__ x, long long x_bytes,
                                                                    const int* position, Blanks blanks, int tokens, int top_k,
                                                                    int words, unsigned char* __restrict__ out,
                                                                    long long out_bytes, int lanes_log2) {
  wait_for_previous();
  if (int(blockIdx.x) < blanks.blocks()) return zero_blanks<B>(blanks, words, out, out_bytes);
  const long long t = (blockIdx.x - blanks.blocks()) * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (t < tokens)
    copy_row<B>(x + t * x_bytes, position + t * top_k, top_k, blanks.rows, words, out, out_bytes, 1 << lanes_log2);
}

template <typename T, int N, int W, bool kWeighted>
__global__ void __launch_bounds__(kRowThreads) combine_rows(const T* __restrict__ y, long long y_stride, long long rows,
                                                            const int* __restrict__ position, const float* __restrict__ weights,
                                                            const T* add, long long add_stride, int tokens, int top_k, int width,
                                                            T* out, long long out_stride, int lanes_log2) {
  constexpr int kSlots = 4;  // rows in flight
  const int lanes = 1 << lanes_log2, step = lanes * W;
  const long long t = blockIdx.x * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (t >= tokens) return;
  for (int c = (threadIdx.x & (lanes - 1)) * W; c < width; c += lanes * N) {
    float acc[N];
    Pack<T, N, W> o;
    o.zero();
    if (add) o.load_rw(add + t * add_stride, c, step, width);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = o.get(e);
    for (int j0 = 0; j0 < top_k; j0 += kSlots) {
      Pack<T, N, W> v[kSlots];
      float w[kSlots];
      bool on[kSlots];
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        const int p = j0 + s < top_k ? position[t * top_k + j0 + s] : -1;
        on[s] = p >= 0 && p < rows;
        if (on[s]) {
          v[s].load(y + p * y_stride, c, step, width);
          w[s] = kWeighted ? weights[t * top_k + j0 + s] : 1.f;
        }
      }
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (on[s]) {
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] += w[s] * v[s].get(e);
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) o.set(e, acc[e]);
    o.store(out + t * out_stride, c, step, width);
  }
}

template <typename T, int N, int W>
__global__ void __launch_bounds__(kRowThreads) combine_grad_rows(const T* __restrict__ grad, long long grad_stride, const T* y,
                                                                 long long y_stride, const int* __restrict__ position,
                                                                 Blanks blanks, const float* __restrict__ weights, int tokens,
                                                                 int top_k, int width, T* grad_y, long long grad_y_stride,
                                                                 float* __restrict__ grad_weights, int lanes_log2) {
  constexpr int kSlots = 8;  // rows in flight, and dot products held
  if (int(blockIdx.x) < blanks.blocks())
    return zero_blanks<W * int(sizeof(T))>(blanks, width / W, reinterpret_cast<unsigned char*>(grad_y),
                                           grad_y_stride * (long long)sizeof(T));
  const long long rows = blanks.rows;
  __shared__ float parts[kRowThreads / 32][kSlots];
  const int lanes = 1 << lanes_log2, step = lanes * W;  // 32 lanes at least
  const long long t = (blockIdx.x - blanks.blocks()) * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const bool live = t < tokens;  // the whole warp; the others take part in the block's barriers
  for (int j0 = 0; j0 < top_k; j0 += kSlots) {
    float dot[kSlots], w[kSlots];
    int p[kSlots];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const bool slot = live && j0 + s < top_k;
      p[s] = slot ? position[t * top_k + j0 + s] : -1;
      if (p[s] >= rows) p[s] = -1;
      w[s] = p[s] >= 0 ? weights[t * top_k + j0 + s] : 0.f;
      dot[s] = 0.f;
    }
    if (live) {
      for (int c = (threadIdx.x & (lanes - 1)) * W; c < width; c += lanes * N) {
        Pack<T, N, W> g, v[kSlots];
        g.zero();
        g.load(grad + t * grad_stride, c, step, width);
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (N != W) v[s].zero();  // columns behind the row
          if (p[s] >= 0) v[s].load_rw(y + p[s] * y_stride, c, step, width);
        }
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (p[s] < 0) continue;
          Pack<T, N, W> o;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            dot[s] += g.get(e) * v[s].get(e);
            o.set(e, w[s] * g.get(e));
          }
          o.store(grad_y + p[s] * grad_y_stride, c, step, width);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) dot[s] = warp_sum(dot[s]);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = lanes >> 5;
    if (warps > 1) {
      __syncthreads();
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (lane == s) parts[warp][s] = dot[s];
      __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (lane == s && live && j0 + s < top_k && warp % warps == 0) {
        float sum = dot[s];
        for (int k = 1; k < warps; ++k) sum += parts[warp + k][s];
        grad_weights[t * top_k + j0 + s] = p[s] >= 0 ? sum : 0.f;
      }
  }
}

template <int N>
struct Count {
  static constexpr int value = N;
};

// f(V constant) with 32 * V >= experts.
template <typename F>
void with_scores(int experts, F&& f) {
  if (experts <= 32) f(Count<1>());
  else if (experts <= 64) f(Count<2>());
  else if (experts <= 128) f(Count<4>());
  else if (experts <= 256) f(Count<8>());
  else if (experts <= 512) f(Count<16>());
  else f(Count<32>());
}

int tail_blocks(bool zero_tail, long long rows) {
  return zero_tail ? int(std::min<long long>(kTailBlocks, ceil_div_ll(rows, kRowThreads / 32))) : 0;
}

}  // namespace

void route_launch(int dtype, RowsIn logits, int tokens, int experts, int top_k, bool normalize, float* weights, int* chosen,
                  cudaStream_t stream) {
  if (tokens == 0) return;
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_scores(experts, [&](auto v) {
      route_tokens<T, decltype(v)::value><<<ceil_div(tokens, kRouteWarps), kRouteWarps * 32, 0, stream>>>(
          static_cast<const T*>(logits.ptr), logits.stride, tokens, experts, top_k, normalize, weights, chosen);
    });
  });
  PSB_LAUNCH_CHECK();
}

void route_grad_launch(int dtype, const float* grad_weights, RowsIn logits, const float* weights, const int* chosen, int tokens,
                       int experts, int top_k, bool normalize, RowsOut grad_logits, cudaStream_t stream) {
  if (tokens == 0) return;
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_scores(experts, [&](auto v) {
      constexpr int V = decltype(v)::value;
      auto kernel = normalize ? route_grad_tokens<T, V, true> : route_grad_tokens<T, V, false>;
      kernel<<<ceil_div(tokens, kRouteWarps), kRouteWarps * 32, 0, stream>>>(
          grad_weights, static_cast<const T*>(logits.ptr), logits.stride, weights, chosen, tokens, experts, top_k,
          static_cast<T*>(grad_logits.ptr), grad_logits.stride);
    });
  });
  PSB_LAUNCH_CHECK();
}

long long dispatch_rows(long long slots, int experts, int align) {
  return (slots + std::min<long long>(experts, slots) * (align - 1)) / align * align;
}

void dispatch_launch(int dtype, RowsIn x, Indices chosen, int tokens, int top_k, int experts, int align, int width, RowsOut out,
                     long long row_count, bool zero_tail, int* position, int* offsets, int* counts, cudaStream_t stream) {
  const long long n = chosen.count;
  const Blanks blanks{offsets, counts, row_count, experts, tail_blocks(zero_tail, row_count), align > 1 ? experts * kPadBlocks : 0};
  const int size = dtype_size(dtype);
  const long long row_bytes = (long long)width * size;
  const bool few = n <= kFewSlots;
  if (!few)
    launch_clusters<expert_order>(sort_blocks(n), 1, experts, stream, chosen.ptr, chosen.wide, n, experts, align, position, offsets,
                                  counts);
  auto run = [&](auto bytes) {
    constexpr int B = decltype(bytes)::value;
    const auto* src = static_cast<const unsigned char*>(x.ptr);
    auto* dst = static_cast<unsigned char*>(out.ptr);
    const int words = int(row_bytes / B), lanes_log2 = few ? row_lanes(words, 1, 5) : row_lanes(words, kRowUnroll, 0);
    const long long blocks = blanks.blocks() + ceil_div_ll(tokens, kRowThreads >> lanes_log2);
    if (few)
      dispatch_few<B><<<grid_x(std::max(1LL, blocks)), kRowThreads, 0, stream>>>(
          src, x.stride * size, chosen.ptr, chosen.wide, int(n), align, position, offsets, counts, blanks, tokens, top_k, words, dst,
          out.stride * size, lanes_log2);
    else
      launch_after(dispatch_rows_kernel<B>, grid_x(blocks), kRowThreads, stream, src, x.stride * size, position, blanks, tokens,
                   top_k, words, dst, out.stride * size, lanes_log2);
  };
  auto fits = [&](int bytes) {
    return row_bytes % bytes == 0 && rows_aligned(x.ptr, x.stride, size, bytes) && rows_aligned(out.ptr, out.stride, size, bytes);
  };
  if (fits(16)) run(Count<16>());
  else if (fits(4)) run(Count<4>());
  else run(Count<2>());
  PSB_LAUNCH_CHECK();
}

void combine_launch(int dtype, RowsIn y, long long rows, const int* position, const float* weights, RowsIn add, int tokens,
                    int top_k, int width, RowsOut out, cudaStream_t stream) {
  if (tokens == 0) return;
  const int size = dtype_size(dtype);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto fits = [&](int bytes) {
      return rows_aligned(y.ptr, y.stride, size, bytes) && rows_aligned(out.ptr, out.stride, size, bytes) &&
             (!add.ptr || rows_aligned(add.ptr, add.stride, size, bytes));
    };
    with_shape<T>(width, fits, [&](auto shape) {
      constexpr int N = decltype(shape)::N, W = decltype(shape)::W;
      const int lanes_log2 = row_lanes(ceil_div(width, N), 2, 0);
      const unsigned blocks = grid_x(ceil_div_ll(tokens, kRowThreads >> lanes_log2));
      auto kernel = weights ? combine_rows<T, N, W, true> : combine_rows<T, N, W, false>;
      kernel<<<blocks, kRowThreads, 0, stream>>>(static_cast<const T*>(y.ptr), y.stride, rows, position, weights,
                                                 static_cast<const T*>(add.ptr), add.stride, tokens, top_k, width,
                                                 static_cast<T*>(out.ptr), out.stride, lanes_log2);
    });
  });
  PSB_LAUNCH_CHECK();
}

void combine_grad_launch(int dtype, RowsIn grad, RowsIn y, long long rows, const int* position, const int* offsets,
                         const int* counts, int experts, const float* weights, int tokens, int top_k, int width, RowsOut grad_y,
                         bool zero_tail, float* grad_weights, cudaStream_t stream) {
  const Blanks blanks{offsets, counts, rows, experts, tail_blocks(zero_tail, rows), experts * kPadBlocks};
  const int size = dtype_size(dtype);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto fits = [&](int bytes) {
      return rows_aligned(grad.ptr, grad.stride, size, bytes) && rows_aligned(y.ptr, y.stride, size, bytes) &&
             rows_aligned(grad_y.ptr, grad_y.stride, size, bytes);
    };
    with_shape<T>(width, fits, [&](auto shape) {
      constexpr int N = decltype(shape)::N, W = decltype(shape)::W;
      const int lanes_log2 = row_lanes(ceil_div(width, N), 8, 5);
      const unsigned blocks = grid_x(blanks.blocks() + ceil_div_ll(tokens, kRowThreads >> lanes_log2));
      combine_grad_rows<T, N, W><<<blocks, kRowThreads, 0, stream>>>(
          static_cast<const T*>(grad.ptr), grad.stride, static_cast<const T*>(y.ptr), y.stride, position, blanks, weights, tokens,
          top_k, width, static_cast<T*>(grad_y.ptr), grad_y.stride, grad_weights, lanes_log2);
    });
  });
  PSB_LAUNCH_CHECK();
}

}  // namespace psb
