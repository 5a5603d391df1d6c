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
// A warp a token; lane l holds the V scores from l * V on in registers, so that a lane
// loads words of 16 bytes where the rows allow it (`words`) and the lanes' order is the
// experts'.  Scores compare as numbers: -0 equals +0, a NaN compares false and is never
// chosen, and -inf (off) lies below kLowest, the least score that can be.  Of equal
// scores the lowest index comes first.
constexpr int kRouteWarps = 8;
constexpr float kLowest = -3.402823466e+38f;

// The largest of a warp's numbers (none of them a NaN).
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Scores a load: all of a lane's, up to 16 bytes.
template <typename T, int V>
constexpr int kScoreWord = V * int(sizeof(T)) < 16 ? V : 16 / int(sizeof(T));

// A lane's scores, -inf behind the last expert.
template <typename T, int V>
__device__ __forceinline__ void load_scores(Pack<T, V, kScoreWord<T, V>>& p, const T* row, int c, int step, int experts, bool words) {
#pragma unroll
  for (int v = 0; v < V; ++v) p.set(v, -INFINITY);
  if (words) p.load(row, c, step, experts);
  else p.load_elements(row, c, step, experts);
}

struct Gathered {
  float2 item[32];  // score and index
  float taken[32];  // scores by rank
};

// The top_k largest of a warp's scores, ranked: g.taken[r] is the score of rank r and
// take(r, index) is called by one lane for every rank r that there is; returns their
// number and sets `top` to the largest (kLowest where there is none).
//
// The k-th largest of the 32 lanes' own maxima (counted once where they are equal) is a
// bound that at least k scores reach, and rarely many more do: those are gathered in
// shared memory, where each lane ranks one of them among all.  Where more than 32 reach
// it, the scores are taken one by one instead.
// 16384 tokens of 256 experts in FP32, top 8: 7.8 us a call with the scores in the L2, 8.9
// with scores from memory (1.9 TB/s); in 16 bits 9.1, as it is bound by instructions (about
// 400 a warp, 75% of the issue slots taken).  A maximum over the warp for each choice took
// 17.3 us; half a warp a token the same as a whole one.
template <int V, typename Take>
__device__ __forceinline__ int top_scores(float (&x)[V], int top_k, Gathered& g, float& top, Take&& take) {
  const int lane = threadIdx.x & 31;
  float best = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) best = fmaxf(best, x[v]);
  float left = best, bound = top = fmaxf(kLowest, warp_max(left));
  for (int j = 1; j < top_k; ++j) {
    left = left == bound ? -INFINITY : left;
    bound = warp_max(left);
  }
  bound = fmaxf(kLowest, bound);
  int mine = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) mine += x[v] >= bound;
  int slot = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, slot, d);
    if (lane >= d) slot += o;
  }
  const int found = __shfl_sync(0xffffffffu, slot, 31);
  if (found <= 32) {
    slot -= mine;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (x[v] >= bound) g.item[slot++] = make_float2(x[v], __int_as_float(lane * V + v));
    if (lane >= found) g.item[lane] = make_float2(-INFINITY, 0.f);
    __syncwarp();
    const float2 own = g.item[lane];
    int rank = 0;
    for (int i = 0; i < found; i += 4) {
      const float4 a = *reinterpret_cast<const float4*>(g.item + i), b = *reinterpret_cast<const float4*>(g.item + i + 2);
      rank += (a.x > own.x) + (a.z > own.x) + (b.x > own.x) + (b.z > own.x);
    }
    // Equal scores have got the same rank, so the ranks add up to less than they should:
    // then, as the slots ascend with the index, the lower slot comes first.
    if (__reduce_add_sync(0xffffffffu, lane < found ? rank : 0) != found * (found - 1) / 2)
      for (int i = 0; i < found; ++i) rank += g.item[i].x == own.x && i < lane;
    if (lane < found && rank < top_k) {
      g.taken[rank] = own.x;
      take(rank, __float_as_int(own.y));
    }
    return min(found, top_k);
  }
  for (int j = 0; j < top_k; ++j) {
    const float largest = warp_max(best);
    if (!(largest >= kLowest)) return j;
    int at = 0x7fffffff;
#pragma unroll
    for (int v = V - 1; v >= 0; --v)
      if (x[v] == largest) at = lane * V + v;
    const int first = __reduce_min_sync(0xffffffffu, at);
    best = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (first == lane * V + v) x[v] = -INFINITY;
      best = fmaxf(best, x[v]);
    }
    if (at == first) {
      g.taken[j] = largest;
      take(j, first);
    }
  }
  return top_k;
}

template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) route_tokens(const T* logits, long long stride, bool words,
                                                                 int tokens, int experts, int top_k, bool normalize,
                                                                 float* weights, int* chosen) {
  __shared__ __align__(16) Gathered gathered[kRouteWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = blockIdx.x * (long long)kRouteWarps + warp;
  wait_for_previous();
  if (t >= tokens) return;
  float x[V], top;
  bool nan = false;
  {
    Pack<T, V, kScoreWord<T, V>> p;
    load_scores<T, V>(p, logits + t * stride, lane * V, kScoreWord<T, V>, experts, words);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      x[v] = p.get(v);
      nan = nan || x[v] != x[v];
    }
  }
  nan = __any_sync(0xffffffffu, nan);
  float sum = 0.f;
  if (!normalize) {
    top = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) top = fmaxf(top, x[v]);
    top = fmaxf(kLowest, warp_max(top));
#pragma unroll
    for (int v = 0; v < V; ++v) sum += expf(x[v] - top);
    sum = warp_sum(sum);
  }
  Gathered& g = gathered[warp];
  const int found = top_scores<V>(x, top_k, g, top, [&](int r, int e) { chosen[t * top_k + r] = e; });
  __syncwarp();
  const float e = lane < found ? expf(g.taken[lane] - top) : 0.f;
  const float total = normalize ? warp_sum(e) : sum;
  if (lane < top_k) {
    // A NaN (or +inf, which makes the total NaN) reaches every place, those without a choice
    // too: a row of NaN alone has no choice that could show it.
    weights[t * top_k + lane] = nan || total != total ? NAN : lane >= found ? 0.f : e / total;
    if (lane >= found) chosen[t * top_k + lane] = -1;
  }
}

// With p the softmax that the weights are shares of, g[e] the gradient of the choice e (0
// where it was not chosen) and G = sum_j g_j w_j:  d logits[e] = p[e] * (g[e] - G).
// Shares of all experts: p from the logits, dense.  Shares of the chosen ones
// (normalize): p is the weights, zero elsewhere, and the logits are not read; a weight that
// is NaN makes its whole row NaN, as a NaN of the scores does in the dense form.  g (or
// w_j (g_j - G)) is spread over the experts in shared memory.  A lane's words stand 32
// words apart, so that a warp writes whole sectors.  16384 tokens of 256 experts in FP32,
// dense: 7.4 us with the scores in the L2, 8.6 from memory (4.1 TB/s), where handing each
// choice round the warp took 9.3; normalized 6.6.
template <typename T, int V, bool kNormalize>
__global__ void __launch_bounds__(kRouteWarps * 32) route_grad_tokens(const float* grad, const T* logits,
                                                                      long long stride, bool words, const float* weights,
                                                                      const int* chosen, int tokens, int experts,
                                                                      int top_k, T* out, long long out_stride) {
  constexpr int W = kScoreWord<T, V>;
  __shared__ __align__(16) float spread[kRouteWarps][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = blockIdx.x * (long long)kRouteWarps + warp;
  wait_for_previous();
  if (t >= tokens) return;
  Pack<T, V, W> x;
  if (!kNormalize) load_scores<T, V>(x, logits + t * stride, lane * W, 32 * W, experts, words);
  int mine = -1;
  float g = 0.f, w = 0.f;
  if (lane < top_k) {
    mine = chosen[t * top_k + lane];
    g = grad[t * top_k + lane];
    w = weights[t * top_k + lane];
  }
  // The dense form has a NaN of the scores in p; here the weights tell of it.
  const float unchosen = kNormalize && __any_sync(0xffffffffu, w != w) ? NAN : 0.f;
  if (mine < 0 || mine >= experts) {
    mine = -1 - lane;
    g = w = 0.f;
  }
  float* own = spread[warp];
#pragma unroll
  for (int v = 0; v < V; ++v) own[v * 32 + lane] = unchosen;
  __syncwarp();
  const float inner = warp_sum(g * w);
  float value = kNormalize ? w * (g - inner) : g;
  const unsigned same = __match_any_sync(0xffffffffu, mine);
  if (__any_sync(0xffffffffu, same & (same - 1)))  // a choice that stands twice: the first takes their sum
    for (int j = 1; j < top_k; ++j) {
      const float other = __shfl_sync(0xffffffffu, value, j);
      if (j > lane && (same >> j & 1)) value += other;
    }
  if (mine >= 0 && lane == __ffs(same) - 1) own[mine] = value;
  __syncwarp();
  float top = -INFINITY, sum = 0.f, p[V];
  if (!kNormalize) {
#pragma unroll
    for (int v = 0; v < V; ++v) top = fmaxf(top, x.get(v));
    top = fmaxf(kLowest, warp_max(top));
#pragma unroll
    for (int v = 0; v < V; ++v) sum += p[v] = expf(x.get(v) - top);
    sum = warp_sum(sum);
    // One rounding to 32 bits more than a division of each p, which took 9.2 to 9.8 us where
    // this takes 7.4 (16384 tokens of 256 experts).
    sum = sum > 0.f ? 1.f / sum : sum;  // a NaN stays
  }
  Pack<T, V, W> o;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float s = own[(v / W * 32 + lane) * W + v % W];
    o.set(v, kNormalize ? s : p[v] * sum * (s - inner));
  }
  if (words) o.store(out + t * out_stride, lane * W, 32 * W, experts);
  else o.store_elements(out + t * out_stride, lane * W, 32 * W, experts);
}

// ---- order of the slots by expert ---------------------------------------------------
__global__ void __launch_bounds__(kSortThreads) expert_order(const void* chosen, bool wide, long long n, int experts,
                                                             int align, int* position, int* offsets,
                                                             int* counts) {
  extern __shared__ __align__(16) unsigned char smem[];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  let_next_start();
  wait_for_previous();
  auto expert = [&](long long i) {
    const long long e = index_at(chosen, wide, i);
    return e >= 0 && e < experts ? int(e) : -1;
  };
  auto widen = [&](uint32_t count) { return (count + uint32_t(align) - 1) / uint32_t(align) * uint32_t(align); };
  sort_pass<int, false, true>(
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

// A token's row to the rows of its choices, by `lanes` threads: read once, written top_k
// times.  Bound by the writes: 8192 tokens of 4096 in 16 bits to 8 experts each take
// 103 us after the order's 9, 6.1 TB/s with the rows up to multiples of 128.
template <int B>
__device__ __forceinline__ void copy_row(const unsigned char* x, const int* position, int top_k, long long rows, int words,
                                         unsigned char* out, long long out_bytes, int lanes) {
  const auto* src = reinterpret_cast<const Word<B>*>(x);
  for (int c = threadIdx.x & (lanes - 1); c < words; c += lanes * kRowUnroll) {
    Word<B> v[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u)
      if (c + u * lanes < words) v[u] = src[c + u * lanes];
    for (int j = 0; j < top_k; ++j) {
      const int p = position[j];
      if (p < 0 || p >= rows) continue;
      auto* dst = reinterpret_cast<Word<B>*>(out + p * out_bytes);
#pragma unroll
      for (int u = 0; u < kRowUnroll; ++u)
        if (c + u * lanes < words) __stcs(dst + c + u * lanes, v[u]);
    }
  }
}

// Few slots: one launch, a block a token, in which every block counts all slots for
// itself, instead of a sort and a copy that waits for it.  1024 slots, rows of 2048 in
// 16 bits: 4.7 us against 8.3; 2048 slots 5.7 against 9.3; 4096 slots of narrow rows
// 15.4 against 8.8, where the counting costs more than the sort.
constexpr int kFewSlots = 2048;

template <int B>
__global__ void __launch_bounds__(kRowThreads) dispatch_few(const unsigned char* x, long long x_bytes,
                                                            const void* chosen, bool wide, int n, int align,
                                                            int* position, int* offsets,
                                                            int* counts, Blanks blanks, int top_k, int words,
                                                            unsigned char* out, long long out_bytes) {
  __shared__ int expert[kFewSlots], count[kMaxExperts], begin[kMaxExperts + 1], place[kMaxTopK];
  __shared__ int warp_total[kRowThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, experts = blanks.experts;
  wait_for_previous();
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
  const int t = blockIdx.x - blanks.blocks();
  if (t * top_k >= n) return;  // the block that is there for no tokens at all
  for (int j = warp; j < top_k; j += kRowThreads / 32) {
    const int slot = t * top_k + j, e = expert[slot];
    int earlier = 0;
    for (int i = lane; i < slot; i += 32) earlier += expert[i] == e;
    earlier = __reduce_add_sync(0xffffffffu, earlier);
    if (lane == 0) position[slot] = place[j] = e < 0 ? -1 : begin[e] + earlier;
  }
  __syncthreads();
  copy_row<B>(x + t * x_bytes, place, top_k, blanks.rows, words, out, out_bytes, kRowThreads);
}

template <int B>
__global__ void __launch_bounds__(kRowThreads) dispatch_rows_kernel(const unsigned char* x, long long x_bytes,
                                                                    const int* position, Blanks blanks, int tokens, int top_k,
                                                                    int words, unsigned char* out,
                                                                    long long out_bytes, int lanes_log2) {
  wait_for_previous();
  if (int(blockIdx.x) < blanks.blocks()) return zero_blanks<B>(blanks, words, out, out_bytes);
  const long long t = (blockIdx.x - blanks.blocks()) * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (t < tokens)
    copy_row<B>(x + t * x_bytes, position + t * top_k, top_k, blanks.rows, words, out, out_bytes, 1 << lanes_log2);
}

// A token's rows are added up in the order of the choices, kSlots of them at a time and
// kTurns stretches of the row, so that a thread has four loads in flight whether a token
// has many rows or two.  Bound by memory: 8192 tokens of 4096 in 16 bits, 8 experts each
// and a residual take 113 us with inputs that alternate, 5.9 TB/s, and 108 with inputs that
// stay (the positions and weights of a batch are read before its rows: 111 otherwise;
// eight rows in flight: 112, and 103 against 81 in 32 bits, where they cost occupancy).
// 6799 tokens with 2 experts each: 32 us with (2, 2), 41 with (4, 1).
template <typename T, int N, int W, int S, bool kWeighted, int kSlots, int kTurns>
__global__ void __launch_bounds__(kRowThreads) combine_rows(const T* y, long long y_stride, long long rows,
                                                            const int* position, const float* weights,
                                                            const T* add, long long add_stride, int tokens, int top_k, int width,
                                                            T* out, long long out_stride, int lanes_log2) {
  wait_for_previous();
  const int lanes = 1 << lanes_log2, step = word_step<W, S>(lanes), turn = lanes * N;
  const long long t = blockIdx.x * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (t >= tokens) return;
  for (int c = first_column<N, W, S>(threadIdx.x & (lanes - 1)); c < width; c += turn * kTurns) {
    float acc[kTurns][N];
    Pack<T, N, W> o[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      o[k].zero();
      if (add) o[k].load(add + t * add_stride, c + k * turn, step, width);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[k][e] = o[k].get(e);
    }
    for (int j0 = 0; j0 < top_k; j0 += kSlots) {
      Pack<T, N, W> v[kTurns][kSlots];
      float w[kSlots];
      int p[kSlots];
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        const bool slot = j0 + s < top_k;
        p[s] = slot ? position[t * top_k + j0 + s] : -1;
        w[s] = kWeighted && slot ? weights[t * top_k + j0 + s] : 1.f;
        if (p[s] >= rows) p[s] = -1;
      }
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (p[s] >= 0)
#pragma unroll
          for (int k = 0; k < kTurns; ++k) v[k][s].load(y + p[s] * y_stride, c + k * turn, step, width);
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (p[s] >= 0) {
#pragma unroll
          for (int k = 0; k < kTurns; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) acc[k][e] += w[s] * v[k][s].get(e);
        }
    }
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
#pragma unroll
      for (int e = 0; e < N; ++e) o[k].set(e, acc[k][e]);
      o[k].store(out + t * out_stride, c + k * turn, step, width);
    }
  }
}

// Sums of K numbers each over a warp: a lane gets that of number lane / (32 / K).  While
// there is more than one number left, half the lanes go on with one half of them and half
// with the other, so eight sums take 9 shuffles, not 40.
template <int K>
__device__ __forceinline__ float sum_slots(float (&d)[K]) {
  const int lane = threadIdx.x & 31;
  int far = 16;
#pragma unroll
  for (int n = K / 2; n > 0; n /= 2, far /= 2) {
    const bool upper = lane & far;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = upper ? d[i + n] : d[i], send = upper ? d[i] : d[i + n];
      d[i] = keep + __shfl_xor_sync(0xffffffffu, send, far);
    }
  }
  float v = d[0];
#pragma unroll
  for (; far > 0; far /= 2) v += __shfl_xor_sync(0xffffffffu, v, far);
  return v;
}

// Both gradients in one pass: the token's gradient row is read once and multiplied with
// each weight on its way out, and with each of its rows of y into a dot product, a warp
// (or more, for few tokens) a token, kSlots rows and kTurns stretches of them in flight.
// Bound by memory: 8192 tokens of 2048 in 16 bits, 8 experts each, take 100 us, 5.8 TB/s
// with the rows up to multiples of 128 (104 without the bound of 80 registers); 6799
// tokens of 4096, 2 experts each, 47 us with (2, 4), 63 with (8, 1).  Ragged rows are
// bound by latency and want more warps instead: 15687 tokens of 1893, one expert each,
// 57 us with (2, 2) in 64 registers, 102 with (2, 4) in 128.
template <typename T, int N, int W, int S, int kSlots, int kTurns>
__global__ void __launch_bounds__(kRowThreads, W == N ? 3 : 4) combine_grad_rows(const T* grad, long long grad_stride, const T* y,
                                                                 long long y_stride, const int* position,
                                                                 Blanks blanks, const float* weights, int tokens,
                                                                 int top_k, int width, T* grad_y, long long grad_y_stride,
                                                                 float* grad_weights, int lanes_log2) {
  wait_for_previous();
  if (int(blockIdx.x) < blanks.blocks())
    return zero_blanks<W * int(sizeof(T))>(blanks, width / W, reinterpret_cast<unsigned char*>(grad_y),
                                           grad_y_stride * (long long)sizeof(T));
  const long long rows = blanks.rows;
  __shared__ float parts[kRowThreads / 32][kSlots];
  const int lanes = 1 << lanes_log2, step = word_step<W, S>(lanes);  // 32 lanes at least
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
      const int turn = lanes * N;
      for (int c = first_column<N, W, S>(threadIdx.x & (lanes - 1)); c < width; c += turn * kTurns) {
        Pack<T, N, W> g[kTurns], v[kTurns][kSlots];
#pragma unroll
        for (int k = 0; k < kTurns; ++k) {
          g[k].zero();  // columns behind the row
          g[k].load(grad + t * grad_stride, c + k * turn, step, width);
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            if (N != W || kTurns > 1) v[k][s].zero();
            if (p[s] >= 0) v[k][s].load(y + p[s] * y_stride, c + k * turn, step, width);
          }
        }
#pragma unroll
        for (int k = 0; k < kTurns; ++k)
#pragma unroll
          for (int s = 0; s < kSlots; ++s) {
            if (p[s] < 0) continue;
            Pack<T, N, W> o;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              dot[s] += g[k].get(e) * v[k][s].get(e);
              o.set(e, w[s] * g[k].get(e));
            }
            o.store(grad_y + p[s] * grad_y_stride, c + k * turn, step, width);
          }
      }
    }
    const float dot_warp = sum_slots<kSlots>(dot);
    constexpr int kEach = 32 / kSlots;  // lanes that end up with a slot's sum
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = lanes >> 5, slot = lane / kEach;
    if (warps > 1) {
      __syncthreads();
      if (lane % kEach == 0) parts[warp][slot] = dot_warp;
      __syncthreads();
    }
    if (lane % kEach == 0 && live && j0 + slot < top_k && warp % warps == 0) {
      float sum = dot_warp;
      for (int k = 1; k < warps; ++k) sum += parts[warp + k][slot];
      const int at = position[t * top_k + j0 + slot];
      grad_weights[t * top_k + j0 + slot] = at >= 0 && at < rows ? sum : 0.f;
    }
  }
}

template <int N>
struct Count {
  static constexpr int value = N;
};

// Calls f(V, words): 32 * V >= experts, and whether every row allows the words
// (fits(bytes): they begin at multiples of so many).
template <typename T, typename Fits, typename F>
void with_scores(int experts, Fits&& fits, F&& f) {
  auto call = [&](auto v) {
    constexpr int W = kScoreWord<T, decltype(v)::value>;
    f(v, experts % W == 0 && fits(W * int(sizeof(T))));
  };
  if (experts <= 32) call(Count<1>());
  else if (experts <= 64) call(Count<2>());
  else if (experts <= 128) call(Count<4>());
  else if (experts <= 256) call(Count<8>());
  else if (experts <= 512) call(Count<16>());
  else call(Count<32>());
}

int tail_blocks(bool zero_tail, long long rows) {
  return zero_tail ? int(std::min<long long>(kTailBlocks, ceil_div_ll(rows, kRowThreads / 32))) : 0;
}

}  // namespace

void route_launch(int dtype, RowsIn logits, int tokens, int experts, int top_k, bool normalize, float* weights, int* chosen,
                  cudaStream_t stream) {
  if (tokens == 0) return;
  const int size = dtype_size(dtype);
  auto fits = [&](int bytes) { return rows_aligned(logits.ptr, logits.stride, size, bytes); };
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_scores<T>(experts, fits, [&](auto v, bool words) {
      launch_after(route_tokens<T, decltype(v)::value>, grid_x(ceil_div_ll(tokens, kRouteWarps)), kRouteWarps * 32, stream,
                   static_cast<const T*>(logits.ptr), logits.stride, words, tokens, experts, top_k, normalize, weights, chosen);
    });
  });
}

void route_grad_launch(int dtype, const float* grad_weights, RowsIn logits, const float* weights, const int* chosen, int tokens,
                       int experts, int top_k, bool normalize, RowsOut grad_logits, cudaStream_t stream) {
  if (tokens == 0) return;
  const int size = dtype_size(dtype);
  auto fits = [&](int bytes) {
    return rows_aligned(logits.ptr, logits.stride, size, bytes) && rows_aligned(grad_logits.ptr, grad_logits.stride, size, bytes);
  };
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_scores<T>(experts, fits, [&](auto v, bool words) {
      constexpr int V = decltype(v)::value;
      auto kernel = normalize ? route_grad_tokens<T, V, true> : route_grad_tokens<T, V, false>;
      launch_after(kernel, grid_x(ceil_div_ll(tokens, kRouteWarps)), kRouteWarps * 32, stream, grad_weights,
                   static_cast<const T*>(logits.ptr), logits.stride, words, weights, chosen, tokens, experts, top_k,
                   static_cast<T*>(grad_logits.ptr), grad_logits.stride);
    });
  });
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
    launch_clusters<expert_order>(sort_blocks(n), 1, sort_smem(experts), stream, chosen.ptr, chosen.wide, n, experts, align, position, offsets,
                                  counts);
  auto run = [&](auto bytes) {
    constexpr int B = decltype(bytes)::value;
    const auto* src = static_cast<const unsigned char*>(x.ptr);
    auto* dst = static_cast<unsigned char*>(out.ptr);
    const int words = int(row_bytes / B), lanes_log2 = row_lanes(words, kRowUnroll, 1, 0, tokens);
    if (few)
      launch_after(dispatch_few<B>, grid_x(std::max(1LL, (long long)blanks.blocks() + tokens)), kRowThreads, stream, src,
                   x.stride * size, chosen.ptr, chosen.wide, int(n), align, position, offsets, counts, blanks, top_k, words, dst,
                   out.stride * size);
    else
      launch_after(dispatch_rows_kernel<B>, grid_x(blanks.blocks() + ceil_div_ll(tokens, kRowThreads >> lanes_log2)), kRowThreads, stream, src, x.stride * size, position, blanks, tokens,
                   top_k, words, dst, out.stride * size, lanes_log2);
  };
  auto fits = [&](int bytes) {
    return row_bytes % bytes == 0 && rows_aligned(x.ptr, x.stride, size, bytes) && rows_aligned(out.ptr, out.stride, size, bytes);
  };
  if (fits(16)) run(Count<16>());
  else if (fits(4)) run(Count<4>());
  else run(Count<2>());
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
      constexpr int N = decltype(shape)::N, W = decltype(shape)::W, S = decltype(shape)::S;
      const int lanes_log2 = row_lanes(width, N, 2, decltype(shape)::kLeastLanesLog2, tokens);
      const unsigned blocks = grid_x(ceil_div_ll(tokens, kRowThreads >> lanes_log2));
      auto run = [&](auto kernel) {
        launch_after(kernel, blocks, kRowThreads, stream, static_cast<const T*>(y.ptr), y.stride, rows, position, weights,
                     static_cast<const T*>(add.ptr), add.stride, tokens, top_k, width, static_cast<T*>(out.ptr), out.stride, lanes_log2);
      };
      if (top_k > 2) run(weights ? combine_rows<T, N, W, S, true, 4, 1> : combine_rows<T, N, W, S, false, 4, 1>);
      else run(weights ? combine_rows<T, N, W, S, true, 2, 2> : combine_rows<T, N, W, S, false, 2, 2>);
    });
  });
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
      constexpr int N = decltype(shape)::N, W = decltype(shape)::W, S = decltype(shape)::S;
      const int lanes_log2 = row_lanes(width, N, 8, 5, tokens);
      const unsigned blocks = grid_x(blanks.blocks() + ceil_div_ll(tokens, kRowThreads >> lanes_log2));
      auto run = [&](auto kernel) {
        launch_after(kernel, blocks, kRowThreads, stream, static_cast<const T*>(grad.ptr), grad.stride, static_cast<const T*>(y.ptr),
                     y.stride, position, blanks, weights, tokens, top_k, width, static_cast<T*>(grad_y.ptr), grad_y.stride, grad_weights,
                     lanes_log2);
      };
      if constexpr (W == N) {
        if (top_k > 4) run(combine_grad_rows<T, N, W, S, 8, 1>);
        else if (top_k > 2) run(combine_grad_rows<T, N, W, S, 4, 2>);
        else run(combine_grad_rows<T, N, W, S, 2, 4>);
      } else {
        if (top_k > 2) run(combine_grad_rows<T, N, W, S, 4, 1>);
        else run(combine_grad_rows<T, N, W, S, 2, 2>);
      }
    });
  });
}

}  // namespace psb
