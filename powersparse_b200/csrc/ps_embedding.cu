// Embedding: rows of a table looked up by token and scaled, and the gradient of the
// table as the sum of the output gradients of each token.
//
//   out[i, :]  = scale * table[t_i, :]
//   grad[v, :] = scale * sum over i with t_i = v of g[i, :]
//
// As products with the one-hot matrix S (S[i, t_i] = 1): out = S * table, and
// grad = S^T * g, a product of the same kind as SpMM whose matrix is new in every
// call.  Its rows are found by sorting the tokens (ps_index_sort.cuh), so each row of
// the gradient is summed without atomics, in an order that no timing changes: the rows of
// a token in the order of the batch, in parts that a chunk, a group of threads or a warp
// adds up, and then the parts.
#include "ps_index_sort.cuh"
#include "ps_rows.cuh"

namespace psb {
namespace {

// ---- lookup ---------------------------------------------------------------------
// 2^lanes_log2 threads a row, kRowUnroll words of it in flight each.  Bound by memory:
// 16384 tokens of 4096 in 16 bits take 32 us with inputs that alternate, 5.9 TB/s of the
// 189 MB that have to move (30 with inputs that stay); 16 tokens 2.1 us, a launch.
constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;

template <typename T, int N, int W, int S>
__global__ void __launch_bounds__(kRowThreads) embedding_rows(const T* table, long long table_stride, long long rows,
                                                              const void* tokens, bool wide, long long n, int width,
                                                              float scale, T* out, long long out_stride,
                                                              int lanes_log2) {
  wait_for_previous();
  const int lanes = 1 << lanes_log2, step = word_step<W, S>(lanes);
  const long long i = blockIdx.x * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (i >= n) return;
  const long long token = index_at(tokens, wide, i);
  const bool inside = token >= 0 && token < rows;
  const T* src = table + (inside ? token : 0) * table_stride;
  if (!inside) scale = 0.f;  // +0, whatever the scale
  T* dst = out + i * out_stride;
  for (int c = first_column<N, W, S>(threadIdx.x & (lanes - 1)); c < width; c += lanes * N * kRowUnroll) {
    Pack<T, N, W> v[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      v[u].zero();
      if (inside) v[u].load(src, c + u * lanes * N, step, width);
    }
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[u].set(e, v[u].get(e) * scale);
      v[u].store_once(dst, c + u * lanes * N, step, width);
    }
  }
}

// ---- gradient: order of the tokens ------------------------------------------------
// A token and its place in the batch.
struct Item {
  uint32_t token, place;
};

// Zeros in `bytes` bytes at p (a multiple of 2), 16 at a time between the ends.
__device__ __forceinline__ void clear(unsigned char* p, long long bytes, int thread, int threads) {
  const long long head = min(bytes, (long long)(-reinterpret_cast<uintptr_t>(p) & 15)), words = (bytes - head) / 16;
  auto* body = reinterpret_cast<uint4*>(p + head);
#pragma unroll 4
  for (long long i = thread; i < words; i += threads) __stcs(body + i, make_uint4(0, 0, 0, 0));
  for (long long i = thread; i < head / 2; i += threads) reinterpret_cast<uint16_t*>(p)[i] = 0;
  auto* tail = reinterpret_cast<uint16_t*>(p + head + words * 16);
  for (long long i = thread; i < (bytes - head - words * 16) / 2; i += threads) tail[i] = 0;
}

// The same word by word for `rows` rows of `words` words, `pitch` bytes apart, but for
// those that are touched (null: none is).
template <int B>
__device__ __forceinline__ void clear_words(unsigned char* p, long long pitch, int words, const unsigned char* touched, int rows,
                                            int thread, int threads) {
  int r = thread / words, c = thread % words;
  const int rows_on = threads / words, words_on = threads % words;
  while (r < rows) {
    if (!touched || !touched[r]) reinterpret_cast<Word<B>*>(p + r * pitch)[c] = Word<B>{};
    r += rows_on;
    c += words_on;
    if (c >= words) {
      c -= words;
      ++r;
    }
  }
}

// Rows of `bytes` bytes: by words of 16 bytes where all rows allow them, a warp a row
// where they do not and are long, else by smaller words.  (39 MB of 320-byte rows: 7 us
// by words, 19 by a warp a row.)
__device__ __forceinline__ void clear_rows(unsigned char* p, long long pitch, long long bytes, const unsigned char* touched, int rows,
                                           int thread, int threads) {
  const auto all = reinterpret_cast<uintptr_t>(p) | uintptr_t(pitch) | uintptr_t(bytes);
  if (all % 16 == 0) return clear_words<16>(p, pitch, int(bytes / 16), touched, rows, thread, threads);
  if (bytes >= 1024) {
    for (int r = thread / 32; r < rows; r += threads / 32)
      if (!touched || !touched[r]) clear(p + r * pitch, bytes, thread % 32, 32);
    return;
  }
  if (all % 4 == 0) return clear_words<4>(p, pitch, int(bytes / 4), touched, rows, thread, threads);
  clear_words<2>(p, pitch, int(bytes / 2), touched, rows, thread, threads);
}

// Rows that a block of `warps` warps clears: about 64 KiB, less where there are few, and
// one a warp at least.
inline int clear_block_rows(long long rows, long long bytes, int warps) {
  const long long block = std::min<long long>(1 << 16, std::max<long long>(1 << 12, rows * bytes / (4 * device_sms())));
  return int(std::max<long long>(warps, block / bytes));
}

// The gradient's rows to be cleared: `rows` stretches of `bytes`, `pitch` bytes apart,
// by blocks of kSortThreads that take kClearBytes or block_rows rows each.
struct Clear {
  unsigned char* ptr;
  long long rows, bytes, pitch;
  int block_rows;
  static constexpr long long kClearBytes = 1 << 18;
  // One stretch where the rows touch.
  __host__ Clear(void* p, long long r, long long b, long long pitch_bytes)
      : ptr(static_cast<unsigned char*>(p)), rows(pitch_bytes == b ? 1 : r), bytes(pitch_bytes == b ? r * b : b), pitch(pitch_bytes),
        block_rows(clear_block_rows(r, b, kSortWarps)) {}
  __host__ long long blocks() const { return rows == 1 ? ceil_div_ll(bytes, kClearBytes) : ceil_div_ll(rows, block_rows); }
  __device__ void run(long long block) const {
    if (rows == 1) {
      const long long begin = block * kClearBytes;
      if (begin < bytes) clear(ptr + begin, min(kClearBytes, bytes - begin), threadIdx.x, kSortThreads);
    } else {
      const long long r = block * block_rows;
      if (r < rows) clear_rows(ptr + r * pitch, pitch, bytes, nullptr, int(min((long long)block_rows, rows - r)), threadIdx.x, kSortThreads);
    }
  }
};

// The rows of a large gradient that the sort leaves to the kernels after it, cleared
// beside their sums: rows [begin, end) that no token names, by blocks of whole warps.
struct Rest {
  unsigned char* ptr;
  const unsigned char* touched;
  long long begin, end, bytes, pitch;
  int block_rows;
  Rest(unsigned char* p, const unsigned char* t, long long b, long long e, long long row_bytes, long long row_pitch, int warps)
      : ptr(p), touched(t), begin(b), end(e), bytes(row_bytes), pitch(row_pitch), block_rows(clear_block_rows(e - b, row_bytes, warps)) {}
  __host__ long long blocks() const { return ceil_div_ll(end - begin, block_rows); }
  __device__ void run(long long block) const {
    const long long r = begin + block * block_rows;
    if (r < end)
      clear_rows(ptr + r * pitch, pitch, bytes, touched + r, int(min((long long)block_rows, end - r)), threadIdx.x, blockDim.x);
  }
};

// The first cluster sorts the tokens; tokens outside [0, rows) and the padding token
// get the key `rows` and come last.  The sorted items are in `a`.  The other clusters
// clear the gradient meanwhile, or the first rows of a large one: rows that no token
// names need it, and what the others cost is hidden, since the sort leaves most of the
// GPU idle.  touched (null unless rows are left to the later kernels): 1 for every token
// that occurs.  counts: two numbers to be set to zero.
__global__ void __launch_bounds__(kSortThreads) embedding_order(const void* tokens, bool wide, long long n,
                                                                long long rows, long long padding, int pass_bits, int passes,
                                                                Item* a, Item* b, int* counts, unsigned char* touched,
                                                                Clear zeros) {
  extern __shared__ __align__(16) unsigned char smem[];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  let_next_start();
  wait_for_previous();
  if (int(blockIdx.x) >= blocks) return zeros.run(blockIdx.x - blocks);
  const int digits = 1 << pass_bits;
  const SortShared sh(smem, digits);
  const Strip strip = warp_strip(n, rank, blocks);
  if (rank == 0 && threadIdx.x < 2) counts[threadIdx.x] = 0;
  if (touched)
    for (long long v = rank * kSortThreads + threadIdx.x; v < rows; v += blocks * kSortThreads) touched[v] = 0;
  for (int pass = 0; pass < passes; ++pass) {
    const bool to_a = ((passes - 1 - pass) & 1) == 0;
    Item* out = to_a ? a : b;
    const Item* in = to_a ? b : a;
    const int shift = pass * pass_bits;
    sort_pass<Item, true, false>(
        sh, digits, pass & 1, strip,
        [&](long long i) -> Item {
          if (pass) return in[i];
          const long long t = index_at(tokens, wide, i);
          return {uint32_t(t >= 0 && t < rows && t != padding ? t : rows), uint32_t(i)};
        },
        [&](Item e) { return int((e.token >> shift) & uint32_t(digits - 1)); }, [](uint32_t count) { return count; },
        [](int, uint32_t, uint32_t) {},
        [&](long long, Item e, uint32_t p) {
          out[p] = e;
          if (touched && pass == 0 && e.token < rows) touched[e.token] = 1;  // cleared before the barrier of the pass
        });
  }
}

// ---- gradient: sums of the sorted rows ----------------------------------------------
// A block takes `chunk` consecutive sorted positions and N columns a thread, and
// adds the gradient rows run by run in 32-bit registers.  A run inside the chunk goes
// to its row; what belongs to a run that crosses a border goes to the chunk's two
// partial rows: [0] for the run that began before the chunk, [1] for one that goes on
// after it.  join_runs adds those up, by a list of the chunks in which such runs begin:
// those of at most kShortRun chunks (at least two) and the longer ones apart, in any order.
constexpr int kShortRun = 4;

struct Joins {
  Item* shorter;  // token and chunk
  Item* longer;
  int* count;  // of the two
};

// Bound by memory where the rows are wide and the table large (16384 tokens of 2048 in
// 16 bits into 131072 rows in 32: 176 us for sort, sums, joins and clearing together, 98%
// of the copy rate).  Ragged rows (50003 of 515 in 16 bits, 47 us in all with inputs that
// alternate, 40 with inputs that stay in the L2) are bound by latency and instructions: 21 us
// for the sort's two passes, about 11 of the 40 for the sums, 8 for the joins.  Eight rows
// in flight and eight blocks an SM: sixteen rows or ten blocks took 2 and 6 us longer there.
constexpr int kSumThreads = 128;
constexpr int kMaxChunk = 64;

template <typename O, int N, int W>
__device__ __forceinline__ void write_sum(O* row, int c, int step, int width, const float (&acc)[N], float scale, bool accumulate) {
  Pack<O, N, W> v;
  v.zero();
  if (accumulate) v.load(row, c, step, width);
#pragma unroll
  for (int e = 0; e < N; ++e) v.set(e, accumulate ? v.get(e) + acc[e] * scale : acc[e] * scale);
  v.store(row, c, step, width);
}

template <typename T, typename O, int N, int W>
__global__ void __launch_bounds__(kSumThreads, 8) sum_runs(const T* grad, long long grad_stride, const Item* items,
                                                           long long n, uint32_t rows, int width, float scale, bool accumulate,
                                                           O* out, long long out_stride, int chunk,
                                                           float* partial, Joins joins, int sum_blocks, int slabs,
                                                           Rest rest) {
  constexpr int kUnroll = 8;
  constexpr uint32_t kNone = 0xffffffffu;
  __shared__ uint32_t key[kMaxChunk + 2], at[kMaxChunk];
  static_assert(kMaxChunk % 32 == 0 && kMaxChunk <= 64);
  let_next_start();
  wait_for_previous();
  if (int(blockIdx.x) >= sum_blocks) return rest.run(blockIdx.x - sum_blocks);
  const long long block = blockIdx.x / slabs, first = block * chunk;
  const int count = int(min((long long)chunk, n - first));
  for (int i = threadIdx.x; i < count + 2; i += blockDim.x) {
    const long long p = first + i - 1;
    const Item item = p >= 0 && p < n ? items[p] : Item{kNone, 0};
    key[i] = item.token;
    if (i >= 1 && i <= count) at[i - 1] = item.place;
  }
  __syncthreads();
  if (blockIdx.x % slabs == 0 && threadIdx.x == 0) {
    const uint32_t token = key[count];
    if (token < rows && key[count + 1] == token && !(key[0] == token && key[1] == token)) {  // begins here and goes on
      const long long far = (block + kShortRun) * chunk;
      const bool longer = far < n && items[far].token == token;
      (longer ? joins.longer : joins.shorter)[atomicAdd(joins.count + longer, 1)] = {token, uint32_t(block)};
    }
  }
  // Where runs end in the chunk, as bits, and how many of its positions name a row (the
  // empty places are sorted behind them): all that the loop asks for each position.
  const int lane = threadIdx.x & 31;
  unsigned long long ends = 0;
  int total = 0;
#pragma unroll
  for (int half = 0; half < kMaxChunk / 32; ++half) {
    const int i = half * 32 + lane;
    const bool on = i < count && key[i + 1] < rows;
    ends |= (unsigned long long)__ballot_sync(0xffffffffu, on && (key[i + 1] != key[i + 2] || i + 1 == count)) << (half * 32);
    total += __popc(__ballot_sync(0xffffffffu, on));
  }
  constexpr int step = 32 * W;
  const int c = first_column<N, W, 32>(blockIdx.x % slabs * blockDim.x + threadIdx.x);
  if (c >= width) return;
  const bool goes_on = key[count] == key[count + 1];
  bool before = key[0] == key[1];  // the current run began before the chunk
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  for (int i = 0; i < total; i += kUnroll) {
    Pack<T, N, W> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      v[u].load(grad + (long long)at[min(i + u, total - 1)] * grad_stride, c, step, width);
    const unsigned here = unsigned(ends >> i) & ((1u << kUnroll) - 1u);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (i + u >= total) break;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += v[u].get(e);
      if (!(here >> u & 1)) continue;
      if (!before && !(goes_on && i + u + 1 == count)) {
        write_sum<O, N, W>(out + (long long)key[i + u + 1] * out_stride, c, step, width, acc, scale, accumulate);
      } else {
        Pack<float, N, W> sum;
#pragma unroll
        for (int e = 0; e < N; ++e) sum.set(e, acc[e]);
        sum.store(partial + (block * 2 + (before ? 0 : 1)) * width, c, step, width);
      }
      before = false;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = 0.f;
    }
  }
}

// The runs that cross a border, 32 * N columns at a time.  Blocks first take the longer
// ones, all their warps one run (every kJoinWarps-th chunk each, then over the warps);
// the `short_blocks` behind them take a short one a warp.
constexpr int kJoinWarps = 16;

template <typename O, int N, int W>
__global__ void __launch_bounds__(kJoinWarps * 32) join_runs(const Item* items, long long n, int width, float scale,
                                                             bool accumulate, O* out, long long out_stride, int chunk,
                                                             const float* partial, Joins joins, int chunks, int long_blocks,
                                                             int short_blocks, int slabs, Rest rest) {
  constexpr int kUnroll = kShortRun;
  __shared__ float sums[kJoinWarps][32 * N];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_previous();
  if (int(blockIdx.x) >= (long_blocks + short_blocks) * slabs) return rest.run(blockIdx.x - (long_blocks + short_blocks) * slabs);
  const int c = blockIdx.x % slabs * 32 * N + lane * W, block = blockIdx.x / slabs;
  float acc[N];
  // Adds the shares of the chunks own + first, own + first + stride, ... (kUnroll of them at
  // most) of the run that begins in chunk `own`; whether the last of them belongs to it.
  auto add = [&](Item join, long long first, int stride) {
    const long long own = join.place;
    Pack<float, N, W> v[kUnroll];
    bool on[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long j = own + first + u * stride;
      const bool inside = j * chunk < n;
      v[u].zero();
      if (inside) v[u].load(partial + (j * 2 + (j == own ? 1 : 0)) * width, c, 32 * W, width);
      on[u] = j == own || (inside && items[j * chunk].token == join.token);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += on[u] ? v[u].get(e) : 0.f;
    return on[kUnroll - 1];
  };
  auto clear_sum = [&] {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
  };
  if (block >= long_blocks) {
    for (int i = (block - long_blocks) * kJoinWarps + warp; i < chunks; i += short_blocks * kJoinWarps) {
      const Item join = joins.shorter[i];  // read beside the count, not after it: there is room for all chunks
      if (i >= joins.count[0]) return;
      clear_sum();
      add(join, 0, 1);
      if (c < width) write_sum<O, N, W>(out + (long long)join.token * out_stride, c, 32 * W, width, acc, scale, accumulate);
    }
    return;
  }
  for (int i = block; i < chunks; i += long_blocks) {
    const Item join = joins.longer[i];
    if (i >= joins.count[1]) return;
    clear_sum();
    for (long long j = warp; add(join, j, kJoinWarps); j += kJoinWarps * kUnroll) {
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sums[warp][e * 32 + lane] = acc[e];
    __syncthreads();
    if (warp == 0 && c < width) {
      for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += sums[w][e * 32 + lane];
      write_sum<O, N, W>(out + (long long)join.token * out_stride, c, 32 * W, width, acc, scale, accumulate);
    }
    __syncthreads();
  }
}

// ---- gradient of few tokens: one launch ---------------------------------------------
// A block for every token of the batch: the first of its kind adds up all of them (the
// others end), where less than a block shares a row every groups-th of them a group of
// threads and then the groups.  Up to kFewTokens / kFewThreads tokens a
// thread are compared, so no sort is needed, and neither are partial rows.  Behind them
// the blocks that clear the rows which no token names.
//
// Taken up to kFewTokens tokens, as every block reads every token, and up to kFewElements
// elements, as the few blocks of one token read all of its rows while the sort's sums
// spread them over the GPU.  Against the sort and its launches, in 16 bits into 4096 rows,
// tokens as text has them (all of one kind; all distinct): 2048 tokens, rows of 256, 11 us
// against 20 (32, 22; 14, 17); 4096 tokens 34 against 21; 2048 tokens, rows of 2048, 30
// against 22 (227, 25; 19, 20); rows of 8192, 512 tokens, 21 against 22 (96, 20; 25, 20), 1024
// tokens 35 against 26 (198, 23; 38, 25) and 2048 tokens 88 against 31 (779, 30; 49, 29).
// Where the table is large its clearing hides the sums of few tokens, and the border lies
// higher: 134M elements, rows of 8192, 600 tokens 52 against 55, 1100 tokens 62 against 56.
constexpr int kFewTokens = 2048;
constexpr long long kFewElements = 5 << 20;
inline bool few_tokens_suffice(long long n, int width) { return n <= kFewTokens && n * width <= kFewElements; }
constexpr int kFewThreads = 256;
constexpr int kFewEach = kFewTokens / kFewThreads;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kLongRun = 64;         // from here on a block's warps share out the rows, not the columns
constexpr int kClearRows = 4096;     // rows a clearing block takes at the most

// The thread's tokens threadIdx.x + k * kFewThreads as rows of the table (-1: none).
__device__ __forceinline__ void few_tokens(const void* tokens, bool wide, int n, long long rows, long long padding,
                                           int (&v)[kFewEach]) {
#pragma unroll
  for (int k = 0; k < kFewEach; ++k) {
    const int i = threadIdx.x + k * kFewThreads;
    const long long t = i < n ? index_at(tokens, wide, i) : -1;
    v[k] = t >= 0 && t < rows && t != padding ? int(t) : -1;
  }
}

template <typename T, typename O, int N, int W, int S>
__global__ void __launch_bounds__(kFewThreads) sum_few(const T* grad, long long grad_stride,
                                                       const void* tokens, bool wide, int n, long long rows,
                                                       long long padding, int width, float scale, bool accumulate,
                                                       O* out, long long out_stride, int block_rows, int lanes_log2,
                                                       int parts) {
  __shared__ union {
    struct {
      unsigned short list[kFewTokens];
      int count[kFewEach * kFewWarps];
      float sums[N][kFewThreads];
    };
    unsigned char touched[kClearRows];
  } sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  wait_for_previous();
  int v[kFewEach];
  if (int(blockIdx.x) >= n * parts) {
    const long long first = (long long)(blockIdx.x - n * parts) * block_rows;
    few_tokens(tokens, wide, n, rows, padding, v);
    for (int r = threadIdx.x; r < block_rows; r += kFewThreads) sh.touched[r] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kFewEach; ++k)
      if (v[k] >= first && v[k] < first + block_rows) sh.touched[v[k] - first] = 1;
    __syncthreads();
    constexpr long long kSize = sizeof(O);
    clear_rows(reinterpret_cast<unsigned char*>(out + first * out_stride), out_stride * kSize, width * kSize, sh.touched,
               int(min((long long)block_rows, rows - first)), threadIdx.x, kFewThreads);
    return;
  }
  const int own = blockIdx.x / parts;
  const long long token = index_at(tokens, wide, own);
  if (token < 0 || token >= rows || token == padding) return;
  few_tokens(tokens, wide, n, rows, padding, v);
  bool earlier = false;
  unsigned same[kFewEach];
#pragma unroll
  for (int k = 0; k < kFewEach; ++k) {
    const bool match = v[k] == int(token);
    earlier = earlier || (match && int(threadIdx.x) + k * kFewThreads < own);
    same[k] = __ballot_sync(0xffffffffu, match);
    if (lane == 0) sh.count[k * kFewWarps + warp] = __popc(same[k]);
  }
  if (__syncthreads_or(earlier)) return;
  // Places of the matches in order: threads' words are in the order of k, then warp, then lane.
  int total = 0, before[kFewEach];
#pragma unroll
  for (int k = 0; k < kFewEach; ++k)
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      if (w == warp) before[k] = total;
      total += sh.count[k * kFewWarps + w];
    }
#pragma unroll
  for (int k = 0; k < kFewEach; ++k)
    if (same[k] >> lane & 1)
      sh.list[before[k] + __popc(same[k] & ((1u << lane) - 1u))] = (unsigned short)(threadIdx.x + k * kFewThreads);
  __syncthreads();

  constexpr int kUnroll = 8;
  const int lanes = total > kLongRun ? 32 : 1 << lanes_log2, groups = kFewThreads / lanes;  // threads a row, rows at a time
  const int group = threadIdx.x / lanes, step = word_step<W, S>(lanes);
  for (int slab = blockIdx.x % parts * lanes * N; slab < width; slab += parts * lanes * N) {
    const int c = slab + first_column<N, W, S>(threadIdx.x & (lanes - 1));
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    for (int i = group; i < total; i += groups * kUnroll) {
      Pack<T, N, W> x[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        x[u].zero();
        if (i + u * groups < total) x[u].load(grad + sh.list[i + u * groups] * grad_stride, c, step, width);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += x[u].get(e);
    }
    if (groups > 1) {
#pragma unroll
      for (int e = 0; e < N; ++e) sh.sums[e][threadIdx.x] = acc[e];
      __syncthreads();
      if (group == 0)
        for (int g = 1; g < groups && g < total; ++g)
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] += sh.sums[e][g * lanes + threadIdx.x];
      __syncthreads();
    }
    if (group == 0) write_sum<O, N, W>(out + token * out_stride, c, step, width, acc, scale, accumulate);
  }
}

// Bytes cleared beside the sort (about 15 us, at 6 TB/s) and beside the joins.
constexpr long long kClearFirst = 96 << 20, kClearLast = 48 << 20;

// Sorted positions a block adds up: more of them make fewer partial rows and joins, but
// fewer threads; where rows are narrow there are few threads a block, and the blocks
// become smaller until the GPU is about a third full.  64 against 32: 65536 tokens in
// rows of 1024 64 against 71 us; 16384 tokens in rows of 2048 188 against 180.
int chunk_of(long long n, int width) {
  int chunk = n >= 32768 ? 64 : n >= 16384 ? 32 : 16;
  const long long threads = ceil_div(width, 8 * 32) * 32;
  while (chunk > 8 && ceil_div_ll(n, chunk) * threads < 65536) chunk /= 2;
  return chunk;
}

constexpr size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

struct Workspace {
  size_t a, b, join_count, shorter, longer, touched, partial, bytes;
  Workspace(long long n, long long rows, int width) {
    const long long chunks = ceil_div_ll(n, chunk_of(n, width));
    a = 0;
    b = a + align_up(size_t(n) * sizeof(Item));
    join_count = b + align_up(size_t(n) * sizeof(Item));
    shorter = join_count + align_up(2 * sizeof(int));
    longer = shorter + align_up(size_t(chunks) * sizeof(Item));
    touched = longer + align_up(size_t(chunks) * sizeof(Item));
    partial = touched + align_up(size_t(rows));
    bytes = partial + align_up(size_t(chunks) * 2 * size_t(width) * sizeof(float));
  }
};

}  // namespace

void embedding_launch(int dtype, RowsIn table, long long rows, int width, Indices tokens, float scale, RowsOut out,
                      cudaStream_t stream) {
  if (tokens.count == 0) return;
  const int size = dtype_size(dtype);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto fits = [&](int bytes) {
      return rows_aligned(table.ptr, table.stride, size, bytes) && rows_aligned(out.ptr, out.stride, size, bytes);
    };
    with_shape<T>(width, fits, [&](auto shape) {
      constexpr int N = decltype(shape)::N, W = decltype(shape)::W, S = decltype(shape)::S;
      const int lanes_log2 = row_lanes(width, N * kRowUnroll, 1, decltype(shape)::kLeastLanesLog2, tokens.count);
      const unsigned blocks = grid_x(ceil_div_ll(tokens.count, kRowThreads >> lanes_log2));
      launch_after(embedding_rows<T, N, W, S>, blocks, kRowThreads, stream, static_cast<const T*>(table.ptr), table.stride, rows,
                   tokens.ptr, tokens.wide, tokens.count, width, scale, static_cast<T*>(out.ptr), out.stride, lanes_log2);
    });
  });
}

size_t embedding_grad_workspace(long long tokens, long long rows, int width) {
  return few_tokens_suffice(tokens, width) ? 0 : Workspace(tokens, rows, width).bytes;
}

void embedding_grad_launch(int grad_dtype, RowsIn grad, Indices tokens, float scale, long long padding, bool accumulate,
                           int out_dtype, RowsOut out, long long rows, int width, void* workspace, cudaStream_t stream) {
  const long long n = tokens.count;
  const int in_size = dtype_size(grad_dtype), out_size = dtype_size(out_dtype), chunk = chunk_of(n, width);
  if (n == 0 && accumulate) return;
  const Workspace at(n, rows, width);
  char* ws = static_cast<char*>(workspace);
  auto* items = reinterpret_cast<Item*>(ws + at.a);
  const Joins joins{reinterpret_cast<Item*>(ws + at.shorter), reinterpret_cast<Item*>(ws + at.longer),
                    reinterpret_cast<int*>(ws + at.join_count)};
  auto* partial = reinterpret_cast<float*>(ws + at.partial);
  const bool few = few_tokens_suffice(n, width);
  const long long row_bytes = (long long)width * out_size;
  // A gradient of more than kClearFirst + kClearLast bytes is cleared in three parts, so
  // that the sums and the joins, too, run beside a part of it.
  const long long pitch = out.stride * out_size, first_rows = kClearFirst / row_bytes, last_rows = kClearLast / row_bytes;
  const bool parts = !few && !accumulate && first_rows + last_rows < rows;
  auto* touched = parts ? reinterpret_cast<unsigned char*>(ws + at.touched) : nullptr;
  auto* bytes = static_cast<unsigned char*>(out.ptr);
  const Rest middle{bytes, touched, first_rows, parts ? rows - last_rows : first_rows, row_bytes, pitch, kSumThreads / 32};
  const Rest last{bytes, touched, middle.end, parts ? rows : middle.end, row_bytes, pitch, kJoinWarps};
  if (!few) {
    const Clear zeros(out.ptr, parts ? first_rows : rows, row_bytes, pitch);
    const int bits = bits_for((unsigned long long)rows), passes = ceil_div(bits, kMaxBits), pass_bits = ceil_div(bits, passes);
    const int blocks = sort_blocks(n);
    const long long clusters = 1 + (accumulate ? 0 : ceil_div_ll(zeros.blocks(), blocks));
    const size_t smem = sort_smem(1 << pass_bits) + stage_smem(n, blocks, sizeof(Item));
    launch_clusters<embedding_order>(blocks, clusters, smem, stream, tokens.ptr, tokens.wide, n, rows, padding, pass_bits,
                                     passes, items, reinterpret_cast<Item*>(ws + at.b), joins.count, touched, zeros);
  }
  auto run = [&](auto t, auto o) {
    using T = decltype(t);
    using O = decltype(o);
    auto fits = [&](int bytes) {
      // A word of the gradient of the table has as many elements, not as many bytes.
      return rows_aligned(grad.ptr, grad.stride, in_size, bytes) &&
             rows_aligned(out.ptr, out.stride, out_size, std::min(16, bytes / in_size * out_size));
    };
    with_shape<T>(width, fits, [&](auto shape) {
      constexpr int N = decltype(shape)::N, W = decltype(shape)::W, S = decltype(shape)::S;
      O* dst = static_cast<O*>(out.ptr);
      if (few) {
        const int block_rows = std::min(kClearRows, clear_block_rows(rows, row_bytes, kFewWarps));
        const int lanes_log2 = row_lanes(width, N, 1, std::max(2, decltype(shape)::kLeastLanesLog2), n);
        // Long rows are shared out among blocks as far as that does not make more than 32 to an SM.
        const int parts = int(std::max(1LL, std::min<long long>(ceil_div(width, N << lanes_log2), 32LL * device_sms() / std::max(1LL, n))));
        const long long blocks = n * parts + (accumulate ? 0 : ceil_div_ll(rows, block_rows));  // n and blocks are not both 0
        launch_after(sum_few<T, O, N, W, S>, grid_x(blocks), kFewThreads, stream, static_cast<const T*>(grad.ptr), grad.stride,
                     tokens.ptr, tokens.wide, int(n), rows, padding, width, scale, accumulate, dst, out.stride, block_rows, lanes_log2,
                     parts);
        return;
      }
      const int chunks = int(ceil_div_ll(n, chunk));
      // As few blocks a row as kSumThreads allows, and no more warps in them than the row fills.
      const int slabs = ceil_div(width, kSumThreads * N), threads = ceil_div(ceil_div(width, slabs * N), 32) * 32;
      const long long sum_blocks = (long long)chunks * slabs;
      launch_after(sum_runs<T, O, N, W>, grid_x(sum_blocks + middle.blocks()), threads, stream, static_cast<const T*>(grad.ptr),
                   grad.stride, items, n, uint32_t(rows), width, scale, accumulate, dst, out.stride, chunk, partial, joins,
                   int(sum_blocks), slabs, middle);
      // At most one run in kShortRun chunks is long; few are.
      const int join_slabs = ceil_div(width, 32 * N);
      const int long_blocks = std::min(ceil_div(chunks, kShortRun), 32);
      const int short_blocks = std::min(ceil_div(chunks, kJoinWarps), std::max(1, 8 * device_sms() / join_slabs));
      launch_after(join_runs<O, N, W>, grid_x((long long)(long_blocks + short_blocks) * join_slabs + last.blocks()), kJoinWarps * 32,
                   stream, items, n, width, scale, accumulate, dst, out.stride, chunk, partial, joins, chunks, long_blocks,
                   short_blocks, join_slabs, last);
    });
  };
  with_type(grad_dtype, [&](auto t) {
    if (out_dtype == grad_dtype) run(t, t);
    else run(t, float());
  });
}

}  // namespace psb
