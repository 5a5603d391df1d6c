// Embedding: rows of a table looked up by token and scaled, and the gradient of the
// table as the sum of the output gradients of each token.
//
//   out[i, :]  = scale * table[t_i, :]
//   grad[v, :] = scale * sum over i with t_i = v of g[i, :]
//
// As products with the one-hot matrix S (S[i, t_i] = 1): out = S * table, and
// grad = S^T * g, a product of the same kind as SpMM whose matrix is new in every
// call.  Its rows are found by sorting the tokens (ps_index_sort.cuh), so each row of
// the gradient is summed in the order of the batch, without atomics.
#include "ps_index_sort.cuh"
#include "ps_rows.cuh"

namespace psb {
namespace {

// ---- lookup ---------------------------------------------------------------------
// 2^lanes_log2 threads a row, kRowUnroll words of it in flight each.
constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;

template <typename T, int N>
__global__ void __launch_bounds__(kRowThreads) embedding_rows(const T* __restrict__ table, long long table_stride, long long rows,
                                                              const void* __restrict__ tokens, bool wide, long long n, int width,
                                                              float scale, T* __restrict__ out, long long out_stride,
                                                              int lanes_log2) {
  const int lanes = 1 << lanes_log2;
  const long long i = blockIdx.x * (long long)(kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (i >= n) return;
  const long long token = index_at(tokens, wide, i);
  const bool inside = token >= 0 && token < rows;
  const T* src = table + (inside ? token : 0) * table_stride;
  T* dst = out + i * out_stride;
  for (int c = (threadIdx.x & (lanes - 1)) * N; c < width; c += lanes * N * kRowUnroll) {
    Pack<T, N> v[kRowUnroll];
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      const int at = c + u * lanes * N;
      v[u].zero();
      if (inside && at < width) v[u].load(src + at);
    }
#pragma unroll
    for (int u = 0; u < kRowUnroll; ++u) {
      const int at = c + u * lanes * N;
      if (at >= width) break;
#pragma unroll
      for (int e = 0; e < N; ++e) v[u].set(e, v[u].get(e) * scale);
      v[u].store(dst + at);
    }
  }
}

// ---- gradient: order of the tokens ------------------------------------------------
// Sorts (token, position in the batch) by token; tokens outside [0, rows) and the
// padding token get the key `rows` and come last.  touched[v] = 1 for every token v
// that occurs (touched may be null).  The sorted pairs are in (key_a, pos_a).
__global__ void __launch_bounds__(kSortThreads) embedding_order(const void* __restrict__ tokens, bool wide, long long n,
                                                                long long rows, long long padding, int pass_bits, int passes,
                                                                uint32_t* key_a, uint32_t* pos_a, uint32_t* key_b, uint32_t* pos_b,
                                                                unsigned char* touched) {
  extern __shared__ uint32_t smem[];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int digits = 1 << pass_bits;
  const SortShared sh(smem, digits);
  const Strip strip = warp_strip(n, rank, blocks);
  uint32_t* row = sh.rows + (threadIdx.x >> 5) * digits;
  if (touched)
    for (long long v = rank * (long long)kSortThreads + threadIdx.x; v < rows; v += (long long)blocks * kSortThreads) touched[v] = 0;
  auto ignore = [](int, uint32_t, uint32_t) {};
  auto same = [](uint32_t count) { return count; };
  for (int pass = 0; pass < passes; ++pass) {
    const bool to_a = ((passes - 1 - pass) & 1) == 0;
    uint32_t *key_out = to_a ? key_a : key_b, *pos_out = to_a ? pos_a : pos_b;
    const uint32_t *key_in = to_a ? key_b : key_a, *pos_in = to_a ? pos_b : pos_a;
    const int shift = pass * pass_bits;
    auto key = [&](long long i) -> uint32_t {
      if (pass) return key_in[i];
      const long long t = index_at(tokens, wide, i);
      return uint32_t(t >= 0 && t < rows && t != padding ? t : rows);
    };
    auto digit = [&](long long i) { return int((key(i) >> shift) & uint32_t(digits - 1)); };
    digit_positions(sh, digits, strip, digit, same, ignore);
    place_digits(strip, row, digit, [&](long long i, int, uint32_t p) {
      const uint32_t k = key(i);
      key_out[p] = k;
      pos_out[p] = pass ? pos_in[i] : uint32_t(i);
      if (pass == 0 && touched && k < rows) touched[k] = 1;  // cleared before the cluster's barrier in digit_positions
    });
    cluster.sync();  // the pass's writes are visible to the cluster
  }
}

// ---- gradient: sums of the sorted rows ----------------------------------------------
// A block takes `chunk` consecutive sorted positions and kSumThreads * N columns, and
// adds the gradient rows run by run in 32-bit registers.  A run inside the chunk goes
// to its row; what belongs to a run that crosses a border goes to the chunk's two
// partial rows: [0] for the run that began before the chunk, [1] for one that goes on
// after it.  join_runs adds those up.
constexpr int kSumThreads = 128;
constexpr int kMaxChunk = 32;

template <typename O, int N>
__device__ __forceinline__ void write_sum(O* at, const float (&acc)[N], float scale, bool accumulate) {
  Pack<O, N> v;
  if (accumulate) {
    v.load_rw(at);
#pragma unroll
    for (int e = 0; e < N; ++e) v.set(e, v.get(e) + acc[e] * scale);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v.set(e, acc[e] * scale);
  }
  v.store(at);
}

template <typename T, typename O, int N>
__global__ void __launch_bounds__(kSumThreads) sum_runs(const T* __restrict__ grad, long long grad_stride,
                                                        const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                        long long n, uint32_t rows, int width, float scale, bool accumulate,
                                                        O* __restrict__ out, long long out_stride, int chunk,
                                                        float* __restrict__ partial) {
  constexpr int kUnroll = 8;
  constexpr uint32_t kNone = 0xffffffffu;
  __shared__ uint32_t key[kMaxChunk + 2], at[kMaxChunk];
  const long long first = blockIdx.x * (long long)chunk;
  const int count = int(min((long long)chunk, n - first));
  for (int i = threadIdx.x; i < count + 2; i += kSumThreads) {
    const long long p = first + i - 1;
    key[i] = p >= 0 && p < n ? keys[p] : kNone;
    if (i >= 1 && i <= count) at[i - 1] = pos[p];
  }
  __syncthreads();
  const int c = (blockIdx.y * kSumThreads + threadIdx.x) * N;
  if (c >= width) return;
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  bool before = key[0] == key[1];  // the current run began before the chunk
  for (int i = 0; i < count; i += kUnroll) {
    Pack<T, N> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u < count && key[i + u + 1] < rows) v[u].load(grad + (long long)at[i + u] * grad_stride + c);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (i + u >= count) break;
      const uint32_t k = key[i + u + 1];
      if (k >= rows) return;  // sorted: nothing but empty places from here on
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += v[u].get(e);
      if (key[i + u + 2] == k && i + u + 1 < count) continue;
      const bool after = key[i + u + 2] == k;
      if (!before && !after) {
        write_sum(out + (long long)k * out_stride + c, acc, scale, accumulate);
      } else {
        Pack<float, N> sum;
#pragma unroll
        for (int e = 0; e < N; ++e) sum.set(e, acc[e]);
        sum.store(partial + (blockIdx.x * 2LL + (before ? 0 : 1)) * width + c);
      }
      before = false;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = 0.f;
    }
  }
}

// The run that begins in chunk blockIdx.x and goes on after it: its partial rows, added
// in order by each of the block's warps (every kJoinWarps-th chunk) and then over the warps.
constexpr int kJoinWarps = 8;

template <typename O, int N>
__global__ void __launch_bounds__(kJoinWarps * 32) join_runs(const uint32_t* __restrict__ keys, long long n, uint32_t rows, int width,
                                                             float scale, bool accumulate, O* __restrict__ out,
                                                             long long out_stride, int chunk, const float* __restrict__ partial) {
  __shared__ float sums[kJoinWarps][32 * N];
  const long long begin = blockIdx.x * (long long)chunk, next = begin + chunk;
  if (next >= n) return;
  const uint32_t k = keys[next - 1];
  if (k >= rows || keys[next] != k) return;
  if (begin > 0 && keys[begin - 1] == k) return;  // the run began in an earlier chunk
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = (blockIdx.y * 32 + lane) * N;
  float acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0.f;
  const long long own = blockIdx.x;
  for (long long j = own + warp; j * chunk < n && (j == own || keys[j * chunk] == k); j += kJoinWarps) {
    if (c < width) {
      Pack<float, N> v;
      v.load(partial + (j * 2 + (j == own ? 1 : 0)) * width + c);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += v.get(e);
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) sums[warp][e * 32 + lane] = acc[e];
  __syncthreads();
  if (warp != 0 || c >= width) return;
  for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += sums[w][e * 32 + lane];
  write_sum(out + (long long)k * out_stride + c, acc, scale, accumulate);
}

// Zeros in every row that no token names (touched null: in every row), a warp a row.
template <typename O, int N>
__global__ void __launch_bounds__(256) zero_rows(const unsigned char* __restrict__ touched, long long rows, int width,
                                                 O* __restrict__ out, long long out_stride) {
  const long long v = blockIdx.x * 8LL + (threadIdx.x >> 5);
  if (v >= rows || (touched && touched[v])) return;
  Pack<O, N> zero;
  zero.zero();
  for (int c = (threadIdx.x & 31) * N; c < width; c += 32 * N) zero.store(out + v * out_stride + c);
}

int chunk_of(long long n) { return n >= 16384 ? 32 : n >= 2048 ? 16 : 4; }

constexpr size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

struct Workspace {
  size_t key_a, pos_a, key_b, pos_b, touched, partial, bytes;
  Workspace(long long n, long long rows, int width) {
    const size_t index = align_up(size_t(n) * sizeof(uint32_t));
    key_a = 0;
    pos_a = key_a + index;
    key_b = pos_a + index;
    pos_b = key_b + index;
    touched = pos_b + index;
    partial = touched + align_up(size_t(rows));
    bytes = partial + align_up(size_t(ceil_div_ll(n, chunk_of(n))) * 2 * size_t(width) * sizeof(float));
  }
};

// f(N constant): elements a thread moves at a time.
template <int N>
struct Count {
  static constexpr int value = N;
};

}  // namespace

void embedding_launch(int dtype, RowsIn table, long long rows, int width, Indices tokens, float scale, RowsOut out,
                      cudaStream_t stream) {
  if (tokens.count == 0) return;
  const int size = dtype_size(dtype);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto per) {
      constexpr int N = decltype(per)::value;
      const int lanes_log2 = std::min(8, std::max(0, log2_up(ceil_div(ceil_div(width, N), kRowUnroll))));
      const unsigned blocks = grid_x(ceil_div_ll(tokens.count, kRowThreads >> lanes_log2));
      embedding_rows<T, N><<<blocks, kRowThreads, 0, stream>>>(static_cast<const T*>(table.ptr), table.stride, rows, tokens.ptr,
                                                               tokens.wide, tokens.count, width, scale, static_cast<T*>(out.ptr),
                                                               out.stride, lanes_log2);
    };
    constexpr int kWide = 16 / sizeof(T);
    if (width % kWide == 0 && rows_aligned(table.ptr, table.stride, size, 16) && rows_aligned(out.ptr, out.stride, size, 16))
      run(Count<kWide>());
    else
      run(Count<1>());
  });
  PSB_LAUNCH_CHECK();
}

size_t embedding_grad_workspace(long long tokens, long long rows, int width) { return Workspace(tokens, rows, width).bytes; }

void embedding_grad_launch(int grad_dtype, RowsIn grad, Indices tokens, float scale, long long padding, bool accumulate,
                           int out_dtype, RowsOut out, long long rows, int width, void* workspace, cudaStream_t stream) {
  const long long n = tokens.count;
  if (n == 0 && accumulate) return;
  const Workspace at(n, rows, width);
  char* ws = static_cast<char*>(workspace);
  auto* keys = reinterpret_cast<uint32_t*>(ws + at.key_a);
  auto* pos = reinterpret_cast<uint32_t*>(ws + at.pos_a);
  auto* touched = n == 0 || accumulate ? nullptr : reinterpret_cast<unsigned char*>(ws + at.touched);
  auto* partial = reinterpret_cast<float*>(ws + at.partial);
  if (n > 0) {
    const int bits = bits_for((unsigned long long)rows), passes = (bits + 9) / 10, pass_bits = (bits + passes - 1) / passes;
    launch_cluster(embedding_order, sort_blocks(n), sort_smem(1 << pass_bits), stream, tokens.ptr, tokens.wide, n, rows, padding,
                   pass_bits, passes, keys, pos, reinterpret_cast<uint32_t*>(ws + at.key_b),
                   reinterpret_cast<uint32_t*>(ws + at.pos_b), touched);
  }
  const int in_size = dtype_size(grad_dtype), out_size = dtype_size(out_dtype), chunk = chunk_of(n);
  auto run = [&](auto t, auto o) {
    using T = decltype(t);
    using O = decltype(o);
    auto with = [&](auto per) {
      constexpr int N = decltype(per)::value;
      O* dst = static_cast<O*>(out.ptr);
      if (!accumulate) {
        zero_rows<O, N><<<grid_x(ceil_div_ll(rows, 8)), 256, 0, stream>>>(touched, rows, width, dst, out.stride);
        PSB_LAUNCH_CHECK();
      }
      if (n == 0) return;
      const unsigned chunks = grid_x(ceil_div_ll(n, chunk));
      const dim3 sums(chunks, unsigned(ceil_div(width, kSumThreads * N)));
      sum_runs<T, O, N><<<sums, kSumThreads, 0, stream>>>(static_cast<const T*>(grad.ptr), grad.stride, keys, pos, n, uint32_t(rows),
                                                          width, scale, accumulate, dst, out.stride, chunk, partial);
      PSB_LAUNCH_CHECK();
      const dim3 joins(chunks, unsigned(ceil_div(width, 32 * N)));
      join_runs<O, N><<<joins, kJoinWarps * 32, 0, stream>>>(keys, n, uint32_t(rows), width, scale, accumulate, dst, out.stride,
                                                             chunk, partial);
      PSB_LAUNCH_CHECK();
    };
    constexpr int kWide = 16 / sizeof(T);
    if (width % kWide == 0 && rows_aligned(grad.ptr, grad.stride, in_size, 16) && rows_aligned(out.ptr, out.stride, out_size, 16))
      with(Count<kWide>());
    else
      with(Count<1>());
  };
  with_type(grad_dtype, [&](auto t) {
    if (out_dtype == grad_dtype) run(t, t);
    else run(t, float());
  });
}

}  // namespace psb
