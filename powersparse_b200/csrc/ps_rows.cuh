// Device helpers of the row operators: element types, vectors of a row, and the
// widest access that the operands allow.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <utility>

#include "powersparse_b200.h"
#include "ps_common.cuh"
#include "ps_rows.h"

namespace psb {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
// One rounding, to nearest even, where a result leaves the 32-bit registers.
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// An element's bits as the word of its size.
__device__ __forceinline__ float from_bits(uint32_t w, float) { return __uint_as_float(w); }
__device__ __forceinline__ __nv_bfloat16 from_bits(uint16_t w, __nv_bfloat16) { return __ushort_as_bfloat16(w); }
__device__ __forceinline__ __half from_bits(uint16_t w, __half) { return __ushort_as_half(w); }
__device__ __forceinline__ uint32_t to_bits(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint16_t to_bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
__device__ __forceinline__ uint16_t to_bits(__half x) { return __half_as_ushort(x); }

// Words of B bytes: what one load or store moves.
template <int B> struct WordOf;
template <> struct WordOf<16> { using type = uint4; };
template <> struct WordOf<8> { using type = uint2; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<2> { using type = uint16_t; };
template <int B> using Word = typename WordOf<B>::type;

// What a thread holds of a row: N elements as N / W words of W, the words `step`
// columns apart (the threads that share the row stand side by side).  Where rows begin
// at multiples of 16 bytes W = N and a word is 16 bytes of T; where they do not, W is
// smaller and the thread still has the same bytes in flight.
template <typename T, int N, int W>
struct Pack {
  static constexpr int kWordBytes = W * int(sizeof(T));
  static constexpr int kPart = kWordBytes < 16 ? kWordBytes : 16;
  static constexpr int kParts = kWordBytes / kPart;
  using Part = Word<kPart>;
  using Element = Word<int(sizeof(T))>;
  union {
    Part w[N / W][kParts];
    unsigned char bytes[N * sizeof(T)];
  };
  // The words at columns c, c + step, ... of a row, as far as they lie below `width`
  // (a word lies below it or not as a whole).
  __device__ __forceinline__ void load(const T* row, int c, int step, int width) {
#pragma unroll
    for (int i = 0; i < N / W; ++i)
      if (c + i * step < width)
#pragma unroll
        for (int k = 0; k < kParts; ++k) w[i][k] = *(reinterpret_cast<const Part*>(row + c + i * step) + k);
  }
  __device__ __forceinline__ void store(T* row, int c, int step, int width) const {
#pragma unroll
    for (int i = 0; i < N / W; ++i)
      if (c + i * step < width)
#pragma unroll
        for (int k = 0; k < kParts; ++k) reinterpret_cast<Part*>(row + c + i * step)[k] = w[i][k];
  }
  // For what this kernel does not read again: it makes room in the caches first (2% of
  // the time of a large lookup or dispatch; the same for loads gained nothing).
  __device__ __forceinline__ void store_once(T* row, int c, int step, int width) const {
#pragma unroll
    for (int i = 0; i < N / W; ++i)
      if (c + i * step < width)
#pragma unroll
        for (int k = 0; k < kParts; ++k) __stcs(reinterpret_cast<Part*>(row + c + i * step) + k, w[i][k]);
  }
  // The same elements one at a time, for rows that do not allow the words.
  __device__ __forceinline__ void load_elements(const T* row, int c, int step, int width) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int at = c + e / W * step + e % W;
      if (at < width) reinterpret_cast<Element*>(bytes)[e] = *reinterpret_cast<const Element*>(row + at);
    }
  }
  __device__ __forceinline__ void store_elements(T* row, int c, int step, int width) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int at = c + e / W * step + e % W;
      if (at < width) reinterpret_cast<Element*>(row + at)[0] = reinterpret_cast<const Element*>(bytes)[e];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N / W; ++i)
#pragma unroll
      for (int k = 0; k < kParts; ++k) w[i][k] = Part{};
  }
  // Single elements stay in registers of their own; in `bytes` two of 16 bits would share one.
  __device__ __forceinline__ float get(int e) const {
    if constexpr (W == 1) return to_float(from_bits(w[e][0], T()));
    else return to_float(reinterpret_cast<const T*>(bytes)[e]);
  }
  __device__ __forceinline__ void set(int e, float x) {
    if constexpr (W == 1) w[e][0] = to_bits(from_float<T>(x));
    else reinterpret_cast<T*>(bytes)[e] = from_float<T>(x);
  }
};

// Every kernel of the row operators is launched so that it may start while the one before
// it in the stream still ends, which hides the launch (a router of 8.3 us: 7.8 us a call
// in a row of them, 10.3 without).  It waits here before it touches any memory, and reads
// with plain loads: the read-only path may hold lines from before the wait, so no pointer
// is __restrict__ and nothing goes by __ldg.  let_next_start() in a kernel whose
// successor is one of these lets the successor's blocks take their places as soon as
// every block of the kernel has its own.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
void launch_after(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  PSB_CUDA(cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...));
}

__device__ __forceinline__ long long index_at(const void* p, bool wide, long long i) {
  return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

inline int dtype_size(int dtype) { return dtype == PS_F32 ? 4 : 2; }

// Whether rows at `ptr`, `stride` elements of `size` bytes apart, all begin at a multiple of `bytes`.
inline bool rows_aligned(const void* ptr, long long stride, int size, int bytes) {
  return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && (stride * size) % bytes == 0;
}

// How the threads of a row share it: N elements a thread and turn, in words of W.  S = 32:
// a warp takes 32 * N columns, its words 32 apart, so that the distances are constants;
// S = 0: for rows that less than a warp shares, the words stand as far apart as there
// are threads.
template <int N_, int W_, int S_>
struct Shape {
  static constexpr int N = N_, W = W_, S = S_;
  // For 32 threads at least where the words are apart by a constant.
  static constexpr int kLeastLanesLog2 = S && W != N ? 5 : 0;
};

// First column of thread t of the row's 2^k lanes in its first turn, and the distance of its words.
template <int N, int W, int S>
__device__ __forceinline__ int first_column(int t) {
  return S ? t / 32 * 32 * N + t % 32 * W : t * W;
}
template <int W, int S>
__device__ __forceinline__ int word_step(int lanes) {
  return S ? S * W : lanes * W;
}

// Calls f(Shape) for rows of `width` elements of type T: words of 16 bytes where
// fits(16) says that every operand's rows allow them, of 4 bytes where fits(4) does,
// else single elements, four words a thread.  fits need not look at the width.
template <typename T, typename Fits, typename F>
void with_shape(int width, Fits&& fits, F&& f) {
  constexpr int kSize = int(sizeof(T)), kN = 16 / kSize, kHalf = 4 / kSize;
  if (width % kN == 0 && fits(16)) {
    f(Shape<kN, kN, 32>());
  } else if (kHalf > 1 && width % kHalf == 0 && fits(4)) {
    if (width > 16 * kN) f(Shape<kN, kHalf, 32>());
    else f(Shape<kN, kHalf, 0>());
  } else {
    if (width > 64) f(Shape<4, 1, 32>());
    else f(Shape<4, 1, 0>());
  }
}

// log2 of the smallest power of two >= v.
inline int log2_up(long long v) {
  int b = 0;
  while ((1LL << b) < v) ++b;
  return b;
}

// log2 of the threads that share a row of `width` elements, `n` of them a thread and
// turn: as many as give a row `turns` turns.  More, while the `rows` leave most of the
// GPU without threads; fewer where the last turn would leave more than a fifth of the
// work empty and the rows fill the GPU's threads twice over.
inline int row_lanes(int width, int n, int turns, int least_log2, long long rows) {
  int lanes = std::min(8, std::max(least_log2, log2_up(ceil_div(ceil_div(width, n), turns))));
  while (lanes < 8 && rows << lanes < 256LL * device_sms() && n << lanes < width) ++lanes;
  while (lanes > std::max(5, least_log2) && rows << lanes >= 4096LL * device_sms() &&
         (long long)ceil_div(width, n << lanes) * (n << lanes) * 4 > 5LL * width)
    --lanes;
  return lanes;
}

inline unsigned grid_x(long long blocks) {
  if (blocks > 0x7fffffffLL) throw std::invalid_argument("too many rows for one launch");
  return unsigned(blocks);
}

// Calls f(T()) with the element type of `dtype`.
template <typename F>
void with_type(int dtype, F&& f) {
  if (dtype == PS_F32) f(float());
  else if (dtype == PS_BF16) f(__nv_bfloat16());
  else f(__half());
}

}  // namespace psb
