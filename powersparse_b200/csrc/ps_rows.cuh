// Device helpers of the row operators: element types, vectors of a row, and the
// widest access that the operands allow.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>

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

// Words of B bytes: what one load or store moves.
template <int B> struct WordOf;
template <> struct WordOf<16> { using type = uint4; };
template <> struct WordOf<8> { using type = uint2; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<2> { using type = uint16_t; };
template <int B> using Word = typename WordOf<B>::type;

// N consecutive elements of a row, moved in words of at most 16 bytes.
template <typename T, int N>
struct Pack {
  static constexpr int kWord = N * int(sizeof(T)) < 16 ? N * int(sizeof(T)) : 16;
  static constexpr int kWords = N * int(sizeof(T)) / kWord;
  union {
    Word<kWord> w[kWords];
    unsigned char bytes[N * sizeof(T)];
  };
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __ldg(reinterpret_cast<const Word<kWord>*>(p) + i);
  }
  // For memory that this kernel also writes.
  __device__ __forceinline__ void load_rw(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = *(reinterpret_cast<const Word<kWord>*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<Word<kWord>*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = Word<kWord>{};
  }
  __device__ __forceinline__ float get(int i) const { return to_float(reinterpret_cast<const T*>(bytes)[i]); }
  __device__ __forceinline__ void set(int i, float x) { reinterpret_cast<T*>(bytes)[i] = from_float<T>(x); }
};

__device__ __forceinline__ long long index_at(const void* p, bool wide, long long i) {
  return wide ? __ldg(static_cast<const long long*>(p) + i) : (long long)__ldg(static_cast<const int*>(p) + i);
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

// log2 of the smallest power of two >= v.
inline int log2_up(long long v) {
  int b = 0;
  while ((1LL << b) < v) ++b;
  return b;
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
