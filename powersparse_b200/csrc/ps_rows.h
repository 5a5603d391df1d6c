// Launchers of the operators on rows chosen by an index that the model makes: the
// embedding (ps_embedding.cu) and the experts' router, dispatch and combine
// (ps_experts.cu).  Arguments are checked by the callers in ps_capi.cu.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace psb {

// A row-major matrix of rows of `width` elements, `stride` elements apart.
struct RowsIn {
  const void* ptr;
  long long stride;
};
struct RowsOut {
  void* ptr;
  long long stride;
};

// Indices as the caller holds them: 32 or 64 bits wide.
struct Indices {
  const void* ptr;
  bool wide;
  long long count;
};

constexpr int kMaxExperts = 1024;  // one digit of the expert order (ps_index_sort.cuh)
constexpr int kMaxTopK = 32;       // a warp keeps one choice a lane

void embedding_launch(int dtype, RowsIn table, long long rows, int width, Indices tokens, float scale, RowsOut out,
                      cudaStream_t stream);

size_t embedding_grad_workspace(long long tokens, long long rows, int width);
void embedding_grad_launch(int grad_dtype, RowsIn grad, Indices tokens, float scale, long long padding, bool accumulate,
                           int out_dtype, RowsOut out, long long rows, int width, void* workspace, cudaStream_t stream);

void route_launch(int dtype, RowsIn logits, int tokens, int experts, int top_k, bool normalize, float* weights, int* chosen,
                  cudaStream_t stream);
void route_grad_launch(int dtype, const float* grad_weights, RowsIn logits, const float* weights, const int* chosen, int tokens,
                       int experts, int top_k, bool normalize, RowsOut grad_logits, cudaStream_t stream);

// Rows that `slots` places can fill at the most when every expert begins at a multiple of `align`.
long long dispatch_rows(long long slots, int experts, int align);
void dispatch_launch(int dtype, RowsIn x, Indices chosen, int tokens, int top_k, int experts, int align, int width, RowsOut out,
                     long long row_count, bool zero_tail, int* position, int* offsets, int* counts, cudaStream_t stream);
void combine_launch(int dtype, RowsIn y, long long rows, const int* position, const float* weights, RowsIn add, int tokens,
                    int top_k, int width, RowsOut out, cudaStream_t stream);
void combine_grad_launch(int dtype, RowsIn grad, RowsIn y, long long rows, const int* position, const int* offsets,
                         const int* counts, int experts, const float* weights, int tokens, int top_k, int width, RowsOut grad_y,
                         bool zero_tail, float* grad_weights, cudaStream_t stream);

}  // namespace psb
