// Launchers of the kernels that sort tokens by expert and bring their rows back (see moe_sort.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

constexpr int kSortMaxTopk = 32;       // a lane of a warp for each entry of a token
constexpr int kSortMaxExperts = 8192;  // counts of all experts lie in shared memory

struct SortTokensArgs {
  const void* x;        // [T, H] rows of row_bytes, x_stride bytes apart
  const void* indices;  // [T, k] int32 or int64 (wide_ids), contiguous
  const float* scale;   // [T, scale_cols], scale_stride elements apart, or null
  void* rows;           // [T k, H]
  float* rows_scale;    // [T k, scale_cols]
  int32_t* offsets;     // [E + 1]
  int32_t* row_of;      // [T, k]
  int32_t* work;        // sort_tokens_work() words, or null where that is 0
  int64_t x_stride, scale_stride;
  int64_t row_bytes;
  int32_t tokens, k, experts, scale_cols;
  int32_t wide_ids, elem_bytes;
};
// Words of workspace that a problem needs (0: one launch counts and copies).
int64_t sort_tokens_work(int64_t tokens, int k, int experts);
cudaError_t launch_sort_tokens(const SortTokensArgs& args, int sms, cudaStream_t stream);

struct UnsortTokensArgs {
  const void* rows;       // [R, H], rows_stride bytes apart
  const float* weights;   // [T, k], or null: all ones
  const int32_t* row_of;  // [T, k]
  void* out;              // [T, H] contiguous
  int64_t rows_stride, num_rows;
  int32_t tokens, k, hidden;
  int dtype;              // 0 fp16, 1 bf16, 2 fp32
};
cudaError_t launch_unsort_tokens(const UnsortTokensArgs& args, int sms, cudaStream_t stream);

struct UnsortBackwardArgs {
  const void* grad;        // [T, H], grad_stride bytes apart
  const void* rows;        // [R, H], rows_stride bytes apart; null where grad_weights is
  const float* weights;    // [T, k], or null: all ones
  const int32_t* row_of;   // [T, k]
  const int32_t* end;      // the number of rows that entries have (offsets + E)
  void* grad_rows;         // [R, H] contiguous, or null
  float* grad_weights;     // [T, k], or null
  int64_t grad_stride, rows_stride, num_rows;
  int32_t tokens, k, hidden;
  int dtype;
};
cudaError_t launch_unsort_tokens_backward(const UnsortBackwardArgs& args, int sms, cudaStream_t stream);

}  // namespace b200
