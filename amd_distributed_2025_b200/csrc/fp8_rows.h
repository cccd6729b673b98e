// Launchers of the kernels that leave e4m3 rows with block scales (see fp8_rows.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

constexpr int kMaxNormCols = 32768;  // a row is held in the registers of one CTA
constexpr int kMaxSiluCols = INT32_MAX - 8192;  // (a team's last round may reach up to 4096 columns behind a row's last block)

// dtype: 0 fp16, 1 bf16, 2 fp32 (x, residual, total, normed; the weight has its own).  Rows are contiguous; strides in
// elements from row to row.  q [rows, cols] and scale [rows, ceil(cols / 128)] are contiguous.
struct RmsNormFp8Args {
  const void* x;
  const void* residual;  // or null
  const void* weight;
  void* total;   // x + residual, or null
  void* normed;  // the normed rows in x's type, contiguous, or null
  void* q;
  float* scale;
  int64_t rows;
  int32_t cols;
  int64_t x_stride, residual_stride, total_stride;
  float eps;
  int dtype, weight_dtype;
};
cudaError_t launch_rms_norm_fp8(const RmsNormFp8Args& args, int sms, cudaStream_t stream);

// x [rows, 2 cols]: gates, then the values that they multiply.
struct SiluMulFp8Args {
  const void* x;
  void* q;
  float* scale;
  int64_t rows;
  int32_t cols;
  int64_t x_stride;
  int dtype;
};
cudaError_t launch_silu_mul_fp8(const SiluMulFp8Args& args, int sms, cudaStream_t stream);

}  // namespace b200
