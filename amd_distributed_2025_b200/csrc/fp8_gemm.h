// Block-scaled fp8 GEMM launcher (see fp8_gemm_sm100.cu).  Counterpart of the stand-alone
// fp8 template in the reference tree (all2all/hip.py:17-59), which serves neither task.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "status.h"

namespace b200 {

struct Fp8GemmArgs {
  const void* a;         // [M, K] e4m3, row-major (K contiguous)
  const void* b;         // [N, K] e4m3, row-major
  const float* a_scale;  // one scale per row of A and 128-wide K block
  const float* b_scale;  // one scale per 128 x 128 block of B
  void* c;               // [M, N] bf16 row-major
  int M, N, K;
  long long as_stride_m, as_stride_k, bs_stride_n, bs_stride_k;  // element strides of the scale tensors
  uint64_t timeout_ns;
  StatusWord* status;  // mapped host memory: where a kernel that gave up on a wait leaves its record
  int sms;
};

// Shared memory of a CTA (it takes all of the tensor memory).
int fp8_gemm_smem(int bn, int splits);

// The tile width and the pairs that share a tile's K, as planned for a problem (for tests).
struct Fp8GemmPlan {
  int bn, splits;
};
Fp8GemmPlan fp8_gemm_plan(int M, int N, int K, int sms);

cudaError_t launch_fp8_gemm(const Fp8GemmArgs& args, cudaStream_t stream);

// The same product for the rows of many experts (see fp8_grouped_sm100.cu): row r of A in [offsets[e], offsets[e + 1]) is
// multiplied by expert e's B.
struct Fp8GroupedArgs {
  const void* a;          // [M, K] e4m3, row-major
  const void* b;          // [E, N, K] e4m3, row-major
  const float* a_scale;   // [M, ceil(K / 128)]
  const float* b_scale;   // [E, ceil(N / 128), ceil(K / 128)]
  const int32_t* offsets; // [E + 1], device memory; cut off at 0 and M, refused where they give more than M rows; one
                          // below another in front of it counts as that
  void* c;                // [M, N] bf16 row-major
  int M, N, K, experts;
  long long as_stride_m, as_stride_k, bs_stride_e, bs_stride_n, bs_stride_k;  // element strides of the scale tensors
  bool zero_rest;         // rows of C in front of offsets[0] and behind offsets[E] are zeroed, else left as they were
  uint64_t timeout_ns;
  StatusWord* status;
  int sms;
};
constexpr int kGroupedMaxExperts = 1024;  // their tables lie in shared memory
// Tokens of a tile as planned for a problem, and the shared memory of a CTA with such tiles (for tests).
int fp8_grouped_tile(int M, int experts);
int fp8_grouped_smem(int tile, int experts);
// Local memory of a thread: anything but 0 is registers that did not suffice, in the loop as a rule.
int fp8_grouped_local_bytes(int tile);
cudaError_t launch_fp8_grouped_gemm(const Fp8GroupedArgs& args, cudaStream_t stream);

// Self-test of the bounded wait: one warp waits for a barrier that nothing signals and leaves its record.
cudaError_t launch_fp8_wait_selftest(StatusWord* status, uint64_t timeout_ns, cudaStream_t stream);

}  // namespace b200
