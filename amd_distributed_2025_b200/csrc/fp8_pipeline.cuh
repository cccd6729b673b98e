// What the fp8 GEMM kernels share: their tensor-core instruction, the bounded wait of their pipelines (Params has
// `timeout_ns` and `status`), packed arithmetic.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "signal.cuh"
#include "sm100_ptx.cuh"
#include "status.h"

namespace b200 {
namespace fp8 {

// Instruction descriptor of tcgen05.mma.kind::f8f6f4 with e4m3 A and B (both K-major) and fp32
// accumulation: bits [4,6) D format (1 = f32), [7,10) A format (0 = e4m3), [10,13) B format,
// [17,23) N >> 3, [24,29) M >> 4.
__device__ __forceinline__ uint32_t make_idesc_e4m3_f32(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void umma_fp8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// `detail` (not 0) tells which wait it was that expired: a hundred for the kind of barrier, plus its index.
template <typename Params>
__device__ __forceinline__ bool fp8_wait(uint32_t bar, uint32_t parity, volatile int* abort, const Params& p, int detail) {
  uint64_t t0 = 0;  // (the clock takes longer to read than most waits last)
  for (uint32_t spins = 1; !ptx::mbar_try_wait(bar, parity); ++spins) {
    if ((spins & 255u) == 0) {
      if (*abort) return false;
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > p.timeout_ns) {
        *abort = detail;
        return false;
      }
    }
  }
  return true;
}

// A CTA in which a wait expired says so on its way out (every warp that knows of it does, and one is enough): what it
// computed is of no use.
template <typename Params>
__device__ __forceinline__ void record_expired(const Params& p, int detail) {
  if (p.status != nullptr && reinterpret_cast<volatile StatusWord*>(p.status)->code == STATUS_OK)
    store_status(p.status, STATUS_TIMEOUT, PHASE_GEMM_PIPELINE, -1, detail, 0, 0);
}

// acc[0..1] += v[0..1] * s
__device__ __forceinline__ void fma2(float2& acc, uint32_t v0, uint32_t v1, float2 ss) {
  const float2 v = make_float2(__uint_as_float(v0), __uint_as_float(v1));
  // (volatile: not before the wait for the tensor memory load that brings v)
  asm volatile("fma.rn.f32x2 %0, %1, %2, %0;"
      : "+l"(reinterpret_cast<unsigned long long&>(acc))
      : "l"(reinterpret_cast<const unsigned long long&>(v)), "l"(reinterpret_cast<const unsigned long long&>(ss)));
}

__device__ __forceinline__ void ld_shared_f4(float* to, uint32_t from) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(to[0]), "=f"(to[1]), "=f"(to[2]), "=f"(to[3])
               : "r"(from)
               : "memory");
}

__device__ __forceinline__ uint32_t pack2(float2 f) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace fp8
}  // namespace b200
