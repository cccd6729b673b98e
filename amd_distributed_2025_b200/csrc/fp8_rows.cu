// Rows for the fp8 tensor cores: e4m3 values with one fp32 scale for each row and 128 columns, the form in which the
// block-scaled GEMMs take their left operand.
//
//   norm      h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * weight
//   silu_mul  y = g / (1 + exp(-g)) * u,  x = [g | u]
//   both      scale = max(max |y| over the block, 1e-30) / 448,  q = e4m3(y / scale), to nearest even
//
// Everything is fp32 between the loads and the conversion.  The maximum carries NaN on (max.NaN), so that a block with a
// NaN has a NaN for its scale and nothing but NaN in it; the floor of 1e-30 keeps the reciprocal of an empty block finite.
// y is multiplied by the reciprocal of the scale, rounded once: a value within 2^-23 of the border between two e4m3 values
// may fall to the other side of it than after a division.
//
// A lane holds eight neighbouring columns of a block (sixteen lanes to a block) where rows are whole aligned 16-byte
// vectors, else every 32nd column (a warp to a block): 2-byte loads and 1-byte stores of a warp stay neighbours.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "fp8_rows.h"
#include "moe_common.cuh"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

using moe::from_f32;
using moe::to_f32;

constexpr int kBlockCols = 128;
constexpr int kNormThreads = 512;  // the most of a team: N = 8 vectors a lane leave 128 registers
constexpr float kE4m3Max = 448.f;
constexpr float kLeastMax = 1e-30f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void unpack8(const int4& raw, float* f, __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = __half22float2(h[j]);
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
}
__device__ __forceinline__ void unpack8(const int4& raw, float* f, __nv_bfloat16) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = __bfloat1622float2(h[j]);
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
}

// Eight values of T as they lie in memory.
template <typename T> struct Raw8 { int4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = __ldcg(reinterpret_cast<const int4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void to_floats(const Raw8<T>& r, float* f) {
  if constexpr (sizeof(T) == 2) {
    unpack8(r.v[0], f, T());
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __int_as_float(r.v[i].x);
      f[4 * i + 1] = __int_as_float(r.v[i].y);
      f[4 * i + 2] = __int_as_float(r.v[i].z);
      f[4 * i + 3] = __int_as_float(r.v[i].w);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* f) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<int4*>(p)[i] = moe::pack_vec<T>(f + i * (16 / (int)sizeof(T)));
}

// How the columns of a row lie in the lanes.  A unit is what a lane has of a block: unit u of a team of lanes.
template <bool VEC>
struct Lanes {
  static constexpr int kPer = VEC ? 8 : 4;           // columns of a unit
  static constexpr int kUnits = kBlockCols / kPer;   // lanes that share a block
  // the first column of unit u, and of element e the distance from it
  static __device__ __forceinline__ int64_t column(int u) {
    return VEC ? (int64_t)u * 8 : (int64_t)(u >> 5) * kBlockCols + (u & 31);
  }
  static __device__ __forceinline__ int step(int e) { return VEC ? e : 32 * e; }

  template <typename T>
  static __device__ __forceinline__ void load(const T* row, int u, int cols, float* f) {
    const int64_t c = column(u);
    if constexpr (VEC) {
      if (c < cols) {
        to_floats<T>(load8<T>(row + c), f);
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) f[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) f[e] = c + step(e) < cols ? to_f32(row[c + step(e)]) : 0.f;
    }
  }
  template <typename T>
  static __device__ __forceinline__ void store(T* row, int u, int cols, const float* f) {
    const int64_t c = column(u);
    if constexpr (VEC) {
      if (c < cols) store8<T>(row + c, f);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (c + step(e) < cols) row[c + step(e)] = from_f32<T>(f[e]);
    }
  }
  // Block scale and e4m3 values of one unit (every lane of the warp takes part; columns behind the row hold zeros).
  static __device__ __forceinline__ void quantise(uint8_t* q_row, float* scale_row, int u, int cols, const float* y) {
    float most = fabsf(y[0]);
#pragma unroll
    for (int e = 1; e < kPer; ++e) most = max_nan(most, fabsf(y[e]));
#pragma unroll
    for (int o = kUnits / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float scale = __fdiv_rn(max_nan(most, kLeastMax), kE4m3Max);
    const float inverse = __frcp_rn(scale);
    const int64_t c = column(u);
    if (c >= cols) return;
    if (u % kUnits == 0) scale_row[u / kUnits] = scale;
    if constexpr (VEC) {
      uint2 packed;
      uint16_t* half = reinterpret_cast<uint16_t*>(&packed);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        half[e] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * e] * inverse, y[2 * e + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<uint2*>(q_row + c) = packed;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (c + step(e) < cols) q_row[c + step(e)] = __nv_cvt_float_to_fp8(y[e] * inverse, __NV_SATFINITE, __NV_E4M3);
    }
  }
};

}  // namespace

// A team of blockDim.x lanes takes a row and keeps it in registers, N units a lane: it is read once.  With blockDim.y > 1
// (short rows) a team is a warp, and the CTA has several.
template <typename T, typename W, bool VEC, int N>
__global__ void __launch_bounds__(kNormThreads) rms_norm_fp8_kernel(const RmsNormFp8Args p) {
  using L = Lanes<VEC>;
  __shared__ float sums[32];
  const int lanes = (int)blockDim.x;
  const int blocks = (p.cols + kBlockCols - 1) / kBlockCols;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < p.rows; row += (int64_t)gridDim.x * blockDim.y) {
    float h[N][L::kPer];
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) L::load(x, i * lanes + (int)threadIdx.x, p.cols, h[i]);
    if (p.residual != nullptr) {
      const T* r = reinterpret_cast<const T*>(p.residual) + row * p.residual_stride;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float f[L::kPer];
        L::load(r, i * lanes + (int)threadIdx.x, p.cols, f);
#pragma unroll
        for (int e = 0; e < L::kPer; ++e) h[i][e] += f[e];
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < L::kPer; ++e) sum = fmaf(h[i][e], h[i][e], sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lanes > 32) {  // (a CTA with a team of several warps has one team)
      if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
      __syncthreads();
      sum = (int)(threadIdx.x & 31) < lanes / 32 ? sums[threadIdx.x & 31] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncthreads();
    }
    if (p.total != nullptr) {
      T* total = reinterpret_cast<T*>(p.total) + row * p.total_stride;
#pragma unroll
      for (int i = 0; i < N; ++i) L::store(total, i * lanes + (int)threadIdx.x, p.cols, h[i]);
    }
    const float rstd = rsqrtf(sum / (float)p.cols + p.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = i * lanes + (int)threadIdx.x;
      float w[L::kPer];
      L::load(reinterpret_cast<const W*>(p.weight), u, p.cols, w);
#pragma unroll
      for (int e = 0; e < L::kPer; ++e) h[i][e] = h[i][e] * rstd * w[e];
      if (p.normed != nullptr) L::store(reinterpret_cast<T*>(p.normed) + row * p.cols, u, p.cols, h[i]);
      L::quantise(reinterpret_cast<uint8_t*>(p.q) + row * p.cols, p.scale + row * blocks, u, p.cols, h[i]);
    }
  }
}

// A team of blockDim.x lanes takes a row, a unit a lane at a time; a CTA has blockDim.y teams.  Teams are whole warps, or
// (vectors only) halves of one.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) silu_mul_fp8_kernel(const SiluMulFp8Args p) {
  using L = Lanes<VEC>;
  const int lanes = (int)blockDim.x;
  const int blocks = (p.cols + kBlockCols - 1) / kBlockCols;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  // all lanes of a warp make the same number of rounds: they meet in the maximum
  for (int64_t row0 = (int64_t)blockIdx.x * blockDim.y; row0 < p.rows; row0 += (int64_t)gridDim.x * blockDim.y) {
    const int64_t row = row0 + threadIdx.y;
    const int cols = row < p.rows ? p.cols : 0;
    const T* gate = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
    for (int u = (int)threadIdx.x; u < blocks * L::kUnits; u += lanes) {
      float g[L::kPer], v[L::kPer];
      L::load(gate, u, cols, g);
      L::load(gate + p.cols, u, cols, v);
#pragma unroll
      for (int e = 0; e < L::kPer; ++e) g[e] = __fdividef(g[e], 1.f + __expf(-g[e])) * v[e];
      L::quantise(reinterpret_cast<uint8_t*>(p.q) + row * p.cols, p.scale + row * blocks, u, cols, g);
    }
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename P>
cudaError_t launch_teams(void (*kernel)(P), int64_t grid, dim3 block, cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, typename W, bool VEC>
cudaError_t norm_units(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  const int units = (p.cols + kBlockCols - 1) / kBlockCols * Lanes<VEC>::kUnits;
  constexpr int kShort = 4 * 32;  // units of a row that one warp takes
  dim3 block;
  int n;
  if (units <= kShort) {
    n = (units + 31) / 32;
    block = dim3(32, 8);
  } else {
    n = std::max(2, (units + kNormThreads - 1) / kNormThreads);
    block = dim3((unsigned)(((units + n - 1) / n + 31) / 32 * 32), 1);
  }
  const int64_t grid = std::min<int64_t>((p.rows + block.y - 1) / block.y, 1 << 30);
  auto go = [&](auto kernel) { return launch_teams(kernel, grid, block, stream, p); };
  if (n <= 1) return go(rms_norm_fp8_kernel<T, W, VEC, 1>);
  if (n <= 2) return go(rms_norm_fp8_kernel<T, W, VEC, 2>);
  if (n <= 4) return go(rms_norm_fp8_kernel<T, W, VEC, 4>);
  if (n <= 8) return go(rms_norm_fp8_kernel<T, W, VEC, 8>);
  if constexpr (!VEC) return go(rms_norm_fp8_kernel<T, W, VEC, 16>);
  return cudaErrorInvalidValue;
}

template <typename T, typename W>
cudaError_t norm_typed(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  const bool vec = p.cols % 8 == 0 && p.x_stride % 8 == 0 && p.residual_stride % 8 == 0 && p.total_stride % 8 == 0 &&
                   aligned16(p.x) && aligned16(p.residual) && aligned16(p.weight) && aligned16(p.total);
  return vec ? norm_units<T, W, true>(p, sms, stream) : norm_units<T, W, false>(p, sms, stream);
}

template <typename T>
cudaError_t norm_weight(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  if (p.weight_dtype == p.dtype) return norm_typed<T, T>(p, sms, stream);
  return p.weight_dtype == 2 ? norm_typed<T, float>(p, sms, stream) : cudaErrorInvalidValue;
}

template <typename T>
cudaError_t silu_typed(const SiluMulFp8Args& p, int sms, cudaStream_t stream) {
  const bool vec = p.cols % 8 == 0 && p.x_stride % 8 == 0 && aligned16(p.x);
  const int units = (p.cols + kBlockCols - 1) / kBlockCols * (vec ? 16 : 32);
  // the largest team of which the least is idle in the last round
  int lanes = 32;
  for (int l = 64; l <= 256; l *= 2)
    if ((units + l - 1) / l * l <= (units + lanes - 1) / lanes * lanes) lanes = l;
  if (units <= 16) lanes = 16;
  const dim3 block((unsigned)lanes, (unsigned)(256 / lanes));
  const int64_t grid = std::min<int64_t>((p.rows + block.y - 1) / block.y, 1 << 30);
  return vec ? launch_teams(silu_mul_fp8_kernel<T, true>, grid, block, stream, p)
             : launch_teams(silu_mul_fp8_kernel<T, false>, grid, block, stream, p);
}

}  // namespace

cudaError_t launch_rms_norm_fp8(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  if (p.rows < 0 || p.cols < 1 || p.cols > kMaxNormCols) return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  switch (p.dtype) {
    case 0: return norm_weight<__half>(p, sms, stream);
    case 1: return norm_weight<__nv_bfloat16>(p, sms, stream);
    case 2: return norm_weight<float>(p, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_silu_mul_fp8(const SiluMulFp8Args& p, int sms, cudaStream_t stream) {
  if (p.rows < 0 || p.cols < 1) return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  switch (p.dtype) {
    case 0: return silu_typed<__half>(p, sms, stream);
    case 1: return silu_typed<__nv_bfloat16>(p, sms, stream);
    case 2: return silu_typed<float>(p, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200
