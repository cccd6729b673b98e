// Rows for the fp8 tensor cores: e4m3 values with one fp32 scale for each row and 128 columns, the form in which the
// block-scaled GEMMs take their left operand.
//
//   norm      h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * weight
//   silu_mul  y = g / (1 + exp(-g)) * u,  x = [g | u]
//   both      scale = max(max |y| over the block, 1e-30) / 448,  q = e4m3(y / scale), to nearest even
//
// Everything is fp32 between the loads and the conversion.  The maximum carries NaN on (max.NaN), so that a block with a
// NaN has a NaN for its scale and nothing but NaN in it; the floor of 1e-30 keeps the reciprocal of an empty block finite.
// The quotient by the scale is a product with the scale's reciprocal (approximate, to a step of fp32) and one step by its
// remainder (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990), in pairs.  Of 94
// million quotients, a third of them within two steps of a border between two e4m3 values, all come out as a division's
// do; the product alone sends 2.8 million to the other side.  What the step takes, us: 16384 x 4096 bf16 73 as before with a
// residual, 48 to 51 without (with rounded reciprocals, value by value, 55); activation, 32761 x 2048 bf16, 52 to 53, and 50
// with its gates in pairs too.
//
// A lane holds 16 neighbouring columns of a block (eight lanes to a block) where rows are whole aligned 32-byte pieces, eight
// (sixteen lanes) where they are 16-byte pieces, else every 32nd column (a warp to a block), so that 2-byte loads and
// 1-byte stores of a warp stay neighbours.
//
// Both are bound by memory where rows are whole pieces.  What that took is few instructions a value: blocks found by
// eight lanes need three shuffles and one reciprocal for 16 values; with eight values to a lane, a division and four shuffles
// for them, and the weight out of L2 for every row, 16384 x 4096 without a residual took as long as the memory takes
// for 2.5 times the bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "fp8_rows.h"
#include "moe_common.cuh"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

using moe::from_f32;
using moe::to_f32;

constexpr int kBlockCols = 128;
// The most lanes of a team: a row that has to be read value by value wants more of them.
template <int PER> constexpr int kNormThreads = PER == 4 ? 1024 : 512;
constexpr float kE4m3Max = 448.f;
constexpr float kLeastMax = 1e-30f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_abs_nan(float a) {
  float r;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float reciprocal(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
// Two operations at once.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return r;
}

// g / (1 + exp(-g)) * u of two values, with the sign changed.  A gate below -87.3 has a sum above 2^126 and counts beside
// values near 1e36: a quarter of the sum still has a reciprocal that is a normal number.  (An exponential that is none adds
// nothing to 1.)
__device__ __forceinline__ float2 minus_silu_mul(float2 g, float2 u) {
  const float2 x = mul2(g, make_float2(-1.44269504f, -1.44269504f));  // log2(e)
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
  const float2 quarter = make_float2(0.25f, 0.25f), sum = fma2(e, quarter, quarter);
  const float2 minus_sigmoid = mul2(make_float2(reciprocal(sum.x), reciprocal(sum.y)), make_float2(-0.25f, -0.25f));
  return mul2(mul2(g, minus_sigmoid), u);
}

// W words of 32 bits from or to global memory, A (4 or 8) at a time where there are as many: the address is a multiple of as
// many bytes.
template <int W, int A>
__device__ __forceinline__ void load_words(uint32_t* w, const void* p) {
  static_assert(W % 4 == 0, "pieces of 16 or 32 bytes");
  if constexpr (W > A) {
    load_words<A, A>(w, p);
    load_words<W - A, A>(w + A, reinterpret_cast<const uint32_t*>(p) + A);
  } else if constexpr (W == 8) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  } else {
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  }
}
template <int W, int A>
__device__ __forceinline__ void store_words(void* p, const uint32_t* w) {
  if constexpr (W > A) {
    store_words<A, A>(p, w);
    store_words<W - A, A>(reinterpret_cast<uint32_t*>(p) + A, w + A);
  } else if constexpr (W == 8) {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p)
                 : "memory");
  } else if constexpr (W == 4) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    static_assert(W == 2, "8, 16 or 32 bytes");
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

__device__ __forceinline__ float2 two_floats(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 two_floats(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t two_packed(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t two_packed(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// How the columns of a row lie in the lanes.  A unit is what a lane has of a block: PER neighbouring columns (16 or 8), or, with
// PER = 4, every 32nd.
template <int PER>
struct Lanes {
  static constexpr bool kVec = PER != 4;
  static constexpr int kUnits = kBlockCols / PER;  // lanes that share a block
  static constexpr int kWords = PER / 2;           // of an access: addresses are multiples of 2 PER bytes
  static __device__ __forceinline__ int column(int u) { return kVec ? u * PER : (u >> 5) * kBlockCols + (u & 31); }

  // A unit as it lies in memory.
  template <typename T> struct Raw { uint32_t w[kVec ? PER * (int)sizeof(T) / 4 : PER]; };

  // (columns behind the row are zeros)
  template <typename T>
  static __device__ __forceinline__ Raw<T> load(const T* row, int u, int cols) {
    Raw<T> r;
    const int c = column(u);
    if constexpr (kVec) {
      if (c < cols) {
        load_words<PER * (int)sizeof(T) / 4, kWords>(r.w, row + c);
      } else {
#pragma unroll
        for (int i = 0; i < PER * (int)sizeof(T) / 4; ++i) r.w[i] = 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) r.w[e] = c + 32 * e < cols ? bits(row[c + 32 * e]) : 0u;
    }
    return r;
  }
  static __device__ __forceinline__ uint32_t bits(float v) { return __float_as_uint(v); }
  static __device__ __forceinline__ uint32_t bits(__half v) { return __half_as_ushort(v); }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }

  template <typename T>
  static __device__ __forceinline__ void floats(const Raw<T>& r, float* f) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if constexpr (sizeof(T) == 4) {
        f[e] = __uint_as_float(r.w[e]);
      } else if constexpr (kVec) {
        if (e % 2 == 0) {
          const float2 v = two_floats(r.w[e / 2], T());
          f[e] = v.x;
          f[e + 1] = v.y;
        }
      } else {
        f[e] = two_floats(r.w[e], T()).x;
      }
    }
  }
  template <typename T>
  static __device__ __forceinline__ void store(T* row, int u, int cols, const float* f) {
    const int c = column(u);
    if constexpr (kVec) {
      if (c >= cols) return;
      uint32_t w[PER * (int)sizeof(T) / 4];
#pragma unroll
      for (int i = 0; i < PER * (int)sizeof(T) / 4; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
        else w[i] = two_packed(f[2 * i], f[2 * i + 1], T());
      }
      store_words<PER * (int)sizeof(T) / 4, kWords>(row + c, w);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (c + 32 * e < cols) row[c + 32 * e] = from_f32<T>(f[e]);
    }
  }
  // Block scale and e4m3 values of one unit (every lane of the warp takes part; columns behind the row hold zeros).  It is
  // given -y: with q = -y * -1 / scale, y's remainder is -(q * scale + -y), and zeros keep their signs through all of it.
  static __device__ __forceinline__ void quantise(uint8_t* q_row, float* scale_row, int u, int cols, const float* minus_y) {
    float most = fabsf(minus_y[0]);
#pragma unroll
    for (int e = 1; e < PER; ++e) most = max_nan(most, fabsf(minus_y[e]));
    if constexpr (kUnits == 32) {
      most = warp_max_abs_nan(most);
    } else {
#pragma unroll
      for (int o = kUnits / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    most = max_nan(most, kLeastMax);
    const float scale = most * (1.f / kE4m3Max), inverse = -reciprocal(scale);  // (normal numbers: most is 1e-30 at least)
    const int c = column(u);
    if (c >= cols) return;
    if (u % kUnits == 0) scale_row[u / kUnits] = scale;
    // (0 for an infinite scale, beside which remainders would be NaN: what is finite becomes a zero)
    const float back = scale < INFINITY ? scale : 0.f;
    uint16_t two[PER / 2];
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) {
      const float2 n = make_float2(minus_y[2 * i], minus_y[2 * i + 1]), by = make_float2(inverse, inverse);
      const float2 q = mul2(n, by);
      two[i] = __nv_cvt_float2_to_fp8x2(fma2(fma2(q, make_float2(back, back), n), by, q), __NV_SATFINITE, __NV_E4M3);
    }
    if constexpr (kVec) {
      uint32_t packed[PER / 4];
#pragma unroll
      for (int i = 0; i < PER / 4; ++i) packed[i] = two[2 * i] | (uint32_t)two[2 * i + 1] << 16;
      store_words<PER / 4, kWords>(q_row + c, packed);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (c + 32 * e < cols) q_row[c + 32 * e] = (uint8_t)(two[e / 2] >> (e % 2 * 8));
    }
  }
};

}  // namespace

// A team of blockDim.x lanes takes a row and keeps it in registers, N units a lane: it is read once.  With blockDim.y > 1
// (short rows) a team is a warp, and the CTA has several.  Teams go from row to row, four times as many as are resident at once:
// that evens out what a few of them lose on memory.  16384 x 4096 bf16 with residual, us: a row to a CTA 108; from row to row,
// the next one under way 81, with the weight out of L1 instead of registers 79, teams as many as are resident 83, four times as
// many 73; without the next one under way 92; a warp to a row 152.
template <typename T, typename W, int PER, int N>
__global__ void __launch_bounds__(kNormThreads<PER>, N == 1 && sizeof(T) == 2 && PER > 4 ? 2 : 1) rms_norm_fp8_kernel(const RmsNormFp8Args p) {
  using L = Lanes<PER>;
  using RawT = typename L::template Raw<T>;
  __shared__ float sums[2][32];
  const int lanes = (int)blockDim.x, u0 = (int)threadIdx.x;
  const int blocks = (p.cols + kBlockCols - 1) / kBlockCols;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  if (row >= p.rows) return;  // (a whole warp, and where a team is more than one, a whole CTA)
  const T* const xs = reinterpret_cast<const T*>(p.x);
  const T* const rs = reinterpret_cast<const T*>(p.residual);
  // Up to two units a lane: the next row is on its way while this one is worked on.
  constexpr bool kAhead = N <= 2;
  constexpr int kKept = kAhead ? N : 1;
  RawT x[kKept], r[kKept];
  auto load_row = [&](int64_t at) {
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      x[i] = L::load(xs + at * p.x_stride, i * lanes + u0, p.cols);
      if (p.residual != nullptr) r[i] = L::load(rs + at * p.residual_stride, i * lanes + u0, p.cols);
    }
  };
  if (kAhead) load_row(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    float h[N][PER];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = i * lanes + u0;
      L::floats(kAhead ? x[i % kKept] : L::load(xs + row * p.x_stride, u, p.cols), h[i]);
      if (p.residual != nullptr) {
        float f[PER];
        L::floats(kAhead ? r[i % kKept] : L::load(rs + row * p.residual_stride, u, p.cols), f);
#pragma unroll
        for (int e = 0; e < PER; ++e) h[i][e] += f[e];
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) sum = fmaf(h[i][e], h[i][e], sum);
    }
    // (total may be x or residual: a lane has read its columns of this row, and nobody else reads them)
    if (p.total != nullptr) {
      T* total = reinterpret_cast<T*>(p.total) + row * p.total_stride;
#pragma unroll
      for (int i = 0; i < N; ++i) L::store(total, i * lanes + u0, p.cols, h[i]);
    }
    if (kAhead && row + step < p.rows) load_row(row + step);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lanes > 32) {  // (a CTA with a team of several warps has one team; rows take turns with the two sets of sums)
      if ((u0 & 31) == 0) sums[turn][u0 >> 5] = sum;
      __syncthreads();
      sum = (u0 & 31) < lanes / 32 ? sums[turn][u0 & 31] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float rstd = rsqrtf(sum / (float)p.cols + p.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = i * lanes + u0;
      float f[PER];
      L::floats(L::load(reinterpret_cast<const W*>(p.weight), u, p.cols), f);  // (out of L1)
#pragma unroll
      for (int e = 0; e < PER; ++e) f[e] = h[i][e] * rstd * f[e];
      if (p.normed != nullptr) L::store(reinterpret_cast<T*>(p.normed) + row * p.cols, u, p.cols, f);
#pragma unroll
      for (int e = 0; e < PER; ++e) f[e] = -f[e];
      L::quantise(reinterpret_cast<uint8_t*>(p.q) + row * p.cols, p.scale + row * blocks, u, p.cols, f);
    }
  }
}

// A team of blockDim.x lanes takes a row, a unit a lane at a time; a CTA has blockDim.y teams.  Teams are whole warps, or parts
// of one that hold whole blocks.
template <typename T, int PER>
__global__ void __launch_bounds__(256) silu_mul_fp8_kernel(const SiluMulFp8Args p) {
  using L = Lanes<PER>;
  const int lanes = (int)blockDim.x;
  const int blocks = (p.cols + kBlockCols - 1) / kBlockCols;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  // All lanes of a CTA make the same number of rounds, over units behind the row as well: a warp's meet in the maximum.
  for (int64_t row0 = (int64_t)blockIdx.x * blockDim.y; row0 < p.rows; row0 += (int64_t)gridDim.x * blockDim.y) {
    const int64_t row = row0 + threadIdx.y;
    const int cols = row < p.rows ? p.cols : 0;
    const T* gate = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
    for (int u0 = 0; u0 < blocks * L::kUnits; u0 += lanes) {
      const int u = u0 + (int)threadIdx.x;
      const auto rg = L::load(gate, u, cols), ru = L::load(gate + p.cols, u, cols);
      float g[PER], v[PER];
      L::floats(rg, g);
      L::floats(ru, v);
#pragma unroll
      for (int e = 0; e < PER; e += 2) {
        const float2 y = minus_silu_mul(make_float2(g[e], g[e + 1]), make_float2(v[e], v[e + 1]));
        g[e] = y.x;
        g[e + 1] = y.y;
      }
      L::quantise(reinterpret_cast<uint8_t*>(p.q) + row * p.cols, p.scale + row * blocks, u, cols, g);
    }
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
namespace {

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

// Columns of a unit, from everything that has to be a multiple of it: sizes and strides in elements, addresses in bytes.
int columns_of_a_unit(int64_t elements, uint64_t addresses) {
  if (elements % 16 == 0 && addresses % 32 == 0) return 16;
  return elements % 8 == 0 && addresses % 16 == 0 ? 8 : 4;
}
uint64_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <typename T, typename W, int PER>
cudaError_t norm_units(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  const int units = (p.cols + kBlockCols - 1) / kBlockCols * Lanes<PER>::kUnits;
  dim3 block;
  int n;
  if (units <= 64) {
    n = (units + 31) / 32;
    block = dim3(32, 8);
  } else {
    n = (units + kNormThreads<PER> - 1) / kNormThreads<PER>;
    block = dim3((unsigned)(((units + n - 1) / n + 31) / 32 * 32), 1);
  }
  const int64_t teams = (p.rows + block.y - 1) / block.y;
  const int threads = (int)(block.x * block.y);
  const auto go = [&](auto n_units) {
    constexpr auto kernel = rms_norm_fp8_kernel<T, W, PER, decltype(n_units)::value>;
    static thread_local int known[kNormThreads<PER> / 32 + 1] = {};  // CTAs that an SM holds, by their size
    int& ctas = known[threads / 32];
    if (ctas == 0 && cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, threads, 0) != cudaSuccess) ctas = 1;
    return launch_teams(kernel, std::min<int64_t>(teams, 4 * (int64_t)sms * std::max(ctas, 1)), block, stream, p);
  };
  if (n <= 1) return go(std::integral_constant<int, 1>());
  if (n <= 2) return go(std::integral_constant<int, 2>());
  if (n <= 4) return go(std::integral_constant<int, 4>());
  if constexpr (PER <= 8) {
    if (n <= 8) return go(std::integral_constant<int, 8>());
  }
  return cudaErrorInvalidValue;
}

template <typename T, typename W>
cudaError_t norm_typed(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  switch (columns_of_a_unit(p.cols | p.x_stride | p.residual_stride | p.total_stride,
                            address(p.x) | address(p.residual) | address(p.weight) | address(p.total))) {
    case 16: return norm_units<T, W, 16>(p, sms, stream);
    case 8: return norm_units<T, W, 8>(p, sms, stream);
    default: return norm_units<T, W, 4>(p, sms, stream);
  }
}

template <typename T>
cudaError_t norm_weight(const RmsNormFp8Args& p, int sms, cudaStream_t stream) {
  if (p.weight_dtype == p.dtype) return norm_typed<T, T>(p, sms, stream);
  return p.weight_dtype == 2 ? norm_typed<T, float>(p, sms, stream) : cudaErrorInvalidValue;
}

template <typename T, int PER>
cudaError_t silu_units(const SiluMulFp8Args& p, int sms, cudaStream_t stream) {
  const int64_t units = (int64_t)((p.cols + kBlockCols - 1) / kBlockCols) * Lanes<PER>::kUnits;
  // the largest team of which no more than a ninth is idle
  int lanes = Lanes<PER>::kUnits;
  for (int l = 2 * lanes; l <= 256; l *= 2)
    if (8 * ((units + l - 1) / l * l) <= 9 * units) lanes = l;
  const dim3 block((unsigned)lanes, (unsigned)(256 / lanes));
  const int64_t grid = std::min<int64_t>((p.rows + block.y - 1) / block.y, 1 << 30);
  return launch_teams(silu_mul_fp8_kernel<T, PER>, grid, block, stream, p);
}

template <typename T>
cudaError_t silu_typed(const SiluMulFp8Args& p, int sms, cudaStream_t stream) {
  switch (columns_of_a_unit(p.cols | p.x_stride, address(p.x))) {
    case 16: return silu_units<T, 16>(p, sms, stream);
    case 8: return silu_units<T, 8>(p, sms, stream);
    default: return silu_units<T, 4>(p, sms, stream);
  }
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
  if (p.rows < 0 || p.cols < 1 || p.cols > kMaxSiluCols) return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  switch (p.dtype) {
    case 0: return silu_typed<__half>(p, sms, stream);
    case 1: return silu_typed<__nv_bfloat16>(p, sms, stream);
    case 2: return silu_typed<float>(p, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200
