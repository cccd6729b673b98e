// Tokens sorted by expert, and their rows back in token order.
//
// Entry i = t k + j of the expert ids [T, k] asks for a row of expert e_i.  Rows are packed expert by expert, inside an
// expert in the order of the entries:
//   row(i) = offsets[e_i] + #{i' < i : e_i' = e_i},   offsets[e] = #{i : e_i < e}
// Entries whose id is not in [0, E) have no row (-1); the rows behind offsets[E] are zero.
//   sort             rows[row(t, j)] = x[t]  (and the same of a scale row)
//   unsort           out[t] = sum_j w[t, j] rows[row(t, j)]; without weights it is the gradient of sort
//   unsort backward  grad_rows[row(t, j)] = w[t, j] grad[t],  grad_w[t, j] = <grad[t], rows[row(t, j)]>
// Sums are fp32, over j upwards, and rounded once; nothing is added by atomics whose order could show in a result (integer
// counts are).
//
// All kernels may start before the previous kernel of the stream has ended: no global memory is touched before
// grid_dep_wait().
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "moe_common.cuh"
#include "moe_sort.h"
#include "per_device.h"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

using namespace moe;

// Copies move vectors V, U of them a lane at a time: the widest that rows, their distance and their addresses allow.
struct Vec32 { uint32_t w[8]; };
template <typename V> struct Copy {
  static constexpr int U = sizeof(V) == 32 ? 1 : sizeof(V) == 16 ? 2 : sizeof(V) == 4 ? 4 : 8;
};
template <typename V>
__device__ __forceinline__ V load_vec(const V* p) { return __ldcg(p); }
template <>
__device__ __forceinline__ Vec32 load_vec<Vec32>(const Vec32* p) {
  Vec32 v;
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p));
  return v;
}
template <typename V>
__device__ __forceinline__ void store_vec(V* p, const V& v) { *p = v; }
template <>
__device__ __forceinline__ void store_vec<Vec32>(Vec32* p, const Vec32& v) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]),
               "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7]), "l"(p)
               : "memory");
}

constexpr int kMaxChunks = 256;  // runs of tokens that are counted

struct SortParams {
  SortTokensArgs a;
  int32_t pieces;      // of a row
  int32_t row_vecs, piece_vecs;
  int32_t vec_ids;               // 1: ids begin at a multiple of 16 bytes
  int32_t chunks, chunk_tokens;  // several launches: runs of tokens that are counted by a CTA each
};

__device__ __forceinline__ int checked_id(long long e, int experts) { return e >= 0 && e < experts ? (int)e : -1; }
__device__ __forceinline__ int expert_of(const SortTokensArgs& a, int64_t i) {
  return checked_id(a.wide_ids ? __ldcg(reinterpret_cast<const long long*>(a.indices) + i)
                               : (long long)__ldcg(reinterpret_cast<const int*>(a.indices) + i),
                    a.experts);
}
// Entries 4 q .. 4 q + 3, from aligned ids.
__device__ __forceinline__ void experts_of(const SortTokensArgs& a, int q, int (&e)[4]) {
  if (a.wide_ids) {
    const longlong2* ids = reinterpret_cast<const longlong2*>(a.indices) + 2 * (int64_t)q;
    const longlong2 u = __ldcg(ids), v = __ldcg(ids + 1);
    e[0] = checked_id(u.x, a.experts), e[1] = checked_id(u.y, a.experts);
    e[2] = checked_id(v.x, a.experts), e[3] = checked_id(v.y, a.experts);
  } else {
    const int4 u = __ldcg(reinterpret_cast<const int4*>(a.indices) + q);
    e[0] = checked_id(u.x, a.experts), e[1] = checked_id(u.y, a.experts);
    e[2] = checked_id(u.z, a.experts), e[3] = checked_id(u.w, a.experts);
  }
}

// counts[0 .. n) in shared memory become exclusive prefix sums; returns their total.  All threads of the CTA.
__device__ __forceinline__ int exclusive_scan(int32_t* counts, int n, int32_t* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
  const int each = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int lo = min(n, tid * each), hi = min(n, lo + each);
  int own = 0;
  for (int i = lo; i < hi; ++i) own += counts[i];
  int upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  int run = before + upto - own;
  for (int i = lo; i < hi; ++i) {
    const int c = counts[i];
    counts[i] = run;
    run += c;
  }
  __syncthreads();
  return total;
}

// One piece of token t's row, and with the first one its scales (two a lane; more are read when they are stored).  Warps ask
// for the next piece before they store the one at hand: a load that is issued behind stores waits for them.
template <typename V>
struct Piece {
  V r[Copy<V>::U];
  float s[2];
};
__device__ __forceinline__ void load_scales(const SortParams& p, int t, float (&s)[2]) {
  if (p.a.scale == nullptr) return;
  const int lane = threadIdx.x & 31;
  const float* scale = p.a.scale + (int64_t)t * p.a.scale_stride;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 32 * u < p.a.scale_cols) s[u] = __ldcg(scale + lane + 32 * u);
}
template <typename V>
__device__ __forceinline__ void load_piece(const SortParams& p, int t, int piece, Piece<V>& to) {
  const int lane = threadIdx.x & 31;
  const V* src = reinterpret_cast<const V*>(reinterpret_cast<const uint8_t*>(p.a.x) + (int64_t)t * p.a.x_stride);
  const int v0 = piece * p.piece_vecs + lane;
  const int v1 = min(p.row_vecs, (piece + 1) * p.piece_vecs);
#pragma unroll
  for (int u = 0; u < Copy<V>::U; ++u)
    if (v0 + 32 * u < v1) to.r[u] = load_vec(src + v0 + 32 * u);
  if (piece == 0) load_scales(p, t, to.s);
}
// Token t's scales, to row `to`.
__device__ __forceinline__ void store_scales(const SortTokensArgs& a, int t, int to, const float (&s)[2]) {
  const int lane = threadIdx.x & 31;
  float* scale = a.rows_scale + (int64_t)to * a.scale_cols;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 32 * u < a.scale_cols) scale[lane + 32 * u] = s[u];
  for (int c = lane + 64; c < a.scale_cols; c += 32) scale[c] = __ldcg(a.scale + (int64_t)t * a.scale_stride + c);
}
// Stores it to the token's k rows; `row` is lane j's: entry j's row.
template <typename V>
__device__ __forceinline__ void store_piece(const SortParams& p, int t, int piece, int row, const Piece<V>& from) {
  const int lane = threadIdx.x & 31;
  const SortTokensArgs& a = p.a;
  const int v0 = piece * p.piece_vecs + lane;
  const int v1 = min(p.row_vecs, (piece + 1) * p.piece_vecs);
  const bool scales = piece == 0 && a.scale != nullptr;
  if (piece == 0 && lane < a.k) a.row_of[(int64_t)t * a.k + lane] = row;
  for (int j = 0; j < a.k; ++j) {
    const int to = __shfl_sync(0xffffffffu, row, j);
    if (to < 0) continue;
    V* dst = reinterpret_cast<V*>(reinterpret_cast<uint8_t*>(a.rows) + (int64_t)to * a.row_bytes);
#pragma unroll
    for (int u = 0; u < Copy<V>::U; ++u)
      if (v0 + 32 * u < v1) store_vec(dst + v0 + 32 * u, from.r[u]);
    if (scales) store_scales(a, t, to, from.s);
  }
}

// Rows [from, to) and their scales are zero: CTA `cta` of `ctas` takes its share.
template <typename V>
__device__ __forceinline__ void zero_rows(void* rows, int64_t row_bytes, float* scales, int scale_cols, int64_t from, int64_t to,
                                          int cta, int ctas) {
  const V zero = {};
  for (int64_t r = from + cta; r < to; r += ctas) {
    V* dst = reinterpret_cast<V*>(reinterpret_cast<uint8_t*>(rows) + r * row_bytes);
    for (int v = threadIdx.x; v < (int)(row_bytes / (int64_t)sizeof(V)); v += blockDim.x) store_vec(dst + v, zero);
    if (scales != nullptr)
      for (int c = threadIdx.x; c < scale_cols; c += blockDim.x) scales[r * scale_cols + c] = 0.f;
  }
}

}  // namespace

// One launch: every CTA counts all entries itself, and ranks its own against each other.
template <typename V>
__global__ void __launch_bounds__(1024) sort_tokens_kernel(const SortParams p) {
  extern __shared__ __align__(16) int32_t smem[];
  __shared__ int32_t warp_sums[32];
  const SortTokensArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, threads = blockDim.x;
  const int P = p.pieces;
  const int64_t items = (int64_t)a.tokens * P;
  const int lo = (int)(items * blockIdx.x / gridDim.x), hi = (int)(items * (blockIdx.x + 1) / gridDim.x);
  const int t0 = lo / P, t1 = hi > lo ? (hi + P - 1) / P : t0;
  const int i0 = t0 * a.k, i1 = t1 * a.k, n = a.tokens * a.k;
  int32_t* start = smem;  // entries of an expert behind the CTA's, then all of them, then the first row
  const int room = (a.experts + 3) & ~3, own = (i1 - i0 + 3) & ~3;
  int32_t* before = start + room;  // own entries and earlier ones
  int32_t* ids = before + room;    // expert of each own entry
  int32_t* rows = ids + own;       // and its row
  for (int e = tid; e < 2 * room; e += threads) smem[e] = 0;
  if (tid < own - (i1 - i0)) ids[i1 - i0 + tid] = -2;
  __syncthreads();
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  int item = lo + (tid >> 5);
  Piece<V> next;  // the warp's first piece is on its way while rows are worked out
  if (item < hi) load_piece(p, item / P, item % P, next);
  auto count = [&](int i, int e) {
    if (e >= 0) atomicAdd((i < i1 ? before : start) + e, 1);
    if (i >= i0 && i < i1) ids[i - i0] = e;
  };
  const int quads = p.vec_ids && n >= 4 * threads ? n >> 2 : 0;
#pragma unroll 2
  for (int q = tid; q < quads; q += threads) {
    int e[4];
    experts_of(a, q, e);
#pragma unroll
    for (int j = 0; j < 4; ++j) count(4 * q + j, e[j]);
  }
  for (int i = 4 * quads + tid; i < n; i += threads) count(i, expert_of(a, i));
  __syncthreads();
  for (int e = tid; e < a.experts; e += threads) start[e] += before[e];
  __syncthreads();
  const int total = exclusive_scan(start, a.experts, warp_sums);
  // an entry's rank is the count up to the CTA's end less the own entries of its expert from it on
  for (int j0 = tid - lane; j0 < i1 - i0; j0 += threads) {
    const int j = j0 + lane;
    const int e = j < i1 - i0 ? ids[j] : -1;
    int from_here = __popc(__match_any_sync(0xffffffffu, e) & (0xffffffffu << lane));
#pragma unroll 4
    for (int q = j0 + 32; q < i1 - i0; q += 4) {
      const int4 later = *reinterpret_cast<const int4*>(ids + q);
      from_here += (later.x == e) + (later.y == e) + (later.z == e) + (later.w == e);
    }
    if (j < i1 - i0) rows[j] = e < 0 ? -1 : start[e] + before[e] - from_here;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int e = tid; e < a.experts; e += threads) a.offsets[e] = start[e];
    if (tid == 0) a.offsets[a.experts] = total;
  }
  for (const int warps = threads >> 5; item < hi; item += warps) {
    const Piece<V> now = next;
    if (item + warps < hi) load_piece(p, (item + warps) / P, (item + warps) % P, next);
    const int t = item / P;
    store_piece(p, t, item - t * P, lane < a.k ? rows[t * a.k - i0 + lane] : -1, now);
  }
  zero_rows<V>(a.rows, a.row_bytes, a.rows_scale, a.scale_cols, total, n, (int)blockIdx.x, (int)gridDim.x);
}

// Two launches, or three, the first: a CTA counts a run of tokens' entries by expert, and ranks them inside the run.  Warps have
// runs of their own inside it, so that order needs no other means than a prefix over warps.
// work: [chunk][expert] counts, [expert] room for their sums, then a rank for each entry.
__global__ void __launch_bounds__(1024) sort_count_kernel(const SortParams p) {
  extern __shared__ __align__(16) int32_t smem[];  // [warp][expert]
  const SortTokensArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
  const int c = blockIdx.x;
  for (int e = tid; e < warps * a.experts; e += blockDim.x) smem[e] = 0;
  __syncthreads();
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int i0 = c * p.chunk_tokens * a.k, i1 = min(a.tokens, (c + 1) * p.chunk_tokens) * a.k;
  const int each = ((i1 - i0 + warps - 1) / warps + 31) & ~31;
  const int w0 = min(i1, i0 + warp * each), w1 = min(i1, w0 + each);
  int32_t* own = smem + warp * a.experts;
  int32_t* ranks = a.work + (int64_t)(p.chunks + 1) * a.experts;
  auto rank_of = [&](int e) {  // among the warp's entries so far (every lane has one, or -1)
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    int rank = 0;
    if (e >= 0) rank = own[e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && (same >> lane) == 1u) own[e] = rank + 1;  // (the last of them)
    __syncwarp();
    return rank;
  };
  constexpr int kHeld = 4;  // entries that a lane keeps until the warps before it are known; beyond them it reads again
  int held_id[kHeld], held_rank[kHeld];
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    const int i = w0 + 32 * r + lane;
    held_id[r] = i < w1 ? expert_of(a, i) : -1;
  }
#pragma unroll
  for (int r = 0; r < kHeld; ++r) held_rank[r] = rank_of(held_id[r]);
  for (int i = w0 + 32 * kHeld + lane; i - lane < w1; i += 32) {
    const int rank = rank_of(i < w1 ? expert_of(a, i) : -1);
    if (i < w1) ranks[i] = rank;
  }
  __syncthreads();
  for (int e = tid; e < a.experts; e += blockDim.x) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < warps; ++w) {
      const int n = smem[w * a.experts + e];
      smem[w * a.experts + e] = run;
      run += n;
    }
    a.work[(int64_t)c * a.experts + e] = run;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    const int i = w0 + 32 * r + lane;
    if (i < w1) ranks[i] = held_id[r] >= 0 ? held_rank[r] + own[held_id[r]] : 0;
  }
  for (int i = w0 + 32 * kHeld + lane; i < w1; i += 32) {
    const int e = expert_of(a, i);
    if (e >= 0) ranks[i] += own[e];
  }
}

// Rows that are short: a CTA adds up the runs' counts, and copies its share of the rows, which lies in one run or two.
//
// Bound by the row stores, which memory takes the slower the more of them are under way in different places: 65536 rows of
// 7168 bytes with scales (8192 tokens, top-8) would take 111 us with 16 to 32 warps an SM, 5 to 8 more with 48, 16 more with 64;
// as bare copies, without the counting and the scales, 93 to 100.  (Scales as a piece of their own, whose loads wait behind the stores
// of others: 8 us more.  In the order of the rows instead of the tokens': 115 and more for the copies alone.)
constexpr int kScatterThreads = 512, kScatterCtas = 2;
template <typename V>
__global__ void __launch_bounds__(kScatterThreads, kScatterCtas) sort_scatter_kernel(const SortParams p) {
  extern __shared__ __align__(16) int32_t smem[];
  __shared__ int32_t warp_sums[32];
  const SortTokensArgs& a = p.a;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warps = threads >> 5;
  const int P = p.pieces;
  const int64_t items = (int64_t)a.tokens * P;
  const int64_t lo = items * blockIdx.x / gridDim.x, hi = items * (blockIdx.x + 1) / gridDim.x;
  const int run = (int)(lo / P) / p.chunk_tokens, t_next = (run + 1) * p.chunk_tokens;
  int32_t* start = smem;              // all entries of an expert, then its first row
  int32_t* base = start + a.experts;  // first row of the share's first run, and of the next
  int32_t* next = base + a.experts;
  for (int e = tid; e < 2 * a.experts; e += threads) smem[e] = 0;
  __syncthreads();
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  const int slices = max(1, threads / a.experts);  // of the runs, which threads of the same expert share
  for (int i = tid; i < slices * a.experts; i += threads) {
    const int e = i % a.experts;
    int all = 0, earlier = 0;
#pragma unroll 8
    for (int q = i / a.experts; q < p.chunks; q += slices) {
      const int n = __ldcg(a.work + (int64_t)q * a.experts + e);
      all += n;
      earlier += q < run ? n : 0;
      if (q == run) next[e] = n;
    }
    atomicAdd(start + e, all);
    atomicAdd(base + e, earlier);
  }
  __syncthreads();
  const int total = exclusive_scan(start, a.experts, warp_sums);
  for (int e = tid; e < a.experts; e += threads) {
    base[e] += start[e];
    next[e] += base[e];
  }
  if (blockIdx.x == 0) {
    for (int e = tid; e < a.experts; e += threads) a.offsets[e] = start[e];
    if (tid == 0) a.offsets[a.experts] = total;
  }
  __syncthreads();
  const int32_t* ranks = a.work + (int64_t)(p.chunks + 1) * a.experts;
  int64_t item = lo + (tid >> 5);
  Piece<V> next_piece;
  int next_id = -1, next_rank = 0;
  auto ask = [&](int64_t i) {
    const int t = (int)(i / P);
    load_piece(p, t, (int)(i - (int64_t)t * P), next_piece);
    if (lane < a.k) {
      next_id = expert_of(a, (int64_t)t * a.k + lane);
      next_rank = __ldcg(ranks + (int64_t)t * a.k + lane);
    }
  };
  if (item < hi) ask(item);
  for (; item < hi; item += warps) {
    const Piece<V> now = next_piece;
    const int t = (int)(item / P);
    const int row = next_id >= 0 ? (t < t_next ? base : next)[next_id] + next_rank : -1;
    if (item + warps < hi) ask(item + warps);
    store_piece(p, t, (int)(item - (int64_t)t * P), row, now);
  }
  zero_rows<V>(a.rows, a.row_bytes, a.rows_scale, a.scale_cols, total, (int64_t)a.tokens * a.k, (int)blockIdx.x, (int)gridDim.x);
}

// Rows that are long, the second launch: for each expert, a run's count becomes that of the runs before it.  Eight warps share
// the runs of 32 experts.
__global__ void __launch_bounds__(256) sort_prefix_kernel(const SortParams p) {
  __shared__ int32_t sums[8][32];
  const SortTokensArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  const int each = (p.chunks + 7) / 8;
  const int q0 = min(p.chunks, warp * each), q1 = e < a.experts ? min(p.chunks, q0 + each) : q0;
  int32_t* counts = a.work + e;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  constexpr int kHeld = kMaxChunks / 8;
  int held[kHeld], own = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held[i] = q0 + i < q1 ? __ldcg(counts + (int64_t)(q0 + i) * a.experts) : 0;
    own += held[i];
  }
  sums[warp][lane] = own;
  __syncthreads();
  int run = 0;
  for (int w = 0; w < warp; ++w) run += sums[w][lane];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    if (q0 + i < q1) counts[(int64_t)(q0 + i) * a.experts] = run;
    run += held[i];
  }
  if (warp == 7 && e < a.experts) counts[(int64_t)p.chunks * a.experts] = run;
}

namespace {

// Entry `lane` of a token on its way to its row: its expert and rank, then what its expert's earlier runs have.
struct Entry {
  int id, rank, base;
  __device__ __forceinline__ void ask(const SortParams& p, int t) {
    const int lane = threadIdx.x & 31;
    id = -1;
    if (lane >= p.a.k) return;
    id = expert_of(p.a, (int64_t)t * p.a.k + lane);
    rank = __ldcg(p.a.work + (int64_t)(p.chunks + 1) * p.a.experts + (int64_t)t * p.a.k + lane);
  }
  __device__ __forceinline__ void ask_base(const SortParams& p, int t) {
    if (id >= 0) base = __ldcg(p.a.work + (int64_t)(t / p.chunk_tokens) * p.a.experts + id);
  }
  __device__ __forceinline__ int row(const int32_t* start) const { return id >= 0 ? start[id] + base + rank : -1; }
};

}  // namespace

// The third: a piece of a row comes into shared memory, and leaves it by a bulk copy for each of the token's rows, one to a lane.
// A warp has room for two pieces: one comes in while the other leaves.  There is one CTA to an SM, and all of them take tokens
// in order together, so that few rows are written at a time, and near one another inside an expert: as bare copies 90 us for
// 65536 rows of 7168 bytes, 97 to 99 when each CTA has a share of its own or an SM has two.  With everything, us, beside the
// kernel above (8192 tokens, top-8, unless said): 7168 bytes and scales 107, 113; 14336 bytes 197, 202; 4096 bytes and scales
// 66, 69; 2048 bytes 40, 37 (which is why rows have to be long); 5000 tokens of 40000 bytes 336, 365; 9000 tokens, top-4 of
// 4096, 4112 bytes 52, 71.  With four warps and pieces of 16 KiB long rows take 2 % less, short ones 12 to 17 % more.
constexpr int kBulkWarps = 8, kBulkPiece = 8192;
__global__ void __launch_bounds__(32 * kBulkWarps) sort_scatter_bulk_kernel(const SortParams p) {
  extern __shared__ __align__(128) int32_t smem[];
  __shared__ int32_t warp_sums[32];
  const SortTokensArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int P = p.pieces;
  const uint32_t slot_bytes = (uint32_t)p.piece_vecs * 16u;
  const uint32_t slots = ptx::smem_u32(smem) + (uint32_t)warp * 2u * slot_bytes;
  int32_t* start = smem + kBulkWarps * 2 * p.piece_vecs * 4;
  const int64_t items = (int64_t)a.tokens * P;
  const int64_t step = (int64_t)gridDim.x * kBulkWarps;
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  int64_t item = (int64_t)warp * gridDim.x + blockIdx.x;
  Entry entry;
  float scales[2];
  auto bring = [&](int64_t i, uint32_t slot) {
    if (i < items) {
      const int t = (int)(i / P), v0 = (int)(i - (int64_t)t * P) * p.piece_vecs, n = min(p.piece_vecs, p.row_vecs - v0);
      const uint8_t* src = reinterpret_cast<const uint8_t*>(a.x) + (int64_t)t * a.x_stride + (int64_t)v0 * 16;
      for (int v = lane; v < n; v += 32) ptx::cp_async_16(slot + (uint32_t)v * 16u, src + (int64_t)v * 16);
    }
    ptx::cp_async_commit();
  };
  auto ask = [&](int64_t i) {
    if (i >= items) return;
    const int t = (int)(i / P);
    entry.ask(p, t);
    if (i % P == 0) load_scales(p, t, scales);
    entry.ask_base(p, t);
  };
  bring(item, slots);
  ask(item);
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) start[e] = __ldcg(a.work + (int64_t)p.chunks * a.experts + e);
  __syncthreads();
  const int total = exclusive_scan(start, a.experts, warp_sums);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.offsets[e] = start[e];
    if (threadIdx.x == 0) a.offsets[a.experts] = total;
  }
  for (uint32_t slot = slots, other = slots + slot_bytes; item < items; item += step) {
    ptx::bulk_wait_group_read<0>();  // the copies out of the other slot have read it
    __syncwarp();
    bring(item + step, other);
    ptx::cp_async_wait_group<1>();
    ptx::fence_proxy_async_smem();
    __syncwarp();
    const int t = (int)(item / P), piece = (int)(item - (int64_t)t * P), v0 = piece * p.piece_vecs;
    const int row = entry.row(start);
    if (row >= 0)
      ptx::bulk_store(reinterpret_cast<uint8_t*>(a.rows) + (int64_t)row * a.row_bytes + (int64_t)v0 * 16, slot,
                      (uint32_t)min(p.piece_vecs, p.row_vecs - v0) * 16u);
    ptx::bulk_commit_group();
    if (piece == 0 && lane < a.k) a.row_of[(int64_t)t * a.k + lane] = row;
    for (int j = 0; piece == 0 && a.scale != nullptr && j < a.k; ++j) {
      const int to = __shfl_sync(0xffffffffu, row, j);
      if (to >= 0) store_scales(a, t, to, scales);
    }
    ask(item + step);
    const uint32_t done = slot;
    slot = other;
    other = done;
  }
  ptx::bulk_wait_group<0>();
  zero_rows<int4>(a.rows, a.row_bytes, a.rows_scale, a.scale_cols, total, (int64_t)a.tokens * a.k, (int)blockIdx.x, (int)gridDim.x);
}

// ---------------------------------------------------------------------------------------
// back to the tokens
// ---------------------------------------------------------------------------------------
namespace {

// What a lane takes of a row at once: sixteen bytes, or one element where rows are not whole aligned 16-byte vectors.
template <typename T, bool VEC> struct Bit;
template <typename T> struct Bit<T, true> {
  static constexpr int N = Vec16<T>::N;
  using Raw = int4;
  static __device__ __forceinline__ void fma(float* acc, const Raw& r, float w) { fma_vec<T>(acc, r, w); }
  static __device__ __forceinline__ Raw pack(const float* acc) { return pack_vec<T>(acc); }
};
template <typename T> struct Bit<T, false> {
  static constexpr int N = 1;
  using Raw = T;
  static __device__ __forceinline__ void fma(float* acc, const Raw& r, float w) { acc[0] = fmaf(to_f32(r), w, acc[0]); }
  static __device__ __forceinline__ Raw pack(const float* acc) { return from_f32<T>(acc[0]); }
};

struct UnsortParams {
  UnsortTokensArgs a;
  int32_t row_vecs, pieces, piece_vecs;
};
struct UnsortBackwardParams {
  UnsortBackwardArgs a;
  int32_t row_vecs;
};

}  // namespace

// A warp takes a piece of a token's row: U vectors a lane of KB rows at a time.  CTAS of a kernel fit an SM.
template <typename T, bool VEC, int KB, int CTAS>
__global__ void __launch_bounds__(256, CTAS) unsort_tokens_kernel(const UnsortParams p) {
  using B = Bit<T, VEC>;
  using Raw = typename B::Raw;
  constexpr int U = VEC ? 2 : 4;
  const UnsortTokensArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t warps = ((int64_t)gridDim.x * blockDim.x) >> 5;
  const int64_t items = (int64_t)a.tokens * p.pieces;
  const uint8_t* rows = reinterpret_cast<const uint8_t*>(a.rows);
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  for (int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; item < items; item += warps) {
    const int t = (int)(item / p.pieces), piece = (int)(item % p.pieces);
    int row = -1;
    float w = 1.f;
    if (lane < a.k) {
      row = __ldcg(a.row_of + (int64_t)t * a.k + lane);
      if (a.weights != nullptr) w = __ldcg(a.weights + (int64_t)t * a.k + lane);
      if (row >= a.num_rows) row = -1;
    }
    Raw* out = reinterpret_cast<Raw*>(reinterpret_cast<T*>(a.out) + (int64_t)t * a.hidden);
    const int v0 = piece * p.piece_vecs, v1 = min(p.row_vecs, v0 + p.piece_vecs);
    for (int vb = v0; vb < v1; vb += 32 * U) {
      float acc[U][B::N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < B::N; ++e) acc[u][e] = 0.f;
      for (int kb = 0; kb < a.k; kb += KB) {
        // all loads leave before the first is used: a lane past the end, or an entry without a row, reads a valid place
        // (its own batch's last vector, row 0) and drops the value
        Raw r[KB][U];
#pragma unroll
        for (int q = 0; q < KB; ++q) {
          const int from = max(__shfl_sync(0xffffffffu, row, min(kb + q, a.k - 1)), 0);
          const Raw* src = reinterpret_cast<const Raw*>(rows + (int64_t)from * a.rows_stride);
#pragma unroll
          for (int u = 0; u < U; ++u) r[q][u] = __ldcg(src + min(vb + lane + 32 * u, v1 - 1));
        }
#pragma unroll
        for (int q = 0; q < KB; ++q) {
          const int from = kb + q < a.k ? __shfl_sync(0xffffffffu, row, kb + q) : -1;
          const float wq = __shfl_sync(0xffffffffu, w, (kb + q) & 31);
          if (from < 0) continue;
#pragma unroll
          for (int u = 0; u < U; ++u) B::fma(acc[u], r[q][u], wq);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (vb + lane + 32 * u < v1) out[vb + lane + 32 * u] = B::pack(acc[u]);
    }
  }
}

// A CTA takes a token.  DOT: the weights' gradient is wanted, so the rows are read.
template <typename T, bool VEC, bool DOT>
__global__ void __launch_bounds__(1024) unsort_tokens_backward_kernel(const UnsortBackwardParams p) {
  using B = Bit<T, VEC>;
  using Raw = typename B::Raw;
  constexpr int KB = 4;
  __shared__ float parts[32][kSortMaxTopk];
  const UnsortBackwardArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
  const int64_t row_bytes = (int64_t)a.hidden * (int64_t)sizeof(T);
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  for (int t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    int row = -1;
    float w = 1.f;
    if (lane < a.k) {
      row = __ldcg(a.row_of + (int64_t)t * a.k + lane);
      if (a.weights != nullptr) w = __ldcg(a.weights + (int64_t)t * a.k + lane);
      if (row >= a.num_rows) row = -1;
    }
    const Raw* grad = reinterpret_cast<const Raw*>(reinterpret_cast<const uint8_t*>(a.grad) + (int64_t)t * a.grad_stride);
    for (int kb = 0; kb < a.k; kb += KB) {
      float dot[KB];
      int from[KB];
      float wq[KB];
#pragma unroll
      for (int q = 0; q < KB; ++q) {
        dot[q] = 0.f;
        from[q] = __shfl_sync(0xffffffffu, row, (kb + q) & 31);
        if (kb + q >= a.k) from[q] = -1;
        wq[q] = __shfl_sync(0xffffffffu, w, (kb + q) & 31);
      }
      for (int v = tid; v < p.row_vecs; v += blockDim.x) {
        const Raw g = grad[v];
        Raw y[KB];
        if (DOT) {
#pragma unroll
          for (int q = 0; q < KB; ++q)
            y[q] = __ldcg(reinterpret_cast<const Raw*>(reinterpret_cast<const uint8_t*>(a.rows) +
                                                       (int64_t)max(from[q], 0) * a.rows_stride) + v);
        }
        float gf[B::N];
#pragma unroll
        for (int e = 0; e < B::N; ++e) gf[e] = 0.f;
        B::fma(gf, g, 1.f);
#pragma unroll
        for (int q = 0; q < KB; ++q) {
          if (from[q] < 0) continue;
          if (DOT) {
            float yf[B::N];
#pragma unroll
            for (int e = 0; e < B::N; ++e) yf[e] = 0.f;
            B::fma(yf, y[q], 1.f);
#pragma unroll
            for (int e = 0; e < B::N; ++e) dot[q] = fmaf(gf[e], yf[e], dot[q]);
          }
          if (a.grad_rows != nullptr) {
            float d[B::N];
#pragma unroll
            for (int e = 0; e < B::N; ++e) d[e] = gf[e] * wq[q];
            reinterpret_cast<Raw*>(reinterpret_cast<uint8_t*>(a.grad_rows) + (int64_t)from[q] * row_bytes)[v] = B::pack(d);
          }
        }
      }
      if (DOT) {
#pragma unroll
        for (int q = 0; q < KB; ++q) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) dot[q] += __shfl_xor_sync(0xffffffffu, dot[q], o);
          if (lane == 0 && kb + q < a.k) parts[warp][kb + q] = dot[q];
        }
      }
    }
    if (DOT) {
      __syncthreads();
      if (tid < a.k) {
        float sum = 0.f;
        for (int i = 0; i < warps; ++i) sum += parts[i][tid];
        a.grad_weights[(int64_t)t * a.k + tid] = sum;
      }
      __syncthreads();
    }
  }
  if (a.grad_rows != nullptr) {
    const int64_t end = max(0, __ldcg(a.end));
    zero_rows<Raw>(a.grad_rows, row_bytes, nullptr, 0, end, a.num_rows, (int)blockIdx.x, (int)gridDim.x);
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
namespace {

constexpr int64_t kOneLaunchEntries = 32768;
constexpr int64_t kBulkRow = 4096;  // bytes of a row that is long (figures at the kernel)
constexpr int kBulkSmem = kBulkWarps * 2 * kBulkPiece;
// Shared memory that keeps a CTA alone on its SM: where two fit, a launch that starts while the one before it still runs may
// put two on the SMs that happen to be free, and none on others.
constexpr int kAloneBytes = 116 * 1024;
constexpr int kCountSmem = 160 * 1024;  // of the counting kernel: a count of every expert for each warp

int sort_chunks(int64_t tokens, int k) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(kMaxChunks, tokens * k / 1024));
}

template <typename V>
cudaError_t sort_typed(SortParams p, int sms, cudaStream_t stream) {
  const SortTokensArgs& a = p.a;
  p.row_vecs = (int)(a.row_bytes / (int64_t)sizeof(V));
  p.piece_vecs = 32 * Copy<V>::U;
  p.pieces = std::max(1, (p.row_vecs + p.piece_vecs - 1) / p.piece_vecs);
  const int64_t items = (int64_t)a.tokens * p.pieces;
  if (a.work == nullptr) {
    if (items > INT32_MAX) return cudaErrorInvalidValue;
    // Every CTA counts all entries: few large ones repeat less of that where there are many.  Up to 16 pieces an SM, one to
    // a warp and one CTA to an SM.
    const int64_t share = (items + sms - 1) / sms;
    const bool few = share <= 16;
    const int threads = few ? 32 * (int)std::max<int64_t>(4, share) : (int64_t)a.tokens * a.k > 2048 ? 1024 : 512;
    const int warps = threads / 32;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((items + warps - 1) / warps, (few ? 1 : 1024 / threads) * (int64_t)sms));
    const int P = p.pieces;
    const int64_t own = ((items + grid - 1) / grid + 2 * P - 2) / P * a.k;  // entries of the tokens that a CTA touches, at most
    const size_t smem = 2 * ((size_t)((a.experts + 3) & ~3) + (size_t)((own + 3) & ~3)) * sizeof(int32_t);
    static OncePerDevice once;
    const cudaError_t opted = once([] { return opt_in(sort_tokens_kernel<V>, kCountSmem, false); });
    if (opted != cudaSuccess) return opted;
    if (smem > kCountSmem) return cudaErrorInvalidValue;
    const size_t alone = few ? std::max<size_t>(smem, kAloneBytes) : smem;
    return ptx::launch_dependent(sort_tokens_kernel<V>, grid, threads, alone, stream, p);
  }
  p.chunks = sort_chunks(a.tokens, a.k);
  p.chunk_tokens = (a.tokens + p.chunks - 1) / p.chunks;
  p.chunks = (a.tokens + p.chunk_tokens - 1) / p.chunk_tokens;
  static OncePerDevice once;
  const cudaError_t opted = once([] {
    cudaError_t e = opt_in(sort_count_kernel, kCountSmem, false);
    if (e == cudaSuccess) e = opt_in(sort_scatter_kernel<V>, 3 * kSortMaxExperts * (int)sizeof(int32_t), false);
    if (e == cudaSuccess) e = opt_in(sort_scatter_bulk_kernel, kBulkSmem + kSortMaxExperts * (int)sizeof(int32_t), false);
    return e;
  });
  if (opted != cudaSuccess) return opted;
  const int warps = std::max(1, std::min(32, kCountSmem / (a.experts * (int)sizeof(int32_t))));
  cudaError_t e = ptx::launch_dependent(sort_count_kernel, p.chunks, 32 * warps, (size_t)warps * a.experts * sizeof(int32_t),
                                        stream, p);
  if (e != cudaSuccess) return e;
  if (sizeof(V) >= 16 && a.row_bytes >= kBulkRow) {
    e = ptx::launch_dependent(sort_prefix_kernel, (a.experts + 31) / 32, 256, 0, stream, p);
    if (e != cudaSuccess) return e;
    p.row_vecs = (int)(a.row_bytes / 16);
    p.pieces = (p.row_vecs * 16 + kBulkPiece - 1) / kBulkPiece;
    p.piece_vecs = (p.row_vecs + p.pieces - 1) / p.pieces;
    const size_t smem = (size_t)kBulkWarps * 2 * p.piece_vecs * 16 + a.experts * sizeof(int32_t);
    return ptx::launch_dependent(sort_scatter_bulk_kernel, sms, 32 * kBulkWarps, std::max<size_t>(smem, kAloneBytes), stream, p);
  }
  // (a share is no longer than a run: there are more CTAs than runs)
  const int grid = (int)std::max<int64_t>(p.chunks, std::min<int64_t>((items + kScatterThreads / 32 - 1) / (kScatterThreads / 32),
                                                                     kScatterCtas * (int64_t)sms));
  return ptx::launch_dependent(sort_scatter_kernel<V>, grid, kScatterThreads, 3 * (size_t)a.experts * sizeof(int32_t), stream, p);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, bool VEC>
cudaError_t unsort_typed(const UnsortTokensArgs& a, int sms, cudaStream_t stream) {
  UnsortParams p;
  p.a = a;
  p.row_vecs = a.hidden / Bit<T, VEC>::N;
  p.piece_vecs = VEC ? 64 : 128;
  p.pieces = (p.row_vecs + p.piece_vecs - 1) / p.piece_vecs;
  // Many pieces: four CTAs to an SM, and twice as many in the grid, which evens out what some lose on memory (bf16, us: 4096
  // tokens, top-6, rows of 8 KiB 50 with as many as would fit with more registers, 39; 2047, top-8 28.8, 25.9; 2047, top-4,
  // 5760 bytes 12.2, 10.8).  Few: every row of a token at once (128 tokens, top-8, 14 KiB 5.4, 4.3).
  const int64_t ctas = ((int64_t)a.tokens * p.pieces + 7) / 8;
  const bool few = ctas <= 2 * (int64_t)sms;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(ctas, 8 * (int64_t)sms));
  const auto go = [&](auto kernel) { return ptx::launch_dependent(kernel, grid, 256, 0, stream, p); };
  if (a.k == 1) return go(unsort_tokens_kernel<T, VEC, 1, 4>);
  if (a.k == 2) return go(unsort_tokens_kernel<T, VEC, 2, 4>);
  if (few) return a.k <= 4 ? go(unsort_tokens_kernel<T, VEC, 4, 2>) : go(unsort_tokens_kernel<T, VEC, 8, 2>);
  return go(unsort_tokens_kernel<T, VEC, 4, 4>);
}

template <typename T>
cudaError_t unsort_vec(const UnsortTokensArgs& a, int sms, cudaStream_t stream) {
  const bool vec = a.hidden % Vec16<T>::N == 0 && a.rows_stride % 16 == 0 && aligned16(a.rows) && aligned16(a.out);
  return vec ? unsort_typed<T, true>(a, sms, stream) : unsort_typed<T, false>(a, sms, stream);
}

template <typename T, bool VEC>
cudaError_t backward_typed(const UnsortBackwardArgs& a, int sms, cudaStream_t stream) {
  UnsortBackwardParams p;
  p.a = a;
  p.row_vecs = a.hidden / Bit<T, VEC>::N;
  // Two vectors a lane, or one where there are few tokens, and then up to 1024 lanes (us: 128 tokens, top-8, 14 KiB 9.7 with two
  // and 256 lanes, 6.1; 256 of them 15.0, with one and 512 lanes 10.4; 4096, top-6, 8 KiB 75.9 with two, 86.5 with one).
  const int each = a.tokens <= 4 * sms ? 1 : 2;
  const int threads = std::max(32, std::min(a.tokens <= sms ? 1024 : 512, (p.row_vecs / each + 31) / 32 * 32));
  const int grid = (int)std::min<int64_t>(std::max(a.tokens, 1), 1 << 30);
  return a.grad_weights != nullptr
             ? ptx::launch_dependent(unsort_tokens_backward_kernel<T, VEC, true>, grid, threads, 0, stream, p)
             : ptx::launch_dependent(unsort_tokens_backward_kernel<T, VEC, false>, grid, threads, 0, stream, p);
}

template <typename T>
cudaError_t backward_vec(const UnsortBackwardArgs& a, int sms, cudaStream_t stream) {
  const bool vec = a.hidden % Vec16<T>::N == 0 && a.grad_stride % 16 == 0 && a.rows_stride % 16 == 0 && aligned16(a.grad) &&
                   aligned16(a.rows) && aligned16(a.grad_rows);
  return vec ? backward_typed<T, true>(a, sms, stream) : backward_typed<T, false>(a, sms, stream);
}

}  // namespace

int64_t sort_tokens_work(int64_t tokens, int k, int experts) {
  if (tokens * k <= kOneLaunchEntries) return 0;
  return (int64_t)(sort_chunks(tokens, k) + 1) * experts + tokens * k;
}

cudaError_t launch_sort_tokens(const SortTokensArgs& a, int sms, cudaStream_t stream) {
  if (a.tokens < 0 || a.k < 1 || a.k > kSortMaxTopk || a.experts < 1 || a.experts > kSortMaxExperts ||
      (int64_t)a.tokens * a.k > INT32_MAX)
    return cudaErrorInvalidValue;
  SortParams p = {};
  p.a = a;
  p.vec_ids = (reinterpret_cast<uintptr_t>(a.indices) & 15u) == 0;
  const uint64_t bits = (uint64_t)a.row_bytes | (uint64_t)a.x_stride | reinterpret_cast<uintptr_t>(a.x) |
                        reinterpret_cast<uintptr_t>(a.rows);
  if (bits % 32 == 0) return sort_typed<Vec32>(p, sms, stream);
  if (bits % 16 == 0) return sort_typed<int4>(p, sms, stream);
  if (bits % 4 == 0) return sort_typed<int>(p, sms, stream);
  if (bits % 2 == 0) return sort_typed<short>(p, sms, stream);
  return sort_typed<signed char>(p, sms, stream);
}

cudaError_t launch_unsort_tokens(const UnsortTokensArgs& a, int sms, cudaStream_t stream) {
  if (a.tokens < 0 || a.k < 1 || a.k > kSortMaxTopk || a.hidden < 1) return cudaErrorInvalidValue;
  if (a.tokens == 0) return cudaSuccess;
  switch (a.dtype) {
    case 0: return unsort_vec<__half>(a, sms, stream);
    case 1: return unsort_vec<__nv_bfloat16>(a, sms, stream);
    case 2: return unsort_vec<float>(a, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_unsort_tokens_backward(const UnsortBackwardArgs& a, int sms, cudaStream_t stream) {
  if (a.tokens < 0 || a.k < 1 || a.k > kSortMaxTopk || a.hidden < 1) return cudaErrorInvalidValue;
  if (a.tokens == 0) return cudaSuccess;
  switch (a.dtype) {
    case 0: return backward_vec<__half>(a, sms, stream);
    case 1: return backward_vec<__nv_bfloat16>(a, sms, stream);
    case 2: return backward_vec<float>(a, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200
