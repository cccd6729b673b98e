// Block-scaled fp8 (e4m3) products of the experts of one GPU, for sm_100a:
//   C[r, n] = sum_kb (A_kb[r, :] . B_e,kb[n, :]) * as[r, kb] * bs[e, n / 128, kb]   for r in [offsets[e], offsets[e + 1])
// Rows of A are sorted by expert and packed; the offsets are device memory, so nothing waits for the host.
//
// An expert has a few rows or a few hundred, and never a whole number of tiles.  The weights take the side of the tensor
// cores' instruction whose size is fixed (a CTA pair has 256 rows of an expert's B, cta_group::2), the tokens the side
// whose size is free: a tile is cut to the rows that its expert has left, in steps of 32.  So the accumulators lie with
// output columns in tensor-memory lanes and tokens in columns.  In that order a token's scale belongs to a column, and read with a
// lane to a row every lane would need the scale of every column.  The epilogue reads 16 lanes x 256 bits instead, which
// gives a thread the same two columns of every eight for each of its four rows: one 16-byte read of scales (already
// multiplied by the weights' scale, and laid out in that order, by the two warps that bring them in) serves sixteen sums.
// The same layout is what stmatrix transposes on the way out, to rows of C.
//
// Every 128-wide K block is multiplied into a tensor-memory buffer of its own; eight epilogue warps (two per lane quarter,
// which take 32-token chunks in turn) multiply by the scales and accumulate in fp32 registers while the next buffer is
// being filled.  Pairs are persistent, and walk the same list of tiles: experts in order, an expert's weight tiles in
// order, its token tiles innermost, so that pairs at work at the same time share weights in L2.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "fp8_gemm.h"
#include "fp8_pipeline.cuh"
#include "gemm_rs.h"
#include "per_device.h"
#include "tensor_map.h"

namespace b200 {

namespace {

using namespace fp8;

constexpr int kRows = 128;  // rows of an expert's B per CTA
constexpr int kBlockK = 128;
constexpr int kWeightBytes = kRows * kBlockK;
constexpr int kChunk = 32;  // tokens of a chunk; a tile is a whole number of them
constexpr int kEpiWarps = 8;
constexpr int kScaleWarps = 2;
constexpr int kThreads = 64 + 32 * (kScaleWarps + kEpiWarps);
constexpr int kLightRegs = 56, kEpiRegs = 224;
static_assert(128 * kLightRegs + 256 * kEpiRegs == kThreads * 168, "not more than the block is launched with");
constexpr int kMaxStages = 12;
constexpr int kMaxBufs = 4;
constexpr int kGroup = 4;       // K blocks whose scales come in together
constexpr int kScaleSlots = 3;
constexpr int kSlabBytes = 16 * 64;  // per epilogue warp: 16 tokens x 32 output columns
constexpr int kBarBytes = 512;
constexpr int kMaxDynamicSmem = 232448 - 256;
constexpr int kTmemCols = 512;
constexpr int kBigBox = 64, kSmallBox = 16;  // rows of a copy of tokens

struct GroupedParams {
  const float* a_scale;
  const float* b_scale;
  const int32_t* offsets;
  __nv_bfloat16* c;
  int M, N, experts, k_blocks, n_tiles;
  long long as_stride_m, as_stride_k, bs_stride_e, bs_stride_n, bs_stride_k;
  int stages;
  int vec_out;     // 1: rows of C are whole aligned 16-byte pieces
  int vec_scales;  // 1: four neighbouring scales of a row of A are an aligned 16-byte piece
  int zero_rest;
  uint64_t timeout_ns;
  StatusWord* status;
};

// What a tile of the list is.
struct Tile {
  int expert, nt;
  int row0, rows;  // of A
  int width;       // rows, rounded up to whole chunks
};

// The experts' rows and the number of tiles up to and including each, in shared memory.
struct Tables {
  int32_t *start, *count, *tiles_end;
};

template <int BT>
struct Walk {
  const Tables& t;
  int n_tiles;
  int e = 0;
  __device__ __forceinline__ Tile at(int tile) {
    while (tile >= t.tiles_end[e]) ++e;
    const int local = tile - (e > 0 ? t.tiles_end[e - 1] : 0);
    const int count = t.count[e];
    const int parts = (count + BT - 1) / BT;
    const int each = ((count + parts - 1) / parts + kChunk - 1) / kChunk * kChunk;  // tiles of an expert are of one size
    Tile r;
    r.expert = e;
    r.nt = local / parts;
    const int part = local - r.nt * parts;
    r.row0 = t.start[e] + part * each;
    r.rows = min(each, count - part * each);
    r.width = (r.rows + kChunk - 1) / kChunk * kChunk;
    return r;
  }
};

// Where a token's scale lies among those of its 16: a lane's four (columns 2 q, 2 q + 1 of both groups of eight) side by side.
__device__ __forceinline__ int scale_place(int token) {
  return (token & ~15) | ((token >> 1 & 3) << 2) | ((token >> 3 & 1) << 1) | (token & 1);
}

}  // namespace

// CH: 32-token chunks of an epilogue warp; a tile has up to 64 * CH tokens.
template <int CH>
__global__ void __launch_bounds__(kThreads, 1)
fp8_grouped_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_big,
                   const __grid_constant__ CUtensorMap map_small, const GroupedParams p) {
  constexpr int kBt = 64 * CH;
  constexpr int kBufs = kBt == 256 ? 2 : kMaxBufs;
  constexpr uint32_t kBufCols = kBt;
  constexpr uint32_t kStageBytes = kWeightBytes + kBt / 2 * kBlockK;
  constexpr uint32_t kSlotBytes = kGroup * kBt * 4;
  extern __shared__ uint8_t smem_raw[];
  __shared__ volatile int abort_flag;
  __shared__ uint32_t tmem_base_shared;
  __shared__ int32_t warp_sums[kThreads / 32];

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int lane = tid & 31;
  const int cta = (int)ptx::cluster_ctarank();

  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t slabs = base + (uint32_t)p.stages * kStageBytes;
  const uint32_t scales = slabs + kEpiWarps * kSlabBytes;
  const uint32_t bars = scales + kScaleSlots * kSlotBytes;
  uint8_t* const tail = smem_raw + (bars + kBarBytes - ptx::smem_u32(smem_raw));
  Tables tables;
  tables.start = reinterpret_cast<int32_t*>(tail);
  tables.count = tables.start + p.experts;
  tables.tiles_end = tables.count + p.experts;
  auto full_bar = [&](uint32_t s) { return bars + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bars + 8u * (kMaxStages + s); };
  auto tfull_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + s); };
  auto tempty_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + kMaxBufs + s); };
  auto sfull_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + 2 * kMaxBufs + s); };
  auto sempty_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + 2 * kMaxBufs + kScaleSlots + s); };

  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < kBufs; ++s) {
      ptx::mbar_init(tfull_bar(s), 1);
      ptx::mbar_init(tempty_bar(s), 2 * kEpiWarps);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      ptx::mbar_init(sfull_bar(s), 32 * kScaleWarps);
      ptx::mbar_init(sempty_bar(s), kEpiWarps);
    }
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
    ptx::prefetch_tensormap(&map_b);
    ptx::prefetch_tensormap(&map_big);
    ptx::prefetch_tensormap(&map_small);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_u32(&tmem_base_shared), kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  ptx::grid_dep_launch();
  ptx::grid_dep_wait();
  // The tables: a run of experts to a thread, then a prefix over threads.
  {
    const int each = (p.experts + kThreads - 1) / kThreads;
    const int lo = min(p.experts, tid * each), hi = min(p.experts, lo + each);
    int own = 0;
    for (int e = lo; e < hi; ++e) {
      const int from = min(max(__ldcg(p.offsets + e), 0), p.M);
      const int to = min(max(__ldcg(p.offsets + e + 1), from), p.M);
      tables.start[e] = from;
      tables.count[e] = to - from;
      own += (to - from + kBt - 1) / kBt * p.n_tiles;
      tables.tiles_end[e] = own;
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    int before = upto - own;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    for (int e = lo; e < hi; ++e) tables.tiles_end[e] += before;
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tcgen05_fence_after();
  const uint32_t tmem_base = tmem_base_shared;
  const int total = tables.tiles_end[p.experts - 1];
  const int first_tile = (int)blockIdx.x >> 1, tile_step = (int)gridDim.x >> 1;
  Walk<kBt> walk{tables, p.n_tiles};

  // All of a CTA's threads come here in the end, each role on its own way: no CTA retires while the other may still signal
  // its barriers.
  auto leave = [&]() {
    if (abort_flag) {
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 200000) __nanosleep(1000);
      if (lane == 0) record_expired(p, abort_flag);
    }
    __syncwarp();
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::cluster_sync_all();
    ptx::tcgen05_fence_after();
    if (warp == 1) ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
  };

  if (warp < 2 + kScaleWarps) {
    ptx::setmaxnreg_dec<kLightRegs>();
    if (warp == 0) {
      uint32_t stage = 0, phase = 0;
      for (int tile = first_tile; tile < total && !abort_flag; tile += tile_step) {
        const Tile t = walk.at(tile);
        const int by = t.expert * p.N + t.nt * 2 * kRows + cta * kRows;
        const int half = t.width / 2;  // tokens that this CTA brings in
        const int ay = t.row0 + cta * half;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!fp8_wait(empty_bar(stage), phase ^ 1u, &abort_flag, p, 100 + (int)stage)) break;
          const uint32_t sa = base + stage * kStageBytes;
          if (ptx::elect_one()) {
            if (cta == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), 2u * (uint32_t)(kWeightBytes + half * kBlockK));
            ptx::tma_load_2d_pair(sa, &map_b, full_bar(stage), kb * kBlockK, by);
            int r = 0;
            for (; r + kBigBox <= half; r += kBigBox)
              ptx::tma_load_2d_pair(sa + kWeightBytes + r * kBlockK, &map_big, full_bar(stage), kb * kBlockK, ay + r);
            for (; r < half; r += kSmallBox)
              ptx::tma_load_2d_pair(sa + kWeightBytes + r * kBlockK, &map_small, full_bar(stage), kb * kBlockK, ay + r);
          }
          __syncwarp();
          if (++stage == (uint32_t)p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == 1) {
      if (cta == 0) {
        uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
        for (int tile = first_tile; tile < total && !abort_flag; tile += tile_step) {
          const Tile t = walk.at(tile);
          const uint32_t idesc = make_idesc_e4m3_f32(256, t.width);
          bool ok = true;
          for (int kb = 0; kb < p.k_blocks && ok; ++kb) {
            ok = fp8_wait(tempty_bar(buf), buf_phase ^ 1u, &abort_flag, p, 200 + (int)buf) &&
                 fp8_wait(full_bar(stage), phase, &abort_flag, p, 300 + (int)stage);
            if (!ok) break;
            ptx::tcgen05_fence_after();
            const uint32_t sa = base + stage * kStageBytes;
            const uint64_t da = ptx::make_smem_desc_k_sw128(sa);
            const uint64_t db = ptx::make_smem_desc_k_sw128(sa + kWeightBytes);
            const uint32_t d = tmem_base + buf * kBufCols;
            if (ptx::elect_one()) {
#pragma unroll
              for (int j = 0; j < kBlockK / 32; ++j)  // 32 fp8 of K = 32 bytes = 2 descriptor address units
                umma_fp8_pair(d, da + 2u * j, db + 2u * j, idesc, j > 0 ? 1u : 0u);
              ptx::umma_commit_pair(empty_bar(stage), 3);
              ptx::umma_commit_pair(tfull_bar(buf), 3);
            }
            __syncwarp();
            if (++stage == (uint32_t)p.stages) {
              stage = 0;
              phase ^= 1u;
            }
            if (++buf == (uint32_t)kBufs) {
              buf = 0;
              buf_phase ^= 1u;
            }
          }
          if (!ok) break;
        }
      }
    } else {
      // ---- scales: those of four K blocks for up to CH tokens a lane, times the weights' --------------------
      const int l = (warp - 2) * 32 + lane;
      uint32_t slot = 0, phase = 0;
      for (int tile = first_tile; tile < total && !abort_flag; tile += tile_step) {
        const Tile t = walk.at(tile);
        const float* bs = p.b_scale + t.expert * p.bs_stride_e + min(t.nt * 2 + cta, (p.N - 1) >> 7) * p.bs_stride_n;
        for (int kb = 0; kb < p.k_blocks; kb += kGroup) {
          float b[kGroup], s[CH][kGroup];
#pragma unroll
          for (int i = 0; i < kGroup; ++i) b[i] = __ldg(bs + min(kb + i, p.k_blocks - 1) * p.bs_stride_k);
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const int token = l + 64 * c;
            const float* as = p.a_scale + (long long)min(t.row0 + token, p.M - 1) * p.as_stride_m;
            if (token >= t.rows) {
#pragma unroll
              for (int i = 0; i < kGroup; ++i) s[c][i] = 0.f;
            } else if (p.vec_scales) {
              const float4 f = __ldg(reinterpret_cast<const float4*>(as + kb));
              s[c][0] = f.x, s[c][1] = f.y, s[c][2] = f.z, s[c][3] = f.w;
            } else {
#pragma unroll
              for (int i = 0; i < kGroup; ++i) s[c][i] = __ldg(as + min(kb + i, p.k_blocks - 1) * p.as_stride_k);
            }
          }
          if (!fp8_wait(sempty_bar(slot), phase ^ 1u, &abort_flag, p, 500 + (int)slot)) break;
          const uint32_t at = scales + slot * kSlotBytes;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const int token = l + 64 * c;
            if (token < t.width) {
#pragma unroll
              for (int i = 0; i < kGroup; ++i)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + (uint32_t)(i * kBt + scale_place(token)) * 4u),
                             "f"(s[c][i] * b[i])
                             : "memory");
            }
          }
          ptx::mbar_arrive(sfull_bar(slot));
          if (++slot == kScaleSlots) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
    }
    leave();
    return;
  }

  // ---- epilogue ----------------------------------------------------------------------------------------------------
  ptx::setmaxnreg_inc<kEpiRegs>();
  const int ew = warp - 2 - kScaleWarps;
  const int q = warp & 3;
  const int side = ew >> 2;  // chunks side, side + 2, ... of a tile
  {
    const uint32_t slab = slabs + (uint32_t)ew * kSlabBytes;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(side * kChunk);
    const uint32_t leader_tempty = ptx::map_cluster(tempty_bar(0), 0);
    const uint32_t scale_at = scales + (uint32_t)(side * kChunk + (lane & 3) * 4) * 4u;
    uint32_t buf = 0, buf_phase = 0, slot = 0, slot_phase = 0;
    bool alive = true;
    for (int tile = first_tile; tile < total && !abort_flag; tile += tile_step) {
      const Tile t = walk.at(tile);
      const int n0 = t.nt * 2 * kRows + cta * kRows + q * 32;
      const int chunks = n0 < p.N ? (t.width / kChunk - side + 1) >> 1 : 0;  // of this warp
      float2 acc[CH][2][4][2];  // [chunk][16 lanes][8 tokens][8 lanes]: the sums of two neighbouring tokens
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[c][x >> 3][x >> 1 & 3][x & 1] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        const int g = kb % kGroup;
        if (g == 0) alive &= fp8_wait(sfull_bar(slot), slot_phase, &abort_flag, p, 600 + (int)slot);
        alive &= fp8_wait(tfull_bar(buf), buf_phase, &abort_flag, p, 400 + (int)buf);
        __syncwarp();
        ptx::tcgen05_fence_after();
        auto done = [&]() {  // the buffer is free for the next products (the warp is converged, and its reads are complete)
          ptx::tcgen05_fence_before();
          ptx::mbar_arrive_remote_if(lane == 0, leader_tempty + 8u * buf);
        };
        if (chunks == 0) done();
        const uint32_t s_at = scale_at + slot * kSlotBytes + (uint32_t)(g * kBt * 4);
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          if (c < chunks) {
            constexpr int kAtOnce = CH > 1 ? 2 : 1;
            uint32_t v[kAtOnce][2][16];
            float s[kAtOnce][8];
#pragma unroll
            for (int d = 0; d < kAtOnce; ++d) {
              // (a chunk behind the tile's last is read and added up too: its columns lie in the buffer, its sums go nowhere)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                ptx::tmem_ld_16x256b_x4(lane_addr + ((uint32_t)(h * 16) << 16) + buf * kBufCols + (c + d) * 2 * kChunk, v[d][h]);
              ld_shared_f4(s[d], s_at + (uint32_t)((c + d) * 2 * kChunk) * 4u);
              ld_shared_f4(s[d] + 4, s_at + (uint32_t)((c + d) * 2 * kChunk + 16) * 4u);
            }
            ptx::tmem_ld_wait();
            if (c + 2 >= chunks) done();
#pragma unroll
            for (int d = 0; d < kAtOnce; ++d)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 ss = make_float2(s[d][2 * i], s[d][2 * i + 1]);
                  fma2(acc[c + d][h][i][0], v[d][h][4 * i], v[d][h][4 * i + 1], ss);
                  fma2(acc[c + d][h][i][1], v[d][h][4 * i + 2], v[d][h][4 * i + 3], ss);
                }
          }
        }
        if (g == kGroup - 1 || kb + 1 == p.k_blocks) {
          __syncwarp();
          ptx::mbar_arrive_if(lane == 0, sempty_bar(slot));
          if (++slot == kScaleSlots) {
            slot = 0;
            slot_phase ^= 1u;
          }
        }
        if (++buf == (uint32_t)kBufs) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      // ---- result: 16 tokens at a time through the slab, 64 bytes of a row to four lanes ---------------------
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (c >= chunks) break;
        const int token0 = (2 * c + side) * kChunk;
#pragma unroll
        for (int i0 = 0; i0 < 4; i0 += 2) {
#pragma unroll
          for (int i = i0; i < i0 + 2; ++i) {
            const int row = (i - i0) * 8 + (lane & 7);  // of the slab: a token
            const uint32_t at = slab + (uint32_t)row * 64u + (uint32_t)(((lane >> 3) ^ (row >> 1 & 3)) << 4);
            ptx::stmatrix_x4_trans(at, pack2(acc[c][0][i][0]), pack2(acc[c][0][i][1]), pack2(acc[c][1][i][0]),
                                   pack2(acc[c][1][i][1]));
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int row = (lane >> 2) + 8 * j, piece = lane & 3;
            uint32_t v[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                         : "r"(slab + (uint32_t)row * 64u + (uint32_t)((piece ^ (row >> 1 & 3)) << 4))
                         : "memory");
            const int token = token0 + i0 * 8 + row, n = n0 + piece * 8;
            if (token < t.rows && n < p.N) {
              __nv_bfloat16* to = p.c + (long long)(t.row0 + token) * p.N + n;
              if (p.vec_out) {
                *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
              } else {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                  if (n + x < p.N) reinterpret_cast<uint16_t*>(to)[x] = (uint16_t)(v[x >> 1] >> (16 * (x & 1)));
              }
            }
          }
          __syncwarp();
        }
      }
    }
    if (p.zero_rest) {  // rows of no expert, a row to a warp
      const int end = min(max(__ldcg(p.offsets + p.experts), 0), p.M);
      for (int row = end + (int)blockIdx.x * kEpiWarps + ew; row < p.M; row += (int)gridDim.x * kEpiWarps) {
        __nv_bfloat16* c = p.c + (long long)row * p.N;
        if (p.vec_out) {
          for (int n = lane * 8; n < p.N; n += 256) *reinterpret_cast<uint4*>(c + n) = make_uint4(0, 0, 0, 0);
        } else {
          for (int n = lane; n < p.N; n += 32) c[n] = __float2bfloat16_rn(0.f);
        }
      }
    }
  }
  leave();
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
namespace {

int tail_bytes(int bt, int experts) {
  return kEpiWarps * kSlabBytes + kScaleSlots * kGroup * bt * 4 + kBarBytes + 3 * 4 * experts;
}
int stage_bytes(int bt) { return kWeightBytes + bt / 2 * kBlockK; }
int stages_of(int bt, int experts) {
  return std::min(kMaxStages, (kMaxDynamicSmem - 1024 - tail_bytes(bt, experts)) / stage_bytes(bt));
}

template <int CH>
cudaError_t launch(const GroupedParams& p, int pairs, int smem, const CUtensorMap& map_b, const CUtensorMap& map_big,
                   const CUtensorMap& map_small, cudaStream_t stream) {
  static OncePerDevice once;
  const cudaError_t opted = once([] { return opt_in(fp8_grouped_kernel<CH>, kMaxDynamicSmem, false); });
  if (opted != cudaSuccess) return opted;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, fp8_grouped_kernel<CH>, map_b, map_big, map_small, p);
}

}  // namespace

int fp8_grouped_tile(int M, int experts) {
  const int mean = M / std::max(experts, 1);
  return mean <= 48 ? 64 : mean <= 96 ? 128 : 256;
}

int fp8_grouped_smem(int tile, int experts) {
  return 1024 + stages_of(tile, experts) * stage_bytes(tile) + tail_bytes(tile, experts);
}

cudaError_t launch_fp8_grouped_gemm(const Fp8GroupedArgs& a, cudaStream_t stream) {
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.K % 16 != 0 || a.experts < 1 || a.experts > kGroupedMaxExperts ||
      (int64_t)a.experts * a.N > INT32_MAX)
    return cudaErrorInvalidValue;
  const int bt = fp8_grouped_tile(a.M, a.experts);
  GroupedParams p = {};
  p.a_scale = a.a_scale;
  p.b_scale = a.b_scale;
  p.offsets = a.offsets;
  p.c = reinterpret_cast<__nv_bfloat16*>(a.c);
  p.M = a.M;
  p.N = a.N;
  p.experts = a.experts;
  p.k_blocks = (a.K + kBlockK - 1) / kBlockK;
  p.n_tiles = (a.N + 2 * kRows - 1) / (2 * kRows);
  p.as_stride_m = a.as_stride_m;
  p.as_stride_k = a.as_stride_k;
  p.bs_stride_e = a.bs_stride_e;
  p.bs_stride_n = a.bs_stride_n;
  p.bs_stride_k = a.bs_stride_k;
  p.stages = stages_of(bt, a.experts);
  p.vec_out = a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.c) & 15u) == 0;
  p.vec_scales = a.as_stride_k == 1 && a.as_stride_m % 4 == 0 && p.k_blocks % 4 == 0 &&
                 (reinterpret_cast<uintptr_t>(a.a_scale) & 15u) == 0;
  p.zero_rest = a.zero_rest;
  p.timeout_ns = a.timeout_ns;
  p.status = a.status;
  // tiles at the most: every expert's last one may be a single row
  const int64_t most = std::min<int64_t>(a.M, a.M / bt + a.experts) * p.n_tiles;
  if (most > INT32_MAX / 2) return cudaErrorInvalidValue;
  const int pairs = (int)std::min<int64_t>(most, std::min(gemm_cluster_capacity(2), a.sms / 2));
  CUtensorMap map_b, map_big, map_small;
  if (!make_tensor_map(&map_b, a.b, (uint64_t)a.experts * a.N, (uint64_t)a.K, 1, kRows, kBlockK, 128) ||
      !make_tensor_map(&map_big, a.a, (uint64_t)a.M, (uint64_t)a.K, 1, kBigBox, kBlockK, 128) ||
      !make_tensor_map(&map_small, a.a, (uint64_t)a.M, (uint64_t)a.K, 1, kSmallBox, kBlockK, 128))
    return cudaErrorInvalidValue;
  const int smem = fp8_grouped_smem(bt, a.experts);
  switch (bt) {
    case 64: return launch<1>(p, pairs, smem, map_b, map_big, map_small, stream);
    case 128: return launch<2>(p, pairs, smem, map_b, map_big, map_small, stream);
    default: return launch<4>(p, pairs, smem, map_b, map_big, map_small, stream);
  }
}

}  // namespace b200
