// Block-scaled fp8 (e4m3) products of the experts of one GPU, for sm_100a:
//   C[r, n] = sum_kb (A_kb[r, :] . B_e,kb[n, :]) * as[r, kb] * bs[e, n / 128, kb]   for r in [offsets[e], offsets[e + 1])
// Rows of A are sorted by expert and packed; the offsets are device memory, so nothing waits for the host.
//
// A CTA pair (cta_group::2) multiplies 256 output columns of an expert by some of its rows.  Which of the two is which side
// of the tensor cores' instruction goes by how many rows there are (two kernels, chosen by the mean):
//   WIDE    Tokens are the rows of the product, 256 of them, or 128 where an expert has no more left.  A token lies in a
//           tensor-memory lane, so its scale is one number to an epilogue thread and K block.
//   else    Output columns are the rows, tokens the side whose size is free: 32 or 64.  What counts is that the weights
//           stream: eight stages of 16 KB of them lie ahead in each SM.  A token's scale belongs to a column then; the
//           epilogue reads 16 lanes x 128 bits of tensor memory at a time, which gives a thread every fourth token, and so eight
//           scales for sixteen sums instead of a scale a sum.  stmatrix turns the result around on its way out.
// Scales come in by two warps, which multiply both operands' and lay them out as the epilogue reads them.
//
// Every 128-wide K block is multiplied into tensor memory of its own: two buffers of 256 columns, each for one K block (256
// tokens), two (128) or four.  Eight epilogue warps, two to a lane quarter, take a buffer out, hand it back, and add it up in
// fp32 registers while the other is being filled.  Pairs are persistent, and walk the same list of tiles: experts in order,
// an expert's in bands, so that pairs at work at the same time share weights and tokens in L2.
//
// What bounds it: few rows, the weights out of memory (256 experts of 2048 x 7168 with 4 rows each: 3.76 GB in 525 to 568 us
// from box to box, 6.6 to 7.2 TB/s, in a row of calls); many rows, the chain of an epilogue warp, as in fp8_gemm (8192 x 4096 x
// 4096, one expert: 122 us, 121 there, 2.25 PFLOP/s); skewed routing (24576 rows over 64 experts of 4096 x 4096, 1 GB of weights)
// is between the two: 478 us at first, 535 to 584 where calls follow on one another for a second: power, at 1.3 to 1.4 GHz.
// What it took, us at 8192 rows of one expert / of 64 experts / at 256 experts with 4 rows each:
//   tokens always on the free side, up to 256 of them, 16 x 256 bits           154 / 232 / 570
//   the next piece out of tensor memory while one is added up                  176 / 208 / 552   (registers spill)
//   256 tokens as rows                                                         128 / 224 / 537
//   16 x 128 bits instead (the tensor memory gives those four times as fast)   127 / 221 / 537
//   buffers emptied at once and handed back before the sums                    120 / 220 / 537
//   128 tokens as rows                                                         123 / 200 / 537
//   bands, the epilogue told its tiles                                         122 / 200 / 537   (24576 skewed: 491 to 478)
// Shared memory is what the free side runs short of: sixteen-byte reads take four passes each beside what the tensor cores
// read (920 cycles for the sums of a buffer that take 240 without them; asked for a half ahead, 650).  A spilled register in
// the loop costs more the more shared memory is taken, as L1 is what is left of it.  L2 prefetches of weights ahead of the
// copies: 530 to 590 and more in the last column.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

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
constexpr int kLightRegs = 40, kEpiRegs = 232;
static_assert(128 * kLightRegs + 256 * kEpiRegs == kThreads * 168, "not more than the block is launched with");
// More stages do not pay: what they take is taken from L1, which the scales come through.
constexpr int kMaxStages = 8, kWideStages = 5;
constexpr int kBufs = 2;        // tensor-memory buffers of 256 columns
constexpr uint32_t kBufCols = 256;
constexpr int kGroup = 4;       // K blocks whose scales come in together
constexpr int kScaleSlots = 4;
constexpr int kSlabBytes = 2048;  // per epilogue warp: 32 tokens x 32 output columns
constexpr int kBarBytes = 512;  // barriers, and behind them notes of what tiles are
constexpr int kNotes = 8, kNotesAt = 256;  // of tiles, 16 bytes each
static_assert(8 * (2 * kMaxStages + 2 * kBufs + 2 * kScaleSlots) <= kNotesAt && kNotesAt + 16 * kNotes <= kBarBytes);
static_assert(kNotes > kScaleSlots + 1, "a tile has a slot of scales at least: no note is written over that is still read");
constexpr int kMaxDynamicSmem = 232448 - 256;
constexpr int kTmemCols = 512;
constexpr int kBigBox = 64, kSmallBox = 16;  // rows of a copy of tokens
constexpr long long kFall = 1ll << 42;  // added to the sum of rows (2^10 counts below 2^31) for an offset below the one before it

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
  int width;       // tokens that are brought in and multiplied: 256, 128, or rows rounded up to whole chunks
};

// The experts' rows and the number of tiles up to and including each, in shared memory.
struct Tables {
  int32_t *start, *count, *tiles_end;
};

// The list: experts in order, an expert's token tiles in bands of at most kBand (all about as wide), a band's weight tiles in
// order, its token tiles innermost.  What pairs at work at the same time read is then small next to what they multiply, as in
// fp8_gemm: without bands the one expert of 24576 rows takes 414 us instead of 364, 476 instead of 414 where calls follow on
// one another for a second, and power is what there is too little of.
//
// A pair's tiles: dealt out in turn, every other round the other way round.  Were it always the same, the token tiles of
// experts with 384 rows each, 256 and 128, would go to even and to odd pairs for good (64 of them: 533 us, 412 to 420).
// (A tile from the front of the list and one from its end in turn, or a run of it to each pair, evens out as much and takes
// L2 its sense: skewed routing 493 and 645 us against 480 then.)
constexpr int kBand = 8;
template <int BT>
struct Walk {
  Tables t;
  int experts, n_tiles;
  // The pair's tile of a round, or -1 behind the last.
  __device__ __forceinline__ int tile_of(int round) const {
    const int pairs = (int)gridDim.x >> 1, pair = (int)blockIdx.x >> 1;
    const int tile = round * pairs + ((round & 1) != 0 ? pairs - 1 - pair : pair);
    return tile < t.tiles_end[experts - 1] ? tile : -1;
  }
  __device__ __forceinline__ Tile at(int tile) const {
    int e = 0;
    for (int above = experts; above - e > 0;) {  // the first whose tiles end behind this one
      const int m = (e + above) >> 1;
      if (t.tiles_end[m] > tile) above = m;
      else e = m + 1;
    }
    const int local = tile - (e > 0 ? t.tiles_end[e - 1] : 0);
    const int count = t.count[e];
    const int parts = (count + BT - 1) / BT;
    Tile r;
    r.expert = e;
    int part = 0;
    r.nt = local;
    if (parts > 1) {
      const int bands = (parts + kBand - 1) / kBand, wide = (parts + bands - 1) / bands;
      const int band = local / (wide * n_tiles), in_band = local - band * wide * n_tiles;
      const int of_band = min(wide, parts - band * wide);
      r.nt = in_band / of_band;
      part = band * wide + in_band - r.nt * of_band;
    }
    r.row0 = t.start[e] + part * BT;
    r.rows = min(BT, count - part * BT);
    r.width = BT == 64 ? (r.rows + kChunk - 1) / kChunk * kChunk : r.rows > kRows ? 2 * kRows : kRows;
    return r;
  }
};

// Where a token's scale lies among those of its chunk: a lane's eight (every fourth token) side by side.
__device__ __forceinline__ int scale_place(int token) { return (token & ~31) | ((token & 3) << 3) | (token >> 2 & 7); }

}  // namespace

// WIDE: tiles of up to 256 tokens, else of up to 64.
template <bool WIDE>
__global__ void __launch_bounds__(kThreads, 1)
fp8_grouped_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_big,
                   const __grid_constant__ CUtensorMap map_small, const GroupedParams p) {
  constexpr int kBt = WIDE ? 256 : 64;
  constexpr uint32_t kStageBytes = kWeightBytes + kBt / 2 * kBlockK;
  constexpr uint32_t kSlotBytes = kGroup * kBt * 4;
  extern __shared__ uint8_t smem_raw[];
  __shared__ volatile int abort_flag;
  __shared__ uint32_t tmem_base_shared;
  __shared__ int32_t warp_sums[kThreads / 32];
  __shared__ long long warp_rows[kThreads / 32];

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
  auto tempty_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + kBufs + s); };
  auto sfull_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + 2 * kBufs + s); };
  auto sempty_bar = [&](uint32_t s) { return bars + 8u * (2 * kMaxStages + 2 * kBufs + kScaleSlots + s); };
  // What the tile of a round is, for the epilogue.
  auto note = [&](int round) { return bars + (uint32_t)(kNotesAt + round % kNotes * 16); };

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
  // The tables: a run of experts to a thread, then a prefix over threads.  Offsets that give more rows than there are would
  // name tiles without end: nothing is computed then, and the record says so.  Fewer rows, with offsets that fall, would give
  // some of them to two experts, whose tiles would write them at the same time: an offset counts as the largest up to it
  // then, which one thread works out.
  {
    const int each = (p.experts + kThreads - 1) / kThreads;
    const int lo = min(p.experts, tid * each), hi = min(p.experts, lo + each);
    int own = 0;
    long long rows = 0;
    for (int e = lo; e < hi; ++e) {
      const int here = __ldcg(p.offsets + e), next = __ldcg(p.offsets + e + 1);
      const int from = min(max(here, 0), p.M);
      const int to = min(max(next, from), p.M);
      tables.start[e] = from;
      tables.count[e] = to - from;
      own += (to - from + kBt - 1) / kBt * p.n_tiles;
      tables.tiles_end[e] = own;
      rows += to - from + (next < here ? kFall : 0);
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rows += __shfl_xor_sync(0xffffffffu, rows, o);
    if (lane == 31) warp_sums[warp] = upto;
    if (lane == 0) warp_rows[warp] = rows;
    __syncthreads();
    int before = upto - own;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    rows = 0;
    for (int w = 0; w < kThreads / 32; ++w) rows += warp_rows[w];
    const bool falls = rows >= kFall;
    rows %= kFall;
    const bool bad = rows > p.M;
    for (int e = lo; e < hi; ++e) tables.tiles_end[e] = bad ? 0 : tables.tiles_end[e] + before;
    if (falls && !bad) {
      __syncthreads();
      if (tid == 0) {
        int from = min(max(__ldcg(p.offsets), 0), p.M), tiles = 0;
        for (int e = 0; e < p.experts; ++e) {
          const int to = min(max(__ldcg(p.offsets + e + 1), from), p.M);
          tables.start[e] = from;
          tables.count[e] = to - from;
          tiles += (to - from + kBt - 1) / kBt * p.n_tiles;
          tables.tiles_end[e] = tiles;
          from = to;
        }
      }
    }
    if (bad && blockIdx.x == 0 && tid == 0 && p.status != nullptr)
      store_status(p.status, STATUS_BAD_INDEX, PHASE_NONE, -1, p.experts, 0, (uint64_t)rows);
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tcgen05_fence_after();
  const uint32_t tmem_base = tmem_base_shared;
  const Walk<kBt> walk{tables, p.experts, p.n_tiles};
  // K blocks that are multiplied into a tensor-memory buffer one beside the other.
  auto steps = [](int width) { return WIDE ? 2 * kRows / width : 4; };

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
      for (int round = 0, tile; (tile = walk.tile_of(round)) >= 0 && !abort_flag; ++round) {
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
        for (int round = 0, tile; (tile = walk.tile_of(round)) >= 0 && !abort_flag; ++round) {
          const Tile t = walk.at(tile);
          const uint32_t idesc = WIDE ? make_idesc_e4m3_f32(t.width, 2 * kRows) : make_idesc_e4m3_f32(2 * kRows, t.width);
          const int step = steps(t.width);
          const uint32_t block_cols = kBufCols / (uint32_t)step;
          bool ok = true;
          for (int kb = 0; kb < p.k_blocks && ok; kb += step) {
            ok = fp8_wait(tempty_bar(buf), buf_phase ^ 1u, &abort_flag, p, 200 + (int)buf);
            ptx::tcgen05_fence_after();
            const int here = min(step, p.k_blocks - kb);
            for (int i = 0; i < here; ++i) {
              ok = ok && fp8_wait(full_bar(stage), phase, &abort_flag, p, 300 + (int)stage);
              if (!ok) break;
              ptx::tcgen05_fence_after();
              const uint32_t sa = base + stage * kStageBytes;
              const uint64_t da = ptx::make_smem_desc_k_sw128(WIDE ? sa + kWeightBytes : sa);
              const uint64_t db = ptx::make_smem_desc_k_sw128(WIDE ? sa : sa + kWeightBytes);
              const uint32_t d = tmem_base + buf * kBufCols + (uint32_t)i * block_cols;
              if (ptx::elect_one()) {
#pragma unroll
                for (int j = 0; j < kBlockK / 32; ++j)  // 32 fp8 of K = 32 bytes = 2 descriptor address units
                  umma_fp8_pair(d, da + 2u * j, db + 2u * j, idesc, j > 0 ? 1u : 0u);
                ptx::umma_commit_pair(empty_bar(stage), 3);
                if (i + 1 == here) ptx::umma_commit_pair(tfull_bar(buf), 3);
              }
              __syncwarp();
              if (++stage == (uint32_t)p.stages) {
                stage = 0;
                phase ^= 1u;
              }
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
      // ---- scales: those of four K blocks for up to two tokens a lane, times the weights' ---------------------
      // WIDE: tokens of this CTA's rows, as they come, once for each block of weights; else in the order in which the
      // epilogue's lanes read them.
      const int l = (warp - 2) * 32 + lane;
      uint32_t slot = 0, phase = 0;
      for (int round = 0, tile; (tile = walk.tile_of(round)) >= 0 && !abort_flag; ++round) {
        const Tile t = walk.at(tile);
        const int last = (p.N - 1) >> 7;
        const float* bs = p.b_scale + t.expert * p.bs_stride_e;
        const float* b0 = bs + min(t.nt * 2 + (WIDE ? 0 : cta), last) * p.bs_stride_n;
        const float* b1 = bs + min(t.nt * 2 + 1, last) * p.bs_stride_n;
        const int token0 = WIDE ? cta * (t.width / 2) : 0;
        // WIDE: the epilogue is told what the tile is, with the tile's first scales.  It bounds the kernel, and working out its
        // tiles itself, twice each, took it 2 to 3 % of its time.
        for (int kb = 0; kb < p.k_blocks; kb += kGroup) {
          float s[2][kGroup];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c == 1 && !(WIDE && t.width == 2 * kRows)) break;
            const int token = token0 + l + 64 * c;
            const float* as = p.a_scale + (long long)min(t.row0 + token, p.M - 1) * p.as_stride_m;
            if (token >= t.rows) {
#pragma unroll
              for (int i = 0; i < kGroup; ++i) s[c][i] = 0.f;
            } else if (p.vec_scales) {
              const float4 f = __ldca(reinterpret_cast<const float4*>(as + kb));
              s[c][0] = f.x, s[c][1] = f.y, s[c][2] = f.z, s[c][3] = f.w;
            } else {
#pragma unroll
              for (int i = 0; i < kGroup; ++i) s[c][i] = __ldca(as + min(kb + i, p.k_blocks - 1) * p.as_stride_k);
            }
          }
          float b[2][kGroup];
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            b[0][i] = __ldca(b0 + min(kb + i, p.k_blocks - 1) * p.bs_stride_k);
            if (WIDE) b[1][i] = __ldca(b1 + min(kb + i, p.k_blocks - 1) * p.bs_stride_k);
          }
          if (!fp8_wait(sempty_bar(slot), phase ^ 1u, &abort_flag, p, 500 + (int)slot)) break;
          const uint32_t at = scales + slot * kSlotBytes;
          if (WIDE && kb == 0 && l == 0)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(note(round)), "r"(t.nt), "r"(t.row0), "r"(t.rows), "r"(t.width)
                         : "memory");
          auto put = [&](int place, const float* f, const float* w) {
#pragma unroll
            for (int i = 0; i < kGroup; ++i)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + (uint32_t)(i * kBt + place) * 4u), "f"(f[i] * w[i]) : "memory");
          };
          if (WIDE) {
            put(l, s[0], b[0]);
            put(kRows + l, s[0], b[1]);
            if (t.width == 2 * kRows) {
              put(l + 64, s[1], b[0]);
              put(kRows + l + 64, s[1], b[1]);
            }
          } else {
            put(scale_place(l), s[0], b[0]);
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
  const int side = ew >> 2;  // which half of the columns (else: which of a tile's two chunks) is this warp's
  {
    const uint32_t slab = slabs + (uint32_t)ew * kSlabBytes;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16);
    const uint32_t leader_tempty = ptx::map_cluster(tempty_bar(0), 0);
    uint32_t bufs = 0, slots = 0;  // used so far: the low bits say which one is next, the bit above them its phase
    bool alive = true;
    auto arrive_done = [&]() {  // the buffer is free for the next products (the warp is converged, and its reads are complete)
      ptx::tcgen05_fence_before();
      ptx::mbar_arrive_remote_if(lane == 0, leader_tempty + 8u * (bufs & 1u));
    };
    auto await_products = [&]() {
      alive &= fp8_wait(tfull_bar(bufs & 1u), bufs >> 1 & 1u, &abort_flag, p, 400 + (int)(bufs & 1u));
      __syncwarp();
      ptx::tcgen05_fence_after();
    };
    auto await_scales = [&]() {
      alive &= fp8_wait(sfull_bar(slots % kScaleSlots), slots / kScaleSlots & 1u, &abort_flag, p, 600 + (int)(slots % kScaleSlots));
      __syncwarp();
    };
    auto free_scales = [&]() {
      __syncwarp();
      ptx::mbar_arrive_if(lane == 0, sempty_bar(slots % kScaleSlots));
      ++slots;
    };
    // 32 tokens x 32 columns leave through the slab, 64 bytes to a token (its four pieces swapped so that neither way meets
    // bank conflicts), in pieces of 16 bytes, four lanes to a token.
    auto piece_at = [&](int row, int piece) { return slab + (uint32_t)row * 64u + (uint32_t)((piece ^ (row >> 1 & 3)) << 4); };
    auto send = [&](int row0, int rows, int n0) {
      __syncwarp();
      rows = min(rows, 32);
      if (p.vec_out) {
        const int n = n0 + (lane & 3) * 8;
        if (n < p.N) {
          __nv_bfloat16* to = p.c + (long long)(row0 + (lane >> 2)) * p.N + n;
#pragma unroll 4
          for (int row = lane >> 2; row < rows; row += 8) {
            uint4 w;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                         : "r"(piece_at(row, lane & 3))
                         : "memory");
            *reinterpret_cast<uint4*>(to) = w;
            to += 8ll * p.N;
          }
        }
      } else if (n0 + lane < p.N) {  // a column to a lane
        uint16_t* to = reinterpret_cast<uint16_t*>(p.c) + (long long)row0 * p.N + n0 + lane;
#pragma unroll 1
        for (int row = 0; row < rows; ++row) {
          uint16_t w;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(piece_at(row, lane >> 3) + (uint32_t)(lane & 7) * 2u) : "memory");
          *to = w;
          to += p.N;
        }
      }
      __syncwarp();
    };
    auto noted = [&](int round) {
      Tile t;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(t.nt), "=r"(t.row0), "=r"(t.rows), "=r"(t.width)
                   : "r"(note(round))
                   : "memory");
      return t;
    };
    for (int round = 0, tile; (tile = walk.tile_of(round)) >= 0 && !abort_flag; ++round) {
      if (WIDE) await_scales();
      const Tile t = WIDE ? noted(round) : walk.at(tile);
      if (WIDE && t.width == 2 * kRows) {
        // ---- tokens in lanes: a lane's scale is its token's times that of its columns' block of weights -------
        // A CTA has 128 of 256 tokens in its lanes; `side` is the block of weights.
        const bool idle = t.rows <= cta * kRows + q * 32 || t.nt * 2 * kRows + side * kRows >= p.N;
        const uint32_t from = lane_addr + (uint32_t)(side * kRows);
        const uint32_t scale_at = scales + (uint32_t)(side * kRows + q * 32 + lane) * 4u;
        float2 acc[4][16];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[c][x] = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          const int g = kb % kGroup;
          if (g == 0) await_scales();
          float s;
          asm volatile("ld.shared.f32 %0, [%1];"
                       : "=f"(s)
                       : "r"(scale_at + slots % kScaleSlots * kSlotBytes + (uint32_t)(g * kBt * 4))
                       : "memory");
          await_products();
          if (!idle) {
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              uint32_t v[2][32];
              ptx::tmem_ld_32x32b_x32(from + (bufs & 1u) * kBufCols + c * 32, v[0]);
              ptx::tmem_ld_32x32b_x32(from + (bufs & 1u) * kBufCols + c * 32 + 32, v[1]);
              ptx::tmem_ld_wait();
              if (c == 2) arrive_done();
#pragma unroll
              for (int d = 0; d < 2; ++d)
#pragma unroll
                for (int x = 0; x < 16; ++x) fma2(acc[c + d][x], v[d][2 * x], v[d][2 * x + 1], make_float2(s, s));
            }
          } else {
            arrive_done();
          }
          ++bufs;
          if (g == kGroup - 1 || kb + 1 == p.k_blocks) free_scales();
        }
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        if (!idle) {
          const Tile t = noted(round);  // (again: what it takes to keep it through the loop is needed there)
          const int first = cta * kRows + q * 32, rows = t.rows - first, n0 = t.nt * 2 * kRows + side * kRows;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (n0 + c * 32 < p.N) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(lane, j)),
                             "r"(pack2(acc[c][4 * j])), "r"(pack2(acc[c][4 * j + 1])), "r"(pack2(acc[c][4 * j + 2])),
                             "r"(pack2(acc[c][4 * j + 3]))
                             : "memory");
              send(t.row0 + first, rows, n0 + c * 32);
            }
          }
        }
        continue;
      }
      if constexpr (WIDE) {
        // ---- the same for up to 128 tokens: a CTA has 64 of them in its lanes, once with each block of weights, whose
        // columns `side` halves; two K blocks to a buffer
        const bool idle = t.rows <= cta * (kRows / 2) + (q & 1) * 32 || t.nt * 2 * kRows + (q >> 1) * kRows + side * 64 >= p.N;
        const uint32_t from = lane_addr + (uint32_t)(side * 64);
        const uint32_t scale_at = scales + (uint32_t)((q >> 1) * kRows + (q & 1) * 32 + lane) * 4u;
        float2 acc[2][16];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[c][x] = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int kb = 0; kb < p.k_blocks; kb += 2) {
          const int g = kb % kGroup;
          if (g == 0) await_scales();
          float s[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            asm volatile("ld.shared.f32 %0, [%1];"
                         : "=f"(s[i])
                         : "r"(scale_at + slots % kScaleSlots * kSlotBytes + (uint32_t)((g + i) * kBt * 4))
                         : "memory");
          const bool both = kb + 1 < p.k_blocks;  // of the buffer's blocks; one that is not there is read as it is, and left
          await_products();
          if (!idle) {
            uint32_t v[4][32];
#pragma unroll
            for (int j = 0; j < 4; ++j) ptx::tmem_ld_32x32b_x32(from + (bufs & 1u) * kBufCols + (j >> 1) * 128 + (j & 1) * 32, v[j]);
            ptx::tmem_ld_wait();
            arrive_done();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (j < 2 || both) {
#pragma unroll
                for (int x = 0; x < 16; ++x) fma2(acc[j & 1][x], v[j][2 * x], v[j][2 * x + 1], make_float2(s[j >> 1], s[j >> 1]));
              }
            }
          } else {
            arrive_done();
          }
          ++bufs;
          if (g == kGroup - 2 || kb + 2 >= p.k_blocks) free_scales();
        }
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        if (!idle) {
          const Tile t = noted(round);
          const int first = cta * (kRows / 2) + (q & 1) * 32, rows = t.rows - first;
          const int n0 = t.nt * 2 * kRows + (q >> 1) * kRows + side * 64;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (n0 + c * 32 < p.N) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(lane, j)),
                             "r"(pack2(acc[c][4 * j])), "r"(pack2(acc[c][4 * j + 1])), "r"(pack2(acc[c][4 * j + 2])),
                             "r"(pack2(acc[c][4 * j + 3]))
                             : "memory");
              send(t.row0 + first, rows, n0 + c * 32);
            }
          }
        }
        continue;
      }
      // ---- output columns in lanes, a chunk of tokens to a warp; four K blocks to a buffer, 64 columns apart ----
      const int n0 = t.nt * 2 * kRows + cta * kRows + q * 32;
      if (n0 >= p.N || side * kChunk >= t.width) {  // nothing of the tile is this warp's
#pragma unroll 1
        for (int kb = 0; kb < p.k_blocks; kb += kGroup) {
          await_scales();
          await_products();
          arrive_done();
          ++bufs;
          free_scales();
        }
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        continue;
      }
      const uint32_t from = lane_addr + (uint32_t)(side * kChunk);
      const uint32_t scale_at = scales + (uint32_t)(side * kChunk + (lane & 3) * 8) * 4u;
      float2 acc[2][8];  // [16 lanes][4 tokens]: the sums of a token for two columns, 8 apart
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[x >> 3][x & 7] = make_float2(0.f, 0.f);
      // Two K blocks at a time.  Their scales are asked for two blocks ahead: beside the tensor cores, which read their
      // operands from shared memory, a load from there takes longer than the sums.
      float s[2][2][8];
      auto fetch = [&](int kb, float (&to)[2][8]) {
        if (kb % kGroup == 0) {
          if (kb > 0) free_scales();
          await_scales();
        }
        const uint32_t s_at = scale_at + slots % kScaleSlots * kSlotBytes + (uint32_t)(kb % kGroup * kBt * 4);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          ld_shared_f4(to[d], s_at + (uint32_t)(d * kBt * 4));
          ld_shared_f4(to[d] + 4, s_at + (uint32_t)(d * kBt * 4) + 16u);
        }
      };
      fetch(0, s[0]);
#pragma unroll 1
      for (int kb0 = 0; kb0 < p.k_blocks; kb0 += kGroup) {
        await_products();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int kb = kb0 + 2 * u;
          if (kb < p.k_blocks) {
            uint32_t v[2][2][16];
#pragma unroll
            for (int d = 0; d < 2; ++d)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                ptx::tmem_ld_16x128b_x8(from + ((uint32_t)(h * 16) << 16) + (bufs & 1u) * kBufCols + (2 * u + d) * 64, v[d][h]);
            ptx::tmem_ld_wait();
            if (u == 1 || kb + 2 >= p.k_blocks) {
              arrive_done();
              ++bufs;
            }
            if (kb + 2 < p.k_blocks) fetch(kb + 2, s[u ^ 1]);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              if (kb + d < p.k_blocks) {  // (the place of a block that is not there is read as it is)
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                  for (int h = 0; h < 2; ++h)
                    fma2(acc[h][i], v[d][h][2 * i], v[d][h][2 * i + 1], make_float2(s[u][d][i], s[u][d][i]));
              }
            }
          }
        }
      }
      free_scales();
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      const int token0 = side * kChunk;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {  // eight tokens (a lane's are four apart), 32 columns
        const auto two = [&](int h, bool upper) {
          return pack2(upper ? make_float2(acc[h][i].y, acc[h][i + 1].y) : make_float2(acc[h][i].x, acc[h][i + 1].x));
        };
        const int token = 4 * i + ((lane & 1) << 2) + (lane >> 1 & 3);
        ptx::stmatrix_x4_trans(piece_at(token, lane >> 3), two(0, false), two(0, true), two(1, false), two(1, true));
      }
      send(t.row0 + token0, t.rows - token0, n0);
    }
    if (p.zero_rest) {  // rows of no expert, in front of the first one's and behind the last one's, a row to a warp
      const int front = tables.start[0], behind = tables.start[p.experts - 1] + tables.count[p.experts - 1];
      for (int i = (int)blockIdx.x * kEpiWarps + ew; i < front + p.M - behind; i += (int)gridDim.x * kEpiWarps) {
        __nv_bfloat16* c = p.c + (long long)(i < front ? i : behind + i - front) * p.N;
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
  return std::min(bt == 64 ? kMaxStages : kWideStages, (kMaxDynamicSmem - 1024 - tail_bytes(bt, experts)) / stage_bytes(bt));
}

template <bool WIDE>
cudaError_t launch(const GroupedParams& p, int pairs, int smem, const CUtensorMap& map_b, const CUtensorMap& map_big,
                   const CUtensorMap& map_small, cudaStream_t stream) {
  static OncePerDevice once;
  const cudaError_t opted = once([] { return opt_in(fp8_grouped_kernel<WIDE>, kMaxDynamicSmem, false); });
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
  return cudaLaunchKernelEx(&cfg, fp8_grouped_kernel<WIDE>, map_b, map_big, map_small, p);
}

}  // namespace

// By the mean, since the counts are on the device.  Tiles of 64 tokens and wide ones, us, 64 experts of 4096 x 4096 / 32 of
// 2048 x 7168:
//   mean rows      48                    56                    64                    72                    100
//   even routing   172, 185 / 81, 89     173, 188 / 88, 89     193, 189 / 85, 91     216, 190 / 99, 91     234, 192 / 102, 92
//   skewed         202, 203 / 90, 88     214, 210 / 99, 94     221, 216 / 97, 96     228, 222 / 107, 97    259, 241 / 116, 105
// At 20 rows, even routing: 164, 180 / 78, 86.
int fp8_grouped_tile(int M, int experts) {
  const int mean = M / std::max(experts, 1);
  return mean <= 64 ? 64 : 256;
}

int fp8_grouped_smem(int tile, int experts) {
  return 1024 + stages_of(tile, experts) * stage_bytes(tile) + tail_bytes(tile, experts);
}

int fp8_grouped_local_bytes(int tile) {
  cudaFuncAttributes a = {};
  const cudaError_t e = tile == 64 ? cudaFuncGetAttributes(&a, fp8_grouped_kernel<false>) : cudaFuncGetAttributes(&a, fp8_grouped_kernel<true>);
  return e == cudaSuccess ? (int)a.localSizeBytes : -1;
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
  return bt == 64 ? launch<false>(p, pairs, smem, map_b, map_big, map_small, stream)
                  : launch<true>(p, pairs, smem, map_b, map_big, map_small, stream);
}

}  // namespace b200
