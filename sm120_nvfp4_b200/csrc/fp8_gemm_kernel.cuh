// FP8 (E4M3) matrix products with one FP32 scale per 128 values of K, for sm_100a.
//
//   Y[r, c] = sum_b SA[r, b] * SB[c / 128, b] * sum_{k in block b} A[r, k] * B[c, k]
//
// A [rows, K] and B [N, K] hold E4M3 codes, K contiguous; a block b is 128 values of K (the last one
// may be shorter). SA has one scale per row and block, SB one per 128 x 128 tile of B: the format of
// FP8 checkpoints and of activations quantised on the fly. Rows come in groups with a B of their own
// (experts), or as one group.
//
// The scales are FP32 numbers, so they cannot go through the tensor core's power-of-two block
// scales: the 128 products of a block are summed by tcgen05.mma (kind::f8f6f4, FP32 in tensor
// memory, four instructions of K = 32), and every block's sums are read back, multiplied by their
// two scales and added to FP32 accumulators in registers ("promotion"). Tensor memory holds several
// of these block sums, so the promotion of one block runs under the MMAs of the next.
//
// Two kernels:
//   fp8_skinny_kernel<BN>  few rows. The weights take the 128-row side of the MMA and BN = 16 .. 128
//                          rows of A the other, so that a row of activations costs a column, not 1/128
//                          of a tile, and what is streamed - the weights - fills whole tiles. K can be
//                          split over a cluster whose CTAs add their partial tiles through distributed
//                          shared memory, in split order.
//   fp8_pair_kernel        many rows: 256 x 256 tiles on CTA pairs (cta_group::2).
// All waits are bounded (ptx::mbar_wait) and reported through the device error word.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gemm_kernel.cuh"

namespace b200 {

constexpr int kFp8BlockK = 128;               // values of K per scale = bytes of K per stage row
constexpr int kFp8Panel = 8;                  // blocks of K whose scales arrive together ...
constexpr int kFp8Panels = 2;                 // ... and panels in shared memory

enum Fp8Out { kOutF16 = 0, kOutF32 = 1, kOutBf16 = 2 };

struct Fp8Params {
  int num_groups;
  int total_rows;             // rows of A and of the output
  int n, k;
  const int* seqlens;         // [G] valid rows per group (device), or nullptr: one group of total_rows
  const int* cu_seqlens;      // [G+1] first row of each group (device)
  const float* a_scale;       // [total_rows, kb]
  const float* b_scale;       // [G, ceil(N/128), kb]
  void* out;                  // [total_rows, n]
  int out_type;               // Fp8Out
  int raster_m;
  int num_stages;
  int scales_by_16;           // scale rows start on 16-byte boundaries: whole panels by 16-byte copies
  int splits;                 // skinny kernel: CTAs of a cluster over K
  int tma_store;
  int* error;
  long long wait_limit;
  int withhold_first_arrival;
};

// Valid rows, first row and tile prefix of every group into shared memory. Row ranges that would
// leave the matrices are cut off. Ends with a __syncthreads().
__device__ __forceinline__ void fp8_group_tables(const Fp8Params& p, int tile_rows, int* s_cu_tiles, int* s_row0,
                                                 int* s_rows) {
  const int G = p.num_groups;
  for (int g = threadIdx.x; g < G; g += blockDim.x) {
    int row0 = p.cu_seqlens ? p.cu_seqlens[g] : 0;
    int rows = p.seqlens ? p.seqlens[g] : p.total_rows;
    if (row0 < 0 || row0 > p.total_rows) { row0 = 0; rows = 0; }
    rows = max(0, min(rows, p.total_rows - row0));
    s_rows[g] = rows;
    s_row0[g] = row0;
    s_cu_tiles[g] = (rows + tile_rows - 1) / tile_rows;
  }
  __syncthreads();
  if (threadIdx.x < 32) {   // exclusive scan, 32 groups at a time
    const int lane = threadIdx.x;
    int carry = 0;
    for (int base = 0; base < G; base += 32) {
      const int v = base + lane < G ? s_cu_tiles[base + lane] : 0;
      int incl = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      if (base + lane < G) s_cu_tiles[base + lane] = carry + incl - v;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_cu_tiles[G] = carry;
  }
  __syncthreads();
}

// Starts the copies of one panel of scales into shared memory, [block][stride] floats: the scales of
// `count` blocks of K from b0 on for ROWS rows, of which the first `valid` exist (the others become
// zeros), and behind them those of TILES column tiles of B. Rows are kb floats apart in memory and of
// any alignment, so the copies are 4 bytes each; eight neighbouring lanes take a row's eight blocks, which
// is one sector (with a row per lane every copy was a sector of its own, and the eight blocks of a panel
// fetched each of them again: the loader could not keep up with the MMAs).
template <int ROWS, int TILES>
__device__ __forceinline__ void fp8_load_scales(uint32_t dst, int stride, const float* a_scale, long long row, int valid, int kb,
                                                int b0, int count, const float* b_scale, int tiles_left, int lane) {
  const int j = lane & 7;
  const bool block_in = j < count;
  const float* src = a_scale + (row + (lane >> 3)) * kb + b0 + j;
  const uint32_t to = dst + static_cast<uint32_t>(j * stride + (lane >> 3)) * 4;
#pragma unroll 8
  for (int r = 0; r < ROWS; r += 4) {
    const bool in = r + (lane >> 3) < valid;
    if (block_in) ptx::cp_async_4(to + 4 * r, in ? src + static_cast<long long>(r) * kb : a_scale, in);
  }
  const int tile = lane >> 3;
  if (tile < TILES && block_in) {
    const bool in = tile < tiles_left;
    ptx::cp_async_4(dst + static_cast<uint32_t>(j * stride + ROWS + tile) * 4, in ? b_scale + static_cast<long long>(tile) * kb + b0 + j : b_scale, in);
  }
}

// One output value, rounded once from FP32.
__device__ __forceinline__ void fp8_store(void* out, int type, long long at, float v) {
  if (type == kOutF16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else if (type == kOutBf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(out)[at] = v;
}

__device__ __forceinline__ uint32_t fp8_pack2(int type, float lo, float hi) {
  if (type == kOutF16) return pack_half2(lo, hi);
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&b);
}

// --------------------------------------------------------------------- few rows

template <int BN>
struct Fp8SkinnyCfg {
  static_assert(BN == 16 || BN == 32 || BN == 64 || BN == 128, "tile of 16 to 128 rows of A");
  static constexpr int kThreads = 256;        // loaders of B, A and the scales, MMA issuer, four promotion warps
  static constexpr int kBuffers = 4;          // block sums in tensor memory
  static constexpr int kTmemCols = kBuffers * BN < 32 ? 32 : kBuffers * BN;
  static constexpr int kWBytes = 128 * kFp8BlockK;
  static constexpr int kXBytes = BN * kFp8BlockK;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kMaxStages = 12;
  static constexpr int kSlotFloats = BN + 4;  // row scales of one block, then the scale of the weights' tile (multiple of 4)
  static constexpr int kRedBytes = 128 * BN * 4;
  static constexpr int fixed_bytes(int groups, int splits) {
    return 1024 + 512 + kFp8Panels * kFp8Panel * kSlotFloats * 4 + 3 * (groups + 1) * 4 + (splits > 1 ? kRedBytes : 0);
  }
  static constexpr int stages_for(int groups, int splits) {
    const int s = (kSmemBudget - fixed_bytes(groups, splits)) / kStageBytes;
    return s > kMaxStages ? kMaxStages : s;
  }
  static constexpr int smem_bytes(int groups, int splits) {
    return fixed_bytes(groups, splits) + stages_for(groups, splits) * kStageBytes;
  }
  static_assert(stages_for(kMaxGroups, 2) >= 4, "pipeline too shallow");
};

template <int BN>
__global__ void __launch_bounds__(256, 1)
fp8_skinny_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                  const Fp8Params p) {
  using Cfg = Fp8SkinnyCfg<BN>;
  constexpr int kLoadW = 0, kMma = 1, kLoadX = 2, kLoadS = 3, kFirstPromoter = 4;
  const int kStages = p.num_stages;
  const int splits = p.splits;
  const int kb = (p.k + kFp8BlockK - 1) / kFp8BlockK;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* red = smem + kStages * Cfg::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(red + (splits > 1 ? Cfg::kRedBytes : 0));
  const uint32_t full_u32 = ptx::smem_u32(bars);                       // operands of a stage have landed
  const uint32_t empty_u32 = full_u32 + 8 * Cfg::kMaxStages;           // ... have been read by the MMAs
  const uint32_t sum_full_u32 = empty_u32 + 8 * Cfg::kMaxStages;       // a block's sums are in tensor memory
  const uint32_t sum_empty_u32 = sum_full_u32 + 8 * Cfg::kBuffers;     // ... have been read
  const uint32_t sc_full_u32 = sum_empty_u32 + 8 * Cfg::kBuffers;      // a block's scales are in their slot
  const uint32_t sc_empty_u32 = sc_full_u32 + 8 * kFp8Panels;
  const uint32_t red_full_u32 = sc_empty_u32 + 8 * kFp8Panels;     // every CTA's part of this CTA's columns
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * Cfg::kMaxStages + 2 * Cfg::kBuffers + 2 * kFp8Panels + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);
  float* slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);
  int* s_cu_tiles = reinterpret_cast<int*>(slots + kFp8Panels * kFp8Panel * Cfg::kSlotFloats);
  int* s_row0 = s_cu_tiles + (p.num_groups + 1);
  int* s_rows = s_row0 + (p.num_groups + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = splits > 1 ? static_cast<int>(ptx::cluster_cta_rank()) : 0;

  if (warp == 0) {
    if (lane == 0) {
      *abort_flag = 0;
      ptx::prefetch_tensormap(&tmap_w);
    }
    for (int s = lane; s < kStages; s += 32) {
      ptx::mbar_init(full_u32 + 8 * s, 2);
      ptx::mbar_init(empty_u32 + 8 * s, 1);
    }
    if (lane < Cfg::kBuffers) {
      ptx::mbar_init(sum_full_u32 + 8 * lane, 1);
      ptx::mbar_init(sum_empty_u32 + 8 * lane, 4);
    }
    if (lane < kFp8Panels) {
      ptx::mbar_init(sc_full_u32 + 8 * lane, 32);
      ptx::mbar_init(sc_empty_u32 + 8 * lane, 4);
    }
    if (lane == 31) ptx::mbar_init(red_full_u32, 1);
    __syncwarp();
    if (lane == 0) ptx::fence_barrier_init();
  } else if (warp == kMma) {
    ptx::tmem_alloc<1>(ptx::smem_u32(tmem_holder), Cfg::kTmemCols);
    ptx::tmem_relinquish<1>();
  } else if (warp == kLoadX && lane == 0) {
    ptx::prefetch_tensormap(&tmap_x);
  }
  ptx::tc_fence_before_sync();
  fp8_group_tables(p, BN, s_cu_tiles, s_row0, s_rows);
  if (splits > 1) ptx::cluster_arrive_relaxed();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;

  const int n_tiles = (p.n + 127) / 128;
  const int total_mt = s_cu_tiles[p.num_groups];
  const int total_tasks = total_mt * n_tiles;
  // a cluster takes one task, a CTA of an unsplit launch as many as come its way
  const int first_task = static_cast<int>(blockIdx.x) / splits;
  const int task_step = splits > 1 ? total_tasks : static_cast<int>(gridDim.x);
  const int b_begin = kb * rank / splits, b_end = kb * (rank + 1) / splits;
  const uint32_t stage_u32 = ptx::smem_u32(smem);
  bool met = false;             // this warp has waited for the cluster's set-up

  if (warp == kLoadW || warp == kLoadX) {
    const bool weights = warp == kLoadW;
    const uint32_t bytes = weights ? Cfg::kWBytes : Cfg::kXBytes;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, withhold = weights && p.withhold_first_arrival != 0 && blockIdx.x == 0;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int row = weights ? t.g * p.n + t.nt * 128 : s_row0[t.g] + t.mt * BN;
      for (int b = b_begin; b < b_end; ++b) {
        if (!ptx::mbar_wait(empty_u32 + 8 * stage, phase ^ 1, abort_flag, kWaitEmpty, p.wait_limit)) { ok = false; break; }
        if (ptx::elect_one()) {
          const uint32_t bar = full_u32 + 8 * stage;
          if (withhold) withhold = false;
          else ptx::mbar_arrive_expect_tx(bar, bytes);
          ptx::tma_load_2d(stage_u32 + stage * Cfg::kStageBytes + (weights ? 0 : Cfg::kWBytes), weights ? &tmap_w : &tmap_x,
                           bar, b * kFp8BlockK, row);
        }
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == kLoadS) {
    int panel = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int row = s_row0[t.g] + t.mt * BN;
      const int valid = min(BN, s_rows[t.g] - t.mt * BN);
      const float* sb = p.b_scale + (static_cast<long long>(t.g) * n_tiles + t.nt) * kb;
      for (int b0 = b_begin; b0 < b_end; b0 += kFp8Panel) {
        if (!ptx::mbar_wait(sc_empty_u32 + 8 * panel, phase ^ 1, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
        fp8_load_scales<BN, 1>(ptx::smem_u32(slots + panel * kFp8Panel * Cfg::kSlotFloats), Cfg::kSlotFloats, p.a_scale, row, valid,
                               kb, b0, b_end - b0, sb, 1, lane);
        ptx::cp_async_mbar_arrive(sc_full_u32 + 8 * panel);
        if (++panel == kFp8Panels) { panel = 0; phase ^= 1; }
      }
    }
    ptx::cp_async_wait_all();
    __syncwarp();
  } else if (warp == kMma) {
    constexpr uint32_t idesc = ptx::make_idesc_e4m3(128, BN);
    const uint32_t lo0 = ptx::kmajor_sw128_desc_lo(stage_u32);
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      for (int b = b_begin; b < b_end; ++b) {
        if (!ptx::mbar_wait(sum_empty_u32 + 8 * buf, buf_phase ^ 1, abort_flag, kWaitAccEmpty, p.wait_limit) ||
            !ptx::mbar_wait(full_u32 + 8 * stage, phase, abort_flag, kWaitFull, p.wait_limit)) { ok = false; break; }
        ptx::tc_fence_after_sync();
        if (ptx::elect_one()) {
          const uint32_t w_lo = lo0 + stage * (Cfg::kStageBytes >> 4);
          const uint32_t x_lo = w_lo + (Cfg::kWBytes >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j)      // 32 values of K = 32 bytes = 2 units of the address field
            ptx::tc_mma_e4m3<1>(tmem_base + buf * BN, w_lo + 2 * j, x_lo + 2 * j, ptx::kKmajorSw128DescHi, idesc, j > 0 ? 1u : 0u);
          ptx::tc_commit<1>(empty_u32 + 8 * stage);
          ptx::tc_commit<1>(sum_full_u32 + 8 * buf);
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1; }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ promotion: lane = row of B (output column), register = row of A
    const int q = warp & 3;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    constexpr int kChunk = BN < 32 ? BN : 32;
    int buf = 0, panel = 0;
    uint32_t buf_phase = 0, panel_phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int valid = min(BN, s_rows[t.g] - t.mt * BN);
      float acc[BN];
#pragma unroll
      for (int c = 0; c < BN; ++c) acc[c] = 0.0f;
      for (int b = b_begin; b < b_end; ++b) {
        const int in_panel = (b - b_begin) & (kFp8Panel - 1);
        if ((in_panel == 0 && !ptx::mbar_wait(sc_full_u32 + 8 * panel, panel_phase, abort_flag, kWaitSlots, p.wait_limit)) ||
            !ptx::mbar_wait(sum_full_u32 + 8 * buf, buf_phase, abort_flag, kWaitAccFull, p.wait_limit)) { ok = false; break; }
        ptx::tc_fence_after_sync();
        const float* sc = slots + (panel * kFp8Panel + in_panel) * Cfg::kSlotFloats;
        const float sb = sc[BN];
#pragma unroll
        for (int c0 = 0; c0 < BN; c0 += kChunk) {
          uint32_t v[kChunk];
          ptx::tmem_ld_cols<kChunk>(lane_addr + buf * BN + c0, v);
          ptx::tmem_ld_wait_regs<kChunk>(v);
#pragma unroll
          for (int c = 0; c < kChunk; c += 4) {
            const float4 sa = *reinterpret_cast<const float4*>(sc + c0 + c);
            acc[c0 + c] = fmaf(__uint_as_float(v[c]), sa.x * sb, acc[c0 + c]);
            acc[c0 + c + 1] = fmaf(__uint_as_float(v[c + 1]), sa.y * sb, acc[c0 + c + 1]);
            acc[c0 + c + 2] = fmaf(__uint_as_float(v[c + 2]), sa.z * sb, acc[c0 + c + 2]);
            acc[c0 + c + 3] = fmaf(__uint_as_float(v[c + 3]), sa.w * sb, acc[c0 + c + 3]);
          }
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        const bool panel_done = in_panel == kFp8Panel - 1 || b + 1 == b_end;
        if (lane == 0) {
          ptx::mbar_arrive(sum_empty_u32 + 8 * buf);
          if (panel_done) ptx::mbar_arrive(sc_empty_u32 + 8 * panel);
        }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
        if (panel_done && ++panel == kFp8Panels) { panel = 0; panel_phase ^= 1; }
      }
      if (!ok) break;
      const int tile_row = q * 32 + lane;
      const int col = t.nt * 128 + tile_row;                      // output column
      const long long out0 = (static_cast<long long>(s_row0[t.g]) + t.mt * BN) * p.n + col;
      if (splits == 1) {
        if (col < p.n) {
#pragma unroll
          for (int c = 0; c < BN; ++c)
            if (c < valid) fp8_store(p.out, p.out_type, out0 + static_cast<long long>(c) * p.n, acc[c]);
        }
      } else {
        // CTA d of the cluster finishes rows [d w, (d + 1) w) of the tile: everybody stores its part
        // into slot `rank` of that CTA's buffer, [slot][row][128 columns], counted in bytes there.
        const int w = (valid + splits - 1) / splits;
        const int mine = max(0, min(w, valid - rank * w));
        if (warp == kFirstPromoter && lane == 0 && mine > 0)
          ptx::mbar_arrive_expect_tx(red_full_u32, static_cast<uint32_t>(splits * mine * 128 * 4));
        ptx::cluster_wait();                                       // every CTA has its barriers
        met = true;
        const uint32_t red_u32 = ptx::smem_u32(red);
        int d = 0, at = 0;
        uint32_t base = ptx::map_to_cta(red_u32, 0), bar = ptx::map_to_cta(red_full_u32, 0);
        int rows_d = min(w, valid);
#pragma unroll
        for (int c = 0; c < BN; ++c) {
          if (c < valid) {
            if (at == w) {
              ++d;
              at = 0;
              base = ptx::map_to_cta(red_u32, d);
              bar = ptx::map_to_cta(red_full_u32, d);
              rows_d = min(w, valid - d * w);
            }
            ptx::st_async_b32(base + static_cast<uint32_t>(((rank * rows_d + at) * 128 + tile_row) * 4), __float_as_uint(acc[c]), bar);
            ++at;
          }
        }
        if (mine > 0) {
          if (!ptx::mbar_wait_cluster(red_full_u32, 0, abort_flag, kWaitPartials, p.wait_limit)) break;
          const float* part = reinterpret_cast<const float*>(red);
          for (int i = 0; i < mine; ++i) {
            float sum = part[i * 128 + tile_row];
            for (int s = 1; s < splits; ++s) sum = __fadd_rn(sum, part[(s * mine + i) * 128 + tile_row]);
            if (col < p.n) fp8_store(p.out, p.out_type, out0 + static_cast<long long>(rank * w + i) * p.n, sum);
          }
        }
      }
    }
    __syncwarp();
  }

  // ---- teardown
  if (splits > 1 && !met) ptx::cluster_wait();     // every thread waits once for the arrival at set-up
  __syncthreads();
  const int aborted = *abort_flag;
  if (splits > 1) ptx::cluster_sync();
  if (aborted != 0) {
    const long long start = clock64();
    while (clock64() - start < (1ll << 22)) {
    }
    if (threadIdx.x == 0 && p.error) atomicCAS(p.error, 0, aborted | (static_cast<int>(blockIdx.x) << 8));
  }
  if (warp == kMma) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<1>(tmem_base, Cfg::kTmemCols);
  }
}

// -------------------------------------------------------------------- many rows

// 256 x 256 tiles on CTA pairs: each CTA loads 128 rows of A and its half of the 256 rows of B, the
// MMAs read both halves, and each CTA's tensor memory receives 128 rows x 256 columns of a block's
// sums. Two such buffers fill the 512 columns of tensor memory. 128 accumulators per thread in eight
// promotion warps need more registers than an even share (65536 / 384 = 168): the other four warps
// give theirs up (72 + 2 x 216 = 504 = 3 x 168).
struct Fp8PairCfg {
  static constexpr int kThreads = 384;
  static constexpr int kBuffers = 2;
  static constexpr int kABytes = 128 * kFp8BlockK;
  static constexpr int kBBytes = 128 * kFp8BlockK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kMaxStages = 6;
  // Scales arrive in panels of four blocks of K, [row][block]: a promotion thread takes its row's four
  // with one 16-byte read. Two more rows hold those of the tile's two 128-column tiles of B.
  static constexpr int kPanel = 4;
  static constexpr int kPanels = 4;
  static constexpr int kPanelFloats = (128 + 2) * kPanel;
  static constexpr int kStagingBytes = 8 * 32 * 128;
  static constexpr int fixed_bytes(int groups) {
    return 1024 + 512 + kPanels * kPanelFloats * 4 + 3 * (groups + 1) * 4 + kStagingBytes;
  }
  static constexpr int stages_for(int groups) {
    const int s = (kSmemBudget - fixed_bytes(groups)) / kStageBytes;
    return s > kMaxStages ? kMaxStages : s;
  }
  static constexpr int smem_bytes(int groups) { return fixed_bytes(groups) + stages_for(groups) * kStageBytes; }
};
static_assert(Fp8PairCfg::stages_for(kMaxGroups) >= 4, "pipeline too shallow");

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(384, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_out, const Fp8Params p) {
  using Cfg = Fp8PairCfg;
  constexpr int kLoadA = 0, kMma = 1, kLoadB = 2, kLoadS = 3, kFirstPromoter = 4;
  const int kStages = p.num_stages;
  const int kb = (p.k + kFp8BlockK - 1) / kFp8BlockK;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* staging = smem + kStages * Cfg::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + Cfg::kStagingBytes);
  // `full`, and `sum_empty` of the first CTA serve the pair; `empty`, `sum_full` exist in both CTAs
  const uint32_t full_u32 = ptx::smem_u32(bars);
  const uint32_t empty_u32 = full_u32 + 8 * Cfg::kMaxStages;
  const uint32_t sum_full_u32 = empty_u32 + 8 * Cfg::kMaxStages;
  const uint32_t sum_empty_u32 = sum_full_u32 + 8 * Cfg::kBuffers;
  const uint32_t sc_full_u32 = sum_empty_u32 + 8 * Cfg::kBuffers;
  const uint32_t sc_empty_u32 = sc_full_u32 + 8 * Cfg::kPanels;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * Cfg::kMaxStages + 2 * Cfg::kBuffers + 2 * Cfg::kPanels);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);
  float* slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);
  int* s_cu_tiles = reinterpret_cast<int*>(slots + Cfg::kPanels * Cfg::kPanelFloats);
  int* s_row0 = s_cu_tiles + (p.num_groups + 1);
  int* s_rows = s_row0 + (p.num_groups + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int cta = static_cast<int>(ptx::cluster_cta_rank());
  const bool leader = cta == 0;

  if (warp == 0) {
    if (lane == 0) {
      *abort_flag = 0;
      ptx::prefetch_tensormap(&tmap_a);
    }
    for (int s = lane; s < kStages; s += 32) {
      ptx::mbar_init(full_u32 + 8 * s, 2);
      ptx::mbar_init(empty_u32 + 8 * s, 1);
    }
    if (lane < Cfg::kBuffers) {
      ptx::mbar_init(sum_full_u32 + 8 * lane, 1);
      ptx::mbar_init(sum_empty_u32 + 8 * lane, 16);    // eight promotion warps of each CTA
    }
    if (lane < Cfg::kPanels) {
      ptx::mbar_init(sc_full_u32 + 8 * lane, 32);
      ptx::mbar_init(sc_empty_u32 + 8 * lane, 8);
    }
    __syncwarp();
    if (lane == 0) ptx::fence_barrier_init();
  } else if (warp == kMma) {
    ptx::tmem_alloc<2>(ptx::smem_u32(tmem_holder), 512);
    ptx::tmem_relinquish<2>();
  } else if (warp == kLoadB && lane == 0) {
    ptx::prefetch_tensormap(&tmap_b);
  } else if (warp == kFirstPromoter && lane == 0 && p.tma_store) {
    ptx::prefetch_tensormap(&tmap_out);
  }
  ptx::tc_fence_before_sync();
  fp8_group_tables(p, 256, s_cu_tiles, s_row0, s_rows);
  ptx::cluster_arrive_relaxed();
  ptx::cluster_wait();                        // the partner's barriers exist
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;

  const int n_tiles = (p.n + 255) / 256;
  const int total_mt = s_cu_tiles[p.num_groups];
  const int total_tasks = total_mt * n_tiles;
  const int first_task = static_cast<int>(blockIdx.x) >> 1, task_step = static_cast<int>(gridDim.x) >> 1;
  const uint32_t stage_u32 = ptx::smem_u32(smem);

  // (each share is set where its code begins: after a join the compiler would hold both to the smaller)
  if (warp < kFirstPromoter) {
  ptx::setmaxnreg_dec<72>();
  if (warp == kLoadA || warp == kLoadB) {
    const bool is_a = warp == kLoadA;
    const CUtensorMap* tmap = is_a ? &tmap_a : &tmap_b;
    const uint32_t full_target = ptx::map_to_cta(full_u32, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, withhold = is_a && p.withhold_first_arrival != 0 && blockIdx.x == 0;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int row = is_a ? s_row0[t.g] + t.mt * 256 + cta * 128 : t.g * p.n + t.nt * 256 + cta * 128;
      for (int b = 0; b < kb; ++b) {
        if (!ptx::mbar_wait(empty_u32 + 8 * stage, phase ^ 1, abort_flag, kWaitEmpty, p.wait_limit)) { ok = false; break; }
        if (ptx::elect_one()) {
          if (withhold) withhold = false;
          else if (leader) ptx::mbar_arrive_expect_tx(full_u32 + 8 * stage, 2 * Cfg::kABytes);   // both CTAs' halves
          ptx::tma_load_2d_pair(stage_u32 + stage * Cfg::kStageBytes + (is_a ? 0 : Cfg::kABytes), tmap,
                                full_target + 8 * stage, b * kFp8BlockK, row);
        }
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == kLoadS) {
    int panel = 0;
    uint32_t phase = 0;
    bool ok = true;
    const int nb = (p.n + 127) / 128;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int row = s_row0[t.g] + t.mt * 256 + cta * 128;
      const int valid = min(128, s_rows[t.g] - t.mt * 256 - cta * 128);     // may be <= 0 in the second CTA
      const float* sb = p.b_scale + (static_cast<long long>(t.g) * nb + 2 * t.nt) * kb;
      for (int b0 = 0; b0 < kb; b0 += Cfg::kPanel) {
        if (!ptx::mbar_wait(sc_empty_u32 + 8 * panel, phase ^ 1, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
        const uint32_t dst = ptx::smem_u32(slots + panel * Cfg::kPanelFloats);
        if (p.scales_by_16) {
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 32) {
            const int c = c0 + lane;
            const bool in = c < valid;
            ptx::cp_async_16(dst + 16 * c, in ? p.a_scale + static_cast<long long>(row + c) * kb + b0 : p.a_scale, in);
          }
          const bool in = 2 * t.nt + lane < nb;
          if (lane < 2) ptx::cp_async_16(dst + 16 * (128 + lane), in ? sb + static_cast<long long>(lane) * kb + b0 : p.b_scale, in);
        } else {
          const int j = lane & 3, r0 = lane >> 2;
          const bool block_in = b0 + j < kb;
#pragma unroll 4
          for (int r = r0; r < 128; r += 8) {
            const bool in = block_in && r < valid;
            ptx::cp_async_4(dst + 4 * (4 * r + j), in ? p.a_scale + static_cast<long long>(row + r) * kb + b0 + j : p.a_scale, in);
          }
          const bool in = block_in && 2 * t.nt + r0 < nb;
          if (r0 < 2) ptx::cp_async_4(dst + 4 * (4 * (128 + r0) + j), in ? sb + static_cast<long long>(r0) * kb + b0 + j : p.b_scale, in);
        }
        ptx::cp_async_mbar_arrive(sc_full_u32 + 8 * panel);
        if (++panel == Cfg::kPanels) { panel = 0; phase ^= 1; }
      }
    }
    ptx::cp_async_wait_all();
    __syncwarp();
  } else if (warp == kMma) {
    if (leader) {
      constexpr uint32_t idesc = ptx::make_idesc_e4m3(256, 256);
      const uint32_t lo0 = ptx::kmajor_sw128_desc_lo(stage_u32);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      for (int task = first_task; task < total_tasks && ok; task += task_step) {
        for (int b = 0; b < kb; ++b) {
          if (!ptx::mbar_wait(full_u32 + 8 * stage, phase, abort_flag, kWaitFull, p.wait_limit) ||
              !ptx::mbar_wait(sum_empty_u32 + 8 * buf, buf_phase ^ 1, abort_flag, kWaitAccEmpty, p.wait_limit)) { ok = false; break; }
          ptx::tc_fence_after_sync();
          if (ptx::elect_one()) {
            const uint32_t a_lo = lo0 + stage * (Cfg::kStageBytes >> 4);
            const uint32_t b_lo = a_lo + (Cfg::kABytes >> 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              ptx::tc_mma_e4m3<2>(tmem_base + buf * 256, a_lo + 2 * j, b_lo + 2 * j, ptx::kKmajorSw128DescHi, idesc, j > 0 ? 1u : 0u);
            ptx::tc_commit<2>(empty_u32 + 8 * stage, 3);
            ptx::tc_commit<2>(sum_full_u32 + 8 * buf, 3);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1; }
          if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
        }
      }
    }
    __syncwarp();
  }
  } else {
    ptx::setmaxnreg_inc<216>();
    // ------------------ promotion: lane = row of the tile, registers = 128 columns (one scale tile of B)
    const int q = warp & 3;
    const int half = (warp - kFirstPromoter) >> 2;
    const uint32_t addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + half * 128;
    const uint32_t stg = ptx::smem_u32(staging) + (warp - kFirstPromoter) * 4096;
    const uint32_t stg_row = stg + lane * 128;
    const uint32_t sum_empty_target = ptx::map_to_cta(sum_empty_u32, 0);
    int buf = 0, panel = 0;
    uint32_t buf_phase = 0, panel_phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      uint64_t acc[64];                      // column pairs, as the packed FMA takes them
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = 0;
      float4 s4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int b = 0; b < kb; ++b) {
        if ((b & (Cfg::kPanel - 1)) == 0) {
          if (!ptx::mbar_wait(sc_full_u32 + 8 * panel, panel_phase, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
          const float4* sc = reinterpret_cast<const float4*>(slots + panel * Cfg::kPanelFloats);
          const float4 sa = sc[q * 32 + lane], sb = sc[128 + half];
          s4 = make_float4(sa.x * sb.x, sa.y * sb.y, sa.z * sb.z, sa.w * sb.w);
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sc_empty_u32 + 8 * panel);
          if (++panel == Cfg::kPanels) { panel = 0; panel_phase ^= 1; }
        }
        const uint64_t s = ptx::pack_f32x2(__float_as_uint(s4.x), __float_as_uint(s4.x));
        s4 = make_float4(s4.y, s4.z, s4.w, s4.x);
        if (!ptx::mbar_wait(sum_full_u32 + 8 * buf, buf_phase, abort_flag, kWaitAccFull, p.wait_limit)) { ok = false; break; }
        ptx::tc_fence_after_sync();
        const uint32_t from = addr + buf * 256;
#pragma unroll
        for (int c0 = 0; c0 < 8; ++c0) {       // 16 columns at a time
          uint32_t v[16];
          ptx::tmem_ld_cols<16>(from + c0 * 16, v);
          ptx::tmem_ld_wait_regs<16>(v);
          if (c0 == 7) {                       // everything has left tensor memory
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if (leader) ptx::mbar_arrive(sum_empty_u32 + 8 * buf);
              else ptx::mbar_arrive_cluster(sum_empty_target + 8 * buf);
            }
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) ptx::fma_f32x2(acc[c0 * 8 + c], ptx::pack_f32x2(v[2 * c], v[2 * c + 1]), s);
        }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
      }
      auto value = [&](int c) { return __uint_as_float(static_cast<uint32_t>(c & 1 ? acc[c >> 1] >> 32 : acc[c >> 1])); };
      if (!ok) break;
      // ---- output: a slab of 32 valid rows leaves through the staging buffer and the store engine,
      // a ragged one by predicated stores
      const int row_in_group = t.mt * 256 + cta * 128 + q * 32;
      const int rows_left = s_rows[t.g] - row_in_group;
      const int map_row = s_row0[t.g] + row_in_group;
      const int col0 = t.nt * 256 + half * 128;
      if (rows_left <= 0 || col0 >= p.n) continue;
      const int elem = p.out_type == kOutF32 ? 4 : 2;
      if (p.tma_store && rows_left >= 32) {
#pragma unroll
        for (int c0 = 0; c0 < 4; ++c0) {                 // 32 columns at a time
          const int col = col0 + c0 * 32;
          if (elem == 4 || (c0 & 1) == 0) {
            if (lane == 0) ptx::bulk_wait_group_read<0>();
            __syncwarp();
          }
          if (elem == 4) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
              ptx::st_shared_v4(stg_row + (static_cast<uint32_t>(u ^ (lane & 7)) << 4), __float_as_uint(value(c0 * 32 + 4 * u)),
                                __float_as_uint(value(c0 * 32 + 4 * u + 1)), __float_as_uint(value(c0 * 32 + 4 * u + 2)),
                                __float_as_uint(value(c0 * 32 + 4 * u + 3)));
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = fp8_pack2(p.out_type, value(c0 * 32 + 8 * u + 2 * i), value(c0 * 32 + 8 * u + 2 * i + 1));
              ptx::st_shared_v4(stg_row + (static_cast<uint32_t>(((c0 & 1) * 4 + u) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
          }
          if (elem == 4 || (c0 & 1) == 1) {
            ptx::fence_proxy_async_smem();
            __syncwarp();
            const int box_col = elem == 4 ? col : col - 32;
            if (lane == 0 && box_col < p.n) {
              ptx::tma_store_2d(&tmap_out, stg, box_col, map_row);
              ptx::bulk_commit_group();
            }
          }
        }
      } else if (lane < rows_left) {
        const long long at = static_cast<long long>(map_row + lane) * p.n;
#pragma unroll
        for (int c = 0; c < 128; c += 8) {               // n is a multiple of 8
          const int col = col0 + c;
          if (col < p.n) {
            if (elem == 4) {
              float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + col);
              dst[0] = make_float4(value(c), value(c + 1), value(c + 2), value(c + 3));
              dst[1] = make_float4(value(c + 4), value(c + 5), value(c + 6), value(c + 7));
            } else {
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at + col) =
                  make_uint4(fp8_pack2(p.out_type, value(c), value(c + 1)), fp8_pack2(p.out_type, value(c + 2), value(c + 3)),
                             fp8_pack2(p.out_type, value(c + 4), value(c + 5)), fp8_pack2(p.out_type, value(c + 6), value(c + 7)));
            }
          }
        }
      }
    }
    if (lane == 0) ptx::bulk_wait_group<0>();            // shared memory must outlive the last box
    __syncwarp();
  }

  // ---- teardown: neither CTA may leave while the other can still signal its barriers
  __syncthreads();
  ptx::cluster_sync();
  const int aborted = *abort_flag;
  if (aborted != 0) {
    const long long start = clock64();
    while (clock64() - start < (1ll << 22)) {
    }
    if (threadIdx.x == 0 && p.error) atomicCAS(p.error, 0, aborted | (static_cast<int>(blockIdx.x) << 8));
  }
  if (warp == kMma) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<2>(tmem_base, 512);
  }
}

}  // namespace b200
