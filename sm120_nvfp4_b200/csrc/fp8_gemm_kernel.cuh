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
constexpr int kFp8ScaleSlots = 8;             // ring of scale vectors

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
  static constexpr int kSlotFloats = BN + 4;  // row scales of one block, then the scale of the weights' tile
  static constexpr int kRedBytes = 128 * BN * 4;
  static constexpr int fixed_bytes(int groups, int splits) {
    return 1024 + 512 + kFp8ScaleSlots * kSlotFloats * 4 + 3 * (groups + 1) * 4 + (splits > 1 ? kRedBytes : 0);
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
  const uint32_t sc_empty_u32 = sc_full_u32 + 8 * kFp8ScaleSlots;
  const uint32_t red_full_u32 = sc_empty_u32 + 8 * kFp8ScaleSlots;     // every CTA's part of this CTA's columns
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * Cfg::kMaxStages + 2 * Cfg::kBuffers + 2 * kFp8ScaleSlots + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);
  float* slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);
  int* s_cu_tiles = reinterpret_cast<int*>(slots + kFp8ScaleSlots * Cfg::kSlotFloats);
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
    if (lane < kFp8ScaleSlots) {
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
    // 4-byte asynchronous copies: the scales of one block are kb floats apart in memory. Rows behind
    // the end are not read and become zeros.
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int row = s_row0[t.g] + t.mt * BN;
      const int valid = min(BN, s_rows[t.g] - t.mt * BN);
      const float* sb = p.b_scale + (static_cast<long long>(t.g) * n_tiles + t.nt) * kb;
      for (int b = b_begin; b < b_end; ++b) {
        if (!ptx::mbar_wait(sc_empty_u32 + 8 * slot, phase ^ 1, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
        const uint32_t dst = ptx::smem_u32(slots + slot * Cfg::kSlotFloats);
#pragma unroll
        for (int c0 = 0; c0 < BN; c0 += 32) {
          const int c = c0 + lane;
          if (c < BN) {
            const bool in = c < valid;
            ptx::cp_async_4(dst + 4 * c, p.a_scale + static_cast<long long>(in ? row + c : row) * kb + b, in);
          }
        }
        if (lane == 0) ptx::cp_async_4(dst + 4 * BN, sb + b, true);
        ptx::cp_async_mbar_arrive(sc_full_u32 + 8 * slot);
        if (++slot == kFp8ScaleSlots) { slot = 0; phase ^= 1; }
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
    int buf = 0, slot = 0;
    uint32_t buf_phase = 0, slot_phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int valid = min(BN, s_rows[t.g] - t.mt * BN);
      float acc[BN];
#pragma unroll
      for (int c = 0; c < BN; ++c) acc[c] = 0.0f;
      for (int b = b_begin; b < b_end; ++b) {
        if (!ptx::mbar_wait(sc_full_u32 + 8 * slot, slot_phase, abort_flag, kWaitSlots, p.wait_limit) ||
            !ptx::mbar_wait(sum_full_u32 + 8 * buf, buf_phase, abort_flag, kWaitAccFull, p.wait_limit)) { ok = false; break; }
        ptx::tc_fence_after_sync();
        const float* sc = slots + slot * Cfg::kSlotFloats;
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
        if (lane == 0) {
          ptx::mbar_arrive(sum_empty_u32 + 8 * buf);
          ptx::mbar_arrive(sc_empty_u32 + 8 * slot);
        }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
        if (++slot == kFp8ScaleSlots) { slot = 0; slot_phase ^= 1; }
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
// give theirs up (56 + 2 x 224 = 504 = 3 x 168 per three warpgroups' lanes).
struct Fp8PairCfg {
  static constexpr int kThreads = 384;
  static constexpr int kBuffers = 2;
  static constexpr int kABytes = 128 * kFp8BlockK;
  static constexpr int kBBytes = 128 * kFp8BlockK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kMaxStages = 6;
  static constexpr int kSlotFloats = 128 + 4;                    // scales of the CTA's rows, of two column tiles
  static constexpr int kStagingBytes = 8 * 32 * 128;
  static constexpr int fixed_bytes(int groups) {
    return 1024 + 512 + kFp8ScaleSlots * kSlotFloats * 4 + 3 * (groups + 1) * 4 + kStagingBytes;
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
  const uint32_t sc_empty_u32 = sc_full_u32 + 8 * kFp8ScaleSlots;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * Cfg::kMaxStages + 2 * Cfg::kBuffers + 2 * kFp8ScaleSlots);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);
  float* slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);
  int* s_cu_tiles = reinterpret_cast<int*>(slots + kFp8ScaleSlots * Cfg::kSlotFloats);
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
      ptx::mbar_init(sum_empty_u32 + 8 * lane, 16);
    }
    if (lane < kFp8ScaleSlots) {
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
  ptx::setmaxnreg_dec<56>();
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
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    const int nb = (p.n + 127) / 128;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      const int row = s_row0[t.g] + t.mt * 256 + cta * 128;
      const int valid = min(128, s_rows[t.g] - t.mt * 256 - cta * 128);     // may be <= 0 in the second CTA
      const float* sb = p.b_scale + (static_cast<long long>(t.g) * nb + 2 * t.nt) * kb;
      for (int b = 0; b < kb; ++b) {
        if (!ptx::mbar_wait(sc_empty_u32 + 8 * slot, phase ^ 1, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
        const uint32_t dst = ptx::smem_u32(slots + slot * Cfg::kSlotFloats);
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 32) {
          const int c = c0 + lane;
          const bool in = c < valid;
          ptx::cp_async_4(dst + 4 * c, p.a_scale + (in ? static_cast<long long>(row + c) * kb + b : 0), in);
        }
        if (lane < 2) {
          const bool in = 2 * t.nt + lane < nb;
          ptx::cp_async_4(dst + 4 * (128 + lane), sb + (in ? static_cast<long long>(lane) * kb : 0) + b, in);
        }
        ptx::cp_async_mbar_arrive(sc_full_u32 + 8 * slot);
        if (++slot == kFp8ScaleSlots) { slot = 0; phase ^= 1; }
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
    ptx::setmaxnreg_inc<224>();
    // ------------------ promotion: lane = row of the tile, registers = 128 columns (one scale tile of B)
    const int q = warp & 3;
    const int half = (warp - kFirstPromoter) >> 2;
    const uint32_t addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + half * 128;
    const uint32_t stg = ptx::smem_u32(staging) + (warp - kFirstPromoter) * 4096;
    const uint32_t stg_row = stg + lane * 128;
    const uint32_t sum_empty_target = ptx::map_to_cta(sum_empty_u32, 0);
    int buf = 0, slot = 0;
    uint32_t buf_phase = 0, slot_phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
      float2 acc[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = make_float2(0.0f, 0.0f);
      for (int b = 0; b < kb; ++b) {
        if (!ptx::mbar_wait(sc_full_u32 + 8 * slot, slot_phase, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
        const float* sc = slots + slot * Cfg::kSlotFloats;
        const float s = sc[q * 32 + lane] * sc[128 + half];
        if (!ptx::mbar_wait(sum_full_u32 + 8 * buf, buf_phase, abort_flag, kWaitAccFull, p.wait_limit)) { ok = false; break; }
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int c0 = 0; c0 < 4; ++c0) {
          uint32_t v[32];
          ptx::tmem_ld_cols<32>(addr + buf * 256 + c0 * 32, v);
          ptx::tmem_ld_wait_regs<32>(v);
          if (c0 == 3) {                       // everything has left tensor memory
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if (leader) ptx::mbar_arrive(sum_empty_u32 + 8 * buf);
              else ptx::mbar_arrive_cluster(sum_empty_target + 8 * buf);
              ptx::mbar_arrive(sc_empty_u32 + 8 * slot);
            }
          }
#pragma unroll
          for (int c = 0; c < 16; ++c)
            acc[c0 * 16 + c] = ptx::fma2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]), s, acc[c0 * 16 + c]);
        }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
        if (++slot == kFp8ScaleSlots) { slot = 0; slot_phase ^= 1; }
      }
      if (!ok) break;
      // ---- output: a slab of 32 valid rows leaves through the staging buffer and the store engine,
      // a ragged one by predicated stores
      const int row_in_group = t.mt * 256 + cta * 128 + q * 32;
      const int rows_left = s_rows[t.g] - row_in_group;
      const int map_row = s_row0[t.g] + row_in_group;
      const int col0 = t.nt * 256 + half * 128;
      if (rows_left <= 0 || col0 >= p.n) continue;
      const int elem = p.out_type == kOutF32 ? 4 : 2;
      const int box = 128 / elem;                        // columns per staged box
      if (p.tma_store && rows_left >= 32) {
#pragma unroll
        for (int c0 = 0; c0 < 4; ++c0) {                 // 32 columns at a time
          const int col = col0 + c0 * 32;
          if (col >= p.n) break;
          if (elem == 4 || (c0 & 1) == 0) {
            if (lane == 0) ptx::bulk_wait_group_read<0>();
            __syncwarp();
          }
          if (elem == 4) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const float2 x = acc[c0 * 16 + 2 * u], y = acc[c0 * 16 + 2 * u + 1];
              ptx::st_shared_v4(stg_row + (static_cast<uint32_t>(u ^ (lane & 7)) << 4), __float_as_uint(x.x),
                                __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = fp8_pack2(p.out_type, acc[c0 * 16 + 4 * u + i].x, acc[c0 * 16 + 4 * u + i].y);
              ptx::st_shared_v4(stg_row + (static_cast<uint32_t>(((c0 & 1) * 4 + u) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
          }
          if (elem == 4 || (c0 & 1) == 1 || col + 32 >= p.n) {
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              ptx::tma_store_2d(&tmap_out, stg, col0 + (c0 * 32 / box) * box, map_row);
              ptx::bulk_commit_group();
            }
          }
        }
      } else if (lane < rows_left) {
        const long long at = static_cast<long long>(map_row + lane) * p.n + col0;
#pragma unroll
        for (int c = 0; c < 64; c += 4) {                // 8 columns: n is a multiple of 8
          if (col0 + 2 * c < p.n) {
            if (elem == 4) {
              float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + 2 * c);
              dst[0] = make_float4(acc[c].x, acc[c].y, acc[c + 1].x, acc[c + 1].y);
              dst[1] = make_float4(acc[c + 2].x, acc[c + 2].y, acc[c + 3].x, acc[c + 3].y);
            } else {
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at + 2 * c) =
                  make_uint4(fp8_pack2(p.out_type, acc[c].x, acc[c].y), fp8_pack2(p.out_type, acc[c + 1].x, acc[c + 1].y),
                             fp8_pack2(p.out_type, acc[c + 2].x, acc[c + 2].y), fp8_pack2(p.out_type, acc[c + 3].x, acc[c + 3].y));
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
