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
//   fp8_skinny_kernel<BN, kWide>  few rows; K can be split over a cluster whose CTAs add their partial
//                          tiles through distributed shared memory, in split order.
//                          kWide = false: the weights take the 128-row side of the MMA and BN = 16 .. 64
//                          rows of A the other, so that a row of activations costs a column, not 1/128
//                          of a tile. A thread then needs BN row scales per block, each read by all
//                          lanes: 512 BN bytes per warp, four cycles per row at 128 bytes per cycle, which
//                          at 128 rows took longer than everything else (0.75 us per block).
//                          kWide = true: 128 rows of A on the 128-row side, one scale per thread.
//   fp8_pair_kernel        many rows: 256 x 256 tiles on CTA pairs (cta_group::2).
//
// What bounds them, measured back to back with cold operands. One row, 4096 x 7168: 7.5 us for 29.4 MB, of which HBM
// takes 4.5; the rest is the first loads' latency, the exchange of partial tiles and the stores. 77 x 1000 x
// 1040: 5.2 us of fixed costs and dependent blocks, as short as Python can issue them. 128 x 4096 x 8192: 14.0 us;
// 16 blocks per CTA at 0.335 us, which is 128 SMs taking 32 KB each from L2 (12.5 TB/s), and the exchange.
// 64 rows over 32 groups of 4096 x 7168: 125 us, HBM (765 MB, 6.1 TB/s; weights of empty groups are not
// read). Many rows: see the pair kernel.
//
// Both start while the kernel before them drains: barriers, tensor memory and descriptors are set up by the time
// that one has ended (one row, 4096 x 7168: 12.3 -> 9.0 us back to back, 4096 x 4096 x 7168 136 -> 129).
//
// Waits on barriers in shared memory are bounded (ptx::mbar_wait_warp: one answer per warp) and reported through the
// device error word. Three others have no limit. The barriers of a cluster: its CTAs run at the same time, and all
// arrive, after a wait that has run out too. griddepcontrol.wait: it ends with the kernel before. The allocation
// of tensor memory, which comes before griddepcontrol.wait: a block of these kernels takes more than 200 of an SM's 228
// KB of shared memory, so no other of them and no four-bit product, which all use more than the rest, can be there
// with tensor memory of its own while this one waits for theirs.
#pragma once

#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gemm_kernel.cuh"

namespace b200 {

constexpr int kFp8BlockK = 128;               // values of K per scale = bytes of K per stage row
constexpr int kFp8Panel = 8;                  // few rows: blocks of K whose scales arrive together ...
constexpr int kFp8Panels = 2;                 // ... and panels of them in shared memory

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
  if (p.seqlens == nullptr) {   // one group of all rows
    if (threadIdx.x == 0) {
      s_rows[0] = p.total_rows;
      s_row0[0] = 0;
      s_cu_tiles[0] = 0;
      s_cu_tiles[1] = (p.total_rows + tile_rows - 1) / tile_rows;
    }
    __syncthreads();
    return;
  }
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
template <int kType>
__device__ __forceinline__ void fp8_store(void* out, long long at, float v) {
  if constexpr (kType == kOutF16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else if constexpr (kType == kOutBf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(out)[at] = v;
}

__device__ __forceinline__ uint32_t fp8_pack2(int type, float lo, float hi) {
  if (type == kOutF16) return pack_half2(lo, hi);
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&b);
}

// Eight consecutive values, 16-byte aligned.
template <int kType, typename Value>
__device__ __forceinline__ void fp8_store8(void* out, long long at, Value value) {
  if constexpr (kType == kOutF32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
    dst[0] = make_float4(value(0), value(1), value(2), value(3));
    dst[1] = make_float4(value(4), value(5), value(6), value(7));
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
        make_uint4(fp8_pack2(kType, value(0), value(1)), fp8_pack2(kType, value(2), value(3)),
                   fp8_pack2(kType, value(4), value(5)), fp8_pack2(kType, value(6), value(7)));
  }
}

// --------------------------------------------------------------------- few rows

template <int BN, bool kWide>
struct Fp8SkinnyCfg {
  static_assert(kWide ? BN == 128 : BN == 16 || BN == 32 || BN == 64, "unsupported tile");
  static constexpr int kTileM = kWide ? 128 : BN;          // rows of A per tile
  static constexpr int kTileN = kWide ? BN : 128;          // rows of B (output columns) per tile
  // promotion: a warp per quarter of tensor memory's lanes and, from 32 rows on, per half of the columns
  static constexpr int kHalves = BN >= 32 ? 2 : 1;
  static constexpr int kPromoters = 4 * kHalves;
  static constexpr int kCols = BN / kHalves;               // accumulators of a promotion thread
  static constexpr int kThreads = 128 + 32 * kPromoters;   // loaders of B and A, MMA issuer, (idle), promotion
  static constexpr int kScales = kTileM * kFp8Panel / (32 * kPromoters);   // scales of a panel per promotion thread
  static constexpr int kBuffers = 4;          // block sums in tensor memory
  static constexpr int kTmemCols = kBuffers * BN < 32 ? 32 : kBuffers * BN;
  static constexpr int kWideBytes = 128 * kFp8BlockK;      // operand on the 128-row side of the MMA
  static constexpr int kNarrowBytes = BN * kFp8BlockK;
  static constexpr int kStageBytes = kWideBytes + kNarrowBytes;
  static constexpr int kMaxStages = 12;
  static constexpr int kSlotFloats = kTileM + 4;           // scales of one block, padded against bank conflicts
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
  static_assert(stages_for(kMaxGroups, 2) >= 4 && stages_for(kMaxGroups, 2) * kStageBytes >= kRedBytes, "ring too small");
  static_assert(smem_bytes(1, 1) > 200 * 1024 && smem_bytes(1, 2) > 200 * 1024, "one block per SM: see the allocation of tensor memory");
};

template <int BN, bool kWide>
__global__ void __launch_bounds__(Fp8SkinnyCfg<BN, kWide>::kThreads, 1)
fp8_skinny_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                  const Fp8Params p) {
  using Cfg = Fp8SkinnyCfg<BN, kWide>;
  constexpr int kLoadWide = 0, kMma = 1, kLoadNarrow = 2, kFirstPromoter = 4;
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
  const uint32_t sc_full_u32 = sum_empty_u32 + 8 * Cfg::kBuffers;      // a panel of scales is in shared memory
  const uint32_t part_full_u32 = sc_full_u32 + 8 * kFp8Panels;         // this CTA's partial tile is in its ring
  const uint32_t red_full_u32 = part_full_u32 + 8;                     // every CTA's part of this CTA's rows
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * Cfg::kMaxStages + 2 * Cfg::kBuffers + kFp8Panels + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);
  float* slots = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);
  int* s_cu_tiles = reinterpret_cast<int*>(slots + kFp8Panels * kFp8Panel * Cfg::kSlotFloats);
  int* s_row0 = s_cu_tiles + (p.num_groups + 1);
  int* s_rows = s_row0 + (p.num_groups + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = splits > 1 ? static_cast<int>(ptx::cluster_cta_rank()) : 0;
  const bool one_group = p.seqlens == nullptr;

  if (warp == 0) {
    if (lane == 0) {
      *abort_flag = 0;
      ptx::prefetch_tensormap(kWide ? &tmap_x : &tmap_w);
    }
    for (int s = lane; s < kStages; s += 32) {
      ptx::mbar_init(full_u32 + 8 * s, 2);
      ptx::mbar_init(empty_u32 + 8 * s, 1);
    }
    if (lane < Cfg::kBuffers) {
      ptx::mbar_init(sum_full_u32 + 8 * lane, 1);
      ptx::mbar_init(sum_empty_u32 + 8 * lane, Cfg::kPromoters);
    }
    if (lane < kFp8Panels) ptx::mbar_init(sc_full_u32 + 8 * lane, Cfg::kPromoters);
    if (lane == 30) ptx::mbar_init(part_full_u32, Cfg::kPromoters);
    if (lane == 31) ptx::mbar_init(red_full_u32, 1);
    if (one_group && lane == 0) {
      s_rows[0] = p.total_rows;
      s_row0[0] = 0;
      s_cu_tiles[0] = 0;
      s_cu_tiles[1] = (p.total_rows + Cfg::kTileM - 1) / Cfg::kTileM;
    }
    __syncwarp();
    if (lane == 0) ptx::fence_barrier_init();
  } else if (warp == kMma) {
    ptx::tmem_alloc<1>(ptx::smem_u32(tmem_holder), Cfg::kTmemCols);
    ptx::tmem_relinquish<1>();
  } else if (warp == kLoadNarrow && lane == 0) {
    ptx::prefetch_tensormap(kWide ? &tmap_w : &tmap_x);
  }
  ptx::tc_fence_before_sync();
  const int b_begin = kb * rank / splits, b_end = kb * (rank + 1) / splits;
  if (warp == (kWide ? kLoadNarrow : kLoadWide) && one_group && splits == 1 && p.total_rows <= Cfg::kTileM) {
    // The first tile of weights on its way into L2 while the kernel before this one drains. Nothing is read that
    // way: should that kernel still write them, L2 has what it wrote, and the loads below take it from there.
    // (16 x 18432 x 7168 25.4 -> 24.1 us, 1 x 65536 x 4096 48.4 -> 45.8. Not where K is split, whose few blocks per
    // CTA are asked for at once anyway: 1 x 4096 x 7168 7.5 -> 7.9.)
    const int b = b_begin + lane;
    if (b < b_end) ptx::tma_prefetch_2d(&tmap_w, b * kFp8BlockK, static_cast<int>(blockIdx.x) / splits * Cfg::kTileN);
  }
  ptx::grid_wait();
  ptx::grid_launch_dependents();
  if (one_group) {
    // the loaders need the barriers only, and start before tensor memory has been allocated
    if (warp == kLoadWide || warp == kLoadNarrow) {
      ptx::named_barrier_sync(3, 64);
      ptx::named_barrier_arrive(4, Cfg::kThreads);
    } else {
      ptx::named_barrier_sync(4, Cfg::kThreads);
    }
  } else {
    fp8_group_tables(p, Cfg::kTileM, s_cu_tiles, s_row0, s_rows);
  }
  __syncwarp();
  if (splits > 1) ptx::cluster_arrive_relaxed();
  ptx::tc_fence_after_sync();

  const int n_tiles = (p.n + Cfg::kTileN - 1) / Cfg::kTileN;
  const int total_mt = s_cu_tiles[p.num_groups];
  const int total_tasks = total_mt * n_tiles;
  // a cluster takes one task, a CTA of an unsplit launch as many as come its way
  const int first_task = static_cast<int>(blockIdx.x) / splits;
  const int task_step = splits > 1 ? total_tasks : static_cast<int>(gridDim.x);
  const uint32_t stage_u32 = ptx::smem_u32(smem);
  // Threads of a cluster wait for each other twice: `met`, this warp has waited for the set-up of the others'
  // barriers; `done`, it has said that it needs nothing of the others any more. Both are the same in all lanes
  // of a warp, on the way out of a wait that has run out too: a lane that took its own way would be counted
  // in the wrong phase.
  bool met = false, done = false;
  // (a single row of tiles needs none of the divisions: they stood 0.6 us before the first load)
  auto decode = [&](int task) {
    if (one_group && total_mt == 1) return TileCoord{0, 0, task, 0};
    return decode_tile(task, total_mt, n_tiles, 1, p.raster_m, s_cu_tiles, p.num_groups);
  };

  if (warp == kLoadWide || warp == kLoadNarrow) {
    const bool wide = warp == kLoadWide, rows_of_a = wide == kWide;
    const uint32_t bytes = wide ? Cfg::kWideBytes : Cfg::kNarrowBytes;
    const CUtensorMap* tmap = rows_of_a ? &tmap_x : &tmap_w;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, withhold = wide && p.withhold_first_arrival != 0 && blockIdx.x == 0;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode(task);
      const int row = rows_of_a ? s_row0[t.g] + t.mt * Cfg::kTileM : t.g * p.n + t.nt * Cfg::kTileN;
      for (int b = b_begin; b < b_end; ++b) {
        if (!ptx::mbar_wait_warp(empty_u32 + 8 * stage, phase ^ 1, abort_flag, kWaitEmpty, p.wait_limit)) { ok = false; break; }
        if (ptx::elect_one()) {
          const uint32_t bar = full_u32 + 8 * stage;
          if (withhold) withhold = false;
          else ptx::mbar_arrive_expect_tx(bar, bytes);
          ptx::tma_load_2d(stage_u32 + stage * Cfg::kStageBytes + (wide ? 0 : Cfg::kWideBytes), tmap, bar, b * kFp8BlockK, row);
        }
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    const uint32_t tmem_base = *tmem_holder;
    constexpr uint32_t idesc = ptx::make_idesc_e4m3(128, BN);
    const uint32_t lo0 = ptx::kmajor_sw128_desc_lo(stage_u32);
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    bool ok = true;
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      for (int b = b_begin; b < b_end; ++b) {
        if (!ptx::mbar_wait_warp(sum_empty_u32 + 8 * buf, buf_phase ^ 1, abort_flag, kWaitAccEmpty, p.wait_limit) ||
            !ptx::mbar_wait_warp(full_u32 + 8 * stage, phase, abort_flag, kWaitFull, p.wait_limit)) { ok = false; break; }
        ptx::tc_fence_after_sync();
        if (ptx::elect_one()) {
          const uint32_t wide_lo = lo0 + stage * (Cfg::kStageBytes >> 4);
          const uint32_t narrow_lo = wide_lo + (Cfg::kWideBytes >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j)      // 32 values of K = 32 bytes = 2 units of the address field
            ptx::tc_mma_e4m3<1>(tmem_base + buf * BN, wide_lo + 2 * j, narrow_lo + 2 * j, ptx::kKmajorSw128DescHi, idesc, j > 0 ? 1u : 0u);
          ptx::tc_commit<1>(empty_u32 + 8 * stage);
          ptx::tc_commit<1>(sum_full_u32 + 8 * buf);
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1; }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp >= kFirstPromoter) {
    // ------------ promotion. kWide: lane = row of A, register = output column; else the other way round
    const int q = warp & 3;
    const int col_first = (warp - kFirstPromoter) / 4 * Cfg::kCols;
    const uint32_t lane_addr = *tmem_holder + (static_cast<uint32_t>(q * 32) << 16) + col_first;
    const int tile_row = q * 32 + lane;
    const int tid = static_cast<int>(threadIdx.x) - 32 * kFirstPromoter;
    // The promotion threads fetch the scales themselves, a panel of eight blocks ahead: into registers
    // while the last panel is used, then, each row scale times that of the weights' tile, into shared memory
    // as [block][rows of A]. Eight neighbouring lanes take the eight blocks of a row, which is one sector.
    // (A loader warp with asynchronous copies had the first panel ready 2000 cycles after the operands.)
    float next_scale[Cfg::kScales], next_w_scale = 0.0f;
    auto fetch_scales = [&](int task, int b0) {
      const TileCoord t = decode(task);
      const int left = s_rows[t.g] - t.mt * Cfg::kTileM;
      const int j = tid & 7;
      const float* src = p.a_scale + static_cast<long long>(s_row0[t.g] + t.mt * Cfg::kTileM) * kb + b0 + j;
      const long long tile = static_cast<long long>(t.g) * ((p.n + 127) / 128) + t.nt * Cfg::kTileN / 128;
      next_w_scale = b0 + j < b_end ? p.b_scale[tile * kb + b0 + j] : 0.0f;
#pragma unroll
      for (int i = 0; i < Cfg::kScales; ++i) {
        const int r = (tid >> 3) + i * (4 * Cfg::kPromoters);
        next_scale[i] = r < left && b0 + j < b_end ? src[static_cast<long long>(r) * kb] : 0.0f;
      }
    };
    int buf = 0, panel = 0;
    uint32_t buf_phase = 0, panel_phase = 0;
    bool ok = true;
    if (first_task < total_tasks && b_begin < b_end) fetch_scales(first_task, b_begin);
    for (int task = first_task; task < total_tasks && ok; task += task_step) {
      const TileCoord t = decode(task);
      // rows of A and output columns of the tile that exist; `valid` are those the registers run over
      const int rows_in = min(Cfg::kTileM, s_rows[t.g] - t.mt * Cfg::kTileM), cols_in = min(Cfg::kTileN, p.n - t.nt * Cfg::kTileN);
      const int valid = kWide ? cols_in : rows_in;
      float acc[Cfg::kCols];
#pragma unroll
      for (int c = 0; c < Cfg::kCols; ++c) acc[c] = 0;
      const float* sc = nullptr;
      // Scales of block b, in shared memory from its panel's first block on. (A warp reaches a panel's buffer
      // again only after all have used it: each arrives at the other panel's barrier in between.)
      auto scales_for = [&](int b) {
        if (((b - b_begin) & (kFp8Panel - 1)) != 0) {
          sc += Cfg::kSlotFloats;
          return true;
        }
        float* to = slots + panel * kFp8Panel * Cfg::kSlotFloats;
#pragma unroll
        for (int i = 0; i < Cfg::kScales; ++i) to[(tid & 7) * Cfg::kSlotFloats + (tid >> 3) + i * (4 * Cfg::kPromoters)] = next_scale[i] * next_w_scale;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(sc_full_u32 + 8 * panel);
        if (b + kFp8Panel < b_end) fetch_scales(task, b + kFp8Panel);
        else if (task + task_step < total_tasks) fetch_scales(task + task_step, b_begin);
        if (!ptx::mbar_wait_warp(sc_full_u32 + 8 * panel, panel_phase, abort_flag, kWaitSlots, p.wait_limit)) return false;
        sc = to;
        if (++panel == kFp8Panels) { panel = 0; panel_phase ^= 1; }
        return true;
      };
      auto sums_ready = [&] {
        if (!ptx::mbar_wait_warp(sum_full_u32 + 8 * buf, buf_phase, abort_flag, kWaitAccFull, p.wait_limit)) return false;
        ptx::tc_fence_after_sync();
        return true;
      };
      auto release_sums = [&] {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(sum_empty_u32 + 8 * buf);
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
      };
      if constexpr (kWide) {
        // The loads run one step of 16 columns ahead of the additions, across blocks too: the first step of
        // the next block is on its way while the last of this one is added. (Steps of 32 spill.)
        constexpr int kSteps = Cfg::kCols / 16;
        static_assert(kSteps % 2 == 0, "the first step of a block uses the first buffer");
        uint32_t v[2][16];
        if (b_begin < b_end) {
          ok = sums_ready();
          if (ok) ptx::tmem_ld_cols<16>(lane_addr + buf * BN, v[0]);
        }
        for (int b = b_begin; b < b_end && ok; ++b) {
          ok = scales_for(b);
          if (!ok) break;
          const float by = sc[tile_row];
#pragma unroll
          for (int step = 0; step < kSteps; ++step) {
            ptx::tmem_ld_wait_regs<16>(v[step & 1]);
            if (step + 1 < kSteps) {
              ptx::tmem_ld_cols<16>(lane_addr + buf * BN + (step + 1) * 16, v[(step + 1) & 1]);
            } else {
              release_sums();
              if (b + 1 < b_end) {
                ok = sums_ready();
                if (!ok) break;
                ptx::tmem_ld_cols<16>(lane_addr + buf * BN, v[0]);
              }
            }
#pragma unroll
            for (int c = 0; c < 16; ++c) acc[step * 16 + c] = fmaf(__uint_as_float(v[step & 1][c]), by, acc[step * 16 + c]);
          }
        }
        ptx::tmem_ld_wait();                                       // nothing may stay in flight after a break
      } else {
        for (int b = b_begin; b < b_end; ++b) {
          ok = scales_for(b) && sums_ready();
          if (!ok) break;
          // all columns first, one wait: the reads of the scales then follow each other without it
          constexpr int kStep = Cfg::kCols < 32 ? 16 : 32;
          static_assert(kStep == Cfg::kCols, "one load");
          uint32_t v[kStep];
          ptx::tmem_ld_cols<kStep>(lane_addr + buf * BN, v);
          ptx::tmem_ld_wait_regs<kStep>(v);
          release_sums();
#pragma unroll
          for (int c = 0; c < kStep; c += 4) {
            const float4 sa = *reinterpret_cast<const float4*>(sc + col_first + c);
            acc[c] = fmaf(__uint_as_float(v[c]), sa.x, acc[c]);
            acc[c + 1] = fmaf(__uint_as_float(v[c + 1]), sa.y, acc[c + 1]);
            acc[c + 2] = fmaf(__uint_as_float(v[c + 2]), sa.z, acc[c + 2]);
            acc[c + 3] = fmaf(__uint_as_float(v[c + 3]), sa.w, acc[c + 3]);
          }
        }
      }
      if (!ok) break;
      auto value = [&](int c) { return acc[c]; };
      const long long out0 = (static_cast<long long>(s_row0[t.g]) + t.mt * Cfg::kTileM) * p.n + t.nt * Cfg::kTileN;
      if (splits == 1) {
        auto store_all = [&](auto type) {
          constexpr int kType = decltype(type)::value;
          if constexpr (kWide) {
            if (tile_row < rows_in) {
              const long long at = out0 + static_cast<long long>(tile_row) * p.n + col_first;
#pragma unroll
              for (int c = 0; c < Cfg::kCols; c += 8)            // n is a multiple of 8
                if (col_first + c < valid) fp8_store8<kType>(p.out, at + c, [&](int j) { return value(c + j); });
            }
          } else if (tile_row < cols_in) {
#pragma unroll
            for (int c = 0; c < Cfg::kCols; ++c)
              if (col_first + c < valid)
                fp8_store<kType>(p.out, out0 + static_cast<long long>(col_first + c) * p.n + tile_row, value(c));
          }
        };
        if (p.out_type == kOutF16) store_all(std::integral_constant<int, kOutF16>());
        else if (p.out_type == kOutBf16) store_all(std::integral_constant<int, kOutBf16>());
        else store_all(std::integral_constant<int, kOutF32>());
      } else {
        // CTA d of the cluster finishes register columns [d w, (d + 1) w) of the tile. Everybody lays its
        // partial tile into its (now idle) operand ring, [register column][128 lanes], and copies slice d into CTA d's buffer,
        // one bulk copy each, counted in bytes on the receiver's barrier. (Asynchronous stores of single
        // words took longer than the product: 64 x 7168 x 2048 14.4 us unsplit, 18.5 split in two.)
        const int w = kWide ? BN / splits : (valid + splits - 1) / splits;
        const int mine = max(0, min(w, valid - rank * w));
        const bool first = warp == kFirstPromoter && lane == 0;
        if (first && mine > 0) ptx::mbar_arrive_expect_tx(red_full_u32, static_cast<uint32_t>((splits - 1) * mine * 512));
#pragma unroll
        for (int c = 0; c < Cfg::kCols; ++c)
          if (col_first + c < valid) reinterpret_cast<float*>(smem)[(col_first + c) * 128 + tile_row] = value(c);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(part_full_u32);
        __syncwarp();                                              // (the barriers of a cluster are for whole warps)
        ptx::cluster_wait();                                       // every CTA has its barriers
        met = true;
        if (!ptx::mbar_wait_warp(part_full_u32, 0, abort_flag, kWaitPartials, p.wait_limit)) break;
        const uint32_t red_u32 = ptx::smem_u32(red);
        if (first) {
          for (int d = 0; d < splits; ++d) {
            const int rows_d = min(w, valid - d * w);
            if (d == rank || rows_d <= 0) continue;
            ptx::bulk_copy_to_cta(ptx::map_to_cta(red_u32 + static_cast<uint32_t>(rank * rows_d * 512), d),
                                  stage_u32 + static_cast<uint32_t>(d * w * 512), static_cast<uint32_t>(rows_d * 512),
                                  ptx::map_to_cta(red_full_u32, d));
          }
        }
        if (mine > 0 && !ptx::mbar_wait_cluster_warp(red_full_u32, 0, abort_flag, kWaitPartials, p.wait_limit)) break;
        __syncwarp();
        ptx::cluster_arrive_relaxed();       // the others' copies have landed here (the wait is in the teardown)
        done = true;
        if (mine > 0) {
          // partial sums in split order, two columns per thread
          auto reduce = [&](auto count) {
            constexpr int kSplits = decltype(count)::value;
            // sum of the partial values at (register column i, 128-side index l .. l + 1), in split order
            auto sum2 = [&](int i, int l) {
              float2 v[kSplits];
#pragma unroll
              for (int s = 0; s < kSplits; ++s) {
                const float* part = s == rank ? reinterpret_cast<const float*>(smem) + (rank * w + i) * 128
                                              : reinterpret_cast<const float*>(red) + (s * mine + i) * 128;
                v[s] = *reinterpret_cast<const float2*>(part + l);
              }
#pragma unroll
              for (int s = 1; s < kSplits; ++s) {
                v[0].x = __fadd_rn(v[0].x, v[s].x);
                v[0].y = __fadd_rn(v[0].y, v[s].y);
              }
              return v[0];
            };
            auto store2 = [&](long long at, float2 v) {              // at is even
              if (p.out_type == kOutF32) *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at) = v;
              else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at) = fp8_pack2(p.out_type, v.x, v.y);
            };
            if constexpr (kWide) {
              // eight columns of a row per thread: neighbouring lanes read neighbouring words, and store 16
              // (32) bytes of their own row; w is a multiple of 8, so are the slices' ends
              for (int x = tid; x < (mine >> 3) * 128; x += 32 * Cfg::kPromoters) {
                const int i = 8 * (x >> 7), l = x & 127;
                float sum[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
#pragma unroll
                  for (int s = 0; s < kSplits; ++s) {
                    const float* part = s == rank ? reinterpret_cast<const float*>(smem) + (rank * w + i + c) * 128
                                                  : reinterpret_cast<const float*>(red) + (s * mine + i + c) * 128;
                    sum[c] = s == 0 ? part[l] : __fadd_rn(sum[c], part[l]);
                  }
                }
                if (l < rows_in) {
                  const long long at = out0 + static_cast<long long>(l) * p.n + rank * w + i;
                  auto eight = [&](int c) { return sum[c]; };
                  if (p.out_type == kOutF32) fp8_store8<kOutF32>(p.out, at, eight);
                  else if (p.out_type == kOutF16) fp8_store8<kOutF16>(p.out, at, eight);
                  else fp8_store8<kOutBf16>(p.out, at, eight);
                }
              }
            } else {
              for (int x = tid; x < mine * 64; x += 32 * Cfg::kPromoters) {
                const int i = x >> 6, l = 2 * (x & 63);
                const float2 v = sum2(i, l);
                if (l < cols_in) store2(out0 + static_cast<long long>(rank * w + i) * p.n + l, v);
              }
            }
          };
          if (splits == 2) reduce(std::integral_constant<int, 2>());
          else if (splits == 4) reduce(std::integral_constant<int, 4>());
          else reduce(std::integral_constant<int, 8>());
        }
      }
    }
    __syncwarp();
  }

  // ---- teardown. A CTA of a cluster must outlive its copies: their receivers arrive after having got them.
  if (splits > 1) {
    if (!met) ptx::cluster_wait();     // every thread waits once for the arrival at set-up ...
    if (!done) ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();               // ... and once for the others' end
  }
  __syncthreads();
  const int aborted = *abort_flag;
  if (aborted != 0) {
    const long long start = clock64();
    while (clock64() - start < (1ll << 22)) {
    }
    if (threadIdx.x == 0 && p.error) atomicCAS(p.error, 0, aborted | (static_cast<int>(blockIdx.x) << 8));
  }
  if (warp == kMma) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<1>(*tmem_holder, Cfg::kTmemCols);
  }
}

// -------------------------------------------------------------------- many rows

// 256 x 256 tiles on CTA pairs: each CTA loads 128 rows of A and its half of the 256 rows of B, the
// MMAs read both halves, and each CTA's tensor memory receives 128 rows x 256 columns of a block's
// sums. Two such buffers fill the 512 columns of tensor memory. 128 accumulators per thread in eight
// promotion warps need more registers than an even share (65536 / 384 = 168): the other four warps
// give theirs up (104 + 2 x 200 = 504 = 3 x 168; 56 / 224 to 104 / 200 differ by what the compiler spills: measured).
//
// 8192^3: 479 us in a burst (2300 TFLOP/s), 561 us sustained (1960 TFLOP/s, 0.71 of twice the measured BF16 rate),
// where power holds the SM clock at 1.46 GHz. The same loads and MMAs with nothing done to their sums take
// 394 / 466 us, bound by the operands' way from L2 (13.7 TB/s); promotion adds one TMEM read and one FMA per
// value and block. 4096 x 4096 x 7168 under counters: tensor pipe 60 % of the cycles, FMA pipe 35 %, issue
// slots 56 %. Tried without gain: MMAs of half the columns (four times as many waits; 527 us), polling
// barriers between MMAs, packed FMAs (their operands cost moves), loads of the next block before this
// one's additions (spills: 535 us), a panel of scales read ahead, wider steps than 16 columns.
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
static_assert(Fp8PairCfg::smem_bytes(1) > 200 * 1024, "one block per SM: see the allocation of tensor memory");

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
  ptx::grid_wait();
  ptx::grid_launch_dependents();
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
  ptx::setmaxnreg_dec<104>();
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
        if (!ptx::mbar_wait_warp(empty_u32 + 8 * stage, phase ^ 1, abort_flag, kWaitEmpty, p.wait_limit)) { ok = false; break; }
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
        if (!ptx::mbar_wait_warp(sc_empty_u32 + 8 * panel, phase ^ 1, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
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
          if (!ptx::mbar_wait_warp(full_u32 + 8 * stage, phase, abort_flag, kWaitFull, p.wait_limit) ||
              !ptx::mbar_wait_warp(sum_empty_u32 + 8 * buf, buf_phase ^ 1, abort_flag, kWaitAccEmpty, p.wait_limit)) { ok = false; break; }
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
    ptx::setmaxnreg_inc<200>();
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
      float acc[128];
#pragma unroll
      for (int c = 0; c < 128; ++c) acc[c] = 0.0f;
      float4 s4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int b = 0; b < kb; ++b) {
        if ((b & (Cfg::kPanel - 1)) == 0) {
          if (!ptx::mbar_wait_warp(sc_full_u32 + 8 * panel, panel_phase, abort_flag, kWaitSlots, p.wait_limit)) { ok = false; break; }
          const float4* sc = reinterpret_cast<const float4*>(slots + panel * Cfg::kPanelFloats);
          const float4 sa = sc[q * 32 + lane], sb = sc[128 + half];
          s4 = make_float4(sa.x * sb.x, sa.y * sb.y, sa.z * sb.z, sa.w * sb.w);
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sc_empty_u32 + 8 * panel);
          if (++panel == Cfg::kPanels) { panel = 0; panel_phase ^= 1; }
        }
        const float s = s4.x;
        s4 = make_float4(s4.y, s4.z, s4.w, s4.x);
        if (!ptx::mbar_wait_warp(sum_full_u32 + 8 * buf, buf_phase, abort_flag, kWaitAccFull, p.wait_limit)) { ok = false; break; }
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
          for (int c = 0; c < 16; ++c) acc[c0 * 16 + c] = fmaf(__uint_as_float(v[c]), s, acc[c0 * 16 + c]);
        }
        if (++buf == Cfg::kBuffers) { buf = 0; buf_phase ^= 1; }
      }
      auto value = [&](int c) { return acc[c]; };
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
            auto eight = [&](int j) { return value(c + j); };
            if (p.out_type == kOutF32) fp8_store8<kOutF32>(p.out, at + col, eight);
            else if (p.out_type == kOutF16) fp8_store8<kOutF16>(p.out, at + col, eight);
            else fp8_store8<kOutBf16>(p.out, at + col, eight);
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
