// Host launchers and C ABI of the FP8 products with a scale per block of 128.
#include <atomic>
#include <cstdint>
#include <mutex>

#include "fp8_gemm_kernel.cuh"
#include "host_common.hpp"
#include "internal.hpp"

namespace b200 {

extern std::atomic<long long> g_wait_limit;
extern std::atomic<int> g_withhold_once;

namespace {

constexpr int kPairTile = 512;
constexpr int kMaxRows = 0x7fffff00;

std::atomic<int> g_fp8_tile{0};
std::atomic<int> g_fp8_splits{0};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

struct Fp8Problem {
  int groups, rows, n, k;
  const void* a;
  const void* b;
  const int* seqlens;
  const int* cu_seqlens;
  int avg_rows;      // rows per group: exact for one group, a hint for several
};

// Largest number of clusters of `ctas` that can be resident at once (not every SM need be pairable).
template <typename Kernel>
int resident_clusters(Kernel kernel, const DeviceInfo& dev, int ctas, int threads, int smem) {
  cudaLaunchConfig_t probe = {};
  probe.gridDim = dim3(static_cast<unsigned>(dev.sm_count / ctas * ctas));
  probe.blockDim = dim3(static_cast<unsigned>(threads));
  probe.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  probe.attrs = attr;
  probe.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &probe) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = dev.sm_count / (2 * ctas);
  }
  return n;
}

// Tiles of `tile_rows` rows: exact for one group, an upper bound for several.
long long row_tiles(const Fp8Problem& q, int tile_rows) {
  const long long exact = (static_cast<long long>(q.rows) + tile_rows - 1) / tile_rows;
  return q.seqlens == nullptr ? exact : static_cast<long long>(q.rows) / tile_rows + (q.rows < q.groups ? q.rows : q.groups);
}

// The same, but what is likely for several: every group ends in a tile that is half empty on average.
long long likely_row_tiles(const Fp8Problem& q, int tile_rows) {
  if (q.seqlens == nullptr) return row_tiles(q, tile_rows);
  const long long tiles = static_cast<long long>(q.rows) / tile_rows + (q.groups + 1) / 2, least = q.rows < q.groups ? q.rows : q.groups;
  return tiles > least ? tiles : least;
}

template <int BN, bool kWide>
int launch_skinny(const Fp8Problem& q, Fp8Params p, int splits, const DeviceInfo& dev, cudaStream_t stream) {
  using Cfg = Fp8SkinnyCfg<BN, kWide>;
  auto kernel = fp8_skinny_kernel<BN, kWide>;
  static std::once_flag once[64];
  static cudaError_t attr_status[64];
  std::call_once(once[dev.device], [&] {
    attr_status[dev.device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget);
  });
  if (attr_status[dev.device] != cudaSuccess) return B200_NVFP4_CUDA_ERROR;
  CUtensorMap tmap_x, tmap_w;
  if (!encode_tmap_2d_u8(&tmap_x, q.a, static_cast<uint64_t>(q.rows), static_cast<uint64_t>(q.k), Cfg::kTileM, kFp8BlockK,
                         CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_2d_u8(&tmap_w, q.b, static_cast<uint64_t>(q.groups) * q.n, static_cast<uint64_t>(q.k), Cfg::kTileN, kFp8BlockK,
                         CU_TENSOR_MAP_SWIZZLE_128B))
    return B200_NVFP4_CUDA_ERROR;
  p.splits = splits;
  p.num_stages = Cfg::stages_for(q.groups, splits);
  p.raster_m = 16;
  const long long tasks = row_tiles(q, Cfg::kTileM) * ((q.n + Cfg::kTileN - 1) / Cfg::kTileN);
  const long long blocks = splits > 1 ? tasks * splits : (tasks < dev.sm_count ? tasks : dev.sm_count);
  return launch_overlapped(kernel, static_cast<unsigned>(blocks < 1 ? 1 : blocks), Cfg::kThreads, static_cast<size_t>(Cfg::smem_bytes(q.groups, splits)),
                           splits, stream, tmap_x, tmap_w, p);
}

int launch_pair(const Fp8Problem& q, Fp8Params p, const DeviceInfo& dev, cudaStream_t stream) {
  using Cfg = Fp8PairCfg;
  static std::once_flag once[64];
  static cudaError_t attr_status[64];
  static int max_pairs[64];
  std::call_once(once[dev.device], [&] {
    cudaError_t e = cudaFuncSetAttribute(fp8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget);
    cudaFuncAttributes attr;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, fp8_pair_kernel);
    // the kernel moves registers between its warpgroups: it must have been launched with all of them
    if (e == cudaSuccess && attr.numRegs * Cfg::kThreads < 104 * 128 + 200 * 256) e = cudaErrorInvalidConfiguration;
    attr_status[dev.device] = e;
    max_pairs[dev.device] = e == cudaSuccess ? resident_clusters(fp8_pair_kernel, dev, 2, Cfg::kThreads, kSmemBudget) : 0;
  });
  if (attr_status[dev.device] != cudaSuccess) return B200_NVFP4_CUDA_ERROR;
  CUtensorMap tmap_a, tmap_b;
  if (!encode_tmap_2d_u8(&tmap_a, q.a, static_cast<uint64_t>(q.rows), static_cast<uint64_t>(q.k), 128, kFp8BlockK,
                         CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_2d_u8(&tmap_b, q.b, static_cast<uint64_t>(q.groups) * q.n, static_cast<uint64_t>(q.k), 128, kFp8BlockK,
                         CU_TENSOR_MAP_SWIZZLE_128B))
    return B200_NVFP4_CUDA_ERROR;
  CUtensorMap tmap_out = tmap_a;
  const bool f32 = p.out_type == kOutF32;
  p.tma_store = q.n >= (f32 ? 32 : 64) &&
                encode_tmap_2d_out(&tmap_out, p.out, static_cast<uint64_t>(q.rows), static_cast<uint64_t>(q.n),
                                   static_cast<uint64_t>(q.n), f32, 32, f32 ? 32 : 64);
  p.scales_by_16 = (q.k + kFp8BlockK - 1) / kFp8BlockK % 4 == 0 && aligned16(p.a_scale) && aligned16(p.b_scale);
  p.splits = 1;
  p.num_stages = Cfg::stages_for(q.groups);
  p.raster_m = 8;
  long long pairs = row_tiles(q, 256) * ((q.n + 255) / 256);
  if (pairs > max_pairs[dev.device]) pairs = max_pairs[dev.device];
  if (pairs < 1) pairs = 1;
  return launch_overlapped(fp8_pair_kernel, static_cast<unsigned>(2 * pairs), Cfg::kThreads, static_cast<size_t>(Cfg::smem_bytes(q.groups)), 1, stream,
                           tmap_a, tmap_b, tmap_out, p);       // (clusters of two by the kernel's own declaration)
}

struct Fp8Choice {
  int tile, splits;      // rows of A per tile (512: 256 x 256 on CTA pairs), CTAs per tile over K
};

// Microseconds that a launch of `tasks` tiles takes, split over K or not: a fixed part, a part per block of 128 of
// K that a CTA goes through, a part for the exchange of partial tiles, once more per round of tiles. The
// constants are fitted to these (rows x N x K, tile / splits: us back to back):
//   77 x 1000 x 1040    16/1 5.5, 16/2 5.4, 32/1 5.9, 32/4 5.2, 64/1 7.4, 64/4 6.5, 128/1 8.5
//   77 x 1024 x 4096    16/2 8.3, 32/2 8.9, 32/4 6.6, 64/4 8.1, 128/4 9.8, 128/1 16.9, pairs 18.8
//   48 x 4096 x 7168    16/1 18.5, 32/2 13.2, 64/2 14.2, 64/4 10.2, 128/2 16.8, 128/4 13.6
//   128 x 4096 x 7168   32/1 20.0, 64/1 23.2, 64/2 16.0, 128/1 24.6, 128/2 17.4, 128/4 14.0; 192 rows: pairs 29.4
//   192 x 7168 x 2048   64/1 16.7 (two rounds), 128/1 11.9, pairs 12.6; 384 rows: 128/1 20.1 (two rounds), pairs 13.5
float fp8_cost(int tile, int splits, long long tasks, int kb, int places) {
  const float fixed = tile == 16 ? 2.8f : tile == 32 ? 2.9f : tile == 64 ? 3.6f : tile == 128 ? 4.3f : 4.0f;
  const float per_task = tile == 16 ? 0.5f : tile == 32 ? 0.6f : tile == 64 ? 0.9f : tile == 128 ? 1.2f : 2.0f;
  const float per_block = tile == 16 ? 0.24f : tile == 32 ? 0.265f : tile == 64 ? 0.33f : tile == 128 ? 0.335f : 0.42f;
  const float exchange = tile == 16 ? 0.7f : tile == 32 ? 0.9f : tile == 64 ? 1.0f : 2.0f;
  const long long rounds = (tasks * splits + places - 1) / places;
  return fixed + static_cast<float>(rounds) * (per_task + per_block * static_cast<float>((kb + splits - 1) / splits)) +
         (splits > 1 ? exchange : 0.0f);
}

// Clusters of 2, 4 and 8 CTAs of the few-row kernel that fit the GPU at once (of 8, fewer than SMs / 8: those of a
// cluster come from one part of the GPU, and sixteen clusters took 9.1 us where 32 of four took 5.8).
const int* few_row_clusters(const DeviceInfo& dev) {
  static std::once_flag once[64];
  static int fit[64][4];
  std::call_once(once[dev.device], [&] {
    auto kernel = fp8_skinny_kernel<16, false>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget) != cudaSuccess) cudaGetLastError();
    for (int i = 1; i < 4; ++i)
      fit[dev.device][i] = resident_clusters(kernel, dev, 1 << i, Fp8SkinnyCfg<16, false>::kThreads, kSmemBudget);
  });
  return fit[dev.device];
}

// Tile and splits. One group, or several whose tiles are likely to fit the GPU at once (16 groups, 100 rows, 1024 x
// 2048: 16/1 8.3, 64/1 10.6; 4 groups, 64 rows, 4096 x 2048: 32/1 8.7, 64/1 10.3): the least estimated time, of all
// tiles (or `tile` alone) unsplit and of those splits that certainly fit at once and leave each CTA two blocks.
// Several groups that do not: the tile that the average group fills to at most three quarters, since groups
// differ; every further tile of a group reads its weights again. 32 groups over 4096 x 7168, us for the average
// row counts 12 / 24 / 40 / 64 / 96 / 128: 16 rows 151 / 226 / - , 32 rows 148 / 157 / 218 / 320, 64 rows 164 /
// 167 / 172 / 256 / 324, 128 rows 177 / 178 / 182 / 185 / 215 / 289, pairs - / - / 216 / 218 / 220 / 219.
Fp8Choice pick_fp8(const Fp8Problem& q, const DeviceInfo& dev, int tile) {
  const int kb = (q.k + kFp8BlockK - 1) / kFp8BlockK;
  const long long columns = (q.n + 127) / 128;
  const bool grouped = q.seqlens != nullptr;
  const int* clusters = few_row_clusters(dev);
  Fp8Choice best{tile == 0 ? kPairTile : tile, 1};
  float least = 3.4e38f;
  for (int t = 16; t <= 128; t *= 2) {
    const long long tasks = likely_row_tiles(q, t) * columns, most = row_tiles(q, t) * columns;
    if ((tile != 0 && tile != t) || (grouped && tasks > dev.sm_count)) continue;
    for (int i = 0; i == 0 || (i < 4 && most <= clusters[i] && kb >= 2 << i); ++i) {
      const int s = 1 << i;
      const float cost = fp8_cost(t, s, tasks, kb, dev.sm_count);
      if (cost < least) {
        least = cost;
        best = {t, s};
      }
    }
  }
  if (tile != 0) return best;
  if (!grouped) {
    if (fp8_cost(kPairTile, 1, row_tiles(q, 256) * ((q.n + 255) / 256), kb, dev.sm_count / 2) < least) best = {kPairTile, 1};
  } else if (least == 3.4e38f) {
    for (int t = 16; t <= 128; t *= 2)
      if (static_cast<long long>(q.avg_rows) * 4 <= t * 3) return {t, 1};
  }
  return best;
}

int fp8_product(const Fp8Problem& q, const void* a_scale, const void* b_scale, void* out, int out_type, cudaStream_t stream) {
  const DeviceInfo& dev = current_device_info();
  if (!dev.ok) return B200_NVFP4_CUDA_ERROR;
  if (!device_supported(dev)) return B200_NVFP4_UNSUPPORTED_DEVICE;
  if (q.rows == 0) return B200_NVFP4_SUCCESS;
  Fp8Params p = {};
  p.num_groups = q.groups;
  p.total_rows = q.rows;
  p.n = q.n;
  p.k = q.k;
  p.seqlens = q.seqlens;
  p.cu_seqlens = q.cu_seqlens;
  p.a_scale = static_cast<const float*>(a_scale);
  p.b_scale = static_cast<const float*>(b_scale);
  p.out = out;
  p.out_type = out_type;
  p.error = device_error_word();
  p.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
  p.withhold_first_arrival = g_withhold_once.exchange(0, std::memory_order_relaxed);
  const int forced = g_fp8_tile.load(std::memory_order_relaxed);
  const Fp8Choice choice = pick_fp8(q, dev, forced);
  if (choice.tile == kPairTile) return launch_pair(q, p, dev, stream);
  const int forced_splits = g_fp8_splits.load(std::memory_order_relaxed);
  const int splits = forced_splits ? forced_splits : choice.splits;
  switch (choice.tile) {
    case 16: return launch_skinny<16, false>(q, p, splits, dev, stream);
    case 32: return launch_skinny<32, false>(q, p, splits, dev, stream);
    case 64: return launch_skinny<64, false>(q, p, splits, dev, stream);
    default: return launch_skinny<128, true>(q, p, splits, dev, stream);
  }
}

bool valid_fp8(int rows, int n, int k, int out_type) {
  // (coordinates of a tile or block that reaches past the end still have to fit 32 bits)
  return rows >= 0 && rows <= kMaxRows && n > 0 && n <= kMaxRows && k > 0 && k <= kMaxRows && (k % 16) == 0 && (n % 8) == 0 &&
         out_type >= kOutF16 && out_type <= kOutBf16;
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_nvfp4_fp8_gemm(int m, int n, int k, const void* a, const void* b, const void* a_scale, const void* b_scale, void* c,
                        int out_type, b200_stream_t stream) {
  using namespace b200;
  if (!valid_fp8(m, n, k, out_type) || a == nullptr || b == nullptr || a_scale == nullptr || b_scale == nullptr ||
      c == nullptr || !aligned16(a) || !aligned16(b) || !aligned16(c) || !aligned4(a_scale) || !aligned4(b_scale))
    return B200_NVFP4_INVALID_ARGUMENT;
  const Fp8Problem q{1, m, n, k, a, b, nullptr, nullptr, m};
  return fp8_product(q, a_scale, b_scale, c, out_type, static_cast<cudaStream_t>(stream));
}

int b200_nvfp4_fp8_grouped_gemm(void* y, const void* x, const void* w, const void* seqlens, const void* cu_seqlens,
                                const void* x_scale, const void* w_scale, int num_group, int m, int n, int k,
                                int num_seq_per_group_avg, int out_type, b200_stream_t stream) {
  using namespace b200;
  if (!valid_fp8(m, n, k, out_type) || num_group <= 0 || num_group > kMaxGroups || y == nullptr || x == nullptr ||
      w == nullptr || seqlens == nullptr || cu_seqlens == nullptr || x_scale == nullptr || w_scale == nullptr ||
      !aligned16(y) || !aligned16(x) || !aligned16(w) || !aligned4(seqlens) || !aligned4(cu_seqlens) || !aligned4(x_scale) ||
      !aligned4(w_scale) || static_cast<long long>(num_group) * n > kMaxRows)
    return B200_NVFP4_INVALID_ARGUMENT;
  const int avg = num_seq_per_group_avg > 0 ? num_seq_per_group_avg : (m + num_group - 1) / num_group;
  const Fp8Problem q{num_group, m, n, k, x, w, static_cast<const int*>(seqlens), static_cast<const int*>(cu_seqlens), avg};
  return fp8_product(q, x_scale, w_scale, y, out_type, static_cast<cudaStream_t>(stream));
}

int b200_nvfp4_fp8_set_tile(int tile, int splits) {
  if ((tile != 0 && tile != 16 && tile != 32 && tile != 64 && tile != 128 && tile != b200::kPairTile) ||
      (splits != 0 && splits != 1 && splits != 2 && splits != 4 && splits != 8))
    return B200_NVFP4_INVALID_ARGUMENT;
  b200::g_fp8_tile.store(tile, std::memory_order_relaxed);
  b200::g_fp8_splits.store(splits, std::memory_order_relaxed);
  return B200_NVFP4_SUCCESS;
}

}  // extern "C"
