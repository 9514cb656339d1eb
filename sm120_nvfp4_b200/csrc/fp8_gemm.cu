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

// CTAs per tile over K: as many as still fit the GPU at once and leave each enough blocks of K to pay for the
// exchange of partial tiles, which grows with the tile (us, tile / splits; 24 x 1024 x 1024: 16/1 6.3,
// 16/4 5.9; 96 x 1024 x 1024: 64/1 7.6, 64/2 8.7; 64 x 7168 x 2048: 64/1 10.6, 64/2 10.3; 128 x 7168 x 2048: 128/1 12.8, 128/2 14.8;
// 128 x 4096 x 7168: 128/1 29.5, 128/4 17.2).
int pick_fp8_splits(const Fp8Problem& q, const DeviceInfo& dev, int tile) {
  const long long tasks = row_tiles(q, tile) * ((q.n + 127) / 128);
  const int kb = (q.k + kFp8BlockK - 1) / kFp8BlockK;
  const int least = tile == 16 ? 2 : (tile == 128 ? 12 : 8);
  for (int s = 8; s >= 2; s /= 2)
    if (tasks * s <= dev.sm_count && kb >= least * s) return s;
  return 1;
}

// Rows of A per tile (512: 256 x 256 on CTA pairs).
//   Groups: the tile that the average group fills to at most three quarters, since groups differ; every
//   further tile of a group reads its weights again. 32 groups over 4096 x 7168, us for the average row
//   counts 12 / 24 / 40 / 64 / 96 / 128: 16 rows 151 / 226 / - , 32 rows 148 / 157 / 218 / 320,
//   64 rows 164 / 167 / 172 / 256 / 324, 128 rows 177 / 178 / 182 / 185 / 215 / 289, pairs - / - / 216 / 218 /
//   220 / 219.
//   One group: the smallest tile that holds all rows up to 64; then 128 rows where K is deep enough to be
//   split (128 x 4096 x 7168: 17.2 us, 64 rows 17.7) or the tiles fit the GPU at once, 64 rows while even
//   those do (128 x 7168 x 2048: 11.0 against 12.8), pairs beyond (384 x 7168 x 2048: 14.3 against 22.0).
int pick_fp8_tile(const Fp8Problem& q, const DeviceInfo& dev) {
  const int rows = q.avg_rows;
  if (q.seqlens != nullptr) {
    for (int tile = 16; tile <= 128; tile *= 2)
      if (static_cast<long long>(rows) * 4 <= tile * 3) return tile;
    return kPairTile;
  }
  for (int tile = 16; tile <= 64; tile *= 2)
    if (rows <= tile) return tile;
  const long long columns = (q.n + 127) / 128;
  if (pick_fp8_splits(q, dev, 128) > 1) return 128;
  if (row_tiles(q, 64) * columns <= dev.sm_count) return 64;
  return row_tiles(q, 128) * columns <= dev.sm_count ? 128 : kPairTile;
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
  const int tile = forced ? forced : pick_fp8_tile(q, dev);
  if (tile == kPairTile) return launch_pair(q, p, dev, stream);
  int splits = g_fp8_splits.load(std::memory_order_relaxed);
  if (splits == 0) splits = pick_fp8_splits(q, dev, tile);
  switch (tile) {
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
