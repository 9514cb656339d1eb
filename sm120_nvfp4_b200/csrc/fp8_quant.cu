// Row quantiser to E4M3 with one FP32 scale per 128 values, optionally with SiLU(gate) * up in front.
//
//   amax_b = max(|x|) over the 128 values of a block, at least 2^-60
//   s_b = RN(amax_b / 448),  q = E4M3(RN(x / s_b))
//
// HBM-bound: 2 bytes read (4 with SiLU) and 1.03 written per value of a 16-bit input. Sixteen lanes
// share a block, eight values each: one 16-byte load (two for FP32), an amax by four shuffles and one
// 8-byte store, all coalesced; a thread works on several blocks so that their loads overlap.
//
// The division: every quotient of a block has the same divisor s, so one correctly rounded reciprocal
// r = RN(1 / s) serves them all by Markstein's sequence (IBM J. Res. Dev. 34(1), 1990): q0 = RN(x r),
// rem = x - q0 s (exact), RN(q0 + rem r) = RN(x / s). The floor of amax keeps rem exact wherever the
// quotient is one E4M3 distinguishes from zero: |q0| >= 2^-11 and s >= 2^-69 leave rem's last bit at
// 2^-126. A block with an infinity or a NaN takes plain divisions, and its scale says so: the
// values times the scale are NaN.
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "host_common.hpp"
#include "internal.hpp"

namespace b200 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 8.67361737988403547e-19f;   // 2^-60

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// v[j] / s for a divisor whose correctly rounded reciprocal is y: Markstein's sequence (see above). The
// signs are chosen so that a quotient of -0 stays -0.
__device__ __forceinline__ float quotient(float v, float s, float y) {
  const float q0 = __fmul_rn(v, y);
  return __fmaf_rn(-__fmaf_rn(q0, s, -v), y, q0);
}

// silu(g) * u = g / (1 + e^-g) * u in IEEE FP32 steps. Inside |g| <= 87 the divisor lies in [1, 2^126], so
// the quotient needs no special cases; outside (or infinite) the eight values take the plain division.
__device__ __forceinline__ void silu_mul8(float (&v)[8], const float (&u)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
  if (top <= 87.0f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = __fadd_rn(1.0f, expf(-v[j]));
      v[j] = __fmul_rn(quotient(v[j], d, __frcp_rn(d)), u[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(__fdiv_rn(v[j], __fadd_rn(1.0f, expf(-v[j]))), u[j]);
  }
}

// `step_rows`, `step_cols`: 16 / kb and 16 % kb, the way from one of a thread's blocks to its next.
template <typename T, bool kSwiglu, int kUnroll>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(uint8_t* __restrict__ q, float* __restrict__ scale, const T* __restrict__ x, int k, uint32_t kb,
                    uint32_t blocks, uint32_t step_rows, uint32_t step_cols) {
  const int lane = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (16u * kUnroll) + (threadIdx.x >> 4);
  float v[kUnroll][8];
  [[maybe_unused]] float u[kUnroll][8];
  long long at[kUnroll];
  bool in[kUnroll];
  uint32_t row = first / kb, col_block = first - row * kb;
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int col = static_cast<int>(col_block) * 128 + lane * 8;
    in[i] = first + 16u * i < blocks && col < k;
    at[i] = static_cast<long long>(row) * k + col;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    if (in[i]) {
      if constexpr (kSwiglu) {
        const T* src = x + at[i] + static_cast<long long>(row) * k;     // rows of 2 k: gate, then up
        load8(src, v[i]);
        load8(src + k, u[i]);
      } else {
        load8(x + at[i], v[i]);
      }
    }
    row += step_rows;
    col_block += step_cols;
    if (col_block >= kb) { col_block -= kb; ++row; }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if constexpr (kSwiglu) {
      if (in[i]) silu_mul8(v[i], u[i]);
    }
    float amax = kAmaxFloor;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[i][j]));
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    const float s = __fdiv_rn(amax, kE4m3Max);
    if (s < __int_as_float(0x7f800000)) {
      const float y = __frcp_rn(s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = quotient(v[i][j], s, y);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = __fdiv_rn(v[i][j], s);
    }
    if (in[i]) {
      *reinterpret_cast<uint2*>(q + at[i]) =
          make_uint2(pack4(v[i][0], v[i][1], v[i][2], v[i][3]), pack4(v[i][4], v[i][5], v[i][6], v[i][7]));
      if (lane == 0) scale[first + 16u * i] = s;
    }
  }
}

template <typename T, bool kSwiglu, int kUnroll>
void launch_blocks(void* q, void* scale, const void* x, int k, uint32_t kb, uint32_t blocks, cudaStream_t stream) {
  constexpr uint32_t kPerBlock = 16u * kUnroll;
  fp8_quantize_kernel<T, kSwiglu, kUnroll><<<(blocks + kPerBlock - 1) / kPerBlock, 256, 0, stream>>>(
      static_cast<uint8_t*>(q), static_cast<float*>(scale), static_cast<const T*>(x), k, kb, blocks, 16u / kb, 16u % kb);
}

template <typename T, bool kSwiglu>
void launch_quantize(void* q, void* scale, const void* x, int k, uint32_t kb, uint32_t blocks, int sms, cudaStream_t stream) {
  // several blocks of 128 per sixteen lanes once that still leaves every SM two thread blocks, else one
  constexpr int kUnroll = kSwiglu ? 1 : 2;
  if (blocks >= static_cast<uint32_t>(sms) * 2u * 16u * kUnroll)
    launch_blocks<T, kSwiglu, kUnroll>(q, scale, x, k, kb, blocks, stream);
  else
    launch_blocks<T, kSwiglu, 1>(q, scale, x, k, kb, blocks, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace b200

extern "C" int b200_nvfp4_fp8_quantize_rows(void* q, void* scale, const void* x, int rows, int k, int input_dtype, int swiglu,
                                            b200_stream_t stream) {
  using namespace b200;
  const long long kb = (static_cast<long long>(k) + 127) / 128;
  if (rows < 0 || k <= 0 || (k % 16) != 0 || q == nullptr || scale == nullptr || x == nullptr || !aligned16(q) ||
      !aligned16(x) || input_dtype < 0 || input_dtype > 2 || rows * kb > 0x7fffffffLL)
    return B200_NVFP4_INVALID_ARGUMENT;
  const DeviceInfo& dev = current_device_info();
  if (!dev.ok) return B200_NVFP4_CUDA_ERROR;
  if (!device_supported(dev)) return B200_NVFP4_UNSUPPORTED_DEVICE;
  if (rows == 0) return B200_NVFP4_SUCCESS;
  const uint32_t blocks = static_cast<uint32_t>(rows * kb);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t kbu = static_cast<uint32_t>(kb);
  switch (input_dtype * 2 + (swiglu != 0)) {
    case 0: launch_quantize<__half, false>(q, scale, x, k, kbu, blocks, dev.sm_count, s); break;
    case 1: launch_quantize<__half, true>(q, scale, x, k, kbu, blocks, dev.sm_count, s); break;
    case 2: launch_quantize<__nv_bfloat16, false>(q, scale, x, k, kbu, blocks, dev.sm_count, s); break;
    case 3: launch_quantize<__nv_bfloat16, true>(q, scale, x, k, kbu, blocks, dev.sm_count, s); break;
    case 4: launch_quantize<float, false>(q, scale, x, k, kbu, blocks, dev.sm_count, s); break;
    default: launch_quantize<float, true>(q, scale, x, k, kbu, blocks, dev.sm_count, s); break;
  }
  count_launch();
  return launch_status();
}
