// Row quantiser to E4M3 with one FP32 scale per 128 values, optionally with SiLU(gate) * up in front.
//
//   amax_b = max(|x|) over the 128 values of a block, at least 2^-60
//   s_b = RN(amax_b / 448),  q = E4M3(RN(x / s_b))
//
// Reads 2 bytes (4 with SiLU) and writes 1.03 per value of a 16-bit input. Eight (or sixteen) lanes share a
// block: 16-byte loads, an amax by three (four) exchanges, one 16-byte (8-byte) store. 32768 x 4096 BF16:
// 69 us, 0.90 of what the bytes take at the measured copy rate. 32768 x 2048 with SiLU: 66 to 69 us in bursts of some
// hundred calls, 0.75 to 0.78 of it, and 73 to 77, 0.67 to 0.70, in runs of a second: 25
// instructions per value, half of them the exponential and the division of the SiLU, at 76 % of the issue
// slots, and the wait for the loads. (Both 2 us more without the overlapped start.)
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
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 8.67361737988403547e-19f;   // 2^-60

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 1 / x to one unit in the last place, x normal.
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// N consecutive values (a multiple of 8 for 16-bit types, of 4 for FP32) in 16-byte loads.
template <int N>
__device__ __forceinline__ void load(const __half* p, float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    const uint4 w = reinterpret_cast<const uint4*>(p)[c];
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
      v[8 * c + 2 * i] = f.x;
      v[8 * c + 2 * i + 1] = f.y;
    }
  }
}

template <int N>
__device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    const uint4 w = reinterpret_cast<const uint4*>(p)[c];
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[8 * c + 2 * i] = __uint_as_float(a[i] << 16);
      v[8 * c + 2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  }
}

template <int N>
__device__ __forceinline__ void load(const float* p, float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N / 4; ++c) {
    const float4 a = reinterpret_cast<const float4*>(p)[c];
    v[4 * c] = a.x; v[4 * c + 1] = a.y; v[4 * c + 2] = a.z; v[4 * c + 3] = a.w;
  }
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Two FP32 operations in one instruction (each lane rounds as the scalar one would).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// v -> -(v / s) for N values whose divisor has the correctly rounded reciprocal y: Markstein's sequence (see
// above). Computed with its sign turned round because then a quotient of -0 stays a zero of the right
// sign; the caller turns the codes' signs back.
template <int N>
__device__ __forceinline__ void minus_quotients(float (&v)[N], float s, float y) {
  const uint64_t s2 = pack2(s, s), y2 = pack2(-y, -y);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const uint64_t x = pack2(v[j], v[j + 1]);
    const uint64_t q0 = mul2(x, y2);
    unpack2(fma2(fma2(q0, s2, x), y2, q0), v[j], v[j + 1]);
  }
}

// silu(g) * u = g / (1 + e^-g) * u. The quotient is Markstein's sequence again, here on the reciprocal
// instruction, which is one unit off at most: its proof leaves the correction 2^-21 of a unit of the quotient off, enough
// to round the other way next to a midpoint. No gate is there: over all 2237399042 FP32 values of g in [-87, 87] the
// result is the IEEE division's to the bit (on B200), so a value does not depend on which of the two ways its
// thread takes. (With the rounded reciprocal 80 us instead of 72.) It is computed with its sign turned
// round for the sake of zeros, as above, and -u turns it back. Gates beyond 87, whose divisor or remainder could
// leave the range, send the thread's values through IEEE divisions (the divisor is below 2^126 otherwise).
template <int N>
__device__ __forceinline__ void silu_mul(float (&v)[N], const float (&u)[N]) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(v[j]));
  if (top <= 87.0f) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = 1.0f + expf(-v[j]);
      const float y = -reciprocal(d);
      const float q0 = __fmul_rn(v[j], y);
      v[j] = __fmul_rn(__fmaf_rn(__fmaf_rn(q0, d, v[j]), y, q0), -u[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = __fmul_rn(__fdiv_rn(v[j], __fadd_rn(1.0f, expf(-v[j]))), u[j]);
  }
}

// Five blocks per SM, 48 registers, for 16-bit types: 32768 x 2048 with SiLU 71.8 -> 67.6 us; FP32 does better with
// the registers it wants (16384 x 2048 with SiLU 46.3, 49.4 held to 48).
// kPer values per thread: 128 / kPer lanes share a block of 128. `step_rows`, `step_cols`: how far the next of a
// thread's kUnroll blocks is, in rows and blocks (the blocks a thread block handles at a time / kb, % kb).
template <typename T, bool kSwiglu, int kPer, int kUnroll>
__global__ void __launch_bounds__(256, kPer == 16 ? 5 : 0)
fp8_quantize_kernel(uint8_t* q, float* scale, const T* x, int k, uint32_t kb,
                    uint32_t blocks, uint32_t step_rows, uint32_t step_cols) {
  constexpr int kLanes = 128 / kPer;
  constexpr uint32_t kAtOnce = 256 / kLanes;
  ptx::grid_wait();
  ptx::grid_launch_dependents();
  const int lane = threadIdx.x & (kLanes - 1);
  const uint32_t first = blockIdx.x * (kAtOnce * kUnroll) + threadIdx.x / kLanes;
  float v[kUnroll][kPer];
  [[maybe_unused]] float u[kSwiglu ? kUnroll : 1][kPer];
  long long at[kUnroll];
  bool in[kUnroll];
  uint32_t row = first / kb, col_block = first - row * kb;
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int col = static_cast<int>(col_block) * 128 + lane * kPer;
    in[i] = first + kAtOnce * i < blocks && col < k;
    at[i] = static_cast<long long>(row) * k + col;
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[i][j] = 0.0f;
    if (in[i]) {
      if constexpr (kSwiglu) {
        const T* src = x + at[i] + static_cast<long long>(row) * k;     // rows of 2 k: gate, then up
        load(src, v[i]);
        load(src + k, u[i]);
      } else {
        load(x + at[i], v[i]);
      }
    }
    row += step_rows;
    col_block += step_cols;
    if (col_block >= kb) { col_block -= kb; ++row; }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if constexpr (kSwiglu) {
      if (in[i]) silu_mul(v[i], u[i]);
    }
    float amax = kAmaxFloor;
#pragma unroll
    for (int j = 0; j < kPer; ++j) amax = max_nan(amax, fabsf(v[i][j]));
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    const float s = __fdiv_rn(amax, kE4m3Max);
    if (s < __int_as_float(0x7f800000)) {
      const float y = __frcp_rn(s);
      minus_quotients(v[i], s, y);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i][j] = -__fdiv_rn(v[i][j], s);
    }
    if (in[i]) {
      uint32_t w[kPer / 4];
#pragma unroll
      for (int j = 0; j < kPer / 4; ++j) w[j] = pack4(v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3]) ^ 0x80808080u;
      if constexpr (kPer == 16) *reinterpret_cast<uint4*>(q + at[i]) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(q + at[i]) = make_uint2(w[0], w[1]);
      if (lane == 0) scale[first + kAtOnce * i] = s;
    }
  }
}

template <typename T, bool kSwiglu, int kPer, int kUnroll>
int launch_blocks(void* q, void* scale, const void* x, int k, uint32_t kb, uint32_t blocks, cudaStream_t stream) {
  constexpr uint32_t kAtOnce = 256u * kPer / 128u, kPerBlock = kAtOnce * kUnroll;
  return launch_overlapped(fp8_quantize_kernel<T, kSwiglu, kPer, kUnroll>, (blocks + kPerBlock - 1) / kPerBlock, 256, 0, 1, stream,
                           static_cast<uint8_t*>(q), static_cast<float*>(scale), static_cast<const T*>(x), k, kb, blocks, kAtOnce / kb,
                           kAtOnce % kb);
}

template <typename T, bool kSwiglu>
int launch_quantize(void* q, void* scale, const void* x, int k, uint32_t kb, uint32_t blocks, int sms, cudaStream_t stream) {
  // Sixteen values per thread halve what a block costs beside its values (index, exchanges, scale); eight
  // where that leaves SMs idle, and for FP32, whose loads would be strided further apart (16384 x 4096: 53.4
  // us with sixteen and one block, 51.3 with eight and two). More blocks per thread cost more
  // occupancy than their overlapped loads bring: 32768 x 4096 BF16 74 us with one, 86 with two; with SiLU
  // 32768 x 2048 88 and 109 (both before later steps).
  constexpr int kPer = sizeof(T) == 2 ? 16 : 8;
  constexpr int kUnroll = sizeof(T) == 4 && !kSwiglu ? 2 : 1;
  if (blocks >= static_cast<uint32_t>(sms) * 2u * 2u * kPer * kUnroll)
    return launch_blocks<T, kSwiglu, kPer, kUnroll>(q, scale, x, k, kb, blocks, stream);
  return launch_blocks<T, kSwiglu, 8, 1>(q, scale, x, k, kb, blocks, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace b200

extern "C" int b200_nvfp4_fp8_quantize_rows(void* q, void* scale, const void* x, int rows, int k, int input_dtype, int swiglu,
                                            b200_stream_t stream) {
  using namespace b200;
  const long long kb = (static_cast<long long>(k) + 127) / 128;
  if (rows < 0 || k <= 0 || k > 0x7fffff00 || (k % 16) != 0 || q == nullptr || scale == nullptr || x == nullptr || !aligned16(q) ||
      !aligned16(x) || (reinterpret_cast<uintptr_t>(scale) & 3u) != 0 || input_dtype < 0 || input_dtype > 2 || rows * kb > 0x7fffffffLL)
    return B200_NVFP4_INVALID_ARGUMENT;
  const DeviceInfo& dev = current_device_info();
  if (!dev.ok) return B200_NVFP4_CUDA_ERROR;
  if (!device_supported(dev)) return B200_NVFP4_UNSUPPORTED_DEVICE;
  if (rows == 0) return B200_NVFP4_SUCCESS;
  const uint32_t blocks = static_cast<uint32_t>(rows * kb);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t kbu = static_cast<uint32_t>(kb);
  switch (input_dtype * 2 + (swiglu != 0)) {
    case 0: return launch_quantize<__half, false>(q, scale, x, k, kbu, blocks, dev.sm_count, s);
    case 1: return launch_quantize<__half, true>(q, scale, x, k, kbu, blocks, dev.sm_count, s);
    case 2: return launch_quantize<__nv_bfloat16, false>(q, scale, x, k, kbu, blocks, dev.sm_count, s);
    case 3: return launch_quantize<__nv_bfloat16, true>(q, scale, x, k, kbu, blocks, dev.sm_count, s);
    case 4: return launch_quantize<float, false>(q, scale, x, k, kbu, blocks, dev.sm_count, s);
    default: return launch_quantize<float, true>(q, scale, x, k, kbu, blocks, dev.sm_count, s);
  }
}
