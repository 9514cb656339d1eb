// Device-side NVFP4 number formats and the dynamic quantiser.
//
// The quantiser follows the reference's act_mul_and_quant_nvfp4_kernel /
// quantize_expert_nvfp4_kernel (src/fused_moe/activation.cu:58-84,141-161): per 16 values,
// scale = UE4M3(amax / 6) with round-to-nearest-even and finite saturation, a non-zero block
// whose scale rounds to zero gets raw scale code 1, payload = E2M1(value / decoded scale).
// The two conversions are the same hardware cvt instructions the reference's device code
// reaches through cutlass::float_ue4m3_t and __nv_fp4x2_e2m1.
#pragma once

#include <cstdint>

#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace b200 {

__device__ __forceinline__ uint8_t ue4m3_encode(float x) {
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
}

// UE4M3 byte (0x00..0x7e) -> FP32, exact.
__device__ __forceinline__ float ue4m3_decode(uint8_t code) {
  const uint32_t c = code;
  if (c < 8u) return static_cast<float>(c) * 0.001953125f;  // subnormals: m * 2^-9
  return __uint_as_float((((c >> 3) + 120u) << 23) | ((c & 7u) << 20));
}

// Two FP32 values -> one byte of packed E2M1 (low nibble = first value), RNE, saturating.
__device__ __forceinline__ uint8_t e2m1x2_encode(float lo, float hi) {
  return static_cast<uint8_t>(__nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest));
}

// exp(x) from explicit fused multiply-adds only, so the bits do not depend on the compiler
// or on a math library: Cody-Waite reduction by ln 2, degree-7 polynomial, scaling by two
// exact powers of two. The CPU oracle evaluates the identical operation sequence. Error is
// below 2 ulp. (The reference calls CUDA's expf, activation.cu:17-19.)
__device__ __forceinline__ float nvfp4_expf(float x) {
  if (x > 88.75f) return __int_as_float(0x7f800000);
  if (x < -104.0f) return 0.0f;
  const float t = __fmul_rn(x, 1.44269504088896341f);
  const float n = rintf(t);
  float r = __fmaf_rn(n, -0.693145751953125f, x);
  r = __fmaf_rn(n, -1.428606765330187045e-06f, r);
  float p = 1.0f / 5040.0f;
  p = __fmaf_rn(p, r, 1.0f / 720.0f);
  p = __fmaf_rn(p, r, 1.0f / 120.0f);
  p = __fmaf_rn(p, r, 1.0f / 24.0f);
  p = __fmaf_rn(p, r, 1.0f / 6.0f);
  p = __fmaf_rn(p, r, 0.5f);
  p = __fmaf_rn(p, r, 1.0f);
  p = __fmaf_rn(p, r, 1.0f);
  const int ni = static_cast<int>(n);
  const int h1 = ni / 2;
  const int h2 = ni - h1;
  const float s1 = __uint_as_float(static_cast<uint32_t>(h1 + 127) << 23);
  const float s2 = __uint_as_float(static_cast<uint32_t>(h2 + 127) << 23);
  return __fmul_rn(__fmul_rn(p, s1), s2);
}

// x / (1 + exp(-x)), IEEE division (activation.cu:17-19).
__device__ __forceinline__ float nvfp4_silu(float x) {
  return __fdiv_rn(x, __fadd_rn(1.0f, nvfp4_expf(-x)));
}

// The same value for |x| <= 87 without nvfp4_expf's range checks (the argument cannot leave the
// range in which the two power-of-two factors are normal) and without a full division. The quotient
// is Markstein's (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", IBM J. Res. Dev. 34(1), 1990): with y = RN(1/d) and q0 = RN(x y), the remainder
// x - d q0 is exact in one fused multiply-add and q0 + remainder * y rounds to RN(x / d). Nothing
// over- or underflows on the way: the divisor lies in [1, 2^126] and the quotient is a normal
// number. Range checks are branches around every one of the sixteen values of a block, which
// serialise their dependency chains (measured: ~270 cycles per value in the GEMM epilogue);
// without them the chains overlap. Bit-identical to nvfp4_silu on every FP16 input in range
// (tested exhaustively).
__device__ __forceinline__ float nvfp4_silu_in_range(float x) {
  const float a = -x;
  const float t = __fmul_rn(a, 1.44269504088896341f);
  const float n = rintf(t);
  float r = __fmaf_rn(n, -0.693145751953125f, a);
  r = __fmaf_rn(n, -1.428606765330187045e-06f, r);
  float p = 1.0f / 5040.0f;
  p = __fmaf_rn(p, r, 1.0f / 720.0f);
  p = __fmaf_rn(p, r, 1.0f / 120.0f);
  p = __fmaf_rn(p, r, 1.0f / 24.0f);
  p = __fmaf_rn(p, r, 1.0f / 6.0f);
  p = __fmaf_rn(p, r, 0.5f);
  p = __fmaf_rn(p, r, 1.0f);
  p = __fmaf_rn(p, r, 1.0f);
  const int ni = static_cast<int>(n);
  const int h1 = ni / 2;
  const int h2 = ni - h1;
  const float s1 = __uint_as_float(static_cast<uint32_t>(h1 + 127) << 23);
  const float s2 = __uint_as_float(static_cast<uint32_t>(h2 + 127) << 23);
  const float d = __fadd_rn(1.0f, __fmul_rn(__fmul_rn(p, s1), s2));
  const float y = __frcp_rn(d);
  const float q0 = __fmul_rn(x, y);
  const float q = __fmaf_rn(__fmaf_rn(-d, q0, x), y, q0);
  // x = -0: the zero remainder would turn the quotient into +0; silu(x) always has the sign of x
  return __uint_as_float((__float_as_uint(q) & 0x7fffffffu) | (__float_as_uint(x) & 0x80000000u));
}

constexpr float kSiluInRangeLimit = 87.0f;

// v[i] = silu(g[i]) * u[i] for one block of 16: the branch-free form, and the plain one for a
// block that holds a gate value outside its range (or an infinity).
__device__ __forceinline__ void silu_mul_block16(const float (&g)[16], const float (&u)[16], float (&v)[16]) {
  float gmax = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    gmax = fmaxf(gmax, fabsf(g[i]));
    v[i] = __fmul_rn(nvfp4_silu_in_range(g[i]), u[i]);
  }
  if (gmax > kSiluInRangeLimit) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __fmul_rn(nvfp4_silu(g[i]), u[i]);
  }
}

// Quantises 16 FP32 values: returns the UE4M3 scale code, writes 8 payload bytes as two
// 32-bit words (little endian, low nibble = even element).
//
// payload = E2M1(RN(value / decoded scale)), the quotient being the IEEE-rounded FP32 division the
// reference performs (activation.cu:77-83). Sixteen divisions by the same divisor are computed
// from one correctly rounded reciprocal r = RN(1 / d): q0 = RN(v r), rem = v - q0 d (exact, one
// FMA), q = RN(q0 + rem r). For a divisor with a 4-bit significand - every decoded UE4M3 scale -
// and quotients in the range E2M1 distinguishes this is the correctly rounded quotient (the
// classical FMA division step; checked exhaustively around all rounding boundaries for all 126
// scales), at 3 instructions per value instead of a division's dozen. A block that contains an
// infinity (amax = inf) takes the plain divisions: inf - inf in the remainder would turn a signed
// infinity into a NaN.
__device__ __forceinline__ uint8_t quantize_block16(const float (&v)[16], uint32_t& lo, uint32_t& hi) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[i]));
  uint8_t code = 0;
  float decoded = 1.0f;
  if (amax > 0.0f) {
    code = ue4m3_encode(__fdiv_rn(amax, 6.0f));
    decoded = ue4m3_decode(code);
    if (!(decoded > 0.0f)) {
      code = 1;
      decoded = 0.001953125f;
    }
  }
  uint32_t w[2] = {0u, 0u};
  if (amax < __int_as_float(0x7f800000)) {
    const float r = __frcp_rn(decoded);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q0 = __fmul_rn(v[2 * i], r);
      float q1 = __fmul_rn(v[2 * i + 1], r);
      q0 = __fmaf_rn(__fmaf_rn(-q0, decoded, v[2 * i]), r, q0);
      q1 = __fmaf_rn(__fmaf_rn(-q1, decoded, v[2 * i + 1]), r, q1);
      // a zero remainder added to a negative zero would give +0: the quotient keeps the dividend's sign
      q0 = __uint_as_float((__float_as_uint(q0) & 0x7fffffffu) | (__float_as_uint(v[2 * i]) & 0x80000000u));
      q1 = __uint_as_float((__float_as_uint(q1) & 0x7fffffffu) | (__float_as_uint(v[2 * i + 1]) & 0x80000000u));
      w[i >> 2] |= static_cast<uint32_t>(e2m1x2_encode(q0, q1)) << (8 * (i & 3));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = e2m1x2_encode(__fdiv_rn(v[2 * i], decoded), __fdiv_rn(v[2 * i + 1], decoded));
      w[i >> 2] |= b << (8 * (i & 3));
    }
  }
  lo = w[0];
  hi = w[1];
  return code;
}

// Byte offset of the scale of (row, k_block) inside one scale region whose K extent spans
// `kt` atoms (kt = ceil(K / 64)); the closed form of the layout the reference addresses
// through Sm1xxBlockScaledConfig<16> (src/fused_moe/scale_layout.cuh:33-41).
__host__ __device__ __forceinline__ long long sf_offset(int row, int k_block, int kt) {
  return (static_cast<long long>(row >> 7) * kt + (k_block >> 2)) * 512 + (row & 31) * 16 +
         ((row & 127) >> 5) * 4 + (k_block & 3);
}

}  // namespace b200
