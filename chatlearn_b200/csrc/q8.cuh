// Device helpers of the 8-bit key/value cache: e4m3 codes, power-of-two scales.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace q8 {

constexpr float kCodeMax = 448.f;                 // largest e4m3 value

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two codes, the first in the low byte; rounds to nearest even, magnitudes above 448 saturate, NaN stays NaN
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// four codes as two pairs of halves (exact: e4m3 is a subset of fp16)
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(codes));
}

// four codes as fp32
__device__ __forceinline__ void unpack_e4m3(uint32_t codes, float* f) {
  uint32_t h[2];
  e4m3x4_to_half2(codes, h[0], h[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// smallest power of two s in [2^-24, 2^64] with amax <= 448 s.  448 = 1.75 * 2^8: with amax = m * 2^x, 1 <= m < 2, the
// exponent is x - 8 where m <= 1.75 and x - 7 above (magnitudes above 448 * 2^64 saturate).
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, -24), 64);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

}  // namespace q8
