// kv_cache_q8.cuh -- the 8-bit K/V cache format shared by the kernels that
// write and read it: e4m3 codes [num_blocks, block_size, n_kv_heads, head_dim]
// and one fp32 scale per (block, KV head); a value is code * scale.
#pragma once

#include <cuda_fp8.h>

#include "tvk_common.cuh"

namespace q8 {

constexpr int kMinScaleExp = -100;  // smallest scale 2^-100: also that of a block of zeros

// The smallest power of two 2^k, k >= kMinScaleExp, with amax <= 448 * 2^k
// (448 = 1.75 * 2^8 is e4m3's largest value); amax finite and >= 0.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t b = __float_as_uint(amax);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);  // subnormals: far below the floor
  e = e < kMinScaleExp ? kMinScaleExp : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Two fp32 values -> two e4m3 codes (low byte: a), nearest, ties to even.
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// Two e4m3 codes (16 bits) -> two halves; every code is a half exactly.
__device__ __forceinline__ uint32_t decode2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}

// Four codes -> four floats.
__device__ __forceinline__ void decode4(uint32_t codes, float* f) {
  const uint32_t lo = decode2(codes), hi = decode2(codes >> 16);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}

}  // namespace q8
