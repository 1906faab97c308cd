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

// Four e4m3 codes -> four halves (lo: codes 0 and 1); every code is a half exactly.
__device__ __forceinline__ void decode4h(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}

// Four codes -> four floats.
__device__ __forceinline__ void decode4(uint32_t codes, float* f) {
  uint32_t lo, hi;
  decode4h(codes, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}

// 3-D tiled TMA load into this CTA's shared memory, completion counted on `bar`.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2), "r"(ptx::smem_u32(bar))
      : "memory");
}

// Asynchronous 4-byte copy global -> shared; zeros when !live (src is not read then).
__device__ __forceinline__ void copy4_async(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
// One arrival on `bar` (counted at its initialisation) once this thread's copies so far have landed.
__device__ __forceinline__ void arrive_after_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ptx::smem_u32(bar)) : "memory");
}

// Two halves -> two e5m2 codes, nearest, ties to even.
__device__ __forceinline__ uint32_t encode2h_e5m2(uint32_t h) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.rn.satfinite.e5m2x2.f16x2 c, %1;\n\tcvt.u32.u16 %0, c;\n\t}" : "=r"(r) : "r"(h));
  return r;
}
__device__ __forceinline__ uint32_t sub2h(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

}  // namespace q8
