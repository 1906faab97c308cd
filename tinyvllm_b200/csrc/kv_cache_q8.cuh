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

// 8x8 transpose of 16-bit elements across a warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// c += a * b, halves in, fp32 sums: 16 x 8 x 16 and 16 x 8 x 8.
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0));
}

}  // namespace q8
