// kv_write_q8.cu -- K/V rows -> paged slots of the 8-bit cache.
//
// For every (block b, KV head h) that a row of the call lands in, K and V apart:
//   started = the call writes the block's row 0: what the block held is dropped
//   old     = started ? 0 : scale[b, h]   (what is not positive and finite counts as 0)
//   now     = max(old, 2^k), k >= -100 the smallest with amax <= 448 * 2^k over
//             the finite values of the call's rows in (b, h)
//   rows of the call: e4m3(x / now), what is not finite as NaN
//   the other rows:   e4m3(code * (old / now)), zeros in a started block
// Scales being powers of two, x / now is exact and a growing scale only moves
// the exponents of the codes already there; they lose nothing until they reach
// e4m3's subnormals.  A call's last row for a slot wins, the others do not count.
//
// One CTA per token finds out whether its token is the first of the call in its
// block (by reading all slots) and if so does the whole block, one warp per (K
// or V, head), so no two CTAs write one block and nothing depends on their order.
#include "kv_cache_q8.cuh"

namespace {

constexpr int kWriteThreads = 256;
constexpr int kMaxBlockSize = 1024;

struct WriteParams {
  const void *k, *v;           // [n_tokens, n_kv_heads, head_dim]
  uint8_t *k_cache, *v_cache;  // codes
  float *k_scale, *v_scale;    // [num_blocks, n_kv_heads]
  const int64_t* slots;  // [n_tokens]
  int n_tokens, n_kv_heads, head_dim, block_size;
  long long n_slots;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x;
    f[1] = a.y;
    f[2] = a.z;
    f[3] = a.w;
    f[4] = b.x;
    f[5] = b.y;
    f[6] = b.z;
    f[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = DT<T>::to_f(h[i]);
  }
}

__device__ __forceinline__ uint2 encode8(const float* f) {
  uint2 c;
  c.x = q8::encode2(f[0], f[1]) | (q8::encode2(f[2], f[3]) << 16);
  c.y = q8::encode2(f[4], f[5]) | (q8::encode2(f[6], f[7]) << 16);
  return c;
}

template <typename T>
__global__ void __launch_bounds__(kWriteThreads) write_kv_q8_kernel(const WriteParams p) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int row_of[kMaxBlockSize];  // last token of the call for each slot of the block, or -1
  __shared__ int first;
  const int t = blockIdx.x, tid = threadIdx.x, bs = p.block_size;
  const long long slot = p.slots[t];
  if (slot < 0 || slot >= p.n_slots) return;
  const long long blk = slot / bs, base = blk * bs;
  if (t > 0) {  // the token before it is in the same block: not the first
    const long long d = p.slots[t - 1] - base;
    if (d >= 0 && d < bs) return;
  }
  for (int i = tid; i < bs; i += kWriteThreads) row_of[i] = -1;
  if (tid == 0) first = t;
  __syncthreads();
  for (int i = tid; i < p.n_tokens; i += kWriteThreads) {
    const long long d = p.slots[i] - base;
    if (d >= 0 && d < bs) {
      atomicMax(&row_of[d], i);
      if (i < t) atomicMin(&first, i);
    }
  }
  __syncthreads();
  if (first != t) return;

  const int warp = tid >> 5, lane = tid & 31;
  const int D8 = p.head_dim / 8, H = p.n_kv_heads;
  const bool started = row_of[0] >= 0;
  for (int pair = blockIdx.y * (kWriteThreads / 32) + warp; pair < 2 * H; pair += gridDim.y * (kWriteThreads / 32)) {
    const int kv = pair & 1, h = pair >> 1;
    const T* x = reinterpret_cast<const T*>(kv ? p.v : p.k) + (size_t)h * p.head_dim;
    uint8_t* codes = (kv ? p.v_cache : p.k_cache) + ((size_t)base * H + h) * p.head_dim;
    float* sp = (kv ? p.v_scale : p.k_scale) + (size_t)blk * H + h;
    float old = started ? 0.f : *sp;
    if (!(old > 0.f && old < INFINITY)) old = 0.f;

    float amax = 0.f;
    for (int i = lane; i < bs * D8; i += 32) {
      const int o = i / D8, c = i - o * D8;
      const int r = row_of[o];
      if (r < 0) continue;
      float f[8];
      load8<T>(x + (size_t)r * H * p.head_dim + c * 8, f);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (isfinite(f[e])) amax = fmaxf(amax, fabsf(f[e]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float now = fmaxf(old, q8::scale_for(amax));
    const float ratio = __fdiv_rn(old, now);
    __syncwarp();  // every lane has read the old scale
    if (lane == 0) *sp = now;
    for (int i = lane; i < bs * D8; i += 32) {
      const int o = i / D8, c = i - o * D8;
      const int r = row_of[o];
      uint2* dst = reinterpret_cast<uint2*>(codes + (size_t)o * H * p.head_dim + c * 8);
      float f[8];
      if (r >= 0) {
        load8<T>(x + (size_t)r * H * p.head_dim + c * 8, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = isfinite(f[e]) ? __fdiv_rn(f[e], now) : __int_as_float(0x7fffffff);
        *dst = encode8(f);
      } else if (started) {
        *dst = make_uint2(0u, 0u);
      } else if (now != old) {
        const uint2 u = *dst;
        q8::decode4(u.x, f);
        q8::decode4(u.y, f + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= ratio;
        *dst = encode8(f);
      }
    }
  }
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

extern "C" int tvk_write_kv_slots_q8(const void* k, const void* v, const int64_t* slots, void* k_cache, void* v_cache,
                                     float* k_scale, float* v_scale, int n_tokens, int n_kv_heads, int head_dim,
                                     int num_blocks, int block_size, int dtype, void* stream) {
  TVK_CHECK_ARG(n_tokens >= 0, "negative n_tokens");
  TVK_CHECK_ARG(n_kv_heads > 0 && num_blocks > 0 && block_size > 0, "sizes must be positive");
  TVK_CHECK_ARG(head_dim > 0 && head_dim % 16 == 0, "head_dim must be a multiple of 16 (got %d)", head_dim);
  TVK_CHECK_ARG((long long)block_size * head_dim < 0x7fffffffLL && (long long)n_kv_heads * head_dim < 0x7fffffffLL,
                "a block's rows exceed the 32-bit index");
  TVK_CHECK_ARG(dtype == TVK_DTYPE_F32 || dtype == TVK_DTYPE_F16 || dtype == TVK_DTYPE_BF16, "unknown dtype %d", dtype);
  if (block_size > kMaxBlockSize) {
    tvk::set_error("block_size %d unsupported (at most %d)", block_size, kMaxBlockSize);
    return TVK_ERR_UNSUPPORTED;
  }
  if (n_tokens == 0) return TVK_OK;
  TVK_CHECK_ARG(k && v && slots && k_cache && v_cache && k_scale && v_scale, "null pointer argument");
  TVK_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(k_cache) && aligned16(v_cache),
                "k, v, k_cache and v_cache must be 16-byte aligned");
  const WriteParams p{k, v, (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, slots, n_tokens, n_kv_heads,
                      head_dim, block_size, (long long)num_blocks * block_size};
  const dim3 grid(n_tokens, 1);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TVK_DTYPE_F16: TVK_CHECK_CUDA(tvk::launch_pdl(write_kv_q8_kernel<__half>, grid, kWriteThreads, 0, s, p)); break;
    case TVK_DTYPE_BF16:
      TVK_CHECK_CUDA(tvk::launch_pdl(write_kv_q8_kernel<__nv_bfloat16>, grid, kWriteThreads, 0, s, p));
      break;
    default: TVK_CHECK_CUDA(tvk::launch_pdl(write_kv_q8_kernel<float>, grid, kWriteThreads, 0, s, p)); break;
  }
  TVK_CHECK_LAUNCH("write_kv_q8");
  return TVK_OK;
}
