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
// A CTA looks after a few neighbouring tokens.  For each that might be the first of
// the call in its block (the token before it lies in another) it reads all slots, which
// says whether it is and which rows the block gets, and if so does the whole block,
// one warp per (K or V, head).  So no two CTAs write one block and nothing depends on
// their order, whatever the slots are; with prompts' runs of slots there is one
// such token per block.  Reading all slots per block costs T^2 / block_size reads from L2: at 8,192
// tokens about a third of the call (33 us for 50 MB of rows and codes), and what bounds calls of
// more than some 30,000 rows.  Few tokens are latency: slot, other slots, rows, store, one
// behind the other (64 rows of 4 heads of 64: 4.7 us, 256 of 8 of 128: 6.5 us).
#include "kv_cache_q8.cuh"

namespace {

constexpr int kWriteThreads = 256;
constexpr int kMaxBlockSize = 1024;
constexpr int kFewTokens = 1024, kChunk = 16;  // tokens per CTA: one up to kFewTokens, else kChunk

struct WriteParams {
  const void *k, *v;           // [n_tokens, n_kv_heads, head_dim]
  uint8_t *k_cache, *v_cache;  // codes
  float *k_scale, *v_scale;    // [num_blocks, n_kv_heads]
  const int64_t* slots;  // [n_tokens]
  int n_tokens, n_kv_heads, head_dim, block_size;
  int chunk;  // tokens a CTA looks after
  long long n_slots;
};

// Eight elements as they lie in memory, and as floats.
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void to_floats(const Raw8<T>& r, float* f) {
  const T* h = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = DT<T>::to_f(h[i]);
}

__device__ __forceinline__ uint2 encode8(const float* f) {
  uint2 c;
  c.x = q8::encode2(f[0], f[1]) | (q8::encode2(f[2], f[3]) << 16);
  c.y = q8::encode2(f[4], f[5]) | (q8::encode2(f[6], f[7]) << 16);
  return c;
}

// Rows of D8 groups of 8 elements, walked 32 groups at a time by a warp.
struct Walk8 {
  int row, c, drow, dc, D8;
  __device__ Walk8(int lane, int D8_) : row(lane / D8_), c(lane % D8_), drow(32 / D8_), dc(32 % D8_), D8(D8_) {}
  __device__ void next() {
    row += drow;
    c += dc;
    if (c >= D8) {
      c -= D8;
      ++row;
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kWriteThreads, 4) write_kv_q8_kernel(const WriteParams p) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int row_of[kMaxBlockSize];   // last token of the call for each slot of the block, or -1
  __shared__ int2 rows[kMaxBlockSize];    // (slot in the block, token) of those there are
  __shared__ int first, n_rows, cands[kChunk], n_cands;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bs = p.block_size;
  const int D = p.head_dim, D8 = D / 8, H = p.n_kv_heads;
  const size_t row_elems = (size_t)H * D;
  if (tid < 32) {
    // the chunk's tokens that the token before them does not share the block with
    const int t = blockIdx.x * p.chunk + lane;
    bool cand = false;
    if (lane < p.chunk && t < p.n_tokens) {
      const long long slot = p.slots[t], before = t > 0 ? p.slots[t - 1] : -1;
      cand = slot >= 0 && slot < p.n_slots && (before < 0 || before / bs != slot / bs);
    }
    const unsigned m = __ballot_sync(0xffffffffu, cand);
    if (cand) cands[__popc(m & ((1u << lane) - 1u))] = t;
    if (lane == 0) n_cands = __popc(m);
  }
  __syncthreads();
  for (int ci = 0; ci < n_cands; ++ci) {
    const int t = cands[ci];
    const long long blk = p.slots[t] / bs, base = blk * bs;
    __syncthreads();  // the block before is done with
    for (int i = tid; i < bs; i += kWriteThreads) row_of[i] = -1;
    if (tid == 0) {
      first = t;
      n_rows = 0;
    }
    __syncthreads();
    auto look = [&](long long slot, int i) {
      const unsigned long long d = (unsigned long long)slot - (unsigned long long)base;
      if (d < (unsigned long long)bs) {
        atomicMax(&row_of[d], i);
        if (i < t) atomicMin(&first, i);
      }
    };
    // two slots a load where they are aligned (an odd last one apart)
    const int pairs = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0 ? p.n_tokens / 2 : 0;
#pragma unroll 8
    for (int i = tid; i < pairs; i += kWriteThreads) {
      const longlong2 two = reinterpret_cast<const longlong2*>(p.slots)[i];
      look(two.x, 2 * i);
      look(two.y, 2 * i + 1);
    }
    for (int i = 2 * pairs + tid; i < p.n_tokens; i += kWriteThreads) look(p.slots[i], i);
    __syncthreads();
    if (first != t) continue;  // the same for all threads
    for (int i = tid; i < bs; i += kWriteThreads)
      if (row_of[i] >= 0) rows[atomicAdd(&n_rows, 1)] = make_int2(i, row_of[i]);
    __syncthreads();

    const int n = n_rows;
    const bool started = row_of[0] >= 0;
    for (int pair = blockIdx.y * (kWriteThreads / 32) + warp; pair < 2 * H; pair += gridDim.y * (kWriteThreads / 32)) {
      const int kv = pair & 1, h = pair >> 1;
      const T* x = reinterpret_cast<const T*>(kv ? p.v : p.k) + (size_t)h * D;
      uint8_t* codes = (kv ? p.v_cache : p.k_cache) + (size_t)base * row_elems + (size_t)h * D;
      float* sp = (kv ? p.v_scale : p.k_scale) + (size_t)blk * H + h;
      float old = started ? 0.f : *sp;
      if (!(old > 0.f && old < INFINITY)) old = 0.f;

      // Both passes read the rows; the second finds them in L1.
      constexpr int kInFlight = 2;  // loads: more would cost the fourth CTA on an SM, which is worth more
      auto for_rows = [&](auto&& use) {
        Walk8 w(lane, D8);
        while (w.row < n) {
          Raw8<T> r[kInFlight];
          int2 at[kInFlight];  // slot in the block (-1: none), group of 8
#pragma unroll
          for (int k = 0; k < kInFlight; ++k) {
            at[k].x = -1;
            if (w.row < n) {
              const int2 row = rows[w.row];
              at[k] = make_int2(row.x, w.c);
              r[k] = load8<T>(x + (size_t)row.y * row_elems + w.c * 8);
            }
            w.next();
          }
#pragma unroll
          for (int k = 0; k < kInFlight; ++k)
            if (at[k].x >= 0) use(r[k], at[k].x, at[k].y);
        }
      };
      float amax = 0.f;
      for_rows([&](const Raw8<T>& r, int, int) {
        float f[8];
        to_floats<T>(r, f);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (isfinite(f[e])) amax = fmaxf(amax, fabsf(f[e]));
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const float now = fmaxf(old, q8::scale_for(amax));
      // Dividing by a power of two is multiplying by its reciprocal; other scales come from the caller only.
      const uint32_t bits = __float_as_uint(now);
      const bool pow2 = (bits & 0x7fffffu) == 0u && bits >= 0x00800000u && bits <= 0x7e800000u;
      const float inv = pow2 ? __uint_as_float(0x7f000000u - bits) : 0.f;
      __syncwarp();  // every lane has read the old scale
      if (lane == 0) *sp = now;

      for_rows([&](const Raw8<T>& r, int slot_in, int c) {
        float f[8];
        to_floats<T>(r, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = pow2 ? f[e] * inv : __fdiv_rn(f[e], now);
          f[e] = isfinite(f[e]) ? y : __int_as_float(0x7fffffff);
        }
        *reinterpret_cast<uint2*>(codes + (size_t)slot_in * row_elems + c * 8) = encode8(f);
      });

      if (n < bs && (started || now != old)) {  // the block's other rows
        const float ratio = __fdiv_rn(old, now);
        Walk8 o(lane, D8);
        while (o.row < bs) {
          uint2 u[4];
          uint2* dst[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool other = o.row < bs && row_of[min(o.row, bs - 1)] < 0;
            dst[k] = other ? reinterpret_cast<uint2*>(codes + (size_t)o.row * row_elems + o.c * 8) : nullptr;
            u[k] = other && !started ? *dst[k] : make_uint2(0u, 0u);
            o.next();
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (!dst[k]) continue;
            float f[8];
            q8::decode4(u[k].x, f);
            q8::decode4(u[k].y, f + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= ratio;
            *dst[k] = started ? make_uint2(0u, 0u) : encode8(f);
          }
        }
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
  TVK_CHECK_ARG(head_dim <= 65536 && n_kv_heads <= 65536, "head_dim and n_kv_heads must be at most 65536");
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
                      head_dim, block_size, n_tokens > kFewTokens ? kChunk : 1, (long long)num_blocks * block_size};
  // a warp per (K or V, head)
  const dim3 grid((n_tokens + p.chunk - 1) / p.chunk, (2 * n_kv_heads + kWriteThreads / 32 - 1) / (kWriteThreads / 32));
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
