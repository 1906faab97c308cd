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
// such token per block.  A warp copies a block's rows to shared memory, all at once in flight, and
// takes the maximum and the codes from there (from registers, two loads at a time and again
// for the codes, 8,192 rows of 8 x 128 took 33 us instead of 22).
//
// Reading all slots per block costs T^2 / block_size reads from L2: at 8,192 tokens 4 of the 22 us (50 MB of
// rows and codes, 2.3 TB/s).  Longer calls make a pass over the slots first that notes, for every 32 tokens, which
// of 64 classes of blocks they write, and read only the slots of groups that may hold a block's
// (8 x 128 fp16: 8,192 rows take 18.8 us either way, 4,096 17.1 instead of 15.4, 16,384 33 instead of 35, 131,072 259
// instead of 538; smallest and largest block per group instead of classes: 821, blocks being anywhere in a pool).
// The rest is issue slots (0.6 of them taken) and the barriers between a block's steps.  A CTA per token
// up to 1,024 tokens, where the chain of loads counts (slot, other slots, rows, store, one behind
// the other: 64 rows of 4 heads of 64 4.2 us, 256 of 8 of 128 5.9 us); beyond, 8 tokens a CTA
// and two (K or V, head) a warp, which halves the reads of slots: 22.3 us, 16 tokens and one 23.9.
#include <type_traits>

#include "kv_cache_q8.cuh"

namespace {

constexpr int kWriteThreads = 256, kWriteCtas = 4;
constexpr int kReadAll = 8192;  // beyond so many tokens a block's rows are looked for by classes of blocks
constexpr int kStage = 256;  // 16-byte vectors of rows that a warp holds in shared memory
constexpr int kMaxBlockSize = 1024;
constexpr int kFewTokens = 1024, kChunk = 8;  // tokens per CTA: one up to kFewTokens, else kChunk

struct WriteParams {
  const void *k, *v;           // [n_tokens, n_kv_heads, head_dim]
  uint8_t *k_cache, *v_cache;  // codes
  float *k_scale, *v_scale;    // [num_blocks, n_kv_heads]
  const int64_t* slots;  // [n_tokens]
  int n_tokens, n_kv_heads, head_dim, block_size;
  int chunk;  // tokens a CTA looks after
  const uint2* classes;  // classes of the blocks of every 32 tokens, or null
  long long n_slots;
};

// Eight elements as floats.
template <typename T>
__device__ __forceinline__ void to_floats(const uint4* u, float* f) {
  uint4 r[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = u[i];
  const T* h = reinterpret_cast<const T*>(r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = DT<T>::to_f(h[i]);
}

// Largest magnitude of the finite ones of eight elements and m.  |x| + 0 |x| is NaN where x is not
// finite, and the maximum passes over NaN.
template <typename T>
__device__ __forceinline__ float amax8(const uint4* u, float m) {
  if constexpr (sizeof(T) == 4) {
    float f[8];
    to_floats<T>(u, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaf(fabsf(f[e]), 0.f, fabsf(f[e])));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint4 r = *u;
    const T2* h = reinterpret_cast<const T2*>(&r);
    T2 zero, best;
    zero.x = zero.y = DT<T>::from_f(0.f);
    best = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T2 x = __habs2(h[i]);
      best = __hmax2(best, __hfma2(x, zero, x));
    }
    return fmaxf(m, fmaxf(DT<T>::to_f(best.x), DT<T>::to_f(best.y)));
  }
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
  __device__ Walk8(int at, int D8_) : row(at / D8_), c(at % D8_), drow(32 / D8_), dc(32 % D8_), D8(D8_) {}
  __device__ void next() {
    row += drow;
    c += dc;
    if (c >= D8) {
      c -= D8;
      ++row;
    }
  }
};

// One of 64 classes of blocks.
__device__ __forceinline__ int class_of(int blk) { return (int)(((uint32_t)blk * 0x9e3779b1u) >> 26); }

// Which classes of blocks every 32 tokens write, a warp each.
__global__ void __launch_bounds__(kWriteThreads) slot_classes_kernel(const int64_t* slots, int n_tokens, int block_size,
                                                                     long long n_slots, uint2* classes) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  const int t = blockIdx.x * kWriteThreads + threadIdx.x;
  const long long slot = t < n_tokens ? slots[t] : -1;
  const bool in = slot >= 0 && slot < n_slots;
  const int c = in ? class_of((int)(slot / block_size)) : 0;
  const uint32_t lo = __reduce_or_sync(0xffffffffu, in && c < 32 ? 1u << c : 0u);
  const uint32_t hi = __reduce_or_sync(0xffffffffu, in && c >= 32 ? 1u << (c - 32) : 0u);
  if ((threadIdx.x & 31) == 0 && t < n_tokens) classes[t / 32] = make_uint2(lo, hi);
}

template <typename T>
__global__ void __launch_bounds__(kWriteThreads, kWriteCtas) write_kv_q8_kernel(const WriteParams p) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int row_of[kMaxBlockSize];   // last token of the call for each slot of the block, or -1
  __shared__ uint16_t rows[kMaxBlockSize];  // the slots of the block that get a row
  __shared__ uint4 stage_s[kWriteThreads / 32][kStage];
  __shared__ int first, n_rows, n_cands;
  __shared__ int2 cands[kChunk];  // (token, its block)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bs = p.block_size;
  const int D = p.head_dim, D8 = D / 8, H = p.n_kv_heads;
  const size_t row_elems = (size_t)H * D;
  if (tid < 32) {
    // the chunk's tokens that the token before them does not share the block with
    const int t = blockIdx.x * p.chunk + lane;
    bool cand = false;
    long long blk = 0;
    if (lane < p.chunk && t < p.n_tokens) {
      const long long slot = p.slots[t], before = t > 0 ? p.slots[t - 1] : -1;
      blk = slot / bs;
      cand = slot >= 0 && slot < p.n_slots && (before < 0 || before / bs != blk);
    }
    const unsigned m = __ballot_sync(0xffffffffu, cand);
    if (cand) cands[__popc(m & ((1u << lane) - 1u))] = make_int2(t, (int)blk);
    if (lane == 0) n_cands = __popc(m);
  }
  __syncthreads();
  for (int ci = 0; ci < n_cands; ++ci) {
    const int t = cands[ci].x, blk = cands[ci].y;
    const long long base = (long long)blk * bs;
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
    if (p.classes) {
      // only the groups of 32 tokens that write a block of this one's class
      const int groups = (p.n_tokens + 31) / 32, c = class_of(blk);
      constexpr int kAtOnce = 4;
      for (int g0 = warp * 32; g0 < groups; g0 += kAtOnce * kWriteThreads) {
        uint2 r[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int g = g0 + k * kWriteThreads + lane;
          r[k] = g < groups ? p.classes[g] : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          for (unsigned m = __ballot_sync(0xffffffffu, ((c < 32 ? r[k].x : r[k].y) >> (c & 31)) & 1u); m; m &= m - 1) {
            const int i = (g0 + k * kWriteThreads + __ffs(m) - 1) * 32 + lane;
            if (i < p.n_tokens) look(p.slots[i], i);
          }
      }
    }
    // two slots a load where they are aligned (an odd last one apart)
    const int to_read = p.classes ? 0 : p.n_tokens;
    const int pairs = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0 ? to_read / 2 : 0;
#pragma unroll 8
    for (int i = tid; i < pairs; i += kWriteThreads) {
      const longlong2 two = reinterpret_cast<const longlong2*>(p.slots)[i];
      look(two.x, 2 * i);
      look(two.y, 2 * i + 1);
    }
    for (int i = 2 * pairs + tid; i < to_read; i += kWriteThreads) look(p.slots[i], i);
    __syncthreads();
    if (first != t) continue;  // the same for all threads
    for (int i = tid; i < bs; i += kWriteThreads)
      if (row_of[i] >= 0) rows[atomicAdd(&n_rows, 1)] = (uint16_t)i;
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

      // The rows in groups of 8 elements, as many at a time as the stage holds: all copies are in flight
      // at once, and each lane reads back its own.  Only rows beyond the stage are fetched again for the second pass.
      constexpr int kVecs = sizeof(T) / 2, kItems = kStage / kVecs;
      uint4* stage = stage_s[warp] + lane * kVecs;
      const int items = n * D8;
      auto fetch = [&](int from) {
        Walk8 w(from + lane, D8);
        for (int i = lane; i < kItems && from + i < items; i += 32, w.next()) {
          const T* src = x + (size_t)row_of[rows[w.row]] * row_elems + w.c * 8;
          uint4* dst = stage + (i - lane) * kVecs;
#pragma unroll
          for (int k = 0; k < kVecs; ++k) ptx::copy16_async(dst + k, reinterpret_cast<const uint4*>(src) + k);
        }
        ptx::wait_copies();
      };
      float amax = 0.f;
      for (int from = 0; from < items; from += kItems) {
        fetch(from);
#pragma unroll 4
        for (int i = lane; i < kItems && from + i < items; i += 32) amax = amax8<T>(stage + (i - lane) * kVecs, amax);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const float now = fmaxf(old, q8::scale_for(amax));
      // Dividing by a power of two is multiplying by its reciprocal; other scales come from the caller only.
      const uint32_t bits = __float_as_uint(now);
      const bool pow2 = (bits & 0x7fffffu) == 0u && bits >= 0x00800000u && bits <= 0x7e800000u;
      const float inv = pow2 ? __uint_as_float(0x7f000000u - bits) : 0.f;
      __syncwarp();  // every lane has read the old scale
      if (lane == 0) *sp = now;

      auto encode_rows = [&](auto scaled) {
        for (int from = 0; from < items; from += kItems) {
          if (items > kItems) fetch(from);
          Walk8 w(from + lane, D8);
#pragma unroll 2
          for (int i = lane; i < kItems && from + i < items; i += 32, w.next()) {
            float f[8];
            to_floats<T>(stage + (i - lane) * kVecs, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = fmaf(f[e], 0.f, scaled(f[e]));  // NaN where f is not finite
            *reinterpret_cast<uint2*>(codes + (size_t)rows[w.row] * row_elems + w.c * 8) = encode8(f);
          }
        }
      };
      if (pow2)
        encode_rows([inv](float f) { return f * inv; });
      else
        encode_rows([now](float f) { return __fdiv_rn(f, now); });

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

extern "C" size_t tvk_write_kv_q8_workspace_size(int n_tokens) {
  return n_tokens > kReadAll ? ((size_t)n_tokens + 31) / 32 * sizeof(uint2) : 0;
}

extern "C" int tvk_write_kv_slots_q8(const void* k, const void* v, const int64_t* slots, void* k_cache, void* v_cache,
                                     float* k_scale, float* v_scale, int n_tokens, int n_kv_heads, int head_dim,
                                     int num_blocks, int block_size, int dtype, void* workspace, size_t workspace_bytes,
                                     void* stream) {
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
  const size_t need = tvk_write_kv_q8_workspace_size(n_tokens);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    tvk::set_error("workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    return TVK_ERR_WORKSPACE;
  }
  TVK_CHECK_ARG(need == 0 || (uintptr_t)workspace % 8 == 0, "workspace must be 8-byte aligned");
  uint2* classes = need > 0 ? (uint2*)workspace : nullptr;
  const long long n_slots = (long long)num_blocks * block_size;
  const WriteParams p{k, v, (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, slots, n_tokens, n_kv_heads,
                      head_dim, block_size, n_tokens > kFewTokens ? kChunk : 1, classes, n_slots};
  // a warp per (K or V, head), in long calls per two of them
  const int per_cta = kWriteThreads / 32 * (n_tokens > kFewTokens ? 2 : 1);
  const dim3 grid((n_tokens + p.chunk - 1) / p.chunk, (2 * n_kv_heads + per_cta - 1) / per_cta);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (classes)
    TVK_CHECK_CUDA(tvk::launch_pdl(slot_classes_kernel, dim3((n_tokens + kWriteThreads - 1) / kWriteThreads), kWriteThreads, 0, s,
                                   slots, n_tokens, block_size, n_slots, classes));
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
