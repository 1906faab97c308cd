// logprobs.cu -- log probabilities of given tokens, the entropy of each row's
// distribution and the row's most likely tokens, in one pass over the logits.
//
//   lse  = m + log(sum_v exp(x_v - m)),  m = max_v x_v
//   logprob[r] = x_token - lse
//   entropy[r] = lse - sum_v p_v x_v = log S - T / S
//                with S = sum exp(x_v - m), T = sum exp(x_v - m) (x_v - m)
//   top[r]     = the K largest logits, equal values in index order
//
// Each thread keeps (m, S, T) in fp32 for the logits it reads, 16 bytes at a
// time, and moves m only when a vector exceeds it.
//
// The K best: after the first tile (512 threads x 4 vectors) the CTA picks a
// threshold that at least K threads' maxima reach, so at least K logits of
// the row do; a logit below it cannot be among the K best.  What reaches it is
// pushed as a 64-bit key (ordered value, inverted index) to shared memory, and
// the K best of those few hundred keys are found by bisection over the keys.
// Rows that keep pushing (sorted or constant logits) run into the buffer's
// limit, are cut back to their K best and go on with an exact threshold.
#include <math.h>

#include "tvk_common.cuh"

namespace {

constexpr int kLpThreads = 512;
constexpr int kLpUnroll = 4;         // 16-byte loads in flight per thread
constexpr int kLpBuf = 2048;         // candidate keys kept in shared memory
constexpr int kLpMaxK = 32;
constexpr int kLpPerThread = kLpBuf / kLpThreads;
constexpr float kLog2e = 1.4426950408889634f;

// fp32 values as unsigned integers of the same order: -0 counts as +0, every
// NaN as one value above +inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o >> 31) ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The larger of all elements of one 16-byte vector, NaN if one is.
template <typename T> __device__ __forceinline__ float vec_max(const uint4& u);
template <> __device__ __forceinline__ float vec_max<float>(const uint4& u) {
  return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
}
template <> __device__ __forceinline__ float vec_max<__half>(const uint4& u) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
  const __half2 c = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return __half2float(__hmax_nan(c.x, c.y));
}
template <> __device__ __forceinline__ float vec_max<__nv_bfloat16>(const uint4& u) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 c = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return __bfloat162float(__hmax_nan(c.x, c.y));
}

// Running sums of one thread: s = sum exp(x - m), t = sum exp(x - m) (x - m).
// x - m is formed before the scaling to base 2, so rows that hold nothing but
// the type's lowest value (masks) neither overflow nor cancel.
struct Sums {
  float m, s, t;
};

// New maximum: m > a.m, or NaN (then everything becomes NaN, as it should).
__device__ __forceinline__ void raise_max(Sums& a, float m) {
  if (a.m == -INFINITY) {  // nothing but -inf so far
    a.s = a.t = m != m ? m : 0.f;
  } else {
    const float d = a.m - m, c = ptx::ex2(d * kLog2e);
    a.t = c == 0.f ? 0.f : c * fmaf(d, a.s, a.t);  // d * s may overflow where c is 0
    a.s *= c;
  }
  a.m = m;
}

__device__ __forceinline__ void add(Sums& a, float x, float m) {
  // exp(-200) is 0 here: -inf adds 0 * -200 to t, not 0 * -inf; NaN stays
  const float d = max_nan(x - m, -200.f);
  const float e = ptx::ex2(d * kLog2e);
  a.s += e;
  a.t = fmaf(e, d, a.t);
}

__device__ __forceinline__ Sums merge(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  r.s = r.t = 0.f;
  const Sums* p[2] = {&a, &b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (p[i]->m == -INFINITY && p[i]->s == 0.f) continue;  // nothing but -inf seen
    const float d = p[i]->m - r.m, c = ptx::ex2(d * kLog2e);
    r.s += p[i]->s * c;
    r.t += c == 0.f ? 0.f : c * fmaf(d, p[i]->s, p[i]->t);
  }
  return r;
}

struct LpParams {
  const void* logits;
  const int32_t* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int32_t* top_tokens;
  long long row_stride;
  int vocab, top_k;
};

struct LpShared {
  unsigned long long keys[kLpBuf];
  unsigned long long best[kLpMaxK];
  Sums part[kLpThreads / 32];
  Sums row;
  int count;
  int wsum[kLpThreads / 32];
};

// Sum of `c` over the CTA (two barriers).
__device__ __forceinline__ int block_count(LpShared& sh, int c) {
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = c;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < kLpThreads / 32; ++i) t += sh.wsum[i];
  __syncthreads();
  return t;
}

// Keeps the K largest keys of the buffer (all of them if there are no more),
// at its front in any order; keys of elements [drop_lo, drop_hi) are dropped
// first.  Returns how many stay; *kth gets the smallest kept key (0 if
// fewer than K).  Every thread of the CTA takes part.
__device__ int keep_best(LpShared& sh, int K, int drop_lo, int drop_hi, unsigned long long* kth) {
  __syncthreads();
  const int n = min(sh.count, kLpBuf);
  unsigned long long mine[kLpPerThread];
  int have = 0;
#pragma unroll
  for (int i = 0; i < kLpPerThread; ++i) {
    const int at = threadIdx.x + i * kLpThreads;
    unsigned long long k = at < n ? sh.keys[at] : 0ull;
    const int idx = (int)(0xffffffffu - (uint32_t)k);
    if (idx >= drop_lo && idx < drop_hi) k = 0ull;
    mine[i] = k;
    have += k != 0ull;
  }
  const int total = block_count(sh, have);
  unsigned long long lo = 1ull;  // every real key is larger than 0
  if (total > K) {
    // bisection: count(key >= lo) >= K always, count(key >= hi) < K
    unsigned long long hi = ~0ull;
    while (hi - lo > 1ull) {
      const unsigned long long mid = lo + ((hi - lo) >> 1);
      int c = 0;
#pragma unroll
      for (int i = 0; i < kLpPerThread; ++i) c += mine[i] >= mid;
      c = block_count(sh, c);
      if (c >= K) {
        lo = mid;
        if (c == K) break;
      } else {
        hi = mid;
      }
    }
  }
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kLpPerThread; ++i)
    if (mine[i] >= lo) sh.keys[atomicAdd(&sh.count, 1)] = mine[i];
  __syncthreads();
  const int kept = sh.count;
  *kth = kept >= K ? lo : 0ull;
  return kept;
}

__device__ __forceinline__ unsigned long long key_of(float x, int idx) {
  return ((unsigned long long)order_of(x) << 32) | (0xffffffffu - (uint32_t)idx);
}

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(const LpParams p) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  constexpr int N = 16 / sizeof(T);
  __shared__ LpShared sh;
  const int K = p.top_k, V = p.vocab, tid = threadIdx.x;
  const long long row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;
  float x_tok = 0.f;
  bool inside = false;  // a token outside the vocabulary has probability 0
  if (tid == 0) {
    sh.count = 0;
    const int tok = p.tokens[row];
    inside = tok >= 0 && tok < V;
    if (inside) x_tok = DT<T>::to_f(x[tok]);
  }
  // Elements before the first 16-byte boundary and after the last whole vector go one to a thread.
  const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nvec = (V - head) / N, tail0 = head + nvec * N;
  const T* xv = x + head;
  Sums a{-INFINITY, 0.f, 0.f};
  unsigned long long tau_key = 0ull;  // only keys above it are candidates
  float tau = -INFINITY;              // only values not below it are
  __syncthreads();

  auto push = [&](float f, int idx) -> bool {  // true: the buffer is getting full
    const unsigned long long k = key_of(f, idx);
    if (k <= tau_key) return false;
    const int at = atomicAdd(&sh.count, 1);
    if (at < kLpBuf) sh.keys[at] = k;
    return at >= kLpBuf / 2;
  };

  {
    const int single = tid < head ? tid : (tid < head + V - tail0 ? tail0 + tid - head : -1);
    if (single >= 0) {
      const float f = DT<T>::to_f(x[single]);
      raise_max(a, f);
      add(a, f, a.m == -INFINITY ? 0.f : a.m);
      if (K > 0) push(f, single);
    }
  }

  for (int base = 0; base < nvec; base += kLpThreads * kLpUnroll) {
    uint4 u[kLpUnroll];
    float vm[kLpUnroll];
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      const int i = base + k * kLpThreads + tid;
      if (i < nvec) u[k] = __ldcs(reinterpret_cast<const uint4*>(xv + (size_t)i * N));
    }
    float tm = -INFINITY;
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      if (base + k * kLpThreads + tid < nvec) {
        vm[k] = vec_max<T>(u[k]);
        tm = max_nan(tm, vm[k]);
        if (!(vm[k] <= a.m)) raise_max(a, vm[k]);
        const float ref = a.m == -INFINITY ? 0.f : a.m;
        const T* h = reinterpret_cast<const T*>(&u[k]);
#pragma unroll
        for (int e = 0; e < N; ++e) add(a, DT<T>::to_f(h[e]), ref);
      }
    }
    if (K == 0) continue;
    if (base == 0) {
      // A value that between K and 2K threads' maxima reach (by bisection; fewer
      // steps than the exact K-th needs): K logits at least are not below it.
      const bool has = tid < nvec;
      const uint32_t o = has ? order_of(tm) : 0u;
      if (__syncthreads_count(has) >= K) {
        uint32_t lo = 0u, hi = 0xffffffffu;
        while (hi - lo > 1u) {
          const uint32_t mid = lo + ((hi - lo) >> 1);
          const int c = __syncthreads_count(has && o >= mid);
          if (c >= K) {
            lo = mid;
            if (c <= 2 * K) break;
          } else {
            hi = mid;
          }
        }
        if (lo) tau = value_of(lo);
      }
    }
    bool full = false;
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      const int i = base + k * kLpThreads + tid;
      if (i < nvec && !(vm[k] < tau)) {
        const T* h = reinterpret_cast<const T*>(&u[k]);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float f = DT<T>::to_f(h[e]);
          if (!(f < tau)) full |= push(f, head + i * N + e);
        }
      }
    }
    if (!__syncthreads_or(full)) continue;
    if (sh.count <= kLpBuf) {
      keep_best(sh, K, 0, 0, &tau_key);
    } else {
      // Keys of this tile were lost: take the tile out and push it again, one
      // element a thread at a time, cutting back whenever the next step might overflow.
      keep_best(sh, K, head + base * N, head + min(base + kLpThreads * kLpUnroll, nvec) * N, &tau_key);
      for (int k = 0; k < kLpUnroll; ++k) {
        const int i = base + k * kLpThreads + tid;
        for (int e = 0; e < N; ++e) {
          if (i < nvec) push(DT<T>::to_f(xv[(size_t)i * N + e]), head + i * N + e);
          __syncthreads();
          const bool cut = sh.count > kLpBuf - kLpThreads;
          __syncthreads();
          if (cut) keep_best(sh, K, 0, 0, &tau_key);
        }
      }
      keep_best(sh, K, 0, 0, &tau_key);
    }
    if (tau_key) tau = value_of((uint32_t)(tau_key >> 32));
  }

  // sums of the row
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
    a = merge(a, b);
  }
  if ((tid & 31) == 0) sh.part[tid >> 5] = a;
  __syncthreads();
  if (tid < 32) {
    a = tid < kLpThreads / 32 ? sh.part[tid] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Sums b;
      b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
      b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
      a = merge(a, b);
    }
    if (tid == 0) sh.row = a;
  }
  __syncthreads();
  const Sums r = sh.row;
  const float log_s = logf(r.s);
  // x - lse; a row of nothing but -inf gives NaN for every token, as the formula does
  auto logprob = [&](float f) -> float { return (f - r.m) - log_s; };
  if (tid == 0) {
    p.logprobs[row] = inside ? logprob(x_tok) : -INFINITY;
    p.entropy[row] = log_s - r.t / r.s;
  }
  if (K > 0) {
    const int n = keep_best(sh, K, 0, 0, &tau_key);
    if (tid < n) {
      const unsigned long long k = sh.keys[tid];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sh.keys[j] > k;
      p.top_logprobs[row * K + rank] = logprob(value_of((uint32_t)(k >> 32)));
      p.top_tokens[row * K + rank] = (int)(0xffffffffu - (uint32_t)k);
    }
  }
}

}  // namespace

extern "C" int tvk_token_logprobs(const void* logits, const int32_t* tokens, float* logprobs, float* entropy,
                                  float* top_logprobs, int32_t* top_tokens, int rows, int vocab,
                                  long long row_stride, int top_k, int dtype, void* stream) {
  TVK_CHECK_ARG(rows >= 0 && vocab > 0 && row_stride >= vocab, "bad shape rows=%d vocab=%d row_stride=%lld", rows,
                vocab, row_stride);
  TVK_CHECK_ARG(top_k >= 0 && top_k <= kLpMaxK && top_k <= vocab, "top_k %d outside [0, min(%d, vocab)]", top_k,
                kLpMaxK);
  TVK_CHECK_ARG(dtype == TVK_DTYPE_F32 || dtype == TVK_DTYPE_F16 || dtype == TVK_DTYPE_BF16, "unknown dtype %d", dtype);
  if (rows == 0) return TVK_OK;
  TVK_CHECK_ARG(logits && tokens && logprobs && entropy && (top_k == 0 || (top_logprobs && top_tokens)),
                "null pointer argument");
  TVK_CHECK_ARG((uintptr_t)logits % tvk::dtype_size(dtype) == 0, "logits must be aligned to their elements");
  LpParams p{logits, tokens, logprobs, entropy, top_logprobs, top_tokens, row_stride, vocab, top_k};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TVK_DTYPE_F16: TVK_CHECK_CUDA(tvk::launch_pdl(token_logprobs_kernel<__half>, rows, kLpThreads, 0, s, p)); break;
    case TVK_DTYPE_BF16:
      TVK_CHECK_CUDA(tvk::launch_pdl(token_logprobs_kernel<__nv_bfloat16>, rows, kLpThreads, 0, s, p));
      break;
    default: TVK_CHECK_CUDA(tvk::launch_pdl(token_logprobs_kernel<float>, rows, kLpThreads, 0, s, p)); break;
  }
  TVK_CHECK_LAUNCH("token_logprobs");
  return TVK_OK;
}
