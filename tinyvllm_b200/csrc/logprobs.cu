// logprobs.cu -- log probabilities of given tokens, the entropy of each row's
// distribution and the row's most likely tokens, in one pass over the logits.
//
//   lse  = m + log(sum_v exp(x_v - m)),  m = max_v x_v
//   logprob[r] = x_token - lse
//   entropy[r] = lse - sum_v p_v x_v = log S - T / S
//                with S = sum exp(x_v - m), T = sum exp(x_v - m) (x_v - m)
//   top[r]     = the K largest logits, equal values in index order
//
// Each thread keeps (m, S, T) in fp32 for the logits it reads, four 16-byte vectors a
// step; its m moves only when a step exceeds it by more than 4 (moving at every new
// maximum, some lane of a warp did so in most steps, which cost a third of the time).
//
// A row to itself (many rows) is a CTA's, whose vectors travel through shared memory a
// step ahead: [2048, 128256] bf16 with one alternative takes 96 us so (5.5 TB/s, 0.84 of
// the measured copy rate; 108 to 113 us called one by one), with loads to registers 145 us, when a warp had nothing in
// flight while it computed (and loads a step ahead in registers 203 us).  Without alternatives
// 86 us; fp32 logits 158 and 161 us, 6.6 TB/s, all that memory gives.  What is left for bf16
// is the exponentials (58 us of the special-function unit) and the candidates' barriers.
// With few rows a cluster of CTAs shares each, and their sums and K best are put
// together by the first over distributed shared memory; they read once and are done, so
// latencies bound them ([1, 128256] bf16 7.0 us, [64, 32000] fp16 with 20 alternatives 8.8 us).
//
// The K best: from the maxima of 64 groups of threads over the first step
// each CTA takes the K-th largest as a threshold, which K logits at least reach; one
// below it is not among the K best.  What reaches it is pushed as a 64-bit key (ordered
// value, inverted index) to shared memory; the same with groups of keys raises the threshold
// after 4, 8 and 16 steps and every 16 from there, and leaves little more than the K best for
// ranking at the end.  [2048, 128256] bf16 takes 124 us with K = 8, 152 with 20, 181 with 32
// (before the buffer's cut was taken out of the loop 127, 157 and 185; with 32 groups and one raise 123, 183 and
// 429): pushing is what it costs.
// Rows that keep pushing (sorted or constant logits) run into the buffer's
// limit, are cut back to their K best and go on with an exact threshold, which what
// comes later has to exceed: 296 constant rows of 256,000 take 100 (fp32) and 106 us (bf16), ordinary
// ones 70 and 55.
#include <math.h>

#include <type_traits>

#include "tvk_common.cuh"

namespace {

constexpr int kLpUnroll = 4;         // 16-byte vectors a thread reads per step
constexpr int kLpFirstSteps = 4, kLpSteps = 16;  // steps before the first look at the candidate buffer, and between two
constexpr float kLpSlack = 4.f;      // a reference may lie this far below its thread's largest logit
constexpr int kLpBuf = 2048;         // candidate keys kept in shared memory
constexpr int kLpMaxK = 32;
constexpr int kLpGroups = 64;        // groups of threads, or of keys, whose maxima give a threshold
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLpFloor = -30000.f, kLpCeiling = 1e38f;  // see add_step

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

// The larger elements of two 16-byte vectors, NaN where one is.
template <typename T> __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
  uint4 r;
  const uint32_t *x = &a.x, *y = &b.x;
  uint32_t* z = &r.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      z[i] = __float_as_uint(max_nan(__uint_as_float(x[i]), __uint_as_float(y[i])));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2 m = __hmax2_nan(*reinterpret_cast<const T2*>(&x[i]), *reinterpret_cast<const T2*>(&y[i]));
      z[i] = *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  return r;
}
// The largest element of one vector, NaN if one is.
template <typename T> __device__ __forceinline__ float vec_max(const uint4& u) {
  const uint4 v = larger<T>(u, make_uint4(u.z, u.w, u.z, u.w));
  if constexpr (sizeof(T) == 4) {
    return max_nan(__uint_as_float(v.x), __uint_as_float(v.y));
  } else {
    const uint4 w = larger<T>(v, make_uint4(v.y, v.y, v.y, v.y));
    const uint16_t lo = (uint16_t)w.x, hi = (uint16_t)(w.x >> 16);
    return DT<T>::to_f(__hmax_nan(*reinterpret_cast<const T*>(&lo), *reinterpret_cast<const T*>(&hi)));
  }
}
// Four bytes of -inf.
template <typename T> __device__ __forceinline__ uint32_t minus_inf() {
  return sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
}

// Element e of a vector, without a register array.
template <typename T> __device__ __forceinline__ T element(const uint4& u, int e) {
  const uint32_t w = sizeof(T) == 4 ? (e == 0 ? u.x : e == 1 ? u.y : e == 2 ? u.z : u.w)
                                    : (e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w);
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const uint16_t b = (uint16_t)(e & 1 ? w >> 16 : w);
    return *reinterpret_cast<const T*>(&b);
  }
}

// Bit e: element e is not below tau (NaN is not).  tau is -inf, NaN or a value of the type.
template <typename T> __device__ __forceinline__ uint32_t not_below(const uint4& u, float tau) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t bits = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= (uint32_t)!(__uint_as_float(w[i]) < tau) << i;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T t = DT<T>::from_f(tau);
    T2 t2;
    t2.x = t2.y = t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = ~__hlt2_mask(*reinterpret_cast<const T2*>(&w[i]), t2);
      bits |= (m & 1u) << (2 * i) | (m >> 31) << (2 * i + 1);
    }
  }
  return bits;
}

// The next larger value of the type (NaN for NaN and +inf).
template <typename T> __device__ __forceinline__ float next_larger(float x) {
  if (x != x) return x;
  x += 0.f;  // +0 for -0
  if constexpr (sizeof(T) == 4) {
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(b >> 31 ? b - 1 : b + 1);
  } else {
    const T t = DT<T>::from_f(x);
    const uint16_t b = *reinterpret_cast<const uint16_t*>(&t), up = b >> 15 ? b - 1 : b + 1;
    return DT<T>::to_f(*reinterpret_cast<const T*>(&up));
  }
}

// Two fp32 values in one register pair, for the packed fp32 instructions.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Elements 2 i and 2 i + 1 of a 16-byte vector.
template <typename T> __device__ __forceinline__ F2 pair_of(const uint4& u, int i);
template <> __device__ __forceinline__ F2 pair_of<float>(const uint4& u, int i) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
  return pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <> __device__ __forceinline__ F2 pair_of<__half>(const uint4& u, int i) {
  const float2 f = __half22float2(reinterpret_cast<const __half2*>(&u)[i]);
  return pack(f.x, f.y);
}
template <> __device__ __forceinline__ F2 pair_of<__nv_bfloat16>(const uint4& u, int i) {
  const uint32_t w = reinterpret_cast<const uint32_t*>(&u)[i];
  return pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// The vector with every element raised to at least -30000 (16-bit types; NaN stays), and for fp32 itself.
template <typename T> __device__ __forceinline__ uint4 floored(const uint4& u) {
  uint4 r = u;
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T low = DT<T>::from_f(kLpFloor);
    T2 low2;
    low2.x = low2.y = low;
    T2* h = reinterpret_cast<T2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low2);
  }
  return r;
}

// Running sums of one thread, even and odd elements apart: s = sum exp(x - m),
// t = sum exp(x - m) u, u = (x - m) / ln 2.
struct Sums {
  float m;
  F2 s, t;
};

// c (t + d s) for a move of the reference by d, c = 2^d; 0 where c is (d s may overflow there).
__device__ __forceinline__ float moved(float c, float d, float s, float t) { return c == 0.f ? 0.f : c * fmaf(d, s, t); }

// New reference: m > a.m, or NaN (then everything becomes NaN, as it should, and stays it: a later step of
// nothing but -inf must not look like a start).
__device__ __forceinline__ void raise_max(Sums& a, float m) {
  if (a.m == -INFINITY) {  // nothing but -inf so far
    const float z = m != m ? m : 0.f;
    a.s = a.t = pack(z, z);
  } else {
    const float d = (a.m - m) * kLog2e, c = ptx::ex2(d);
    const float2 s = unpack(a.s), t = unpack(a.t);
    a.t = pack(moved(c, d, s.x, t.x), moved(c, d, s.y, t.y));
    a.s = mul2(a.s, pack(c, c));
  }
  a.m = max_nan(a.m, m);
}

// With any reference.  x - m is formed before the scaling to base 2, so rows that hold nothing
// but the type's lowest value (masks) neither overflow nor cancel.
__device__ __forceinline__ void add_pair(Sums& a, F2 x) {
  const float ref = a.m == -INFINITY ? 0.f : a.m;
  // 2^-300 is 0 here: -inf adds 0 * -300 to t, not 0 * -inf; NaN stays
  const float2 d = unpack(add2(x, pack(-ref, -ref)));
  const F2 u = pack(max_nan(d.x * kLog2e, -300.f), max_nan(d.y * kLog2e, -300.f));
  const float2 v = unpack(u);
  const F2 e = pack(ptx::ex2(v.x), ptx::ex2(v.y));
  a.s = add2(a.s, e);
  a.t = fma2(e, u, a.t);
}

// A step's vectors.  With an ordinary reference (almost always) 16-bit elements are floored two
// at a time: what lies below -30000 weighs nothing beside it, and no product with -inf arises (up to a
// reference of 1e38: beyond, (x - m) log2 e may pass the fp32 range, which add_pair looks after).
// The first n vectors; ALL: every one, without a branch between them.
template <typename T, bool ALL>
__device__ __forceinline__ void add_step(Sums& a, const uint4 (&u)[kLpUnroll], int n) {
  constexpr int N = 16 / sizeof(T);
  if (sizeof(T) == 2 && a.m > kLpFloor + 1000.f && a.m < kLpCeiling) {
    const F2 scale = pack(kLog2e, kLog2e), minus_m = pack(-a.m, -a.m);
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      if (!ALL && k >= n) break;
      const uint4 w = floored<T>(u[k]);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        const F2 y = mul2(add2(pair_of<T>(w, e), minus_m), scale);
        const float2 v = unpack(y);
        const F2 z = pack(ptx::ex2(v.x), ptx::ex2(v.y));
        a.s = add2(a.s, z);
        a.t = fma2(z, y, a.t);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      if (!ALL && k >= n) break;
#pragma unroll
      for (int e = 0; e < N / 2; ++e) add_pair(a, pair_of<T>(u[k], e));
    }
  }
}

// Sums relative to one maximum.
struct RowSums {
  float m, s, t;
};
// a's sums with the reference moved to m >= a.m.
__device__ __forceinline__ RowSums at_max(const RowSums& a, float m) {
  if (a.m == -INFINITY && a.s == 0.f) return RowSums{m, 0.f, 0.f};  // nothing but -inf seen
  const float d = (a.m - m) * kLog2e, c = ptx::ex2(d);
  return RowSums{m, a.s * c, moved(c, d, a.s, a.t)};
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

// NT: threads of a CTA.  A row to itself gets 256 (four CTAs on an SM: a row's serial end hides
// behind three others' loads), a cluster's share 512, read straight to registers: each thread has two
// steps or so, so there is nothing to run ahead of.  With loads to registers [2048, 128256] bf16 took 145 us with 256 and
// 152 with 512, one row of it on 8 CTAs 8.4 and 7.4, 37 x 50,001 fp32 on 4 CTAs each 10.5 and 9.3; those
// 37 rows took 9.8 through shared memory.
template <int NT>
struct LpShared {
  unsigned long long keys[kLpBuf];
  unsigned long long best[kLpMaxK];  // this CTA's K best, in order
  RowSums sums;                      // and its part of the row's sums
  RowSums all_sums[8];
  float part[NT / 32][2];
  alignas(16) uint32_t group_max[kLpGroups];
  uint32_t at_k;
  int count, n_best;
  int wsum[NT / 32];
};

// Sum of `c` over the CTA (two barriers).
template <int NT>
__device__ __forceinline__ int block_count(LpShared<NT>& sh, int c) {
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = c;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) t += sh.wsum[i];
  __syncthreads();
  return t;
}

// Keeps the K largest keys of the buffer (all of them if there are no more),
// at its front in any order; keys of elements [drop_lo, drop_hi) are dropped
// first.  sh.count says how many stay.  Returns the smallest kept key (0 if fewer than
// K), which is an element's and never below what it was.  Every thread of the CTA takes part.
// Not inlined, and the threshold by value: its few calls otherwise cost the loop around them registers and code
// ([2048, 128256] bf16 100.9 us inlined with the threshold through a pointer, 95.7 so; fp32 no difference).
template <int NT>
__device__ __noinline__ unsigned long long keep_best(LpShared<NT>& sh, int K, int drop_lo, int drop_hi) {
  __syncthreads();
  const int n = min(sh.count, kLpBuf);
  unsigned long long mine[(kLpBuf / NT)];
  int have = 0;
#pragma unroll
  for (int i = 0; i < (kLpBuf / NT); ++i) {
    const int at = threadIdx.x + i * NT;
    unsigned long long k = at < n ? sh.keys[at] : 0ull;
    const int idx = (int)(0xffffffffu - (uint32_t)k);
    if (idx >= drop_lo && idx < drop_hi) k = 0ull;
    mine[i] = k;
    have += k != 0ull;
  }
  const int total = block_count(sh, have);
  unsigned long long lo = 1ull;  // every real key is larger than 0
  if (total > K) {
    // bisection: count(key >= lo) >= K always, count(key >= hi) < K (or hi is the largest key there is, a NaN at the
    // row's start: then one more than K may stay)
    unsigned long long hi = ~0ull;
    while (hi - lo > 1ull) {
      const unsigned long long mid = lo + ((hi - lo) >> 1);
      int c = 0;
#pragma unroll
      for (int i = 0; i < (kLpBuf / NT); ++i) c += mine[i] >= mid;
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
  for (int i = 0; i < (kLpBuf / NT); ++i)
    if (mine[i] >= lo) sh.keys[atomicAdd(&sh.count, 1)] = mine[i];
  __syncthreads();
  const int kept = sh.count;
  unsigned long long least = kept >= K ? ~0ull : 0ull;
  for (int i = 0; kept >= K && i < kept; ++i) least = min(least, sh.keys[i]);
  __syncthreads();  // all have read the count before anyone pushes again
  return least;
}

__device__ __forceinline__ unsigned long long key_of(float x, int idx) {
  return ((unsigned long long)order_of(x) << 32) | (0xffffffffu - (uint32_t)idx);
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same shared variable in another CTA of the cluster.
template <typename P>
__device__ __forceinline__ const P* of_cta(const P* x, uint32_t rank) {
  uint64_t r;
  asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(x)), "r"(rank));
  return reinterpret_cast<const P*>(r);
}

// Sum and maximum over the CTA, the same in every thread.
template <int NT>
__device__ __forceinline__ float block_max(LpShared<NT>& sh, float x) {
  float w;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(w) : "f"(x));
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5][0] = w;
  __syncthreads();
  float m = sh.part[0][0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) m = fmaxf(m, sh.part[i][0]);
  __syncthreads();
  return m;
}

// The K-th largest of sh.group_max (0: fewer than K groups have anything); for the whole CTA, after
// every group has put its maximum there.
template <int NT>
__device__ __forceinline__ uint32_t kth_of_groups(LpShared<NT>& sh, int K) {
  __syncthreads();
  if (K == 1) {  // every warp for itself
    const uint32_t* g = sh.group_max + (threadIdx.x & 31);
    static_assert(kLpGroups == 64, "two a lane");
    return __reduce_max_sync(0xffffffffu, max(g[0], g[32]));
  }
  if (threadIdx.x < kLpGroups) {  // a warp or two
    const uint32_t mine = sh.group_max[threadIdx.x];
    int above = 0, not_below = 0;  // mine is the K-th largest where above < K <= not_below
#pragma unroll
    for (int j = 0; j < kLpGroups; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&sh.group_max[j]);
      above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      not_below += (o.x >= mine) + (o.y >= mine) + (o.z >= mine) + (o.w >= mine);
    }
    if (above < K && K <= not_below) sh.at_k = mine;  // the same value, where several have it
  }
  __syncthreads();
  return sh.at_k;
}

// A value that K keys of the buffer at least reach (0: none found), by groups of keys.  Between a barrier
// before it and its own last one nothing is pushed.
template <int NT>
__device__ uint32_t reached_by_k(LpShared<NT>& sh, int K) {
  const int tid = threadIdx.x;
  if (tid < kLpGroups) sh.group_max[tid] = 0u;
  __syncthreads();
  const int n = min(sh.count, kLpBuf);
  for (int i = tid; i < n; i += NT) atomicMax(&sh.group_max[i % kLpGroups], (uint32_t)(sh.keys[i] >> 32));
  return kth_of_groups(sh, K);
}

// The K best keys of the buffer, in order, into sh.best; fewer if there are no more.
template <int NT>
__device__ void select_best(LpShared<NT>& sh, int K) {
  const int tid = threadIdx.x;
  __syncthreads();
  int n = sh.count;
  if (n > 32) {
    const uint32_t least = n <= 2 * NT ? reached_by_k(sh, K) : 0u;
    bool few = false;
    if (least) {
      const unsigned long long k0 = tid < n ? sh.keys[tid] : 0ull;
      const unsigned long long k1 = tid + NT < n ? sh.keys[tid + NT] : 0ull;
      const bool in0 = (uint32_t)(k0 >> 32) >= least, in1 = (uint32_t)(k1 >> 32) >= least;
      if (tid == 0) sh.count = 0;
      __syncthreads();
      if (in0) sh.keys[atomicAdd(&sh.count, 1)] = k0;
      if (in1) sh.keys[atomicAdd(&sh.count, 1)] = k1;
      __syncthreads();
      n = sh.count;
      few = n <= NT;  // many only where many are equal
    }
    if (!few) {
      keep_best(sh, K, 0, 0);
      n = sh.count;
    }
  }
  if (tid < n) {
    const unsigned long long k = sh.keys[tid];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += sh.keys[j] > k;
    if (rank < K) sh.best[rank] = k;
  }
  if (tid == 0) sh.n_best = n < K ? n : K;
}

// One cluster (of one CTA or more) per row.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_logprobs_kernel(const LpParams p) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
  constexpr int N = 16 / sizeof(T);
  __shared__ LpShared<NT> sh;
  const int K = p.top_k, V = p.vocab, tid = threadIdx.x, lane = tid & 31;
  const uint32_t ctas = cluster_size(), rank = blockIdx.x % ctas;
  const long long row = blockIdx.x / ctas;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;
  if (tid == 0) sh.count = 0;
  // Elements before the first 16-byte boundary and after the last whole vector go one to a thread.
  const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int all_vec = (V - head) / N, tail0 = head + all_vec * N;
  const T* xv = x + head;
  const int v0 = (int)((long long)all_vec * rank / ctas), v1 = (int)((long long)all_vec * (rank + 1) / ctas);
  Sums a{-INFINITY, pack(0.f, 0.f), pack(0.f, 0.f)};
  unsigned long long tau_key = 0ull;  // only keys above it are candidates
  float tau = -INFINITY;              // only values not below it are
  // Each thread's vectors of a step travel to places of its own in shared memory while it works on those of
  // the step before: no other thread reads them, so no barrier is needed, and no register waits for them.
  constexpr bool kRing = NT == 256;
  extern __shared__ uint4 ring[];  // [2][kLpUnroll][NT]
  auto fetch = [&](int half, int base) {
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      const int i = base + k * NT + tid;
      if (i < v1) ptx::copy16_async(ring + (half * kLpUnroll + k) * NT + tid, xv + (size_t)i * N);
    }
    ptx::commit_copies();
  };
  int half = 0;
  if constexpr (kRing) fetch(0, v0);
  // The row's token and its logit, wanted at the end only: asked for behind the first vectors.
  int tok = -1;
  if (tid == 0 && rank == 0) tok = p.tokens[row];
  __syncthreads();

  auto push = [&](float f, int idx) -> bool {  // true: the buffer is getting full
    const unsigned long long k = key_of(f, idx);
    if (k <= tau_key) return false;
    const int at = atomicAdd(&sh.count, 1);
    if (at < kLpBuf) sh.keys[at] = k;
    return at >= kLpBuf / 2;
  };

  const bool inside = tok >= 0 && tok < V;  // a token outside the vocabulary has probability 0
  const float x_tok = inside ? DT<T>::to_f(x[tok]) : 0.f;
  if (rank == 0) {
    const int single = tid < head ? tid : (tid < head + V - tail0 ? tail0 + tid - head : -1);
    if (single >= 0) {
      const float f = DT<T>::to_f(x[single]);
      raise_max(a, f);
      add_pair(a, pack(f, -INFINITY));
      if (K > 0) push(f, single);
    }
  }

  constexpr int kFirst = kLpFirstSteps * kLpUnroll * NT, kMost = kLpSteps * kLpUnroll * NT;
  for (int from = v0, to; from < v1; from = to) {
    to = min(from + min(max(kFirst, from - v0), kMost), v1);  // after 4, 8, 16 and every 16 further steps
    bool full = false;
    for (int base = from; base < to; base += kLpUnroll * NT) {
      uint4 u[kLpUnroll];  // -inf where there is no vector
      if constexpr (kRing) {
        fetch(half ^ 1, base + kLpUnroll * NT);  // into the places read in the step before
        ptx::wait_copies_but<1>();
      }
#pragma unroll
      for (int k = 0; k < kLpUnroll; ++k) {
        const int i = base + k * NT + tid;
        u[k] = make_uint4(minus_inf<T>(), minus_inf<T>(), minus_inf<T>(), minus_inf<T>());
        if (i < to) u[k] = kRing ? ring[(half * kLpUnroll + k) * NT + tid] : __ldcs(reinterpret_cast<const uint4*>(xv + (size_t)i * N));
      }
      half ^= 1;
      uint4 all = larger<T>(u[0], u[1]);
#pragma unroll
      for (int k = 2; k < kLpUnroll; ++k) all = larger<T>(all, u[k]);
      const float tm = vec_max<T>(all);
      if (!(tm <= a.m + kLpSlack)) raise_max(a, tm);
      if (base + kLpUnroll * NT <= to)
        add_step<T, true>(a, u, kLpUnroll);
      else
        add_step<T, false>(a, u, (to - base + NT - 1) / NT);
      if (K == 0) continue;
      if (base == v0) {
        // The K-th largest of the maxima of the groups of threads: K logits at least are not below it.
        const uint32_t o = tid < v1 - v0 ? order_of(tm) : 0u;
        uint32_t top = o;
#pragma unroll
        for (int d = 1; d < NT / kLpGroups; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (tid % (NT / kLpGroups) == 0) sh.group_max[tid / (NT / kLpGroups)] = top;
        const uint32_t at_k = kth_of_groups(sh, K);
        if (at_k) tau = value_of(at_k);  // 0: fewer than K groups have elements
      }
      if (tm < tau) continue;
#pragma unroll
      for (int k = 0; k < kLpUnroll; ++k) {
        const int i = base + k * NT + tid;
        if (i < to && !(vec_max<T>(u[k]) < tau)) {
          for (uint32_t bits = not_below<T>(u[k], tau); bits; bits &= bits - 1) {
            const int e = __ffs(bits) - 1;
            full |= push(DT<T>::to_f(element<T>(u[k], e)), head + i * N + e);
          }
        }
      }
    }
    if (K == 0) continue;
    if (!__syncthreads_or(full)) {
      if (to < v1) {
        const bool many = sh.count > 2 * K;
        __syncthreads();  // all have read it before anyone pushes again
        const uint32_t least = many ? reached_by_k(sh, K) : 0u;
        if (least) tau = value_of(least);
      }
      continue;
    }
    if (sh.count <= kLpBuf) {
      tau_key = keep_best(sh, K, 0, 0);
    } else {
      // Keys of these steps were lost: take the steps out and push them again, one
      // element a thread at a time, cutting back whenever the next push might overflow.
      tau_key = keep_best(sh, K, head + from * N, head + to * N);
      for (int base = from; base < to; base += NT) {
        const int i = base + tid;
        for (int e = 0; e < N; ++e) {
          if (i < to) push(DT<T>::to_f(xv[(size_t)i * N + e]), head + i * N + e);
          __syncthreads();
          const bool cut = sh.count > kLpBuf - NT;
          __syncthreads();
          if (cut) tau_key = keep_best(sh, K, 0, 0);
        }
      }
      tau_key = keep_best(sh, K, 0, 0);
    }
    if (tau_key) {
      // All that follows has larger indices than the K-th best, so ties with that are no candidates; unless it is one of the
      // elements behind the last whole vector.
      tau = value_of((uint32_t)(tau_key >> 32));
      if ((int)(0xffffffffu - (uint32_t)tau_key) < head + to * N) tau = next_larger<T>(tau);
    }
  }

  // This CTA's sums: the largest reference first, then every thread's sums relative to it.
  {
    const float m = block_max(sh, a.m);
    const float2 s2 = unpack(a.s), t2 = unpack(a.t);
    const RowSums mine = at_max(RowSums{a.m, s2.x + s2.y, t2.x + t2.y}, m);
    float s = mine.s, t = mine.t;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0) {
      sh.part[tid >> 5][0] = s;
      sh.part[tid >> 5][1] = t;
    }
    __syncthreads();
    if (tid == 0) {
      s = t = 0.f;
#pragma unroll
      for (int i = 0; i < NT / 32; ++i) {
        s += sh.part[i][0];
        t += sh.part[i][1];
      }
      sh.sums = RowSums{m, s, t};
    }
  }
  if (K > 0) select_best(sh, K);
  if (ctas > 1)
    cluster_sync();
  else
    __syncthreads();

  if (rank == 0) {
    // All CTAs' sums and K best to this one's shared memory, then the row's by every thread that writes
    // something.  (A CTA's places behind its last key hold 0, which no key is.)
    const int n_all = (int)ctas * K;
    if (tid < (int)ctas) sh.all_sums[tid] = *of_cta(&sh.sums, tid);
    if (tid < n_all) {
      const uint32_t c = tid / K;
      const int i = tid % K;
      sh.keys[tid] = i < *of_cta(&sh.n_best, c) ? of_cta(sh.best, c)[i] : 0ull;
    }
    __syncthreads();
    RowSums r = sh.all_sums[0];
    for (uint32_t c = 1; c < ctas; ++c) {
      const RowSums other = sh.all_sums[c];
      const float m = fmaxf(r.m, other.m);
      const RowSums x0 = at_max(r, m), x1 = at_max(other, m);
      r = RowSums{m, x0.s + x1.s, x0.t + x1.t};
    }
    const float log_s = logf(r.s);
    // x - lse; a row of nothing but -inf gives NaN for every token, as the formula does
    auto logprob = [&](float f) -> float { return (f - r.m) - log_s; };
    if (tid == 0) {
      p.logprobs[row] = inside ? logprob(x_tok) : -INFINITY;
      p.entropy[row] = log_s - kLn2 * (r.t / r.s);
    }
    // The row's K best are those of all CTAs' K best that fewer than K others exceed.
    if (tid < n_all && sh.keys[tid] != 0ull) {
      const unsigned long long k = sh.keys[tid];
      int place = 0;
      for (int j = 0; j < n_all; ++j) place += sh.keys[j] > k;
      if (place < K) {
        p.top_logprobs[row * K + place] = logprob(value_of((uint32_t)(k >> 32)));
        p.top_tokens[row * K + place] = (int)(0xffffffffu - (uint32_t)k);
      }
    }
  }
  if (ctas > 1) cluster_sync();  // no CTA ends while its shared memory is read
}

template <typename T, int NT>
cudaError_t launch_nt(const LpParams& p, int rows, int ctas, cudaStream_t stream) {
  constexpr int kRingBytes = NT == 256 ? 2 * kLpUnroll * NT * 16 : 0;
  auto kern = token_logprobs_kernel<T, NT>;
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = tvk::allow_smem(kern, kRingBytes, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ctas);
  cfg.blockDim = NT;
  cfg.dynamicSmemBytes = kRingBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tvk::pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

// CTAs per row: as many as keep all rows resident at once, but none with less than a vector per
// thread.  Two CTAs of 512 threads fit on each of 148 SMs, but clusters of 8 do not fill every GPC:
// 37 fp32 rows of 50,001 take 14.6 us on 8 CTAs each (two waves) and 9.7 on 4.
template <typename T>
cudaError_t launch_logprobs(const LpParams& p, int rows, cudaStream_t stream) {
  const long long vecs = (long long)p.vocab * (long long)sizeof(T) / 16;
  int ctas = 8;
  while (ctas > 1 && ((long long)rows * ctas > 256 || vecs < (long long)ctas * 512)) ctas >>= 1;
  return ctas == 1 ? launch_nt<T, 256>(p, rows, 1, stream) : launch_nt<T, 512>(p, rows, ctas, stream);
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
  const LpParams p{logits, tokens, logprobs, entropy, top_logprobs, top_tokens, row_stride, vocab, top_k};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TVK_DTYPE_F16: TVK_CHECK_CUDA(launch_logprobs<__half>(p, rows, s)); break;
    case TVK_DTYPE_BF16: TVK_CHECK_CUDA(launch_logprobs<__nv_bfloat16>(p, rows, s)); break;
    default: TVK_CHECK_CUDA(launch_logprobs<float>(p, rows, s)); break;
  }
  TVK_CHECK_LAUNCH("token_logprobs");
  return TVK_OK;
}
