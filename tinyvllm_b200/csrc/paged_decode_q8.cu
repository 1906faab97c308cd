// paged_decode_q8.cu -- paged-decode attention over the 8-bit K/V cache
// (e4m3 codes with one fp32 scale per block and KV head, K and V apart):
//
//   s_t = k_scale[blk(t), h] * (q . kcode_t) / sqrt(D)
//   out = sum_t softmax(s)_t * v_scale[blk(t), h] * vcode_t,   t < min(context, table)
//
// The scales never touch the codes: a score is scaled after its dot product and
// a block's share of the output after its P.V, both in fp32, so codes go to the
// arithmetic exactly (every e4m3 value is a half) whatever the scales are.
//
// Work split.  The live tokens of all (sequence, KV head) units are laid out on
// one line in tiles of 64 tokens (plus a few tiles' worth per unit for its start
// and end) and cut into equal pieces, one per CTA; heads of a sequence lie next
// to each other.  Every CTA works its piece out of the context lengths alone.  A
// unit that lies in one piece is written at once; one cut by a border leaves fp32
// partials (max, sum, unnormalised output) in the workspace, and the CTA that
// arrives last at the unit's counter adds them up in CTA order, so the result does
// not depend on who that is.  Nobody waits for anybody.
#include <math.h>

#include "kv_cache_q8.cuh"

namespace {

constexpr int kTile = 64;            // tokens per tile of the work line
constexpr int kSimtTile = 32;        // tokens the simt kernel stages at a time
constexpr int kMaxGroup = 16;        // query heads per KV head
constexpr int kMaxCtas = 592;        // pieces a call is cut into at most (four CTAs on each of 148 SMs)
constexpr int kUnitTiles = 2;        // what a unit's start and end count as on the work line
constexpr int kMinPiece = 4;         // shortest piece, in tiles
constexpr int kSlotFloats = 2240;    // partials of one cut unit: rows * (D + 2), at most 64 * 34, 32 * 66 or 16 * 130

struct Q8Params {
  const void* q;
  void* out;
  const int32_t* block_tables;
  const int32_t* context_lens;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int* status;
  float* part;     // [2 * kMaxCtas][kSlotFloats]
  int* counters;   // [batch * n_kv_heads], zero between calls
  int batch, n_heads, n_kv_heads, group, block_size, num_blocks, max_blocks;
  int max_ctx_tokens;
  float scale_log2;  // log2(e) / sqrt(head_dim)
};

__device__ __forceinline__ int effective_ctx(const Q8Params& p, int b) {
  const int c = p.context_lens[b];
  return c < 0 ? 0 : (c < p.max_ctx_tokens ? c : p.max_ctx_tokens);
}
__device__ __forceinline__ int tiles_of(int ctx) { return (ctx + kTile - 1) / kTile; }

// One CTA's share of one unit: tokens [tok0, tok1) of (b, h).  A unit without
// context is one share with tok0 == tok1 and n_parts 1.
struct Share {
  int b, h, ctx, tok0, tok1;
  int n_parts;    // CTAs that share the unit
  int first_cta;  // the first of them
};

// Walks the units of this CTA's piece.  `heads` = units per sequence.  All
// members are the same in every lane of the calling warp.
struct Walker {
  long long x0, x1, total;
  int pieces, heads;
  int b, h, ctx;
  long long at;  // line position where unit (b, h) starts

  // The whole warp calls this.
  __device__ void start(const Q8Params& p, int heads_, int lane) {
    heads = heads_;
    long long sum = 0;
    for (int i = lane; i < p.batch; i += 32) sum += tiles_of(effective_ctx(p, i)) + kUnitTiles;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    total = sum * heads;
    pieces = (int)min((long long)gridDim.x, (total + kMinPiece - 1) / kMinPiece);
    b = p.batch;
    if ((int)blockIdx.x >= pieces) return;
    x0 = total * blockIdx.x / pieces;
    x1 = total * (blockIdx.x + 1) / pieces;
    // the sequence that holds x0
    long long before = 0;
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
      const int i = i0 + lane;
      const int c = i < p.batch ? effective_ctx(p, i) : 0;
      const long long w = i < p.batch ? (long long)(tiles_of(c) + kUnitTiles) * heads : 0;
      long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > x0);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = i0 + l;
        ctx = __shfl_sync(0xffffffffu, c, l);
        at = before + __shfl_sync(0xffffffffu, incl - w, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    const int w = tiles_of(ctx) + kUnitTiles;
    h = (int)((x0 - at) / w);
    at += (long long)h * w;
  }

  // The CTA whose piece holds line position x.
  __device__ int cta_of(long long x) const { return (int)(((x + 1) * pieces - 1) / total); }

  // The next share of the piece; false when there is none left.
  __device__ bool next(const Q8Params& p, Share& s) {
    while (b < p.batch && at < x1) {
      const int tiles = tiles_of(ctx);
      const long long lo = max(x0 - at, 0LL), hi = min(x1 - at, (long long)tiles);
      const bool mine = tiles ? lo < hi : lo == 0;
      s.b = b;
      s.h = h;
      s.ctx = ctx;
      s.tok0 = (int)lo * kTile;
      s.tok1 = min((int)hi * kTile, ctx);
      s.first_cta = blockIdx.x;
      s.n_parts = 1;
      if (tiles && (lo > 0 || hi < tiles)) {
        s.first_cta = cta_of(at);
        s.n_parts = cta_of(at + tiles - 1) - s.first_cta + 1;
      }
      if (!tiles) s.tok0 = s.tok1 = 0;
      at += tiles + kUnitTiles;
      if (++h == heads) {
        h = 0;
        ++b;
        if (b < p.batch) ctx = effective_ctx(p, b);
      }
      if (mine) return true;
    }
    return false;
  }
};

// Where this CTA leaves its partials of a cut unit.  A CTA is the first of at
// most one cut unit (the last of its piece) and a later one of at most one (the
// first of its piece), so two slots do.
__device__ __forceinline__ float* part_slot(const Q8Params& p, int cta, bool is_first) {
  return p.part + (size_t)(cta * 2 + (is_first ? 1 : 0)) * kSlotFloats;
}

// The end of a share, by the NT threads that hold it: `m`, `l` [rows] and `o`
// [rows][D] in shared memory (o unnormalised, relative to m), rows = query heads
// from row0 on of sequence s.b.  Writes the output rows, or the partials, or as the
// last to arrive the sum of all partials.  `flag` is a shared int; `sync` a
// barrier of the NT threads.
template <typename T, int D, int NT, typename Sync>
__device__ void finish_share(const Q8Params& p, const Share& s, int unit, int rows, int row0, const float* m,
                             const float* l, const float* o, int* flag, int tid, Sync sync) {
  T* out = reinterpret_cast<T*>(p.out) + ((size_t)s.b * p.n_heads + row0) * D;
  if (s.n_parts == 1) {
    for (int i = tid; i < rows * D; i += NT) out[i] = DT<T>::from_f(o[i] / l[i / D]);
    return;
  }
  float* mine = part_slot(p, blockIdx.x, (int)blockIdx.x == s.first_cta);
  for (int i = tid; i < rows * D; i += NT) __stcg(mine + i, o[i]);
  for (int i = tid; i < rows; i += NT) {
    __stcg(mine + rows * D + i * 2, m[i]);
    __stcg(mine + rows * D + i * 2 + 1, l[i]);
  }
  __threadfence();
  sync();
  if (tid == 0) {
    const bool last = atomicAdd(p.counters + unit, 1) == s.n_parts - 1;
    if (last) p.counters[unit] = 0;
    *flag = last;
    __threadfence();
  }
  sync();
  if (!*flag) return;
  for (int i = tid; i < rows * D; i += NT) {
    const int r = i / D;
    float M = -INFINITY;
    for (int c = 0; c < s.n_parts; ++c)
      M = fmaxf(M, __ldcg(part_slot(p, s.first_cta + c, c == 0) + rows * D + r * 2));
    float L = 0.f, A = 0.f;
    for (int c = 0; c < s.n_parts; ++c) {
      const float* src = part_slot(p, s.first_cta + c, c == 0);
      const float w = exp2f(__ldcg(src + rows * D + r * 2) - M);
      L = fmaf(__ldcg(src + rows * D + r * 2 + 1), w, L);
      A = fmaf(__ldcg(src + i), w, A);
    }
    out[i] = DT<T>::from_f(A / L);
  }
}

// -----------------------------------------------------------------------------
// SIMT kernel: any query type, any block size; fp32 CUDA-core arithmetic on
// 32-token tiles staged in shared memory.
// -----------------------------------------------------------------------------
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_decode_q8_simt_kernel(const Q8Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int DP = D + 4;
  constexpr int MAXK = kMaxGroup * D / 128;
  __shared__ __align__(16) float qs[kMaxGroup * D];
  __shared__ __align__(16) float ks[kSimtTile][DP];
  __shared__ __align__(16) float vs[kSimtTile][DP];
  __shared__ float ps[kMaxGroup][kSimtTile];
  __shared__ float corr_s[kMaxGroup], mfin[kMaxGroup], lfin[kMaxGroup];
  __shared__ int flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.group, bs = p.block_size, Hkv = p.n_kv_heads;
  Walker w;
  w.start(p, Hkv, lane);
  Share s;
  while (w.next(p, s)) {
    T* out = reinterpret_cast<T*>(p.out) + ((size_t)s.b * p.n_heads + s.h * G) * D;
    if (s.ctx == 0) {
      for (int i = tid; i < G * D; i += 128) out[i] = DT<T>::from_f(0.f);
      continue;
    }
    __syncthreads();
    const T* q = reinterpret_cast<const T*>(p.q) + ((size_t)s.b * p.n_heads + s.h * G) * D;
    for (int i = tid; i < G * D; i += 128) qs[i] = DT<T>::to_f(q[i]);
    const int32_t* bt = p.block_tables + (size_t)s.b * p.max_blocks;
    float acc[MAXK];
#pragma unroll
    for (int k = 0; k < MAXK; ++k) acc[k] = 0.f;
    float m_own[kMaxGroup / 4], l_own[kMaxGroup / 4];  // heads warp, warp + 4, ...
#pragma unroll
    for (int i = 0; i < kMaxGroup / 4; ++i) {
      m_own[i] = -INFINITY;
      l_own[i] = 0.f;
    }
    for (int t0 = s.tok0; t0 < s.tok1; t0 += kSimtTile) {
      __syncthreads();
      for (int i = tid; i < kSimtTile * (D / 4); i += 128) {
        const int t = i / (D / 4), d4 = (i % (D / 4)) * 4;
        float kf[4] = {0.f, 0.f, 0.f, 0.f}, vf[4] = {0.f, 0.f, 0.f, 0.f};
        const int tok = t0 + t;
        if (tok < s.tok1) {
          const int blk = __ldg(bt + tok / bs);
          if (blk >= 0 && blk < p.num_blocks) {
            const size_t off = (((size_t)blk * bs + tok % bs) * Hkv + s.h) * D + d4;
            q8::decode4(*reinterpret_cast<const uint32_t*>(p.k_cache + off), kf);
            q8::decode4(*reinterpret_cast<const uint32_t*>(p.v_cache + off), vf);
            const float sk = p.k_scale[(size_t)blk * Hkv + s.h], sv = p.v_scale[(size_t)blk * Hkv + s.h];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              kf[e] *= sk;
              vf[e] *= sv;
            }
          }
        }
        *reinterpret_cast<float4*>(&ks[t][d4]) = make_float4(kf[0], kf[1], kf[2], kf[3]);
        *reinterpret_cast<float4*>(&vs[t][d4]) = make_float4(vf[0], vf[1], vf[2], vf[3]);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kMaxGroup / 4; ++i) {
        const int gh = warp + 4 * i;
        if (gh < G) {
          float x = 0.f;
#pragma unroll 8
          for (int d = 0; d < D; d += 4) {
            const float4 kk = *reinterpret_cast<const float4*>(&ks[lane][d]);
            const float4 qq = *reinterpret_cast<const float4*>(&qs[gh * D + d]);
            x = fmaf(qq.x, kk.x, x);
            x = fmaf(qq.y, kk.y, x);
            x = fmaf(qq.z, kk.z, x);
            x = fmaf(qq.w, kk.w, x);
          }
          x = (t0 + lane < s.tok1) ? x * p.scale_log2 : -INFINITY;
          float mx = x;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const float mn = fmaxf(m_own[i], mx);
          const float corr = exp2f(m_own[i] - mn);
          const float pv = exp2f(x - mn);
          float sum = pv;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          l_own[i] = l_own[i] * corr + sum;
          m_own[i] = mn;
          ps[gh][lane] = pv;
          if (lane == 0) corr_s[gh] = corr;
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < MAXK; ++k) {
        const int idx = tid + 128 * k;
        if (idx < G * D) {
          const int gh = idx / D, d = idx % D;
          float a = acc[k] * corr_s[gh];
#pragma unroll 8
          for (int t = 0; t < kSimtTile; ++t) a = fmaf(ps[gh][t], vs[t][d], a);
          acc[k] = a;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kMaxGroup / 4; ++i) {
      const int gh = warp + 4 * i;
      if (gh < G && lane == 0) {
        mfin[gh] = m_own[i];
        lfin[gh] = l_own[i];
      }
    }
    // the query rows are done with: their place takes the output sums
#pragma unroll
    for (int k = 0; k < MAXK; ++k) {
      const int idx = tid + 128 * k;
      if (idx < G * D) qs[idx] = acc[k];
    }
    __syncthreads();
    finish_share<T, D, 128>(p, s, s.b * Hkv + s.h, G, s.h * G, mfin, lfin, qs, &flag, tid, [] { __syncthreads(); });
  }
}

template <typename T>
int launch_simt(const Q8Params& p, int head_dim, cudaStream_t stream) {
  const long long most = (long long)p.batch * p.n_kv_heads * ((p.max_ctx_tokens + kTile - 1) / kTile + kUnitTiles);
  const long long pieces = (most + kMinPiece - 1) / kMinPiece;
  const int grid = (int)(pieces < kMaxCtas ? pieces : kMaxCtas);
  switch (head_dim) {
    case 32: TVK_CHECK_CUDA(tvk::launch_pdl(paged_decode_q8_simt_kernel<T, 32>, grid, 128, 0, stream, p)); break;
    case 64: TVK_CHECK_CUDA(tvk::launch_pdl(paged_decode_q8_simt_kernel<T, 64>, grid, 128, 0, stream, p)); break;
    default: TVK_CHECK_CUDA(tvk::launch_pdl(paged_decode_q8_simt_kernel<T, 128>, grid, 128, 0, stream, p)); break;
  }
  TVK_CHECK_LAUNCH("paged_decode_q8_simt");
  return TVK_OK;
}

}  // namespace

extern "C" size_t tvk_paged_decode_q8_workspace_size(int batch, int n_kv_heads) {
  size_t units = batch > 0 && n_kv_heads > 0 ? (size_t)batch * n_kv_heads : 0;
  return tvk::kWorkspaceHeader + (size_t)2 * kMaxCtas * kSlotFloats * sizeof(float) + units * sizeof(int);
}

extern "C" int tvk_paged_decode_attention_q8(const void* q, const void* k_cache, const void* v_cache,
                                             const float* k_scale, const float* v_scale, const int32_t* block_tables,
                                             const int32_t* context_lens, void* out, int batch, int n_heads,
                                             int n_kv_heads, int head_dim, int block_size, int num_blocks,
                                             int max_blocks, int max_context_len, int dtype, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  TVK_CHECK_ARG(batch >= 0, "batch must be >= 0 (got %d)", batch);
  TVK_CHECK_ARG(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0,
                "n_heads (%d) must be a positive multiple of n_kv_heads (%d)", n_heads, n_kv_heads);
  TVK_CHECK_ARG(n_heads / n_kv_heads <= kMaxGroup, "n_heads / n_kv_heads = %d exceeds %d", n_heads / n_kv_heads,
                kMaxGroup);
  TVK_CHECK_ARG(block_size > 0 && num_blocks > 0 && max_blocks > 0,
                "block_size, num_blocks and max_blocks must be positive");
  TVK_CHECK_ARG((long long)max_blocks * block_size < 0x7fffffffLL, "a table spans more than 2^31 tokens");
  TVK_CHECK_ARG((long long)batch * n_kv_heads * ((long long)max_blocks * block_size / kTile + 1 + kUnitTiles) < 0x7fffffffLL,
                "batch x KV heads x table tiles exceeds the 32-bit work index");
  TVK_CHECK_ARG(dtype == TVK_DTYPE_F32 || dtype == TVK_DTYPE_F16 || dtype == TVK_DTYPE_BF16, "unknown dtype %d", dtype);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) {
    tvk::set_error("head_dim %d unsupported (32, 64 or 128)", head_dim);
    return TVK_ERR_UNSUPPORTED;
  }
  if (batch == 0) return TVK_OK;
  TVK_CHECK_ARG(q && k_cache && v_cache && k_scale && v_scale && block_tables && context_lens && out,
                "null pointer argument");
  TVK_CHECK_ARG(((uintptr_t)q % 16 == 0) && ((uintptr_t)k_cache % 16 == 0) && ((uintptr_t)v_cache % 16 == 0) &&
                    ((uintptr_t)out % 4 == 0),
                "q, k_cache and v_cache must be 16-byte aligned");
  const size_t need = tvk_paged_decode_q8_workspace_size(batch, n_kv_heads);
  if (!workspace || workspace_bytes < need) {
    tvk::set_error("workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    return TVK_ERR_WORKSPACE;
  }
  TVK_CHECK_ARG((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  Q8Params p{};
  p.q = q;
  p.out = out;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.k_cache = (const uint8_t*)k_cache;
  p.v_cache = (const uint8_t*)v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.status = (int*)workspace;
  p.part = (float*)((uint8_t*)workspace + tvk::kWorkspaceHeader);
  p.counters = (int*)(p.part + (size_t)2 * kMaxCtas * kSlotFloats);
  p.batch = batch;
  p.n_heads = n_heads;
  p.n_kv_heads = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.max_blocks = max_blocks;
  int blocks = max_blocks;
  if (max_context_len >= 0) {
    const int cut = (int)(((long long)max_context_len + block_size - 1) / block_size);
    blocks = cut < max_blocks ? cut : max_blocks;
  }
  p.max_ctx_tokens = blocks * block_size;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TVK_DTYPE_F16: return launch_simt<__half>(p, head_dim, s);
    case TVK_DTYPE_BF16: return launch_simt<__nv_bfloat16>(p, head_dim, s);
    default: return launch_simt<float>(p, head_dim, s);
  }
}
