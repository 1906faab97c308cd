// paged_decode_q8.cu -- paged-decode attention over the 8-bit K/V cache
// (e4m3 codes with one fp32 scale per block and KV head, K and V apart):
//
//   s_t = k_scale[blk(t), h] * (q . kcode_t) / sqrt(D)
//   out = sum_t softmax(s)_t * v_scale[blk(t), h] * vcode_t,   t < min(context, table)
//
// The scales never touch the codes: a score is scaled after its dot product, and
// a block's v_scale goes into the weights of its tokens, both in fp32.
//
// Work split.  The live tokens of all (sequence, KV head) units are laid out on
// one line in tiles of tokens (plus two tiles' worth per unit for its start and
// end), heads of a sequence next to each other, and cut into equal pieces, one per CTA,
// which every CTA works out from the context lengths alone.  A unit of few tiles
// belongs whole to the piece that it starts in.  A longer one that a border cuts
// leaves fp32 partials (max, sum, unnormalised output) by piece in the workspace, and
// the CTA that arrives last at the unit's counter adds them up in piece order, so the
// result does not depend on who that is.  Nobody waits for anybody.  (Leaving the
// line's last fifth to the CTAs that are done first, in smaller pieces by ticket, was
// no gain: 256 sequences of 128-4096 tokens 229 us instead of 208, long ones 82 instead of 57,
// for the joins of many parts.)
#include <math.h>

#include <type_traits>

#include "kv_cache_q8.cuh"
#include "sm100_umma.cuh"

namespace {

constexpr int kSimtTile = 128;       // tokens the simt kernel's four warps go through at a time, and its tile of the work line
constexpr int kSimtWhole = 2;        // its units of up to so many tiles are not cut
constexpr int kTcTile = 128;         // the same for the tensor-core kernel: the rows of a matrix instruction
constexpr int kTcWhole = 6;          // joining parts costs as much as 4 to 5 tiles in a row
constexpr int kMaxGroup = 16;        // query heads per KV head
constexpr int kSimtCtas = 592;       // four CTAs on each of 148 SMs (with 16 query heads two fit, and the others follow as those end)
constexpr int kTcCtas = 296;         // two CTAs on each SM
constexpr int kMaxPieces = kSimtCtas;
constexpr int kUnitTiles = 2;        // what a unit's start and end count as on the work line
constexpr int kMaxParts = 4;         // units per (sequence, KV head) at most, where groups are split
constexpr int kSlotFloats = 2080;    // partials of one cut unit: rows * (D + 2), at most 16 * 130

struct Q8Params {
  const void* q;
  void* out;
  const int32_t* block_tables;
  const int32_t* context_lens;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int* status;
  float* part;     // [2 * kMaxPieces][kSlotFloats]
  int* counters;   // [batch * n_kv_heads * kMaxParts], zero between calls
  int batch, n_heads, n_kv_heads, group, block_size, num_blocks, max_blocks;
  int max_ctx_tokens;
  int team;                    // tensor-core kernel: CTAs that walk one piece, each its own unit of every group
  float scale_log2;            // log2(e) / sqrt(head_dim)
  int n_stages;                // ring depth of the tensor-core kernel
  unsigned long long wait_ns;  // wall-time limit of every mbarrier wait
  int dtype;                   // of q and out
  int drop_loads;              // wait-limit test: the producer issues nothing, so waits run out
};

__device__ __forceinline__ int effective_ctx(const Q8Params& p, int b) {
  const int c = p.context_lens[b];
  return c < 0 ? 0 : (c < p.max_ctx_tokens ? c : p.max_ctx_tokens);
}
__host__ __device__ __forceinline__ int tiles_of(int ctx, int tile) { return (ctx + tile - 1) / tile; }

// One piece's share of one unit: tokens [tok0, tok1) of (b, h).  A unit without
// context is one share with tok0 == tok1.
struct Share {
  int b, h, ctx, tok0, tok1;
  int piece;
  int n_parts;      // pieces that share the unit
  int first_piece;  // the first of them
};

// The line and its equal pieces.
struct Cut {
  long long total;
  int pieces;

  __device__ void make(long long total_, int ctas) {
    total = total_;
    pieces = (int)(total < ctas ? total : ctas);
  }
  __device__ long long start(int i) const { return total * i / pieces; }
  __device__ int piece_of(long long x) const { return (int)(((x + 1) * pieces - 1) / total); }
};

// Walks the units of one piece.  `heads` = units per sequence.  WHOLE: units of up to so
// many tiles are never cut.
template <int TILE, int WHOLE>
struct Walker {
  long long x0, x1;  // the piece
  long long at;      // line position where unit (b, h) starts
  int b, h, ctx, next_ctx, piece;

  // Length of the line; the whole warp calls this.
  static __device__ long long line(const Q8Params& p, int heads, int lane) {
    long long sum = 0;
    for (int i = lane; i < p.batch; i += 32) sum += tiles_of(effective_ctx(p, i), TILE) + kUnitTiles;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum * heads;
  }

  // To the unit that holds the start of piece i; the whole warp calls this.
  __device__ void seek(const Q8Params& p, const Cut& cut, int heads, int i_piece, int lane) {
    piece = i_piece;
    x0 = cut.start(i_piece);
    x1 = cut.start(i_piece + 1);
    long long before = 0;
    b = p.batch;
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
      const int i = i0 + lane;
      const int c = i < p.batch ? effective_ctx(p, i) : 0;
      const long long w = i < p.batch ? (long long)(tiles_of(c, TILE) + kUnitTiles) * heads : 0;
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
    if (b >= p.batch) return;
    const int w = tiles_of(ctx, TILE) + kUnitTiles;
    h = (int)((x0 - at) / w);
    at += (long long)h * w;
    next_ctx = b + 1 < p.batch ? effective_ctx(p, b + 1) : 0;
  }

  // The next share of the piece; false when there is none left.
  __device__ bool next(const Q8Params& p, const Cut& cut, int heads, Share& s) {
    while (b < p.batch && at < x1) {
      const int tiles = tiles_of(ctx, TILE);
      long long lo = max(x0 - at, 0LL), hi = min(x1 - at, (long long)tiles);
      bool mine = lo < hi;
      s.n_parts = 1;
      if (tiles <= WHOLE) {
        mine = lo == 0;  // it starts here
        hi = tiles;
      } else if (mine && (lo > 0 || hi < tiles)) {
        s.first_piece = cut.piece_of(at);
        s.n_parts = cut.piece_of(at + tiles - 1) - s.first_piece + 1;
      }
      s.b = b;
      s.h = h;
      s.ctx = ctx;
      s.piece = piece;
      s.tok0 = (int)lo * TILE;
      s.tok1 = min((int)hi * TILE, ctx);
      at += tiles + kUnitTiles;
      if (++h == heads) {
        h = 0;
        ++b;
        ctx = next_ctx;
        next_ctx = b + 1 < p.batch ? effective_ctx(p, b + 1) : 0;  // not needed before the next sequence
      }
      if (mine) return true;
    }
    return false;
  }
};

// Where a CTA leaves its partials of a cut unit.  Its piece is the first of at most
// one cut unit (its last) and a later one of at most one (its first), so two slots do.
__device__ __forceinline__ float* part_slot(const Q8Params& p, int cta, bool is_first) {
  return p.part + (size_t)(cta * 2 + (is_first ? 1 : 0)) * kSlotFloats;
}
__device__ __forceinline__ float* part_of(const Q8Params& p, const Share& s, int c) {
  return part_slot(p, s.first_piece + c, c == 0);
}

// Counts the arrival of a share of a cut unit whose partials the calling threads
// have just stored with __stcg; true in all of them for the last to arrive.
// `flag` is a shared int; `sync` a barrier of these threads.
template <typename Sync>
__device__ bool last_to_arrive(const Q8Params& p, const Share& s, int unit, int* flag, int tid, Sync sync) {
  __threadfence();
  sync();
  if (tid == 0) {
    const bool last = atomicAdd(p.counters + unit, 1) == s.n_parts - 1;
    if (last) p.counters[unit] = 0;
    *flag = last;
    __threadfence();
  }
  sync();
  return *flag != 0;
}

// Element i (of row r) of a cut unit's output from all its partials, each
// [n_o] unnormalised sums and then (max, sum) of every row.
__device__ __forceinline__ float joined(const Q8Params& p, const Share& s, int n_o, int i, int r) {
  float M = -INFINITY;
  for (int c = 0; c < s.n_parts; ++c) M = fmaxf(M, __ldcg(part_of(p, s, c) + n_o + r * 2));
  float L = 0.f, A = 0.f;
#pragma unroll 4
  for (int c = 0; c < s.n_parts; ++c) {
    const float* src = part_of(p, s, c);
    const float w = exp2f(__ldcg(src + n_o + r * 2) - M);
    L = fmaf(__ldcg(src + n_o + r * 2 + 1), w, L);
    A = fmaf(__ldcg(src + i), w, A);
  }
  return A / L;
}

// Largest value of a warp (NaN only where all are).
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// -----------------------------------------------------------------------------
// SIMT kernel: any query type, any block size; fp32 CUDA-core arithmetic.
//
// Each of four warps goes through 32-token tiles of its own (every fourth of the share), whose
// codes it copies to its part of shared memory: K of the next tile while it works on the weights,
// V of the next while on the scores.  Scores: a lane per token, 16 codes at a time decoded to
// registers and used for all GM query heads, whose elements are broadcast from shared memory (one
// such read per four products).  Output: a lane per D / 32 dims, the weights (v_scale in them) broadcast
// likewise.  Running maxima and sums are the warp's own; the four are put together at the end.
//
// Broadcast reads and products bound it: fp32, 16 sequences of 128-4096 tokens, 32/4 heads of 64 33 us, 8 with
// 32/8 of 128 35 us (1.1 TB/s), 64 with 16/1 of 128 107-114 us, 4 sequences of 17-255 with 32/4 of 64 9.2 us.  (Codes decoded
// to floats in shared memory by the whole CTA, a head per warp, took 60, 79, 174 and 14.5 us.)
// -----------------------------------------------------------------------------
constexpr int kSimtWarpTile = 32;

template <int D, int GM>
struct SimtLayout {
  static constexpr int kPitch = D + 16;  // bytes of a row of codes: rows of 8 lanes in different banks
  static constexpr int kCodes = kSimtWarpTile * kPitch;
  static constexpr int kWarp = 2 * kCodes + 2 * kSimtWarpTile * 4 + kSimtWarpTile * GM * 4;  // K, V, scales, weights
  static constexpr int kBytes = GM * D * 4 + 4 * kWarp;
  static_assert(GM * D * 4 + GM * 8 <= kWarp, "a warp's sums take the place of its tiles");
};

__device__ __forceinline__ float load_as_float(const void* x, size_t i, int dtype) {
  if (dtype == TVK_DTYPE_F32) return static_cast<const float*>(x)[i];
  if (dtype == TVK_DTYPE_F16) return DT<__half>::to_f(static_cast<const __half*>(x)[i]);
  return DT<__nv_bfloat16>::to_f(static_cast<const __nv_bfloat16*>(x)[i]);
}
__device__ __forceinline__ void store_from_float(void* x, size_t i, float v, int dtype) {
  if (dtype == TVK_DTYPE_F32)
    static_cast<float*>(x)[i] = v;
  else if (dtype == TVK_DTYPE_F16)
    static_cast<__half*>(x)[i] = DT<__half>::from_f(v);
  else
    static_cast<__nv_bfloat16*>(x)[i] = DT<__nv_bfloat16>::from_f(v);
}

// CTAs on an SM: four; two with the sums of 16 heads (64 sequences with 16/1 heads take 118 us with three and 107 with two).
template <int D, int GM>
__global__ void __launch_bounds__(128, GM == 16 ? 2 : 4) paged_decode_q8_simt_kernel(const Q8Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  using L = SimtLayout<D, GM>;
  constexpr int DV = D / 32;
  extern __shared__ __align__(16) uint8_t simt_smem[];
  __shared__ int flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* qs = reinterpret_cast<float*>(simt_smem);  // [GM][D]
  uint8_t* mine = simt_smem + GM * D * 4 + warp * L::kWarp;
  uint8_t* codes[2] = {mine, mine + L::kCodes};
  float* scales = reinterpret_cast<float*>(mine + 2 * L::kCodes);  // [K, V][token]
  float* ps = scales + 2 * kSimtWarpTile;                          // [token][GM]
  const int G = p.group, bs = p.block_size, Hkv = p.n_kv_heads;
  using Walk = Walker<kSimtTile, kSimtWhole>;
  Cut cut;
  cut.make(Walk::line(p, Hkv, lane), gridDim.x);
  if ((int)blockIdx.x >= cut.pieces) return;
  Walk w;
  w.seek(p, cut, Hkv, blockIdx.x, lane);
  Share s;
  while (w.next(p, cut, Hkv, s)) {
    const size_t out0 = ((size_t)s.b * p.n_heads + s.h * G) * D;
    if (s.ctx == 0) {
      for (int i = tid; i < G * D; i += 128) store_from_float(p.out, out0 + i, 0.f, p.dtype);
      continue;
    }
    __syncthreads();
    for (int i = tid; i < GM * D; i += 128) qs[i] = i < G * D ? load_as_float(p.q, out0 + i, p.dtype) : 0.f;
    __syncthreads();
    const int32_t* bt = p.block_tables + (size_t)s.b * p.max_blocks;
    const int step = 4 * kSimtWarpTile;
    // this lane's block of the tile at t0, -1 where there is none
    auto block_of = [&](int t0) -> int {
      const int blk = t0 + lane < s.tok1 ? __ldg(bt + (t0 + lane) / bs) : -1;
      return blk < p.num_blocks ? blk : -1;
    };
    // K (kv 0) or V codes and scales of the tile at t0, one group of copies; zeros where there are none
    auto issue = [&](int kv, int t0, int blk) {
      const uint8_t* pool = kv ? p.v_cache : p.k_cache;
      constexpr int kChunks = D / 16, kRows = 32 / kChunks;  // 16-byte chunks of a row, rows at a time
      const size_t row = ((size_t)(blk < 0 ? 0 : blk) * bs + (t0 + lane) % bs) * Hkv + s.h;
#pragma unroll
      for (int r = 0; r < kSimtWarpTile; r += kRows) {
        const int t = r + lane / kChunks;
        const size_t at = __shfl_sync(0xffffffffu, (unsigned long long)row, t);
        const bool live = __shfl_sync(0xffffffffu, blk, t) >= 0;
        ptx::copy16_async_or_zeros(ptx::smem_u32(codes[kv] + t * L::kPitch + lane % kChunks * 16), pool + at * D + lane % kChunks * 16, live);
      }
      const float* src = kv ? p.v_scale : p.k_scale;
      q8::copy4_async(ptx::smem_u32(scales + kv * kSimtWarpTile + lane), blk >= 0 ? src + (size_t)blk * Hkv + s.h : src, blk >= 0);
      ptx::commit_copies();
    };
    float acc[GM][DV], m[GM], l[GM];
#pragma unroll
    for (int h = 0; h < GM; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int k = 0; k < DV; ++k) acc[h][k] = 0.f;
    }
    const int first = s.tok0 + warp * kSimtWarpTile;
    int blk = first < s.tok1 ? block_of(first) : -1;
    if (first < s.tok1) {
      issue(0, first, blk);
      issue(1, first, blk);
    }
    for (int t0 = first; t0 < s.tok1; t0 += step) {
      const int next = block_of(t0 + step);  // all -1 behind the end: the copies are zeros that nobody reads
      ptx::wait_copies_but<1>();
      __syncwarp();
      float x[GM];
#pragma unroll
      for (int h = 0; h < GM; ++h) x[h] = 0.f;
#pragma unroll 1
      for (int d = 0; d < D; d += 16) {
        const uint4 c = *reinterpret_cast<const uint4*>(codes[0] + lane * L::kPitch + d);
        float f[16];
        q8::decode4(c.x, f);
        q8::decode4(c.y, f + 4);
        q8::decode4(c.z, f + 8);
        q8::decode4(c.w, f + 12);
#pragma unroll
        for (int h = 0; h < GM; ++h)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 q4 = *reinterpret_cast<const float4*>(qs + h * D + d + e);
            x[h] = fmaf(q4.x, f[e], x[h]);
            x[h] = fmaf(q4.y, f[e + 1], x[h]);
            x[h] = fmaf(q4.z, f[e + 2], x[h]);
            x[h] = fmaf(q4.w, f[e + 3], x[h]);
          }
      }
      const float sk = scales[lane] * p.scale_log2;
      const bool live = t0 + lane < s.tok1;
      __syncwarp();  // every lane has read K and its scale
      issue(0, t0 + step, next);
      float corr[GM];
      ptx::wait_copies_but<1>();
      const float sv = scales[kSimtWarpTile + lane];
#pragma unroll
      for (int h = 0; h < GM; ++h) {
        x[h] = live ? x[h] * sk : -INFINITY;
        const float mn = fmaxf(m[h], warp_max(x[h]));
        corr[h] = exp2f(m[h] - mn);
        m[h] = mn;
        const float pv = exp2f(x[h] - mn);
        l[h] = fmaf(l[h], corr[h], pv);
        x[h] = live ? pv * sv : 0.f;
      }
#pragma unroll
      for (int h = 0; h < GM; h += 4)
        *reinterpret_cast<float4*>(ps + lane * GM + h) = make_float4(x[h], x[h + 1], x[h + 2], x[h + 3]);
      __syncwarp();  // weights and V are there
#pragma unroll
      for (int h = 0; h < GM; ++h)
#pragma unroll
        for (int k = 0; k < DV; ++k) acc[h][k] *= corr[h];
#pragma unroll 2
      for (int t = 0; t < kSimtWarpTile; ++t) {
        const uint8_t* at = codes[1] + t * L::kPitch + lane * DV;
        const uint32_t c = DV == 4 ? *reinterpret_cast<const uint32_t*>(at) : DV == 2 ? *reinterpret_cast<const uint16_t*>(at) : *at;
        float f[4];
        q8::decode4(c, f);
#pragma unroll
        for (int h = 0; h < GM; h += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(ps + t * GM + h);
#pragma unroll
          for (int k = 0; k < DV; ++k) {
            acc[h][k] = fmaf(w4.x, f[k], acc[h][k]);
            acc[h + 1][k] = fmaf(w4.y, f[k], acc[h + 1][k]);
            acc[h + 2][k] = fmaf(w4.z, f[k], acc[h + 2][k]);
            acc[h + 3][k] = fmaf(w4.w, f[k], acc[h + 3][k]);
          }
        }
      }
      __syncwarp();  // every lane has read V and the weights
      issue(1, t0 + step, next);
    }
    // The warps' sums, relative to each warp's maxima, in place of its tiles.
    ptx::wait_copies();
    __syncwarp();
    float* sums = reinterpret_cast<float*>(mine);  // [GM][D], then (maximum, sum) of every head
#pragma unroll
    for (int h = 0; h < GM; ++h) {
      float sum = l[h];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
      for (int k = 0; k < DV; ++k) sums[h * D + lane * DV + k] = acc[h][k];
      if (lane == 0) {
        sums[GM * D + h * 2] = m[h];
        sums[GM * D + h * 2 + 1] = sum;
      }
    }
    __syncthreads();
    float* part = s.n_parts == 1 ? nullptr : part_slot(p, s.piece, s.piece == s.first_piece);
    const float* all = reinterpret_cast<const float*>(simt_smem + GM * D * 4);
    constexpr int kStride = L::kWarp / 4;
    for (int i = tid; i < G * D; i += 128) {
      const int h = i / D;
      float M = -INFINITY, A = 0.f, Ls = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) M = fmaxf(M, all[k * kStride + GM * D + h * 2]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = exp2f(all[k * kStride + GM * D + h * 2] - M);
        A = fmaf(all[k * kStride + i], f, A);
        Ls = fmaf(all[k * kStride + GM * D + h * 2 + 1], f, Ls);
      }
      if (part) {
        __stcg(part + i, A);
        if (i % D == 0) {
          __stcg(part + G * D + h * 2, M);
          __stcg(part + G * D + h * 2 + 1, Ls);
        }
      } else {
        store_from_float(p.out, out0 + i, A / Ls, p.dtype);
      }
    }
    if (part && last_to_arrive(p, s, s.b * Hkv + s.h, &flag, tid, [] { __syncthreads(); }))
      for (int i = tid; i < G * D; i += 128) store_from_float(p.out, out0 + i, joined(p, s, G * D, i, i / D), p.dtype);
  }
}

// -----------------------------------------------------------------------------
// tcgen05 kernel: 16-bit queries; block sizes 8, 16, 32, 64 and multiples of 128.
//
// A unit is HP = 128 / D neighbouring KV heads of one sequence, so that a token's
// codes are one 128-byte row whatever D is, and up to GP query heads of each
// (larger groups take several units).  The codes are matrix operands as TMA
// lands them, 128 tokens a tile:
//   S^T [128 tokens, 4 GP] = K . Q^T         per KV head; K rows are K-major (128 B swizzle)
//   O^T [128 dims, 4 GP HP] += V^T . P^T     V rows read M-major; all heads at once, a head's
//                                            dims times other heads' columns are not read
// and what has more bits than e4m3 comes in parts, each a column (slot) of its own:
//  * a query row, scaled by a power of two to a maximum in [2^7, 2^8), is
//    q1 + q2 + q3 + 2^-8 q4, each part the e4m3 of what is left: 4 significant bits
//    a part, exact for fp16 and bf16 down to 2^-18 of 2^7, i.e. 2^-25 of the maximum;
//  * a weight 2^(s + log2 v_scale - M), at most 2^15, is p1 + p2 + 2^-8 (p3 + p4), each part the
//    e5m2 of what is left: three significant bits and the sign of the rest make four bits a part, and
//    e5m2's five exponent bits reach from 2^15 to 2^-16, so that a long tail behind one heavy
//    token counts.  After p1 what is left is a half (2^-15 of the weight, 2^-25 at least), which the
//    others hold exactly; the largest weight counts as 2^11..2^15.  (Three parts in e4m3, the first of a
//    weight as a half, end at 2^-23 of the largest: weights below that, nearly all of a long tail, were
//    lost, and the output was off by up to half of sum p|v|.)
// The matrix unit sums in fp32.  So nothing is converted per K/V element: the work of
// the CUDA cores is per (token, query head).  (Decoding the codes to halves for
// mma.sync took 470 instructions per 16 tokens and 265 us where this took 218 us in
// its first form: 256 sequences of 128-4096 tokens, 32/8 heads of 128.  mma.sync on e4m3
// itself is emulated on this architecture and took longer still.)
//
// Now that call takes 184-198 us (from box to box), 5.7-6.1 TB/s of codes and scales, 0.87-0.92
// of the measured copy rate: memory bounds units of 4 heads.  With 8 heads a unit
// 5.3 TB/s, with 16 2.6 TB/s (32/4 and 32/2 heads of 128, the same sequences):
// there the softmax warps' work per (token, query head) bounds it, about half of that
// the parts of a weight and their byte stores.  (The fourth part costs nothing at 4 heads a unit, 3 % at
// 8 and 10 % at 16: 102.9 -> 106.4 and 99.6 -> 110.2 us.)
//
// Roles: warp 0 streams K tiles (TMA) and their scales (4-byte asynchronous
// copies), warp 3 V; warp 1 issues the products; warp 2 splits the query rows of the next share;
// warps 4-7, a thread per token, turn S^T into weights, keep the sums of weights, and
// at a share's end, a thread per dim, read O^T and write the output.
// K and V tiles go through one ring of 16 KB slots in the order the products take
// them, K(0) K(1) V(0) K(2) V(1) ..., so that a K tile's slot is free again as soon as
// its S^T is there and not only after the weights and P.V.
// M and the reference R of the sums are per query head, the same in all threads.
// They move only when a weight would pass 2^15 (or a sum's term 2^64); then O^T is rescaled.
// -----------------------------------------------------------------------------
constexpr int kTcThreads = 256;
// Tiles whose scales are kept.  A producer writes a tile's scales once it has the tile's slot, which is free when
// the product of the tile at least (kSlots - 1) / 2 before is done; S^T being double, the softmax is at most two
// tiles behind that: 7 slots make 5 tiles in all.
constexpr int kScaleRing = 8;
constexpr float kLowPart = 0.00390625f;  // 2^-8
constexpr float kTopWeight = 11.f, kMostWeight = 15.f;  // log2 of what the largest weight counts as: when a reference is set, and at most

template <int D, int GP>
struct TcLayout {
  static constexpr int HP = 128 / D;
  static constexpr int HG = HP * GP;                    // query heads of a unit
  static constexpr int NS = 4 * GP;                     // columns of S^T of one KV head: (part, head)
  static constexpr int NO = 4 * HG;                     // columns of O^T: (part, KV head, head)
  static constexpr int kOCol = 2 * HP * NS;             // after two buffers of S^T
  static constexpr int kTmemCols = kOCol + NO <= 64 ? 64 : kOCol + NO <= 128 ? 128 : 256;
  static constexpr int kSlot = kTcTile * 128;           // K or V codes of a tile
  static constexpr int kQ = HP * NS * 128;              // query parts, one row of 128 B per column
  static constexpr int kQBufs = HG == 16 ? 1 : 2;
  static constexpr int kP = NO * 128;                   // weight parts: one row of 128 tokens per column
  static constexpr int kScale = 2 * HP * 16 * 4;        // K and V, HP heads, <= 16 blocks
  static constexpr int kMisc = 1536, kBars = 320;
  static constexpr int kFixed = kQBufs * kQ + 2 * kP + kScaleRing * kScale + kMisc + kBars + 1024;
  static constexpr int kSlots = (113 * 1024 - kFixed) / kSlot;  // two CTAs on an SM
  static constexpr int kQOff = kSlots * kSlot;
  static constexpr int kPOff = kQOff + kQBufs * kQ;
  static constexpr int kScaleOff = kPOff + 2 * kP;
  static constexpr int kMiscOff = kScaleOff + kScaleRing * kScale;
  static constexpr int kBarOff = kMiscOff + kMisc;
  static constexpr int kBytes = kBarOff + kBars + 1024;
  static_assert(HG <= 16 && kOCol + NO <= 256 && kSlots >= 5 && kSlots <= 7, "sizes");
  static_assert((2 * kSlots + kScaleRing + 15) * 8 <= kBars, "barriers");
  static_assert(HG * (D + 2) <= kSlotFloats, "partials");
  static_assert(2 * kP / 4 >= HG * 8, "room for the join's factors of some parts at a time");
};

// Byte of row r of a tile with 128-byte rows in the 128-byte swizzle.
__device__ __forceinline__ uint32_t swz128(int r, int byte) {
  return r * 128 + ((((byte >> 4) ^ (r & 7)) & 7) << 4) + (byte & 15);
}

// Four neighbouring values -> q1, q2, q3 and 2^8 (what is left), e4m3, four bytes each.
__device__ __forceinline__ void split_query(float (&x)[4], uint32_t (&w)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k == 3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= 256.f;
    }
    w[k] = q8::encode2(x[0], x[1]) | (q8::encode2(x[2], x[3]) << 16);
    float f[4];
    q8::decode4(w[k], f);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] -= f[i];
  }
}

// Two weights (neighbouring heads of a token) -> p1, p2, 2^8 p3 and 2^8 p4 of both, e5m2, two bytes each.  An e5m2 is the
// upper byte of a half.  The first remainder is exact in fp32 and is rounded to a half; from there all is exact.
__device__ __forceinline__ void split_weights(float a, float b, uint32_t (&c)[4]) {
  auto as_halves = [](uint32_t codes) { return __byte_perm(codes, 0u, 0x1404); };
  c[0] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E5M2);
  uint32_t h = as_halves(c[0]);
  const float2 top = __half22float2(*reinterpret_cast<const __half2*>(&h));
  uint32_t r = DT<__half>::pack2(a - top.x, b - top.y);
  c[1] = q8::encode2h_e5m2(r);
  r = q8::sub2h(r, as_halves(c[1]));
  const __half2 up = __hmul2(*reinterpret_cast<const __half2*>(&r), __float2half2_rn(256.f));
  r = *reinterpret_cast<const uint32_t*>(&up);
  c[2] = q8::encode2h_e5m2(r);
  c[3] = q8::encode2h_e5m2(q8::sub2h(r, as_halves(c[2])));
}

// Or of a flag over the 128 threads of warps 4-7.
__device__ __forceinline__ bool any_of_128(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

// mbar_wait by a whole warp, one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned long long limit_ns) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, limit_ns));
}

// One byte to shared memory.  No memory clobber, so that the loads of the next head may pass it: for
// bytes that only the matrix unit reads, after a proxy fence (which is ordered behind it).
__device__ __forceinline__ void store_byte(uint32_t addr, uint32_t x) {
  asm volatile("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tst.shared.u8 [%0], h;\n\t}" ::"r"(addr), "r"(x));
}

template <typename T, int D, int GP>
__global__ void __launch_bounds__(kTcThreads, 2)
    paged_decode_q8_tc_kernel(const Q8Params p, const __grid_constant__ CUtensorMap tm_k,
                              const __grid_constant__ CUtensorMap tm_v) {
  using L = TcLayout<D, GP>;
  constexpr int HP = L::HP, HG = L::HG, SL = L::kSlots, QB = L::kQBufs;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base_u32 = (raw + 1023u) & ~1023u;
  uint8_t* base = smem_raw + (base_u32 - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::kBarOff);
  uint64_t* full_bar = bars;                 // [SL] slot's tile landed
  uint64_t* empty_bar = full_bar + SL;       // [SL] slot's products done
  uint64_t* sc_full = empty_bar + SL;        // [kScaleRing] a tile's scales landed
  uint64_t* s_full = sc_full + kScaleRing;   // [2] S^T written
  uint64_t* s_empty = s_full + 2;            // [2] S^T and the tile's scales read
  uint64_t* p_full = s_empty + 2;            // [2] weights written
  uint64_t* p_empty = p_full + 2;            // [2] P.V done
  uint64_t* q_full = p_empty + 2;            // [QB] query parts written
  uint64_t* q_empty = q_full + 2;            // [QB] the share's S^T all done, query factors read
  uint64_t* o_empty = q_empty + 2;           // O^T read
  uint64_t* drain = o_empty + 1;             // after a wait that ran out: every product issued is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  // misc: per head {limit of s + log2 v_scale, limit of s, M, R}, query factors [2][16], warp results
  // [4][16][2], two factors per head [16][2], a flag
  float4* ref_s = reinterpret_cast<float4*>(base + L::kMiscOff);
  float* hs_s = reinterpret_cast<float*>(ref_s + 16);
  float* red_s = hs_s + 32;
  float2* c_s = reinterpret_cast<float2*>(red_s + 128);
  int* flag = reinterpret_cast<int*>(c_s + 16);
  Share* cut_s = reinterpret_cast<Share*>(flag + 4);  // [2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < SL; ++i) {
      ptx::mbar_init(&full_bar[i], 1);
      ptx::mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < kScaleRing; ++i) ptx::mbar_init(&sc_full[i], 64);  // every lane of both producers
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&s_empty[i], 4);
      ptx::mbar_init(&p_full[i], 4);
      ptx::mbar_init(&p_empty[i], 1);
      ptx::mbar_init(&q_full[i], 1);
      ptx::mbar_init(&q_empty[i], 5);
    }
    ptx::mbar_init(o_empty, 4);
    ptx::mbar_init(drain, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    umma::tmem_alloc(tmem_slot, L::kTmemCols);
    umma::tmem_relinquish();
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int G = p.group, Hkv = p.n_kv_heads;
  const int pairs = (Hkv + HP - 1) / HP, splits = (G + GP - 1) / GP;
  const int units = pairs * splits;
  const int rows = p.block_size < kTcTile ? p.block_size : kTcTile;  // rows of one TMA box
  const int nb = kTcTile / rows;                                     // blocks of a tile
  Share s;
  using Walk = Walker<kTcTile, kTcWhole>;
  Cut cut;
  const int team = p.team, groups = units / team, mate = blockIdx.x % team;  // groups of units per sequence
  cut.make(Walk::line(p, groups, lane), gridDim.x / team);
  Walk w;
  w.b = p.batch;
  if ((int)blockIdx.x / team < cut.pieces) w.seek(p, cut, groups, blockIdx.x / team, lane);
  // The next share, with s.h as the unit of this CTA.
  auto next_share = [&]() -> bool {
    if (!w.next(p, cut, groups, s)) return false;
    s.h = s.h * team + mate;
    return true;
  };
  // Slot of the n-th tile of the ring's order and the parity of its round.
  auto slot_of = [](uint32_t n) { return n % SL; };
  auto round_of = [](uint32_t n) { return (n / SL) & 1; };
  // Places of K and V of tile number t in that order.
  auto k_at = [](uint32_t t) { return t == 0 ? 0u : 2 * t - 1; };
  // V(t) follows K(t + 1) if there is one: the last tile's V closes the order.
  auto v_at = [](uint32_t t) { return 2 * t + 2; };

  if (warp == 0 || warp == 3) {
    // ---------------- producers: warp 0 K, warp 3 V ----------------
    // (One warp for both took 2500 cycles a tile, 60 of them per box, and was what bounded the kernel.)
    const bool is_v = warp == 3;
    const CUtensorMap* tm = is_v ? &tm_v : &tm_k;
    const float* scale_src = is_v ? p.v_scale : p.k_scale;
    if (lane == 0) ptx::prefetch_tmap(tm);
    const int nb_shift = 31 - __clz(nb), j = lane & (nb - 1);  // nb is a power of two; this lane's block of a tile
    const int tiles_per_block = rows == kTcTile ? p.block_size / kTcTile : 1;
    uint32_t it = 0;
    bool ok = true;
    // One code tile into the ring: lane j holds the id of the tile's block j.
    auto load = [&](uint32_t n, int live, int x, int row, int blk) {
      const uint32_t sl = slot_of(n);
      ok = ok && warp_wait(&empty_bar[sl], round_of(n) ^ 1, p.wait_ns);
      if (!ok || p.drop_loads) return;
      if (lane == 0) ptx::mbar_arrive_expect_tx(&full_bar[sl], (uint32_t)(live * rows * 128));
      __syncwarp();
      if (lane < live)
        q8::tma_load_3d(base_u32 + sl * L::kSlot + lane * rows * 128, tm, &full_bar[sl], x, row, blk);
    };
    // V(t) follows K(t + 1) in the ring, so it is loaded once it is known whether there is one.
    int v_live = 0, v_x = 0, v_row = 0, v_blk = 0;
    while (ok && next_share()) {
      const int pair = s.h / splits;
      const int32_t* bt = p.block_tables + (size_t)s.b * p.max_blocks;
      const int blk_end = (s.tok1 + p.block_size - 1) / p.block_size;
      constexpr int W = 4;  // ids of 128 blocks at a time, one per lane and register
      int win = -W * 32, id[W];
      // the first block of the tile, and the tile's number in it where a block holds several
      int first = s.tok0 / kTcTile * nb / tiles_per_block, sub = s.tok0 / kTcTile % tiles_per_block;
      for (int t0 = s.tok0; ok && t0 < s.tok1; t0 += kTcTile) {
        if (is_v && it > 0) load(v_at(it - 1), v_live, v_x, v_row, v_blk);  // before this tile's ids are waited for
        if (first + nb > win + W * 32) {
          win = first;
#pragma unroll
          for (int r = 0; r < W; ++r) {
            const int i = win + r * 32 + lane;
            id[r] = i < blk_end ? __ldg(bt + i) : -1;
          }
        }
        const int live = min(nb, blk_end - first);
        const int rel = first + j - win;
        int blk = -1;
#pragma unroll
        for (int r = 0; r < W; ++r) {
          const int v = __shfl_sync(0xffffffffu, id[r], rel & 31);
          blk = (rel >> 5) == r ? v : blk;
        }
        if (!is_v) load(k_at(it), live, pair * 128, sub * kTcTile, blk);
        if (ok && !p.drop_loads) {
          // scales [K, V][HP][nb]: this lane's block, heads by turns
          const uint32_t scales = base_u32 + L::kScaleOff + (it % kScaleRing) * L::kScale + (is_v ? HP * nb * 4 : 0);
          for (int hp = lane >> nb_shift; hp < HP; hp += 32 >> nb_shift) {
            const int head = pair * HP + hp;
            const bool in = j < live && blk >= 0 && blk < p.num_blocks && head < Hkv;
            q8::copy4_async(scales + (hp * nb + j) * 4, in ? scale_src + (size_t)blk * Hkv + head : scale_src, in);
          }
          q8::arrive_after_copies(&sc_full[it % kScaleRing]);
        }
        v_live = live;
        v_x = pair * 128;
        v_row = sub * kTcTile;
        v_blk = blk;
        ++it;
        if (++sub == tiles_per_block) {
          sub = 0;
          first += nb;
        }
      }
    }
    // The last V's place is the one that no further K takes.
    if (is_v && it > 0) load(v_at(it - 1) - 1, v_live, v_x, v_row, v_blk);
    if (!ok && lane == 0) atomicExch(p.status, tvk::kStatusWaitTimeout);
    // No copy is in flight when the CTA ends, whatever became of the others.
    const uint32_t total = 2 * it;
    // (After a wait that ran out the last copy was issued before it, a whole limit ago.)
    for (uint32_t n = total > SL ? total - SL : 0; n < total && ok && !p.drop_loads; ++n)
      if ((n == total - 1 || (n > 0 && n % 2 == 0)) == is_v) ok = warp_wait(&full_bar[slot_of(n)], round_of(n), p.wait_ns);
  } else if (warp == 1) {
    // ---------------- matrix issue: S^T of a tile, then P.V of the one before ----------------
    constexpr uint32_t idesc_s = umma::idesc_e4m3(128, L::NS, false);
    constexpr uint32_t idesc_o = umma::idesc_e4m3(128, L::NO, true, true);
    uint32_t it = 0, share = 0;
    bool ok = true;
    // The P.V that is due: tile, place of its V, whether it starts its share, the share.
    bool due = false, due_first = false;
    uint32_t due_tile = 0, due_at = 0, due_share = 0;
    auto pv_ready = [&]() -> bool {
      return __all_sync(0xffffffffu, ptx::mbar_test(&p_full[due_tile & 1], (due_tile >> 1) & 1) &&
                                         ptx::mbar_test(&full_bar[slot_of(due_at)], round_of(due_at)) &&
                                         (!due_first || ptx::mbar_test(o_empty, (due_share & 1) ^ 1)));
    };
    auto issue_pv = [&]() {
      const uint32_t b = due_tile & 1, sl = slot_of(due_at);
      umma::fence_after_sync();
      if (lane == 0) {
        const uint32_t va = base_u32 + sl * L::kSlot, pa = base_u32 + L::kPOff + b * L::kP;
#pragma unroll
        for (int k = 0; k < kTcTile / 32; ++k)
          umma::mma_f8_ss(tmem + L::kOCol, umma::smem_desc_sw128(va + k * 32 * 128, 0, 1024),
                          umma::smem_desc_sw128(pa + k * 32, 0, 1024), idesc_o, !(due_first && k == 0));
        umma::commit(&empty_bar[sl]);
        umma::commit(&p_empty[b]);
      }
      __syncwarp();
      due = false;
    };
    while (ok && next_share()) {
      if (s.tok0 == s.tok1) continue;
      const uint32_t qb = share % QB;
      for (int t0 = s.tok0; ok && t0 < s.tok1; t0 += kTcTile) {
        // S^T of this tile and P.V of the one before, whichever can go first.
        const uint32_t b = it & 1, n = k_at(it), sl = slot_of(n);
        bool scored = false;
        const uint64_t since = ptx::globaltimer();
        while (!scored || due) {
          if (!scored &&
              __all_sync(0xffffffffu, ptx::mbar_test(&full_bar[sl], round_of(n)) &&
                                          ptx::mbar_test(&s_empty[b], ((it >> 1) & 1) ^ 1) &&
                                          (t0 != s.tok0 || ptx::mbar_test(&q_full[qb], (share / QB) & 1)))) {
            umma::fence_after_sync();
            if (lane == 0) {
              const uint32_t ka = base_u32 + sl * L::kSlot, qa = base_u32 + L::kQOff + qb * L::kQ;
#pragma unroll
              for (int hp = 0; hp < HP; ++hp)
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
                  umma::mma_f8_ss(tmem + (b * HP + hp) * L::NS, umma::smem_desc_sw128(ka + hp * D + k * 32, 0, 1024),
                                  umma::smem_desc_sw128(qa + hp * L::NS * 128 + k * 32, 0, 1024), idesc_s, k > 0);
              umma::commit(&s_full[b]);
              umma::commit(&empty_bar[sl]);
              if (t0 + kTcTile >= s.tok1) umma::commit(&q_empty[qb]);
            }
            __syncwarp();
            scored = true;
          }
          if (due && pv_ready()) issue_pv();
          if ((!scored || due) && __any_sync(0xffffffffu, ptx::globaltimer() - since > p.wait_ns)) {
            ok = false;
            break;
          }
        }
        due = ok;
        due_tile = it;
        due_at = v_at(it);
        due_first = t0 == s.tok0;
        due_share = share;
        ++it;
      }
      ++share;
    }
    if (ok && due) {
      --due_at;  // no K behind the last tile
      const uint64_t since = ptx::globaltimer();
      while (!pv_ready() && ok) ok = !__any_sync(0xffffffffu, ptx::globaltimer() - since > p.wait_ns);
      if (ok) issue_pv();
      ok = ok && warp_wait(&p_empty[due_tile & 1], (due_tile >> 1) & 1, p.wait_ns);  // nothing runs when TMEM is freed
    }
    if (!ok) {
      if (lane == 0) {
        atomicExch(p.status, tvk::kStatusWaitTimeout);
        umma::commit(drain);
      }
      __syncwarp();
      warp_wait(drain, 0, p.wait_ns);
    }
  } else if (warp == 2) {
    // ---------------- query rows of each share, in parts ----------------
    constexpr int LPR = D / 4;     // lanes per row, four elements each
    constexpr int RPW = 32 / LPR;  // rows at a time
    uint32_t share = 0;
    bool ok = true;
    while (ok && next_share()) {
      if (s.tok0 == s.tok1) continue;
      const uint32_t qb = share % QB;
      const int pair = s.h / splits, g0 = (s.h % splits) * GP;
      // row i = (KV head, query head) of the unit
      uint2 u[HG / RPW];
#pragma unroll
      for (int i = 0; i < HG / RPW; ++i) {
        const int r = i * RPW + lane / LPR, hp = r / GP, h = g0 + r % GP, head = pair * HP + hp;
        u[i] = make_uint2(0u, 0u);
        if (h < G && head < Hkv)
          u[i] = *reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(p.q) +
                                                 ((size_t)s.b * p.n_heads + (size_t)head * G + h) * D + (lane % LPR) * 4);
      }
      ok = warp_wait(&q_empty[qb], ((share / QB) & 1) ^ 1, p.wait_ns);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < HG / RPW; ++i) {
        const int r = i * RPW + lane / LPR, hp = r / GP, h = r % GP;
        const T* e4 = reinterpret_cast<const T*>(&u[i]);
        float x[4], mx = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = DT<T>::to_f(e4[k]);
          mx = fmaxf(mx, fabsf(x[k]));
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        int e = (int)(__float_as_uint(mx) >> 23);  // 2^(e - 127) <= mx
        e = e < 8 ? 8 : e;
        // to [2^7, 2^8); a row with an infinity is NaN altogether, as its softmax is
        const float up = e == 255 ? __int_as_float(0x7fffffff) : __uint_as_float((uint32_t)(261 - e) << 23);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] *= up;
        uint32_t parts[4];
        split_query(x, parts);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint32_t*>(base + L::kQOff + qb * L::kQ + hp * L::NS * 128 +
                                       swz128(k * GP + h, (lane % LPR) * 4)) = parts[k];
        if (lane % LPR == 0) hs_s[qb * 16 + r] = __uint_as_float((uint32_t)(e - 7) << 23) * p.scale_log2;
      }
      umma::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&q_full[qb]);
      ++share;
    }
    if (!ok && lane == 0) atomicExch(p.status, tvk::kStatusWaitTimeout);
  } else if (warp >= 4) {
    // ---------------- weights (thread = token), output (thread = dim) ----------------
    const int wq = warp - 4, tid = threadIdx.x - 128;
    const uint32_t lane_addr = tmem + ((uint32_t)(wq * 32) << 16);
    const int my_block = tid / rows;            // block of this thread's token
    const int my_hp = tid / D, dim = tid % D;   // KV head and dim of this thread's row of O^T
    uint32_t it = 0, share = 0;
    bool dead = false;  // a wait ran out: go through the motions, so that every counter is met
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!dead && !warp_wait(bar, parity, p.wait_ns)) {
        if (lane == 0) atomicExch(p.status, tvk::kStatusWaitTimeout);
        dead = true;
      }
    };
    // The first query head of a share that this thread's rows of O^T belong to; Hq or more: none.
    auto head_of = [&](const Share& x) -> int {
      const int kvh = x.h / splits * HP + my_hp;
      return kvh < Hkv ? kvh * G + x.h % splits * GP : p.n_heads;
    };
    auto heads_of = [&](const Share& x) { return min(GP, G - x.h % splits * GP); };  // per KV head
    // The next share with tokens; the rows of those without are zeros.
    auto next_live = [&]() -> bool {
      while (next_share()) {
        if (s.ctx > 0) return true;
        const int head0 = head_of(s);
        T* out = reinterpret_cast<T*>(p.out) + ((size_t)s.b * p.n_heads + head0) * D + dim;
        for (int h = 0; head0 < p.n_heads && h < heads_of(s); ++h) out[(size_t)h * D] = DT<T>::from_f(0.f);
      }
      return false;
    };
    // A piece has at most two shares of cut units, its first and its last.  Arriving at their units'
    // counters takes round trips to memory, so it is left to the piece's end.
    int n_cut = 0;
    bool more = next_live();
    while (more) {
      const Share cur = s;
      more = next_live();  // before this one is worked on, to know this CTA's last tile
      const int nh = heads_of(cur);
      const uint32_t qb = share % QB;
      if (tid < HG) {  // heads beyond the group never ask for new references
        const float lim = tid % GP < nh ? -INFINITY : INFINITY;
        ref_s[tid] = make_float4(lim, lim, -INFINITY, -INFINITY);
      }
      wait(&q_full[qb], (share / QB) & 1);
      float hs[HG], l[HG];
#pragma unroll
      for (int i = 0; i < HG; ++i) {
        hs[i] = hs_s[qb * 16 + i];
        l[i] = 0.f;
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&q_empty[qb]);
      ptx::named_barrier_sync(1, 128);  // the references are set

      for (int t0 = cur.tok0; t0 < cur.tok1; t0 += kTcTile) {
        const uint32_t b = it & 1;
        const bool live = t0 + tid < cur.tok1;
        wait(&sc_full[it % kScaleRing], (it / kScaleRing) & 1);
        const float* sc = reinterpret_cast<const float*>(base + L::kScaleOff + (it % kScaleRing) * L::kScale);
        float ks[HP], lv[HP];  // k_scale and log2 v_scale of this thread's token
#pragma unroll
        for (int hp = 0; hp < HP; ++hp) {
          ks[hp] = sc[hp * nb + my_block];
          lv[hp] = live ? __log2f(sc[(HP + hp) * nb + my_block]) : 0.f;
        }
        wait(&s_full[b], (it >> 1) & 1);
        umma::fence_after_sync();
        float x[HG];  // scores, base 2
        bool raise = false;
#pragma unroll
        for (int hp = 0; hp < HP; ++hp) {
          float c0[GP], c1[GP], c2[GP], c3[GP];
          const uint32_t at = lane_addr + (b * HP + hp) * L::NS;
          umma::ld_32x32b<GP>(at, c0);
          umma::ld_32x32b<GP>(at + GP, c1);
          umma::ld_32x32b<GP>(at + 2 * GP, c2);
          umma::ld_32x32b<GP>(at + 3 * GP, c3);
          umma::ld_wait();
#pragma unroll
          for (int h = 0; h < GP; ++h) {
            const int i = hp * GP + h;
            const float sum = fmaf(c3[h], kLowPart, c2[h] + c1[h]) + c0[h];
            x[i] = live ? sum * (ks[hp] * hs[i]) : -INFINITY;
            const float2 lim = *reinterpret_cast<const float2*>(&ref_s[i]);
            raise |= (x[i] + lv[hp] > lim.x) | (x[i] > lim.y);
          }
        }
        umma::fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&s_empty[b]);
        if (any_of_128(raise)) {
          // New references: the largest weight so far counts as 2^11, the largest term of a sum as 1.
#pragma unroll
          for (int i = 0; i < HG; ++i) {
            const float a = warp_max(x[i] + lv[i / GP]), c = warp_max(x[i]);
            if (lane == 0) *reinterpret_cast<float2*>(red_s + (wq * 16 + i) * 2) = make_float2(a, c);
          }
          ptx::named_barrier_sync(1, 128);
          if (tid < HG) {
            const float4 was = ref_s[tid];
            float nm = was.z, nr = was.w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 top = *reinterpret_cast<const float2*>(red_s + (k * 16 + tid) * 2);
              nm = fmaxf(nm, top.x - kTopWeight);
              nr = fmaxf(nr, top.y);
            }
            c_s[tid] = make_float2(nm == -INFINITY ? 1.f : ptx::ex2(was.z - nm), nr == -INFINITY ? 1.f : ptx::ex2(was.w - nr));
            const bool used = tid % GP < nh;
            ref_s[tid] = make_float4(used ? nm + kMostWeight : INFINITY, used ? nr + 64.f : INFINITY, nm, nr);
          }
          if (t0 != cur.tok0) wait(&p_empty[b ^ 1], ((it - 1) >> 1) & 1);  // P.V of the tile before: O^T is at rest
          ptx::named_barrier_sync(1, 128);
          umma::fence_after_sync();
#pragma unroll
          for (int i = 0; i < HG; ++i) l[i] *= c_s[i].y;
          if (t0 != cur.tok0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float o[GP];
              const uint32_t at = lane_addr + L::kOCol + k * HG + my_hp * GP;
              umma::ld_32x32b<GP>(at, o);
              umma::ld_wait();
#pragma unroll
              for (int h = 0; h < GP; ++h) o[h] *= c_s[my_hp * GP + h].x;
              umma::st_32x32b<GP>(at, o);
            }
            umma::st_wait();
            umma::fence_before_sync();
          }
        }
        // Weights, their sums, and their parts as rows of P^T: this thread's token is byte tid.
        wait(&p_empty[b], ((it >> 1) & 1) ^ 1);
        const uint32_t pw = base_u32 + L::kPOff + b * L::kP + tid;
#pragma unroll
        for (int hp = 0; hp < HP; ++hp)
#pragma unroll
          for (int h = 0; h < GP; h += 2) {  // heads beyond the group too: a branch would cost more
            float wt[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int i = hp * GP + h + k;
              const float2 ref = *reinterpret_cast<const float2*>(&ref_s[i].z);
              l[i] += ptx::ex2(x[i] - ref.y);
              wt[k] = ptx::ex2(x[i] + lv[hp] - (ref.x == -INFINITY ? 0.f : ref.x));
            }
            uint32_t cs[4];
            split_weights(wt[0], wt[1], cs);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // swz128(row, tid): the row's part of the swizzle is an exclusive or of constants
              const int row = k * HG + hp * GP + h;
              store_byte((pw ^ ((row & 7) << 4)) + row * 128, cs[k]);
              store_byte((pw ^ (((row + 1) & 7) << 4)) + (row + 1) * 128, cs[k] >> 8);
            }
          }
        // What lies behind the context has no weight, but may be NaN: zeros for V.
        if (t0 + kTcTile > cur.tok1) {
          const bool last = !more && t0 + kTcTile >= cur.tok1;
          const uint32_t n = v_at(it) - (last ? 1 : 0);
          wait(&full_bar[slot_of(n)], round_of(n));
          if (!live) {
            uint4* v = reinterpret_cast<uint4*>(base + slot_of(n) * L::kSlot + tid * 128);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        umma::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&p_full[b]);
        ++it;
      }

      // ---------------- the share's end ----------------
#pragma unroll
      for (int i = 0; i < HG; ++i) {
        float sum = l[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) red_s[wq * 16 + i] = sum;
      }
      wait(&p_empty[(it - 1) & 1], ((it - 1) >> 1) & 1);
      umma::fence_after_sync();
      float o[GP];
      {
        float a[GP], c[GP];
        const uint32_t at = lane_addr + L::kOCol + my_hp * GP;
        umma::ld_32x32b<GP>(at + 2 * HG, a);
        umma::ld_32x32b<GP>(at + 3 * HG, c);
        umma::ld_wait();
#pragma unroll
        for (int h = 0; h < GP; ++h) c[h] += a[h];
        umma::ld_32x32b<GP>(at, o);
        umma::ld_32x32b<GP>(at + HG, a);
        umma::ld_wait();
#pragma unroll
        for (int h = 0; h < GP; ++h) o[h] += fmaf(c[h], kLowPart, a[h]);
      }
      umma::fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(o_empty);
      ++share;
      ptx::named_barrier_sync(1, 128);
      // Per head: what brings O^T from M to R, and the sum of weights; a whole unit's output is their quotient.
      float* part = cur.n_parts == 1 ? nullptr : part_slot(p, blockIdx.x, cur.piece == cur.first_piece);
      if (tid < HG) {
        const float2 ref = *reinterpret_cast<const float2*>(&ref_s[tid].z);
        const float sum = (red_s[tid] + red_s[16 + tid]) + (red_s[32 + tid] + red_s[48 + tid]);
        const float f = ref.x == -INFINITY ? 0.f : ptx::ex2(ref.x - ref.y);
        c_s[tid].x = part ? f : f / sum;
        if (part) __stcg(reinterpret_cast<float2*>(part + HG * D + tid * 2), make_float2(ref.y, sum));
      }
      ptx::named_barrier_sync(1, 128);
      const int r0 = my_hp * GP, head0 = head_of(cur);
      if (part) {
#pragma unroll
        for (int h = 0; h < GP; ++h)
          __stcg(part + (r0 + h) * D + dim, o[h] * c_s[r0 + h].x);
        if (tid == 0) cut_s[n_cut & 1] = cur;
        ++n_cut;
      } else if (head0 < p.n_heads) {
        T* out = reinterpret_cast<T*>(p.out) + ((size_t)cur.b * p.n_heads + head0) * D + dim;
#pragma unroll
        for (int h = 0; h < GP; ++h)
          if (h < nh) out[(size_t)h * D] = DT<T>::from_f(o[h] * c_s[r0 + h].x);
      }
    }

    // ---------------- cut units: arrive, and where this is the last to, add the parts up ----------------
    for (int i = 0; i < n_cut; ++i) {
      auto sync = [] { ptx::named_barrier_sync(1, 128); };
      sync();  // cut_s is written
      const Share cur = cut_s[i];
      if (!last_to_arrive(p, cur, cur.b * units + cur.h, flag, tid, sync)) continue;
      const int r0 = my_hp * GP, head0 = head_of(cur), nh = heads_of(cur), n_parts = cur.n_parts;
      // First the factor of every part and row, 8 threads a row, then the rows' weighted sums.  The
      // weight buffers are free (their products are done): they take the factors.
      const float* parts = part_slot(p, cur.first_piece * team + mate, false);
      auto at_part = [&](int c) { return c == 0 ? kSlotFloats : c * team * 2 * kSlotFloats; };  // as part_slot places them
      float* f = reinterpret_cast<float*>(base + L::kPOff);
      constexpr int kAtOnce = 2 * L::kP / 4 / HG;
      const int row = tid >> 3;
      const bool has = row < HG;
      const float* ml_row = parts + HG * D + row * 2;
      float M = -INFINITY, Ls = 0.f;
      float2 ml = make_float2(-INFINITY, 0.f);  // of one of the first 8 parts, read once
      if (has && (tid & 7) < n_parts) ml = __ldcg(reinterpret_cast<const float2*>(ml_row + at_part(tid & 7)));
      M = ml.x;
      for (int c = (tid & 7) + 8; has && c < n_parts; c += 8) M = fmaxf(M, __ldcg(ml_row + at_part(c)));
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
      float acc[GP];
#pragma unroll
      for (int h = 0; h < GP; ++h) acc[h] = 0.f;
      for (int c0 = 0; c0 < n_parts; c0 += kAtOnce) {
        const int n = min(n_parts - c0, kAtOnce);
        for (int c = tid & 7; has && c < n; c += 8) {
          const float2 x = c0 + c < 8 ? ml : __ldcg(reinterpret_cast<const float2*>(ml_row + at_part(c0 + c)));
          const float e = exp2f(x.x - M);
          f[c * HG + row] = e;
          Ls = fmaf(x.y, e, Ls);
        }
        sync();
        constexpr int U = GP >= 8 ? 4 : 8;  // parts whose sums are in flight together
        const float* src = parts + r0 * D + dim;
        for (int c = 0; c < n; c += U) {
          float v[U][GP];
#pragma unroll
          for (int k = 0; k < U; ++k) {
            const float* at = src + at_part(c0 + min(c + k, n - 1));
#pragma unroll
            for (int h = 0; h < GP; ++h) v[k][h] = __ldcg(at + h * D);
          }
#pragma unroll
          for (int k = 0; k < U; ++k)
#pragma unroll
            for (int h = 0; h < GP; ++h)
              acc[h] = fmaf(v[k][h], c + k < n ? f[(c + k) * HG + r0 + h] : 0.f, acc[h]);
        }
        sync();
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) Ls += __shfl_xor_sync(0xffffffffu, Ls, d);
      if (has && (tid & 7) == 0) red_s[row] = Ls;
      sync();
      T* out = reinterpret_cast<T*>(p.out) + ((size_t)cur.b * p.n_heads + head0) * D + dim;
#pragma unroll
      for (int h = 0; h < GP; ++h)
        if (head0 < p.n_heads && h < nh) out[(size_t)h * D] = DT<T>::from_f(acc[h] / red_s[r0 + h]);
      sync();  // red_s and the factors may be written again
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    umma::fence_after_sync();
    umma::tmem_dealloc(tmem, L::kTmemCols);
  }
}

template <int D, int GM>
int launch_simt_gm(const Q8Params& p, cudaStream_t stream) {
  using L = SimtLayout<D, GM>;
  auto kern = paged_decode_q8_simt_kernel<D, GM>;
  static std::atomic<unsigned long long> allowed{0};
  TVK_CHECK_CUDA(tvk::allow_smem(kern, L::kBytes, allowed));
  const long long most = (long long)p.batch * p.n_kv_heads * (tiles_of(p.max_ctx_tokens, kSimtTile) + kUnitTiles);
  const int grid = (int)(most < kSimtCtas ? most : kSimtCtas);
  TVK_CHECK_CUDA(tvk::launch_pdl(kern, grid, 128, L::kBytes, stream, p));
  TVK_CHECK_LAUNCH("paged_decode_q8_simt");
  return TVK_OK;
}

template <int D>
int launch_simt_d(const Q8Params& p, cudaStream_t stream) {
  if (p.group <= 4) return launch_simt_gm<D, 4>(p, stream);
  return p.group <= 8 ? launch_simt_gm<D, 8>(p, stream) : launch_simt_gm<D, 16>(p, stream);
}

int launch_simt(const Q8Params& p, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return launch_simt_d<32>(p, stream);
    case 64: return launch_simt_d<64>(p, stream);
    default: return launch_simt_d<128>(p, stream);
  }
}

template <typename T, int D, int GP>
int launch_tc(const Q8Params& p, cudaStream_t stream) {
  using L = TcLayout<D, GP>;
  tvk::EncodeTiledFn encode = tvk::encode_tiled_fn();
  if (!encode) {
    tvk::set_error("cuTensorMapEncodeTiled is not available from the driver");
    return TVK_ERR_CUDA;
  }
  // A row of the box is 128 bytes: HP heads, of which the last may lie beyond the tensor and read as zeros.
  const cuuint64_t row = (cuuint64_t)p.n_kv_heads * D;
  const cuuint64_t dims[3] = {row, (cuuint64_t)p.block_size, (cuuint64_t)p.num_blocks};
  const cuuint64_t strides[2] = {row, row * p.block_size};
  const cuuint32_t box[3] = {128u, (cuuint32_t)(p.block_size < kTcTile ? p.block_size : kTcTile), 1u};
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  CUtensorMap tm[2];
  for (int i = 0; i < 2; ++i) {
    const CUresult r = encode(&tm[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(i ? p.v_cache : p.k_cache), dims,
                              strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
      tvk::set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
      return TVK_ERR_CUDA;
    }
  }
  auto kern = paged_decode_q8_tc_kernel<T, D, GP>;
  static std::atomic<unsigned long long> allowed{0};
  TVK_CHECK_CUDA(tvk::allow_smem(kern, L::kBytes, allowed));
  const int units = (p.n_kv_heads + L::HP - 1) / L::HP * ((p.group + GP - 1) / GP);
  // Teams of up to 8 CTAs on neighbouring units of the same tokens: what they read lies side by side in
  // the pool, and they read it at about the same time.
  int team = units < 8 ? units : 8;
  while (units % team) --team;
  const long long most = (long long)p.batch * (units / team) * (tiles_of(p.max_ctx_tokens, kTcTile) + kUnitTiles);
  const int pieces = (int)(most < kTcCtas / team ? most : kTcCtas / team);
  Q8Params q = p;
  q.team = team;
  TVK_CHECK_CUDA(tvk::launch_pdl(kern, pieces * team, kTcThreads, L::kBytes, stream, q, tm[0], tm[1]));
  TVK_CHECK_LAUNCH("paged_decode_q8_tc");
  return TVK_OK;
}

// 16-bit queries on the tensor cores where 128-token tiles are whole blocks or lie in one.
// Query heads per unit (GP): as few as hold the group, but no more than 16 over the HP KV heads.
// Calls that would leave most CTAs idle take units of 4 all the same: their tiles take half the
// time, and the second reading of K and V comes from L2.  That is, of 4-head units either at
// most 64 (32/4 heads of 64: one sequence of 512 tokens 12.9 -> 9.9 us, 8 of 8,192 22.5 -> 20.9),
// or no more than there are CTAs, none of them cut as far as the tables' width tells (64 sequences of 40-640 with tables
// of 40 blocks: 17.8 -> 15.9; an engine's 64 blocks may hold longer contexts, and such calls take units of 8).
// 32 sequences of 1,024 or 2,048 lose by it (17.4 -> 18.5, 20.6 -> 22.4).
template <typename T>
int launch_16bit(const Q8Params& p, int head_dim, cudaStream_t stream) {
  const int bs = p.block_size;
  if (!(bs == 8 || bs == 16 || bs == 32 || bs == 64 || bs % kTcTile == 0)) return launch_simt(p, head_dim, stream);
  if (head_dim == 32) return launch_tc<T, 32, 4>(p, stream);
  const int pairs = head_dim == 64 ? (p.n_kv_heads + 1) / 2 : p.n_kv_heads;
  const long long units = (long long)p.batch * pairs * ((p.group + 3) / 4);
  const bool idle = units <= 64 || (units <= kTcCtas && tiles_of(p.max_ctx_tokens, kTcTile) <= kTcWhole);
  if (head_dim == 64) return p.group <= 4 || idle ? launch_tc<T, 64, 4>(p, stream) : launch_tc<T, 64, 8>(p, stream);
  if (p.group <= 4 || idle) return launch_tc<T, 128, 4>(p, stream);
  return p.group <= 8 ? launch_tc<T, 128, 8>(p, stream) : launch_tc<T, 128, 16>(p, stream);
}

}  // namespace

extern "C" size_t tvk_paged_decode_q8_workspace_size(int batch, int n_kv_heads) {
  const size_t units = batch > 0 && n_kv_heads > 0 ? (size_t)batch * n_kv_heads * kMaxParts : 0;
  return tvk::kWorkspaceHeader + (size_t)2 * kMaxPieces * kSlotFloats * sizeof(float) + units * sizeof(int);
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
  TVK_CHECK_ARG((long long)max_blocks * block_size <= 0x7fffff00LL, "a table spans more than 2^31 - 256 tokens");
  TVK_CHECK_ARG((long long)batch * n_kv_heads * ((long long)max_blocks * block_size / kSimtTile + 1 + kUnitTiles) < 0x7fffffffLL,
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
                "q, k_cache and v_cache must be 16-byte aligned, out 4-byte");
  // a query row is read by every CTA that shares its sequence, whoever has written its output by then
  const uintptr_t q0 = (uintptr_t)q, o0 = (uintptr_t)out;
  const uintptr_t extent = (uintptr_t)batch * n_heads * head_dim * tvk::dtype_size(dtype);
  TVK_CHECK_ARG(q0 + extent <= o0 || o0 + extent <= q0, "out must not overlap q");
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
  p.counters = (int*)(p.part + (size_t)2 * kMaxPieces * kSlotFloats);
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
  p.dtype = dtype;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  const tvk::WaitTest wt = tvk::take_wait_test();
  p.wait_ns = wt.armed ? wt.limit_ns : tvk::kDefaultWaitNs;
  p.drop_loads = wt.armed ? 1 : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TVK_DTYPE_F16: return launch_16bit<__half>(p, head_dim, s);
    case TVK_DTYPE_BF16: return launch_16bit<__nv_bfloat16>(p, head_dim, s);
    default: return launch_simt(p, head_dim, s);
  }
}
