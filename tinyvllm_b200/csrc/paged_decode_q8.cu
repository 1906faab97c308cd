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

#include <atomic>
#include <type_traits>

#include "kv_cache_q8.cuh"

namespace {

constexpr int kTile = 64;            // tokens per tile of the work line
constexpr int kSimtTile = 32;        // tokens the simt kernel stages at a time
constexpr int kMaxGroup = 16;        // query heads per KV head
constexpr int kMaxCtas = 592;        // pieces a call is cut into at most (four CTAs on each of 148 SMs)
constexpr int kTcCtas = 296;         // the same for the tensor-core kernel: two CTAs on each SM
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
  float scale_log2;            // log2(e) / sqrt(head_dim)
  int n_stages;                // ring depth of the tensor-core kernel
  unsigned long long wait_ns;  // wall-time limit of every mbarrier wait
  int drop_loads;              // wait-limit test: the producer issues nothing, so waits run out
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

// The end of a cut unit's share, by the NT threads that have just stored its
// partials with __stcg (o [rows][D], then m, l [rows][2]): counts the arrival, and
// the last to arrive adds the parts up and writes the output rows (query heads from
// row0 on).  `flag` is a shared int; `sync` a barrier of the NT threads.
template <typename T, int D, int NT, typename Sync>
__device__ void join_parts(const Q8Params& p, const Share& s, int unit, int rows, int row0, int* flag, int tid, Sync sync) {
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
  T* out = reinterpret_cast<T*>(p.out) + ((size_t)s.b * p.n_heads + row0) * D;
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
    if (s.n_parts == 1) {
      for (int i = tid; i < G * D; i += 128) out[i] = DT<T>::from_f(qs[i] / lfin[i / D]);
      continue;
    }
    float* mine = part_slot(p, blockIdx.x, (int)blockIdx.x == s.first_cta);
    for (int i = tid; i < G * D; i += 128) __stcg(mine + i, qs[i]);
    for (int i = tid; i < G; i += 128) {
      __stcg(mine + G * D + i * 2, mfin[i]);
      __stcg(mine + G * D + i * 2 + 1, lfin[i]);
    }
    join_parts<T, D, 128>(p, s, s.b * Hkv + s.h, G, s.h * G, &flag, tid, [] { __syncthreads(); });
  }
}

// -----------------------------------------------------------------------------
// Tensor-core kernel: 16-bit queries; block sizes 8, 16, 32 and multiples of 64.
//
// A unit is HP neighbouring KV heads of one sequence (HP * D bytes a token, 128
// where the head count allows), so that one TMA row is a whole 128-byte line also
// for small heads.  One producer warp streams 64-token tiles of codes (and their
// scales, by 4-byte asynchronous copies, and at a share's start its query rows)
// through a ring of stages; four consumer warps take 16 tokens of a tile each:
//   S^T [16 tokens, 8 heads] = K . Q^T    A = codes as halves, straight from their rows
//   P^T                       = 2^(S^T - m) as halves, transposed in registers
//   O^T [D, 8 heads]         += v_scale * (V^T . P^T)
// Tokens and dims, not heads, are the 16-row side of the products: at 4 to 8
// query heads per KV head that halves the matrix instructions and the accumulators.
// The order of the k index of a product is free, so a lane takes 16 neighbouring
// bytes of its row as four k steps and nothing is shuffled; for V a byte
// permute pairs the same dim of two tokens.
// -----------------------------------------------------------------------------
template <int ROWB>
__device__ __forceinline__ uint32_t row_off(int t, int byte) {  // as the TMA swizzle of ROWB-byte rows lays it
  const int x = ROWB == 128 ? (t & 7) : ROWB == 64 ? ((t >> 1) & 3) : ((t >> 2) & 1);
  return t * ROWB + ((((byte >> 4) ^ x) << 4) | (byte & 15));
}

constexpr int kTcThreads = 160;
constexpr int kScaleFloats = 64;  // scales per stage: K and V, HP <= 4 heads, <= 8 blocks

template <int D, int HP>
struct TcLayout {
  static constexpr int ROWB = D * HP;
  static constexpr int kPart = kTile * ROWB;  // K (or V) codes of a stage
  // stage = K codes, V codes, scales, query rows
  static __host__ __device__ int q_bytes(int group) { return HP * group * D * 2; }
  static __host__ __device__ int scales_off(int n_stages) { return n_stages * 2 * kPart; }
  static __host__ __device__ int q_off(int n_stages) { return scales_off(n_stages) + n_stages * kScaleFloats * 4; }
  static __host__ __device__ int merge_off(int n_stages, int group) { return q_off(n_stages) + n_stages * q_bytes(group); }
  // merge: o [4][HP * group][D], m, l and weights [4][HP * group], one flag
  static __host__ __device__ int bar_off(int n_stages, int group) {
    return merge_off(n_stages, group) + 4 * HP * group * (D + 3) * 4 + 16;
  }
  static __host__ __device__ int bytes(int n_stages, int group) { return bar_off(n_stages, group) + n_stages * 16 + 1024; }
};

template <typename T, int D, int HP, int NT, bool BS8>
__global__ void __launch_bounds__(kTcThreads, 2)
    paged_decode_q8_tc_kernel(const Q8Params p, const __grid_constant__ CUtensorMap tm_k,
                              const __grid_constant__ CUtensorMap tm_v) {
  using L = TcLayout<D, HP>;
  constexpr int ROWB = L::ROWB;
  constexpr int KS = D / 16;  // k steps of S, and 16-dim tiles of O
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t base_u32 = (raw + 1023u) & ~1023u;
  uint8_t* base = smem_raw + (base_u32 - raw);
  const int G = p.group, NS = p.n_stages;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(base + ((L::bar_off(NS, G) + 7) & ~7));
  uint64_t* empty_bar = full_bar + NS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(&full_bar[s], 33);  // the byte count, and every producer lane's scales
      ptx::mbar_init(&empty_bar[s], 4);
    }
    ptx::fence_mbar_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int heads = p.n_kv_heads / HP;
  Walker w;
  w.start(p, heads, lane);
  Share s;
  int stage = 0;
  uint32_t phase = 0;

  if (warp == 4) {
    // ---------------- producer ----------------
    if (lane == 0) {
      ptx::prefetch_tmap(&tm_k);
      ptx::prefetch_tmap(&tm_v);
    }
    const int rows = p.block_size < kTile ? p.block_size : kTile;  // rows of one TMA box
    const int nb = kTile / rows;                                   // blocks of a tile
    const int q_bytes = L::q_bytes(G);
    bool running = true;
    while (running && w.next(p, s)) {
      const int32_t* bt = p.block_tables + (size_t)s.b * p.max_blocks;
      const int blk_end = (s.tok1 + p.block_size - 1) / p.block_size;
      constexpr int W = 4;  // ids of 128 blocks at a time, one per lane and register
      int win = -W * 32, id[W];
      for (int t0 = s.tok0; t0 < s.tok1; t0 += kTile) {
        const int first = t0 / p.block_size;
        if (first + nb > win + W * 32) {
          win = first;
#pragma unroll
          for (int r = 0; r < W; ++r) {
            const int i = win + r * 32 + lane;
            id[r] = i < blk_end ? __ldg(bt + i) : -1;
          }
        }
        if (!ptx::mbar_wait(&empty_bar[stage], phase ^ 1, p.wait_ns)) {
          if (lane == 0) atomicExch(p.status, tvk::kStatusWaitTimeout);
          running = false;
          break;
        }
        if (!p.drop_loads) {
          const int live = min(nb, blk_end - first);
          if (lane == 0) {
            uint32_t tx = (uint32_t)(live * rows * ROWB * 2);
            if (t0 == s.tok0) tx += q_bytes;
            ptx::mbar_arrive_expect_tx(&full_bar[stage], tx);
            if (t0 == s.tok0)
              ptx::bulk_load(base + L::q_off(NS) + stage * q_bytes,
                             reinterpret_cast<const uint8_t*>(p.q) + ((size_t)s.b * p.n_heads + (size_t)s.h * HP * G) * D * 2,
                             (uint32_t)q_bytes, &full_bar[stage]);
          }
          __syncwarp();
          // lane = block of the tile (up to 8) and, for the scales, head and K / V
          const uint32_t codes = base_u32 + stage * 2 * L::kPart;
          const uint32_t scales = base_u32 + L::scales_off(NS) + stage * kScaleFloats * 4;
          for (int i0 = 0; i0 < nb * 2 * HP; i0 += 32) {
            const int i = i0 + lane, j = i % nb, kv = (i / nb) & 1, hp = i / (2 * nb);
            const int rel = first + j - win;
            int blk = -1;
#pragma unroll
            for (int r = 0; r < W; ++r) {
              const int v = __shfl_sync(0xffffffffu, id[r], rel & 31);
              blk = (rel >> 5) == r ? v : blk;
            }
            if (i < nb * 2 * HP) {
              const bool in = j < live && blk >= 0 && blk < p.num_blocks;
              const float* src = kv ? p.v_scale : p.k_scale;
              q8::copy4_async(scales + ((kv * HP + hp) * nb + j) * 4,
                              in ? src + (size_t)blk * p.n_kv_heads + s.h * HP + hp : src, in);
              if (hp == 0 && j < live)
                q8::tma_load_3d(codes + kv * L::kPart + j * rows * ROWB, kv ? &tm_v : &tm_k, &full_bar[stage],
                                s.h * HP * D, t0 % p.block_size, blk);
            }
          }
          q8::arrive_after_copies(&full_bar[stage]);
        }
        if (++stage == NS) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // No copy is in flight when the CTA ends, whatever became of the consumers.
    for (int i = 0; i < NS && !p.drop_loads; ++i) {
      if (!ptx::mbar_wait(&full_bar[stage], phase ^ 1, p.wait_ns)) break;
      if (++stage == NS) {
        stage = 0;
        phase ^= 1;
      }
    }
    return;
  }

  // ---------------- consumers ----------------
  const int g = lane >> 2, tig = lane & 3;
  const int nb = p.block_size < kTile ? kTile / p.block_size : 1;
  const int R = HP * G;  // output rows of a unit
  float* co = reinterpret_cast<float*>(base + L::merge_off(NS, G));
  float* cm = co + 4 * R * D;
  float* cl = cm + 4 * R;
  float* cw = cl + 4 * R;
  int* flag = reinterpret_cast<int*>(cw + 4 * R);
  // Row r of an 8-token group is token tok_of(r): an order in which the lanes of one
  // shared-memory access fall on different banks.
  auto tok_of = [](int r) { return HP == 1 ? r : HP == 2 ? (r >> 1) | ((r & 1) << 2) : ((r & 3) << 1) | (r >> 2); };
  const int tk = tok_of(g), tv0 = tok_of(2 * tig), tv1 = tok_of(2 * tig + 1);
  bool dead = false;  // a wait ran out: go through the motions, so that every counter is met

  while (w.next(p, s)) {
    if (s.ctx == 0) {
      T* out = reinterpret_cast<T*>(p.out) + ((size_t)s.b * p.n_heads + s.h * R) * D;
      for (int i = threadIdx.x; i < R * D; i += 128) out[i] = DT<T>::from_f(0.f);
      continue;
    }
    uint32_t qb[HP][NT][KS][2];
    float o[HP][NT][KS][4], m[HP][NT][2], l[HP][NT][2], hs[HP][NT][2];
#pragma unroll
    for (int hp = 0; hp < HP; ++hp)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[hp][n][i][0] = o[hp][n][i][1] = o[hp][n][i][2] = o[hp][n][i][3] = 0.f;
          qb[hp][n][i][0] = qb[hp][n][i][1] = 0u;
        }
        m[hp][n][0] = m[hp][n][1] = -INFINITY;
        l[hp][n][0] = l[hp][n][1] = 0.f;
        hs[hp][n][0] = hs[hp][n][1] = p.scale_log2;
      }
    for (int t0 = s.tok0; t0 < s.tok1; t0 += kTile) {
      if (!dead && !ptx::mbar_wait(&full_bar[stage], phase, p.wait_ns)) {
        if (lane == 0) atomicExch(p.status, tvk::kStatusWaitTimeout);
        dead = true;
      }
      if (t0 == s.tok0 && !dead) {
        // Query rows as the B operand: lane (g, tig) holds head g, the dims of its K bytes.
        const uint8_t* qs = base + L::q_off(NS) + stage * L::q_bytes(G);
#pragma unroll
        for (int hp = 0; hp < HP; ++hp)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int head = n * 8 + g;
            if (head < G) {
              const uint2* src = reinterpret_cast<const uint2*>(qs + ((size_t)(hp * G + head) * D + tig * (D / 4)) * 2);
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                const uint2 u = src[i];
                qb[hp][n][i][0] = u.x;
                qb[hp][n][i][1] = u.y;
              }
            }
            if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
              // bf16 -> half, each head's row by a power of two that brings its largest value to
              // 2^14..2^15: exact but for values under 2^-28 of that, undone after the product.
              float mx = 0.f;
#pragma unroll
              for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  mx = fmaxf(mx, fabsf(__uint_as_float(qb[hp][n][i][k] << 16)));
                  mx = fmaxf(mx, fabsf(__uint_as_float(qb[hp][n][i][k] & 0xffff0000u)));
                }
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
              int e = (int)(__float_as_uint(mx) >> 23);
              e = e < 15 ? 15 : e;
              const float up = __uint_as_float((uint32_t)(268 - e) << 23);
              const float down = __uint_as_float((uint32_t)(e - 14) << 23) * p.scale_log2;
#pragma unroll
              for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const uint32_t u = qb[hp][n][i][k];
                  qb[hp][n][i][k] =
                      DT<__half>::pack2(__uint_as_float(u << 16) * up, __uint_as_float(u & 0xffff0000u) * up);
                }
              hs[hp][n][0] = __shfl_sync(0xffffffffu, down, tig * 8);
              hs[hp][n][1] = __shfl_sync(0xffffffffu, down, tig * 8 + 4);
            }
          }
      }
      const int left = s.tok1 - t0 - warp * 16;  // live tokens from this warp's first row on
      if (left > 0 && !dead) {
        const uint8_t* kp = base + stage * 2 * L::kPart + warp * 16 * ROWB;
        const uint8_t* vp = kp + L::kPart;
        const float* sc = reinterpret_cast<const float*>(base + L::scales_off(NS) + stage * kScaleFloats * 4);
        const int j0 = warp * 16 / (kTile / nb);  // block of this warp's first row
        const bool partial = left < 16;
#pragma unroll
        for (int hp = 0; hp < HP; ++hp) {
          // ---- S^T = K Q^T
          float st[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) st[n][0] = st[n][1] = st[n][2] = st[n][3] = 0.f;
          uint32_t ka[D / 16], kb[D / 16];  // D / 4 bytes of rows g and g + 8
          if constexpr (D >= 64) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              const uint32_t off = row_off<ROWB>(tk, hp * D + tig * (D / 4) + c * 16);
              const uint4 a = *reinterpret_cast<const uint4*>(kp + off);
              const uint4 b = *reinterpret_cast<const uint4*>(kp + off + 8 * ROWB);
              ka[c * 4] = a.x, ka[c * 4 + 1] = a.y, ka[c * 4 + 2] = a.z, ka[c * 4 + 3] = a.w;
              kb[c * 4] = b.x, kb[c * 4 + 1] = b.y, kb[c * 4 + 2] = b.z, kb[c * 4 + 3] = b.w;
            }
          } else {
            const uint32_t off = row_off<ROWB>(tk, hp * D + tig * 8);
            const uint2 a = *reinterpret_cast<const uint2*>(kp + off);
            const uint2 b = *reinterpret_cast<const uint2*>(kp + off + 8 * ROWB);
            ka[0] = a.x, ka[1] = a.y, kb[0] = b.x, kb[1] = b.y;
          }
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const uint32_t a0 = q8::decode2(ka[i]), a2 = q8::decode2(ka[i] >> 16);
            const uint32_t a1 = q8::decode2(kb[i]), a3 = q8::decode2(kb[i] >> 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) q8::mma16(st[n], a0, a1, a2, a3, qb[hp][n][i][0], qb[hp][n][i][1]);
          }
          // ---- scores, running maximum, weights
          const float ks0 = sc[hp * nb + j0], ks1 = BS8 ? sc[hp * nb + j0 + 1] : ks0;
          const float vs0 = sc[(HP + hp) * nb + j0], vs1 = BS8 ? sc[(HP + hp) * nb + j0 + 1] : vs0;
          uint32_t pb[NT][2];
          bool raise = false;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            st[n][0] *= ks0 * hs[hp][n][0];
            st[n][1] *= ks0 * hs[hp][n][1];
            st[n][2] *= ks1 * hs[hp][n][0];
            st[n][3] *= ks1 * hs[hp][n][1];
            if (partial) {
              if (tk >= left) st[n][0] = st[n][1] = -INFINITY;
              if (tk + 8 >= left) st[n][2] = st[n][3] = -INFINITY;
            }
            raise |= fmaxf(st[n][0], st[n][2]) > m[hp][n][0] + 8.f || fmaxf(st[n][1], st[n][3]) > m[hp][n][1] + 8.f;
          }
          // The maximum moves only when a score passes it by more than 2^8: weights stay
          // below 2^8 (a half holds 2^16), and most tiles rescale nothing.
          if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float mx = fmaxf(st[n][k], st[n][k + 2]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                mx = fmaxf(m[hp][n][k], mx);
                const float c = mx == -INFINITY ? 1.f : ptx::ex2(m[hp][n][k] - mx);
                m[hp][n][k] = mx;
                l[hp][n][k] *= c;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                  o[hp][n][i][k] *= c;
                  o[hp][n][i][k + 2] *= c;
                }
              }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float pr[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) pr[k] = ptx::ex2(st[n][k] - m[hp][n][k & 1]);
            l[hp][n][0] += pr[0] + pr[2];
            l[hp][n][1] += pr[1] + pr[3];
            pb[n][0] = q8::transpose8x8(DT<__half>::pack2(pr[0], pr[1]));
            pb[n][1] = q8::transpose8x8(DT<__half>::pack2(pr[2], pr[3]));
          }
          // ---- O^T += v_scale (V^T P^T); lane (g, tig): D / 8 bytes of tokens tv0, tv1 and those + 8
          constexpr int VW = D / 32;  // 32-bit words of a token
          uint32_t v[4][VW];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int t = (k & 1 ? tv1 : tv0);
            const uint8_t* src = vp + row_off<ROWB>(t, hp * D + g * (D / 8)) + (k >> 1) * 8 * ROWB;
            if constexpr (VW == 4) {
              const uint4 u = *reinterpret_cast<const uint4*>(src);
              v[k][0] = u.x, v[k][1] = u.y, v[k][2] = u.z, v[k][3] = u.w;
            } else if constexpr (VW == 2) {
              const uint2 u = *reinterpret_cast<const uint2*>(src);
              v[k][0] = u.x, v[k][1] = u.y;
            } else {
              v[k][0] = *reinterpret_cast<const uint32_t*>(src);
            }
            if (partial && t + (k >> 1) * 8 >= left) {  // what lies behind the context may be NaN
#pragma unroll
              for (int x = 0; x < VW; ++x) v[k][x] = 0u;
            }
          }
#pragma unroll
          for (int x = 0; x < VW; ++x)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t sel = half ? 0x7362 : 0x5140;
              const uint32_t lo = __byte_perm(v[0][x], v[1][x], sel), hi = __byte_perm(v[2][x], v[3][x], sel);
              const uint32_t a0 = q8::decode2(lo), a1 = q8::decode2(lo >> 16);
              const uint32_t a2 = q8::decode2(hi), a3 = q8::decode2(hi >> 16);
              const int i = x * 2 + half;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                if constexpr (BS8) {
                  float acc1[4] = {0.f, 0.f, 0.f, 0.f};
                  q8::mma8(acc, a0, a1, pb[n][0]);
                  q8::mma8(acc1, a2, a3, pb[n][1]);
#pragma unroll
                  for (int k = 0; k < 4; ++k) o[hp][n][i][k] = fmaf(vs1, acc1[k], o[hp][n][i][k]);
                } else {
                  q8::mma16(acc, a0, a1, a2, a3, pb[n][0], pb[n][1]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) o[hp][n][i][k] = fmaf(vs0, acc[k], o[hp][n][i][k]);
              }
            }
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&empty_bar[stage]);
      if (++stage == NS) {
        stage = 0;
        phase ^= 1;
      }
    }

    // ---------------- the share's end: merge the four warps ----------------
    ptx::named_barrier_sync(1, 128);  // all have read the previous merge
#pragma unroll
    for (int hp = 0; hp < HP; ++hp)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float sum = l[hp][n][k];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const int head = n * 8 + tig * 2 + k;
          if (head >= G) continue;
          const int r = warp * R + hp * G + head;
          if (g == 0) {
            cm[r] = m[hp][n][k];
            cl[r] = sum;
          }
          float2* dst = reinterpret_cast<float2*>(co + (size_t)r * D + g * (D / 8));
#pragma unroll
          for (int i = 0; i < KS; ++i) dst[i] = make_float2(o[hp][n][i][k], o[hp][n][i][k + 2]);
        }
    ptx::named_barrier_sync(1, 128);
    T* out = reinterpret_cast<T*>(p.out) + ((size_t)s.b * p.n_heads + s.h * R) * D;
    float* mine = s.n_parts == 1 ? nullptr : part_slot(p, blockIdx.x, (int)blockIdx.x == s.first_cta);
    for (int i = threadIdx.x; i < R * D; i += 128) {
      const int r = i / D;
      float M = cm[r];
#pragma unroll
      for (int x = 1; x < 4; ++x) M = fmaxf(M, cm[x * R + r]);
      float Lsum = 0.f, A = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        // a warp without tokens in this share has m = -inf and adds nothing
        const float e = cm[x * R + r] == -INFINITY ? 0.f : ptx::ex2(cm[x * R + r] - M);
        Lsum = fmaf(cl[x * R + r], e, Lsum);
        A = fmaf(co[(size_t)x * R * D + i], e, A);
      }
      if (!mine) {
        out[i] = DT<T>::from_f(A / Lsum);
      } else {
        __stcg(mine + i, A);
        if (i % D == 0) {
          __stcg(mine + R * D + r * 2, M);
          __stcg(mine + R * D + r * 2 + 1, Lsum);
        }
      }
    }
    if (mine)
      join_parts<T, D, 128>(p, s, s.b * heads + s.h, R, s.h * R, flag, threadIdx.x, [] { ptx::named_barrier_sync(1, 128); });
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

constexpr int kSmemPerCta = 112 * 1024;  // two CTAs on an SM

template <typename T, int D, int HP, int NT, bool BS8>
int launch_tc(Q8Params p, cudaStream_t stream) {
  using L = TcLayout<D, HP>;
  tvk::EncodeTiledFn encode = tvk::encode_tiled_fn();
  if (!encode) {
    tvk::set_error("cuTensorMapEncodeTiled is not available from the driver");
    return TVK_ERR_CUDA;
  }
  const cuuint64_t row = (cuuint64_t)p.n_kv_heads * D;
  const cuuint64_t dims[3] = {row, (cuuint64_t)p.block_size, (cuuint64_t)p.num_blocks};
  const cuuint64_t strides[2] = {row, row * p.block_size};
  const cuuint32_t box[3] = {(cuuint32_t)L::ROWB, (cuuint32_t)(p.block_size < kTile ? p.block_size : kTile), 1u};
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUtensorMapSwizzle sw = L::ROWB == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                : L::ROWB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                : CU_TENSOR_MAP_SWIZZLE_32B;
  CUtensorMap tm[2];
  for (int i = 0; i < 2; ++i) {
    const CUresult r = encode(&tm[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(i ? p.v_cache : p.k_cache), dims,
                              strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
      tvk::set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
      return TVK_ERR_CUDA;
    }
  }
  // as many stages as fit twice on an SM, 8 at most
  p.n_stages = 2;
  while (p.n_stages < 8 && L::bytes(p.n_stages + 1, p.group) <= kSmemPerCta) ++p.n_stages;
  const int smem = L::bytes(p.n_stages, p.group);
  auto kern = paged_decode_q8_tc_kernel<T, D, HP, NT, BS8>;
  int dev = 0;
  TVK_CHECK_CUDA(cudaGetDevice(&dev));
  static std::atomic<unsigned long long> attr_set{0};  // one bit per device
  if (dev >= 64 || !(attr_set.load() >> dev & 1)) {
    TVK_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerCta));
    if (dev < 64) attr_set.fetch_or(1ull << dev);
  }
  const long long most =
      (long long)p.batch * (p.n_kv_heads / HP) * ((p.max_ctx_tokens + kTile - 1) / kTile + kUnitTiles);
  const long long pieces = (most + kMinPiece - 1) / kMinPiece;
  const int grid = (int)(pieces < kTcCtas ? pieces : kTcCtas);
  TVK_CHECK_CUDA(tvk::launch_pdl(kern, grid, kTcThreads, smem, stream, p, tm[0], tm[1]));
  TVK_CHECK_LAUNCH("paged_decode_q8_tc");
  return TVK_OK;
}

template <typename T, int D, int HP>
int launch_heads(const Q8Params& p, cudaStream_t stream) {
  const bool bs8 = p.block_size == 8;
  if (p.group <= 8) return bs8 ? launch_tc<T, D, HP, 1, true>(p, stream) : launch_tc<T, D, HP, 1, false>(p, stream);
  return bs8 ? launch_tc<T, D, HP, 2, true>(p, stream) : launch_tc<T, D, HP, 2, false>(p, stream);
}

// 16-bit queries on the tensor cores where 64-token tiles are whole blocks or lie in one.
template <typename T>
int launch_16bit(const Q8Params& p, int head_dim, cudaStream_t stream) {
  const int bs = p.block_size;
  if (!(bs == 8 || bs == 16 || bs == 32 || bs % kTile == 0)) return launch_simt<T>(p, head_dim, stream);
  if (head_dim == 128) return launch_heads<T, 128, 1>(p, stream);
  if (head_dim == 64)
    return p.n_kv_heads % 2 == 0 ? launch_heads<T, 64, 2>(p, stream) : launch_heads<T, 64, 1>(p, stream);
  return p.n_kv_heads % 4 == 0 ? launch_heads<T, 32, 4>(p, stream) : launch_heads<T, 32, 1>(p, stream);
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
  const tvk::WaitTest wt = tvk::take_wait_test();
  p.wait_ns = wt.armed ? wt.limit_ns : tvk::kDefaultWaitNs;
  p.drop_loads = wt.armed ? 1 : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TVK_DTYPE_F16: return launch_16bit<__half>(p, head_dim, s);
    case TVK_DTYPE_BF16: return launch_16bit<__nv_bfloat16>(p, head_dim, s);
    default: return launch_simt<float>(p, head_dim, s);
  }
}
