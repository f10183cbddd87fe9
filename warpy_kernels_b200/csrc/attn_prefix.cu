// Attention of a batch of sequences over one shared prefix of keys and each sequence's own keys behind it: FP8 (e4m3) and
// BF16, head dimension 64 and 128, for decoding (few queries per sequence).
//
//   out = softmax(scale . q [K_prefix ; K_own]^T) [V_prefix ; V_own]
//
// Attending sequence by sequence reads the prefix once per sequence.  Here the query rows of ALL sequences that share a KV
// head are stacked, 128 to a tile, and go over the prefix together; the rows of one sequence (its group of query heads
// times its queries) go over its own keys.  Both are the same work: a unit is up to 128 rows and a range of 64-key tiles,
// S = Q.K^T and O += P.V with 128 x 64 tiles on tcgen05.  A sequence's few rows leave most of a tile empty, which costs
// nothing: those units wait for memory (a tile of 128 x 64 takes the tensor pipe 512 cycles, its keys 700 at an SM's share
// of the memory bandwidth), and the warps of empty rows skip the softmax.
//
// Work division: all tiles of all units form one line, prefix first, that is cut into as many equal pieces as CTAs fit the
// GPU (a tile of own keys counts more than one of the prefix).  Lengths are read on the device.  A CTA's piece of a unit is
// a segment; every segment leaves a partial result (O / l and the log-sum-exp of its rows, fp32) and a second kernel, set up
// beside the first, adds up the segments of every row, in the order of the line.
//
// One CTA (two per SM, 320 threads): warp 0 TMA producer, warp 1 issues the products, two softmax groups of four warps take
// the tiles in turn, one thread per row: the structure of attn_fwd_bf16.cu, persistent over its segments.  P is bf16 and
// overwrites its scores in tensor memory.  FP8: scores from e4m3 (kind::f8f6f4); V tiles are converted to bf16 (exact) in
// shared memory by the group that has the tile, so that P keeps 8 bits.
//
// Numerics: logits in base 2; the row reference is the maximum of the segment's first tile (bf16 has the exponent range to
// leave it there).  A segment in which a row rises more than 2^60 above its reference is gone through again at the end of
// its CTA, with the maxima it then knows.
#include <math.h>

#include "common.cuh"
#include "host_common.h"
#include "softmax16.cuh"

namespace wk {
namespace {

constexpr int X_ROWS = 128;  // rows of a tile
constexpr int X_KEYS = 64;   // keys of a tile
constexpr int X_THREADS = 320;
constexpr int X_SOFTMAX = 256;
constexpr int X_TMEM_COLS = 256;
constexpr int X_S_COLS = 64;  // buffer b at column 64 b; P over its first 32
constexpr int X_O_COL = 128;
constexpr float X_MAX_EXP = 60.f;
constexpr int X_CUM = 1024;   // sequences whose tile counts are kept in shared memory
constexpr int X_FLAGS = 512;  // segments of a CTA that are told apart when they are gone through again

struct PrefixParams {
  const uint8_t* q;
  const float* q_descale;
  const float* kp_descale;
  const float* vp_descale;
  const float* k_descale;
  const float* v_descale;
  const int* seqused;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_strides[3];  // bytes
  int64_t out_strides[3], lse_strides[2];
  int B, Hq, Hkv, group, Nq, P, S;
  int rows_all;      // stacked rows of a KV head: B . group . Nq
  int rows_own;      // of one sequence
  int own_slot;      // rows that a partial result of own keys has room for: min(128, rows_own)
  int units_p;       // Hkv . ceil(rows_all / 128), 0 without a prefix
  int blocks_p;      // ceil(rows_all / 128)
  int blocks_own;    // ceil(rows_own / 128)
  int tiles_p;       // of the prefix
  int ctas;          // grid of the main kernel
  int weight_p, weight_own;
  int causal, lse_natural;
  float scale_log2;  // softmax_scale . log2(e)
  int* cum;          // [B + 1] tiles of own keys before each sequence
  float* part;       // [row slot][DH]
  float* part_lse;   // [row slot]
  float* part_top;   // [row slot] largest score
  int* status;
};

// The line of tiles and its division.
struct Line {
  int Wp, W;   // weight of the prefix, of everything
  int G;       // pieces
  int wp, ws;  // weight of a tile
};
__device__ __forceinline__ Line make_line(const PrefixParams& p, int own_tiles) {
  Line l;
  const int per_seq = p.Hkv * p.blocks_own;
  const int tp = p.units_p * p.tiles_p, ts = own_tiles * per_seq;
  const bool few = tp + ts <= 4 * p.ctas;  // then the tiles are dealt out as evenly as they are
  l.wp = few ? 1 : p.weight_p, l.ws = few ? 1 : p.weight_own;
  l.Wp = tp * l.wp;
  l.W = l.Wp + ts * l.ws;
  l.G = min(p.ctas, l.W / max(l.wp, l.ws));  // every piece is at least one tile long
  return l;
}
__device__ __forceinline__ int piece_start(const Line& l, int c) {
  return static_cast<int>(static_cast<int64_t>(l.W) * c / l.G);
}
// The piece that weight x lies in.
__device__ __forceinline__ int owner(const Line& l, int x) {
  return static_cast<int>((static_cast<int64_t>(x + 1) * l.G - 1) / l.W);
}

struct Segment {
  bool own;
  int b, h;        // sequence (own keys) and KV head
  int row0, rows;  // of the unit's row space: stacked rows of the head, or rows of the sequence
  int tile0, tiles;
  int keys;        // length of the key range that tiles count in
  int64_t slot;    // first row slot
};

// The segments of piece c, one after the other.
struct Walker {
  const PrefixParams& p;
  const Line& l;
  const int* cum;
  int c, x, x1, b;
  __device__ __forceinline__ Walker(const PrefixParams& p, const Line& l, const int* cum, int c)
      : p(p), l(l), cum(cum), c(c), x(0), x1(0), b(-1) {
    if (c < l.G) x = piece_start(l, c), x1 = piece_start(l, c + 1);
  }
  __device__ __forceinline__ bool next(Segment& s) {
    while (x < x1) {
      int base, w, total;
      if (x < l.Wp) {
        w = l.wp, total = p.tiles_p;
        const int u = x / (total * w);
        base = u * total * w;
        s.own = false;
        s.h = u / p.blocks_p, s.b = 0;
        s.row0 = (u - s.h * p.blocks_p) * X_ROWS;
        s.rows = min(X_ROWS, p.rows_all - s.row0);
        s.keys = p.P;
        s.slot = static_cast<int64_t>(u + c) * X_ROWS;
      } else {
        w = l.ws;
        const int per_seq = p.Hkv * p.blocks_own;
        const int y = (x - l.Wp) / w;  // a tile (x need not be at its start: rounding down stays in it)
        if (b < 0) {  // the last sequence that starts at or before y
          int lo = 0, hi = p.B - 1;
          while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (cum[mid] * per_seq <= y) lo = mid; else hi = mid - 1;
          }
          b = lo;
        }
        while (cum[b + 1] * per_seq <= y) ++b;
        const int first = cum[b] * per_seq;
        total = cum[b + 1] - cum[b];
        const int u = (y - first) / total;
        base = l.Wp + (first + u * total) * w;
        s.own = true;
        s.b = b, s.h = u / p.blocks_own;
        s.row0 = (u - s.h * p.blocks_own) * X_ROWS;
        s.rows = min(X_ROWS, p.rows_own - s.row0);
        s.keys = p.seqused ? max(0, min(p.S, p.seqused[b])) : p.S;
        s.slot = static_cast<int64_t>(p.units_p + p.ctas) * X_ROWS + static_cast<int64_t>(b * per_seq + u + c) * p.own_slot;
      }
      s.tile0 = (x - base + w - 1) / w;
      const int end = min(total, (x1 - base + w - 1) / w);
      s.tiles = end - s.tile0;
      x = end == total ? base + total * w : x1;
      if (s.tiles > 0) return true;
    }
    return false;
  }
};

// Exclusive sums of the sequences' tile counts, by the whole CTA; `cum` is in shared or global memory.
__device__ __forceinline__ void sum_tiles(const PrefixParams& p, int* cum, int* warp_sums) {
  const int per = (p.B + X_THREADS - 1) / X_THREADS, b0 = threadIdx.x * per, b1 = min(p.B, b0 + per);
  auto tiles = [&](int b) {
    const int n = p.seqused ? max(0, min(p.S, p.seqused[b])) : p.S;
    return (n + X_KEYS - 1) / X_KEYS;
  };
  int sum = 0;
  for (int b = b0; b < b1; ++b) sum += tiles(b);
  int scan = sum;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int i = 1; i < 32; i *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, scan, i);
    if (lane >= i) scan += other;
  }
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  int at = scan - sum;
  for (int w = 0; w < warp; ++w) at += warp_sums[w];
  for (int b = b0; b < b1; ++b) {
    cum[b] = at;
    at += tiles(b);
  }
  if (b1 == p.B && b0 < p.B) cum[p.B] = at;
  __syncthreads();
}

template <bool FP8, int DH>
struct PrefixCfg {
  static constexpr int SIZE = FP8 ? 1 : 2;
  static constexpr int SPANS = FP8 ? 1 : DH / 64;      // 128-byte spans of a K row
  static constexpr int V_SPANS = DH / 64;              // of a V row in bf16
  static constexpr int Q_SPAN = X_ROWS * 128;          // bytes
  static constexpr int KV_SPAN = X_KEYS * 128;
  static constexpr int Q_BYTES = SPANS * Q_SPAN;
  static constexpr int K_BYTES = SPANS * KV_SPAN;      // of a stage; V as loaded likewise
  static constexpr int V16_BYTES = V_SPANS * KV_SPAN;
  static constexpr int STAGES = FP8 ? 3 : DH == 64 ? 4 : 2;
  static constexpr int Q_AT = 0;
  static constexpr int K_AT = Q_BYTES;
  static constexpr int V_AT = K_AT + STAGES * K_BYTES;
  static constexpr int V16_AT = V_AT + STAGES * K_BYTES;  // FP8 only: two buffers
  static constexpr int X_AT = V16_AT + (FP8 ? 2 * V16_BYTES : 0);
  // exchange: row reference, then l and largest score of each group; segments to go through again; warp sums
  static constexpr int FLAG_AT = X_AT + 5 * X_ROWS * 4;
  static constexpr int CUM_AT = FLAG_AT + X_FLAGS / 8 + 64;
  static constexpr int BAR_AT = CUM_AT + (X_CUM + 4) * 4;
  static constexpr int SMEM = BAR_AT + 8 * (4 * STAGES + 8) + 16 + 1024;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Four e4m3 codes -> two words of bf16 pairs, exact.  The code's exponent and mantissa moved to where bf16 has them are
// the value times 2^-120, subnormals included; one product puts that right.  The NaN codes would come out as 480.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  uint32_t x[2] = {__byte_perm(w, 0, 0x1404), __byte_perm(w, 0, 0x3424)};  // codes in the high bytes of the halves
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[i] = (x[i] & 0x80008000u) | ((x[i] >> 4) & 0x07f007f0u);
    x[i] = mul_bf16x2(x[i], 0x7b807b80u);  // 2^120
  }
  if ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (((w >> (8 * i)) & 0x7f) == 0x7f) x[i / 2] |= 0x7fffu << (16 * (i & 1));
  }
  lo = x[0], hi = x[1];
}

template <bool FP8, int DH>
__global__ void __launch_bounds__(X_THREADS, 2)
attn_prefix_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ PrefixParams p) {
  using C = PrefixCfg<FP8, DH>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_ptr = smem_raw + (smem - smem_u32(smem_raw));
  const uint32_t bars = smem + C::BAR_AT;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (ST + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * ST + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * ST + s); };
  const uint32_t misc = bars + 8u * 4 * ST;
  auto s_full = [&](int b) { return misc + 8u * b; };
  auto p_full = [&](int b) { return misc + 8u * (2 + b); };
  const uint32_t q_full = misc + 8u * 4, o_full = misc + 8u * 5, o_free = misc + 8u * 6, tmem_slot = misc + 8u * 7;
  volatile uint32_t* flags = reinterpret_cast<volatile uint32_t*>(smem_ptr + C::FLAG_AT);
  int* warp_sums = reinterpret_cast<int*>(smem_ptr + C::FLAG_AT + X_FLAGS / 8);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), FP8 ? X_SOFTMAX / 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_full(i), X_SOFTMAX / 2);
    }
    mbar_init(q_full, X_SOFTMAX);
    mbar_init(o_full, 1);
    mbar_init(o_free, X_SOFTMAX);
    mbar_fence_init();
  }
  if (threadIdx.x < X_FLAGS / 32) flags[threadIdx.x] = 0;
  if (warp == 1) {
    tmem_alloc(tmem_slot, X_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  pdl_launch_dependents();
  pdl_wait();
  // every CTA writes the same counts where they do not fit shared memory; the combining kernel reads them from there
  int* cum = p.B <= X_CUM ? reinterpret_cast<int*>(smem_ptr + C::CUM_AT) : p.cum;
  sum_tiles(p, cum, warp_sums);
  if (blockIdx.x == 0 && cum != p.cum)
    for (int i = threadIdx.x; i <= p.B; i += X_THREADS) p.cum[i] = cum[i];
  const Line line = make_line(p, cum[p.B]);

  int J = 0;       // tiles of the segments before this one
  int n_seg = 0;   // segments before this one, over both passes
  bool ok = true;  // no wait of this thread's role has given up
  for (int pass = 0; pass < 2; ++pass) {
    Walker walk(p, line, cum, blockIdx.x);
    Segment s;
    for (int i = 0; walk.next(s); ++i) {
      const int flag = min(i, X_FLAGS - 1);
      if (pass && !(flags[flag / 32] >> (flag % 32) & 1)) continue;
      if (warp == 0) {
        if (lane == 0) {
          const CUtensorMap* mk = s.own ? &map_k : &map_kp;
          const CUtensorMap* mv = s.own ? &map_v : &map_vp;
          for (int j = 0; ok && j < s.tiles; ++j) {
            const int st = (J + j) % ST;
            const uint32_t ph = ((J + j) / ST) & 1;
            const int key0 = (s.tile0 + j) * X_KEYS;
            ok = mbar_wait(k_empty(st), ph ^ 1, p.status, WK_ERR_TIMEOUT_EMPTY);
            if (!ok) break;
            mbar_expect_tx(k_full(st), C::K_BYTES);
            for (int c = 0; c < C::SPANS; ++c)
              tma_load_4d(smem + C::K_AT + st * C::K_BYTES + c * C::KV_SPAN, mk, k_full(st), 64 * c, key0, s.h, s.b);
            ok = mbar_wait(v_empty(st), ph ^ 1, p.status, WK_ERR_TIMEOUT_EMPTY);
            if (!ok) break;
            mbar_expect_tx(v_full(st), C::K_BYTES);
            for (int c = 0; c < C::SPANS; ++c)
              tma_load_4d(smem + C::V_AT + st * C::K_BYTES + c * C::KV_SPAN, mv, v_full(st), 64 * c, key0, s.h, s.b);
          }
        }
        __syncwarp();
      } else if (warp == 1) {
        const bool mine = elect_one();
        constexpr uint32_t idesc_qk = FP8 ? make_idesc(0, 0, 0, 0, X_ROWS, X_KEYS) : make_idesc(1, 1, 0, 0, X_ROWS, X_KEYS);
        constexpr uint32_t idesc_pv = make_idesc(1, 1, 0, 1, X_ROWS, DH);
        const uint64_t q_desc = smem_desc_sw128(smem + C::Q_AT, 16, 1024);
        ok = ok && mbar_wait_warp(q_full, n_seg & 1, p.status, WK_ERR_TIMEOUT_LOAD);
        // the tensor pipe runs in issue order: the scores also wait for the product that last read their buffer
        auto issue_qk = [&](int j) {
          const int st = (J + j) % ST;
          ok = ok && mbar_wait_warp(k_full(st), ((J + j) / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD);
          if (!ok) return;
          tc_fence_after();
          const uint64_t k_desc = smem_desc_sw128(smem + C::K_AT + st * C::K_BYTES, 16, 1024);
          const uint32_t d = tmem + ((J + j) & 1) * X_S_COLS;
          if (mine) {
#pragma unroll
            for (int k = 0; k < DH * C::SIZE / 32; ++k) {  // 32 bytes of the head dimension
              const uint64_t a = q_desc + (k >> 2) * (C::Q_SPAN >> 4) + 2 * (k & 3);
              const uint64_t b = k_desc + (k >> 2) * (C::KV_SPAN >> 4) + 2 * (k & 3);
              if (FP8) mma_f8_ss(d, a, b, idesc_qk, k != 0);
              else mma_f16_ss(d, a, b, idesc_qk, k != 0);
            }
            tc_commit(s_full((J + j) & 1));
            tc_commit(k_empty(st));
          }
        };
        issue_qk(0);
        if (s.tiles > 1) issue_qk(1);
        // O of the segment before has been read
        if (n_seg > 0) ok = ok && mbar_wait_warp(o_free, (n_seg - 1) & 1, p.status, WK_ERR_TIMEOUT_TMEM);
        for (int j = 0; ok && j < s.tiles; ++j) {
          const int st = (J + j) % ST, buf = (J + j) & 1;
          ok = mbar_wait_warp(p_full(buf), ((J + j) >> 1) & 1, p.status, WK_ERR_TIMEOUT_P);
          if (!FP8) ok = ok && mbar_wait_warp(v_full(st), ((J + j) / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD);
          if (!ok) break;
          tc_fence_after();
          const uint64_t v_desc = smem_desc_sw128(
              FP8 ? smem + C::V16_AT + buf * C::V16_BYTES : smem + C::V_AT + st * C::K_BYTES, C::KV_SPAN, 1024);
          if (mine) {
#pragma unroll
            for (int k = 0; k < X_KEYS / 16; ++k)
              mma_f16_ts(tmem + X_O_COL, tmem + buf * X_S_COLS + 8 * k, v_desc + 128 * k, idesc_pv, (j | k) != 0);
            if (!FP8) tc_commit(v_empty(st));
            if (j == s.tiles - 1) tc_commit(o_full);
          }
          if (j + 2 < s.tiles) issue_qk(j + 2);
        }
        __syncwarp();
      } else {
        const int quad = warp & 3, grp = (warp - 2) >> 2;
        const int t = threadIdx.x - 64;
        const int r = quad * 32 + lane;  // row of the tile = lane of tensor memory
        const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t s_tmem = tmem + lane_addr + grp * X_S_COLS;
        {
          // the unit's rows of Q, swizzled like a TMA tile; every product that read the last ones has completed
          constexpr int PIECES = DH * C::SIZE / 16;
          for (int x = t; x < s.rows * PIECES; x += X_SOFTMAX) {
            const int row = x / PIECES, c = x % PIECES;
            int m = s.row0 + row, b = s.b;
            if (!s.own) b = m / p.rows_own, m -= b * p.rows_own;
            const int g = m / p.Nq, n = m - g * p.Nq;
            const uint8_t* src = p.q + b * p.q_strides[0] + (s.h * p.group + g) * p.q_strides[1] + n * p.q_strides[2] + 16 * c;
            cp_async16(smem + C::Q_AT + (c >> 3) * C::Q_SPAN + row * 128 + (((c & 7) ^ (row & 7)) << 4), src);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          mbar_arrive(q_full);
        }
        const bool live = r < s.rows, warp_live = quad * 32 < s.rows;
        int b = s.b, limit = s.keys - 1;  // last key of the range that the row sees
        {
          int m = s.row0 + min(r, s.rows - 1);
          if (!s.own) b = m / p.rows_own, m -= b * p.rows_own;
          if (p.causal) {
            const int used = s.own ? s.keys : p.seqused ? max(0, min(p.S, p.seqused[b])) : p.S;
            limit = min(limit, (s.own ? 0 : p.P) + m % p.Nq + used - p.Nq);
          }
        }
        float beta = p.scale_log2, v_scale = 1.f;
        if (FP8) {
          beta *= p.q_descale[b * p.Hkv + s.h] * (s.own ? p.k_descale[b * p.Hkv + s.h] : p.kp_descale[s.h]);
          v_scale = s.own ? p.v_descale[b * p.Hkv + s.h] : p.vp_descale[s.h];
        }
        const uint32_t x_ref = smem + C::X_AT + r * 4;
        auto x_group = [&](int g) { return x_ref + (1 + 2 * g) * X_ROWS * 4; };
        const int64_t slot = s.slot + r;
        float m_ref = pass && live ? p.part_top[slot] : -INFINITY, top = -INFINITY, l = 0.f;
        bool met = false;
        for (int j = (J + grp) & 1; j < s.tiles; j += 2) {
          const int tile = J + j;
          ok = ok && mbar_wait_warp(s_full(grp), (tile >> 1) & 1, p.status, WK_ERR_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          const int key0 = (s.tile0 + j) * X_KEYS;
          const bool masked = __any_sync(0xffffffffu, key0 + X_KEYS - 1 > limit);
          const int last = limit - key0;  // columns beyond it are masked
          if (j == 0 && pass == 0) {
            float m = -INFINITY;
            if (warp_live) {
#pragma unroll 1
              for (int c = 0; c < 2; ++c) {
                uint32_t raw[32];
                tmem_ld32(s_tmem + c * 32, raw);
                tc_wait_ld();
                if (masked) {
#pragma unroll
                  for (int x = 0; x < 32; ++x)
                    if (c * 32 + x > last) raw[x] = 0xff800000u;
                }
                m = fmaxf(m, block_max(raw) * beta);
              }
            }
            m_ref = m;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(x_ref), "f"(m) : "memory");
          }
          if (!met) {
            asm volatile("bar.sync 1, 256;" ::: "memory");
            met = true;
            if (j != 0 && pass == 0) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(m_ref) : "r"(x_ref) : "memory");
          }
          const int st = tile % ST;
          if (FP8) {
            // this tile of V to bf16: a thread takes half a row.  Rows behind the last key become zeros, whatever the cache
            // holds there: 0 . V has to be 0.
            ok = mbar_wait_warp(v_full(st), (tile / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD);
            if (!ok) break;
            constexpr int HALF = DH / 32;  // 16-byte pieces of half a row
            const int row = r >> 1;
            const uint32_t src = smem + C::V_AT + st * C::K_BYTES + row * 128;
            const uint32_t dst = smem + C::V16_AT + grp * C::V16_BYTES + row * 128;
            const bool there = key0 + row < s.keys;
#pragma unroll
            for (int c = 0; c < HALF; ++c) {
              const int piece = (r & 1) * HALF + c;
              uint32_t w[4], o[8];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                           : "r"(src + ((piece ^ (row & 7)) << 4)));
#pragma unroll
              for (int x = 0; x < 4; ++x) e4m3x4_to_bf16(there ? w[x] : 0u, o[2 * x], o[2 * x + 1]);
              const uint32_t to = dst + (piece >> 2) * C::KV_SPAN;
              const int at = (2 * piece) & 7;
              sts128(to + ((at ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
              sts128(to + (((at + 1) ^ (row & 7)) << 4), o[4], o[5], o[6], o[7]);
            }
            mbar_arrive(v_empty(st));
            fence_proxy_async_smem();
          } else if (key0 + X_KEYS > s.keys) {
            ok = mbar_wait_warp(v_full(st), (tile / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD);
            if (!ok) break;
            const int row = r >> 1;
            if (key0 + row >= s.keys && (r & 1) < C::V_SPANS) {
              const uint32_t at = smem + C::V_AT + st * C::K_BYTES + (r & 1) * C::KV_SPAN + row * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) sts128(at + 16 * c, 0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          if (warp_live) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t raw[32];
              tmem_ld32(s_tmem + c * 32, raw);
              tc_wait_ld();
              if (masked) {
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (c * 32 + x > last) raw[x] = 0xff800000u;
              }
              top = fmaxf(top, block_max(raw) * beta);
              const float bias = m_ref > -INFINITY ? -m_ref : 0.f;
              uint32_t w[16];
              float sum;
              softmax_block(raw, beta, bias, w, sum);
              l += sum;
              uint32_t lo[8], hi[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) lo[x] = w[x], hi[x] = w[8 + x];
              tmem_st8(s_tmem + c * 16, lo);
              tmem_st8(s_tmem + c * 16 + 8, hi);
            }
            tc_wait_st();
          }
          tc_fence_before();
          mbar_arrive(p_full(grp));
        }
        if (!met) {  // no tile, or a wait gave up: the other group waits for the meeting all the same
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (pass == 0) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(m_ref) : "r"(x_ref) : "memory");
        }
        ok = ok && mbar_wait_warp(o_full, n_seg & 1, p.status, WK_ERR_TIMEOUT_MMA);
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(x_group(grp)), "f"(l) : "memory");
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(x_group(grp) + X_ROWS * 4), "f"(top) : "memory");
        asm volatile("bar.sync 1, 256;" ::: "memory");
        float l2, top2;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(l2) : "r"(x_group(grp ^ 1)) : "memory");
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(top2) : "r"(x_group(grp ^ 1) + X_ROWS * 4) : "memory");
        l += l2;
        top = fmaxf(top, top2);
        if (ok) {
          tc_fence_after();
          const float inv = l > 0.f ? v_scale / l : l == l ? 0.f : l;  // NaN stays
          float* dst = p.part + slot * DH + grp * (DH / 2);
          if (warp_live) {
#pragma unroll
            for (int c = 0; c < DH / 64; ++c) {
              uint32_t v[32];
              tmem_ld32(tmem + lane_addr + X_O_COL + grp * (DH / 2) + c * 32, v);
              tc_wait_ld();
              if (live)
#pragma unroll
                for (int x = 0; x < 8; ++x)
                  reinterpret_cast<float4*>(dst + c * 32)[x] =
                      make_float4(__uint_as_float(v[4 * x]) * inv, __uint_as_float(v[4 * x + 1]) * inv,
                                  __uint_as_float(v[4 * x + 2]) * inv, __uint_as_float(v[4 * x + 3]) * inv);
              __syncwarp();
            }
          }
          if (live && grp == 0) {
            p.part_lse[slot] = l == 0.f ? -INFINITY : m_ref + log2f(l);
            p.part_top[slot] = top;
            if (pass == 0 && top - m_ref > X_MAX_EXP)
              atomicOr(const_cast<uint32_t*>(flags) + flag / 32, 1u << (flag % 32));
          }
        }
        tc_fence_before();
        mbar_arrive(o_free);
        __syncwarp();
      }
      J += s.tiles;
      ++n_seg;
    }
    __syncthreads();  // flags and largest scores are there
    if (pass == 0) {
      bool any = false;
      for (int i = 0; i < X_FLAGS / 32; ++i) any |= flags[i] != 0;
      if (!any) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, X_TMEM_COLS);
  }
}

// Adds up the segments of every row.  WARPS warps for a row, a row of a CTA's 8 / WARPS.
template <int DH, int WARPS>
__global__ void __launch_bounds__(256)
attn_prefix_combine_kernel(const __grid_constant__ PrefixParams p) {
  constexpr int COLS = DH / 32;  // per lane
  __shared__ float part_o[8][DH], part_m[8], part_l[8];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int row = blockIdx.x * (8 / WARPS) + warp / WARPS, share = warp % WARPS;
  const int rows = p.B * p.Hq * p.Nq;
  const bool live = row < rows;
  int b = 0, head = 0, n = 0;
  float m = -INFINITY, l = 0.f, o[COLS];
#pragma unroll
  for (int i = 0; i < COLS; ++i) o[i] = 0.f;
  auto add = [&](int64_t slot) {
    const float x = __ldcg(p.part_lse + slot);
    float v[COLS];
    const float* src = p.part + slot * DH + lane * COLS;
    if (COLS == 4) {
      const float4 w = __ldcg(reinterpret_cast<const float4*>(src));
      v[0] = w.x, v[1] = w.y, v[COLS - 2] = w.z, v[COLS - 1] = w.w;
    } else {
      const float2 w = __ldcg(reinterpret_cast<const float2*>(src));
      v[0] = w.x, v[1] = w.y;
    }
    const float top = fmaxf(m, x);
    const float f = m > -INFINITY ? exp2f(m - top) : 0.f, g = x == -INFINITY ? 0.f : exp2f(x - top);
    l = l * f + g;
#pragma unroll
    for (int i = 0; i < COLS; ++i) o[i] = o[i] * f + v[i] * g;
    m = top;
  };
  if (live) {
    n = row % p.Nq;
    head = row / p.Nq % p.Hq;
    b = row / p.Nq / p.Hq;
    const Line line = make_line(p, __ldcg(p.cum + p.B));
    const int h = head / p.group, own = (head - h * p.group) * p.Nq + n;  // row among the sequence's
    if (p.units_p > 0) {
      const int stacked = b * p.rows_own + own;
      const int u = h * p.blocks_p + stacked / X_ROWS, x = u * p.tiles_p * line.wp;
      const int c0 = owner(line, x), c1 = owner(line, x + (p.tiles_p - 1) * line.wp);
      for (int c = c0 + share; c <= c1; c += WARPS) add(static_cast<int64_t>(u + c) * X_ROWS + stacked % X_ROWS);
    }
    const int before = __ldcg(p.cum + b), tiles = __ldcg(p.cum + b + 1) - before;
    if (tiles > 0) {
      const int per_seq = p.Hkv * p.blocks_own, u = h * p.blocks_own + own / X_ROWS;
      const int x = line.Wp + (before * per_seq + u * tiles) * line.ws;
      const int c0 = owner(line, x), c1 = owner(line, x + (tiles - 1) * line.ws);
      for (int c = c0 + share; c <= c1; c += WARPS)
        add(static_cast<int64_t>(p.units_p + p.ctas) * X_ROWS + static_cast<int64_t>(b * per_seq + u + c) * p.own_slot + own % X_ROWS);
    }
  }
  if (WARPS > 1) {
#pragma unroll
    for (int i = 0; i < COLS; ++i) part_o[warp][lane * COLS + i] = o[i];
    if (lane == 0) part_m[warp] = m, part_l[warp] = l;
    __syncthreads();
    if (share) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part_m[warp + w]);
    m = top, l = 0.f;
#pragma unroll
    for (int i = 0; i < COLS; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float x = part_m[warp + w], f = x == -INFINITY ? 0.f : exp2f(x - top);
      l += part_l[warp + w] * f;
#pragma unroll
      for (int i = 0; i < COLS; ++i) o[i] += part_o[warp + w][lane * COLS + i] * f;
    }
  }
  if (!live) return;
  const bool empty = l == 0.f;
  const float inv = empty ? 0.f : 1.f / l;
  __nv_bfloat16* dst = p.out + b * p.out_strides[0] + head * p.out_strides[1] + n * p.out_strides[2] + lane * COLS;
  if (COLS == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[COLS - 2] * inv, o[COLS - 1] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[0] * inv, o[1] * inv);
  if (p.lse && lane == 0) {
    const float x = empty ? INFINITY : m + log2f(l);
    p.lse[b * p.lse_strides[0] + head * p.lse_strides[1] + n] = p.lse_natural ? x * 0.6931471805599453f : x;
  }
}

struct Sizes {
  int rows_own, own_slot, blocks_own, blocks_p, units_p, tiles_p, tiles_own, ctas;
  int64_t row_slots, cum_bytes, bytes;
};

// false if the problem is beyond the kernels' 32-bit counts.
bool sizes_of(int B, int Hq, int Hkv, int Nq, int P, int S, int d, int sms, Sizes& z) {
  const int64_t rows_own = static_cast<int64_t>(Hq / Hkv) * Nq, rows_all = rows_own * B;
  if (rows_all * Hkv > INT32_MAX / 2) return false;
  z.rows_own = static_cast<int>(rows_own);
  z.own_slot = rows_own < X_ROWS ? z.rows_own : X_ROWS;
  z.blocks_own = static_cast<int>((rows_own + X_ROWS - 1) / X_ROWS);
  z.blocks_p = static_cast<int>((rows_all + X_ROWS - 1) / X_ROWS);
  z.tiles_p = P / X_KEYS + (P % X_KEYS != 0);
  z.tiles_own = S / X_KEYS + (S % X_KEYS != 0);
  z.units_p = z.tiles_p ? Hkv * z.blocks_p : 0;
  const int64_t units_own = static_cast<int64_t>(B) * Hkv * z.blocks_own;
  const int64_t tiles = static_cast<int64_t>(z.units_p) * z.tiles_p + units_own * z.tiles_own;
  if (tiles > INT32_MAX / 16) return false;
  z.ctas = static_cast<int>(tiles < 2 * sms ? (tiles > 0 ? tiles : 1) : 2 * sms);
  z.row_slots = static_cast<int64_t>(z.units_p + z.ctas) * X_ROWS + (units_own + z.ctas) * z.own_slot;
  z.cum_bytes = (static_cast<int64_t>(B) * 4 + 4 + 15) / 16 * 16;
  z.bytes = z.cum_bytes + z.row_slots * (d + 2) * 4;
  return true;
}

template <bool FP8, int DH>
int launch_prefix(const CUtensorMap (&maps)[4], PrefixParams& p, cudaStream_t stream) {
  using C = PrefixCfg<FP8, DH>;
  static_assert(2 * (C::SMEM + 1024) <= 228 * 1024, "two CTAs per SM");
  const void* fn = reinterpret_cast<const void*>(attn_prefix_kernel<FP8, DH>);
  if (allow_smem(fn, C::SMEM)) return WK_E_CUDA;
  if (int bad = launch_pdl(fn, dim3(p.ctas), X_THREADS, C::SMEM, stream, 1,
                           {const_cast<CUtensorMap*>(&maps[0]), const_cast<CUtensorMap*>(&maps[1]),
                            const_cast<CUtensorMap*>(&maps[2]), const_cast<CUtensorMap*>(&maps[3]), &p}))
    return bad;
  // few rows have many segments each: a CTA for a row
  const int rows = p.B * p.Hq * p.Nq;
  if (rows <= 8 * 148)
    return launch_pdl(reinterpret_cast<const void*>(attn_prefix_combine_kernel<DH, 8>), dim3(rows), 256, 0, stream, 1, {&p});
  return launch_pdl(reinterpret_cast<const void*>(attn_prefix_combine_kernel<DH, 1>), dim3((rows + 7) / 8), 256, 0, stream, 1,
                    {&p});
}

}  // namespace
}  // namespace wk

extern "C" int64_t wk_attn_fwd_shared_prefix_workspace_bytes(int B, int Hq, int Hkv, int Nq, int P, int S, int d) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Nq <= 0 || P < 0 || S < 0 || (d != 64 && d != 128)) return 0;
  const int sms = wk::sm_count();
  wk::Sizes z;
  return sms > 0 && wk::sizes_of(B, Hq, Hkv, Nq, P, S, d, sms, z) ? z.bytes : 0;
}

extern "C" int wk_attn_fwd_shared_prefix(const wk_attn_prefix_args* a, void* stream) {
  using namespace wk;
  if (!a) return WK_E_ARG;
  if (a->B <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->Nq <= 0 || a->P < 0 || a->S < 0) return WK_E_ARG;
  if (a->d != 64 && a->d != 128) return WK_E_ARG;
  if (!a->q || !a->out || (a->P && (!a->k_prefix || !a->v_prefix)) || (a->S && (!a->k || !a->v))) return WK_E_ARG;
  const bool fp8 = a->fp8 != 0;
  if (fp8 && (!a->q_descale || (a->P && (!a->k_prefix_descale || !a->v_prefix_descale)) ||
              (a->S && (!a->k_descale || !a->v_descale))))
    return WK_E_ARG;
  if (!fp8 && (a->q_descale || a->k_descale || a->v_descale || a->k_prefix_descale || a->v_prefix_descale)) return WK_E_ARG;
  if (!(a->softmax_scale > 0.f)) return WK_E_ARG;
  const int size = fp8 ? 1 : 2;
  auto rows_ok = [](const void* base, const int64_t* st, int bytes, int unit) {
    if (reinterpret_cast<uintptr_t>(base) % unit) return false;
    for (int i = 0; i < 3; ++i)
      if (st[i] <= 0 || st[i] * bytes % unit) return false;
    return true;
  };
  if (!rows_ok(a->q, a->q_strides, size, 16) || !rows_ok(a->out, a->out_strides, 2, 8)) return WK_E_ARG;
  if (a->P && (!rows_ok(a->k_prefix, a->k_prefix_strides, size, 16) || !rows_ok(a->v_prefix, a->v_prefix_strides, size, 16)))
    return WK_E_ARG;
  if (a->S && (!rows_ok(a->k, a->k_strides, size, 16) || !rows_ok(a->v, a->v_strides, size, 16))) return WK_E_ARG;
  if (int unsupported = require_sm100()) return unsupported;
  const int sms = sm_count();
  Sizes z;
  if (sms <= 0) return WK_E_CUDA;
  if (!sizes_of(a->B, a->Hq, a->Hkv, a->Nq, a->P, a->S, a->d, sms, z)) return WK_E_ARG;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < z.bytes) return WK_E_ARG;
  PrefixParams p = {};
  p.status = status_word();
  if (!p.status) return WK_E_CUDA;

  CUtensorMap maps[4] = {};
  const void* bases[4] = {a->k_prefix, a->v_prefix, a->k, a->v};
  const int64_t* strides[4] = {a->k_prefix_strides, a->v_prefix_strides, a->k_strides, a->v_strides};
  const uint32_t box[4] = {fp8 ? 128u : 64u, X_KEYS, 1, 1};
  for (int i = 0; i < 4; ++i) {
    const int len = i < 2 ? a->P : a->S;
    if (!len) continue;  // no tile of it is ever loaded
    const uint64_t dims[4] = {static_cast<uint64_t>(a->d), static_cast<uint64_t>(len), static_cast<uint64_t>(a->Hkv),
                              static_cast<uint64_t>(i < 2 ? 1 : a->B)};
    const uint64_t str[3] = {static_cast<uint64_t>(strides[i][2]) * size, static_cast<uint64_t>(strides[i][1]) * size,
                             static_cast<uint64_t>(strides[i][0]) * size};
    if (int bad = encode_tmap(&maps[i], fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, bases[i], dims,
                              str, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return bad;
  }
  p.q = static_cast<const uint8_t*>(a->q);
  p.q_descale = a->q_descale, p.kp_descale = a->k_prefix_descale, p.vp_descale = a->v_prefix_descale;
  p.k_descale = a->k_descale, p.v_descale = a->v_descale;
  p.seqused = a->seqused_k;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  for (int i = 0; i < 3; ++i) p.q_strides[i] = a->q_strides[i] * size, p.out_strides[i] = a->out_strides[i];
  p.lse_strides[0] = a->lse_strides[0], p.lse_strides[1] = a->lse_strides[1];
  p.B = a->B, p.Hq = a->Hq, p.Hkv = a->Hkv, p.group = a->Hq / a->Hkv, p.Nq = a->Nq, p.P = a->P, p.S = a->S;
  p.rows_own = z.rows_own, p.rows_all = z.rows_own * a->B, p.own_slot = z.own_slot;
  p.units_p = z.units_p, p.blocks_p = z.blocks_p, p.blocks_own = z.blocks_own, p.tiles_p = z.tiles_p, p.ctas = z.ctas;
  p.weight_p = 1, p.weight_own = 2;
  p.causal = a->causal, p.lse_natural = a->lse_natural;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.cum = static_cast<int*>(a->workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + z.cum_bytes);
  p.part_lse = p.part + z.row_slots * a->d;
  p.part_top = p.part_lse + z.row_slots;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp8) return a->d == 64 ? launch_prefix<true, 64>(maps, p, st) : launch_prefix<true, 128>(maps, p, st);
  return a->d == 64 ? launch_prefix<false, 64>(maps, p, st) : launch_prefix<false, 128>(maps, p, st);
}
