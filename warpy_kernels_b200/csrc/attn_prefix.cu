// Attention of a batch of sequences over one shared prefix of keys and each sequence's own keys behind it: FP8 (e4m3) and
// BF16, head dimension 64 and 128, for decoding (few queries per sequence).
//
//   out = softmax(scale . q [K_prefix ; K_own]^T) [V_prefix ; V_own]
//
// Attending sequence by sequence reads the prefix once per sequence.  Here the query rows of ALL sequences that share a KV
// head are stacked, 128 to a tile, and go over the prefix together; the rows of one sequence (its group of query heads
// times its queries) go over its own keys.
//
// Own keys come first, and leave parts: O / l and the log-sum-exp of every row, fp32.  Few rows a sequence take a kernel on
// mma.sync whose warps work by themselves, more the tensor-core kernel below, one CTA for 128 of them (own_by_rows).
// The prefix: a unit is 128 stacked rows, and S = Q.K^T and O += P.V go by 128 x 64 tiles on tcgen05.  A unit's tiles are
// divided over the CTAs of a cluster, which meet in distributed shared memory, add the own keys' parts and write the output.
// Where units are few, several clusters share one; then they leave parts too, and a last kernel adds up all of them.  The
// prefix kernel is set up and runs beside the one for own keys and waits for its end before it reads its parts.
//
// One CTA of the tensor-core kernel (two per SM, 320 threads): warp 0 TMA producer, warp 1 issues the products, two softmax
// groups of four warps take the tiles in turn, one thread per row: the structure of attn_fwd_bf16.cu.  P has 16 bits and
// overwrites its scores in tensor memory.  BF16: P is bf16.  FP8: scores from e4m3 (kind::f8f6f4); V tiles become f16 (exact)
// in shared memory, by the group that has the tile and while its scores are computed, and P is f16.
//
// Numerics: logits in base 2; statistics, sums and parts in fp32.  P is rounded to 16 bits for the tensor core: by 2^-8 of
// itself in bf16, 2^-11 in f16; the row sums take it before that.  Tensor-core kernel: the row reference is the maximum of
// the CTA's first tile; a CTA in which a row rises more than 2^60 above it (bf16 has the exponent range) goes through its
// keys once more, with the maxima it then knows.  FP8: f16 P is stored times 2^3 and may rise 2^12; one below 2^-17 of the
// reference is off by 2^-28 of it at most.  Kernel for few rows: the reference moves when a score exceeds it by more than 1;
// P is bf16, or f16 times 2^14 for FP8 inputs, whose K and V become f16 (exact).
//
// What bounds it.  The prefix kernel: 1090 cycles per 128 x 64 tile and SM, where the exponentials need 512 and the products
// 400 to 640 (ncu: MUFU 50 %, tensor pipe 37 %, issue slots 52 %): the chain scores -> P -> product with two groups in each
// of two CTAs (at 96 registers a thread, 12 to 152 bytes of them read back from local memory).  128 sequences, 64 / 8 heads,
// so 1024 stacked rows of each of 8 heads, over 32768 keys: 135 us FP8, 141 us bf16 a call (1020 / 975 TFLOP/s).  (V to bf16
// by integer arithmetic instead, behind the scores: 164 where the present form then took 130; 128-key tiles in one CTA per
// SM, tensor memory read ahead, waits that poll: no faster.)
// Those are for logits of 1.5 nats' spread.  In FP8 a rise of 2^12 is 8.3 nats: with a wider spread more CTAs go through their
// keys twice.  The same call at 1.5, 2, 2.5, 3 and 4 nats: 139, 189, 227, 256, 257 us FP8, 144 to 145 bf16 (2^60).
// Own keys: their bytes in bf16 (97 us for 537 MB), the latency of a warp's instructions in FP8 (64 us for 268 MB).
// Whole calls, inputs from HBM: 16 sequences, 64 / 8 heads, 8192 shared and up to 1024 own bf16 keys 26.5 us; 128 sequences,
// 32768 and up to 2048 FP8 keys 200 to 210 us; 24 sequences, 32 / 8 heads, 5 queries, 4096 and up to 512 bf16 keys 38 us;
// 64 sequences, 32 heads, 2048 and up to 300 FP8 keys 33.5 us.
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "host_common.h"
#include "pair.cuh"
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
// How far (as a power of two) a row may rise above its reference before the CTA goes through its keys again, and what P is
// stored times: bf16 has the exponent range, f16 (FP8 inputs) needs a larger P for the small probabilities.
constexpr float X_MAX_EXP = 60.f, X_MAX_EXP_F16 = 12.f, X_SHIFT_F16 = 3.f, X_SHIFT_AGAIN = 14.f;
constexpr int X_CLUSTER = 16;  // largest cluster
constexpr int X_PAD = 4;       // values between rows in the exchange: lanes with neighbouring rows write without conflicts

constexpr int Y_START = 1;  // what a unit of the kernel for few rows weighs beside its steps
constexpr int Y_WARPS = 4;
constexpr int Y_ROWS = 16;      // rows of one of its units, at most
constexpr int Y_CUM = 1024;     // sequences whose weights are summed in shared memory
constexpr int OWN_PARTS = 32;   // parts of a unit of own keys, at most

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
  int64_t q_strides[3];                    // bytes
  int64_t out_strides[3], lse_strides[2];  // elements
  int B, Hq, Hkv, group, Nq, P, S;
  int rows_all;    // stacked rows of a KV head: B . group . Nq
  int rows_own;    // of one sequence
  int blocks_p;    // units of a KV head's stacked rows
  int tiles_p;     // of the prefix
  int cluster;     // CTAs of a cluster
  int splits;      // clusters that share a unit
  int by_rows;     // own keys go to the kernel for few rows
  int blocks_own;  // units of a sequence's rows: 16 rows each, or 128
  int own_slot;    // rows of one of their parts
  int pieces;      // by_rows: pieces that the line of units may be cut into,
  int least;       // and how long they are at least: no unit then has more than OWN_PARTS parts
  int causal, lse_natural;
  float scale_log2;  // softmax_scale . log2(e)
  int* cum;          // [B + 1] by_rows: weight of the sequences' units before each of them
  int* lengths;      // [B] by_rows: own keys of the sequences
  float* part;       // O / l of row slots [DH]: the prefix's, 128 a unit and split, then those of own keys
  float* part_lse;   // [row slot]
  int64_t own_parts;  // first row slot of own keys
  int* status;
};

// Own keys of sequence b.
__device__ __forceinline__ int own_keys(const PrefixParams& p, int b) {
  return p.seqused ? max(0, min(p.S, __ldcg(p.seqused + b))) : p.S;
}

// A line of W units of weight, cut into G pieces whose lengths differ by one at most.
struct Pieces {
  int W, G;
  int size, longer;  // of a piece; how many (the first ones) are one longer
  __device__ __forceinline__ Pieces(int weight, int most, int least) {
    W = weight, G = max(min(most, W / least), 1);
    size = W / G;
    longer = W - size * G;
  }
  __device__ __forceinline__ int start(int c) const { return c * size + min(c, longer); }
  // The piece that weight x lies in.
  __device__ __forceinline__ int owner(int x) const {
    const int edge = longer * (size + 1);
    return x < edge ? x / (size + 1) : longer + (x - edge) / size;
  }
};
// First row slot of the part that a piece leaves of a unit of own keys.
__device__ __forceinline__ int64_t own_slot_of(const PrefixParams& p, int unit, int piece) {
  return p.own_parts + static_cast<int64_t>(unit + piece) * p.own_slot;
}

// The parts that own keys have left of a row (row `own` of sequence b at KV head h): their row slots are
// first + i . distance.
struct OwnParts {
  int64_t first;
  int count, distance;
  __device__ __forceinline__ OwnParts(const PrefixParams& p, int b, int h, int own) : first(0), count(0), distance(p.own_slot) {
    if (!p.S) return;
    if (p.by_rows) {
      const int all = __ldcg(p.cum + p.B), before = __ldcg(p.cum + b), weight = __ldcg(p.cum + b + 1) - before;
      if (weight <= Y_START) return;
      const int per_seq = p.Hkv * p.blocks_own, u = h * p.blocks_own + own / Y_ROWS, x = before * per_seq + u * weight;
      const Pieces line(all * per_seq, p.pieces, p.least);
      const int c = line.owner(x + Y_START);
      count = line.owner(x + weight - 1) - c + 1;
      first = own_slot_of(p, b * per_seq + u, c) + own % Y_ROWS;
    } else if (own_keys(p, b)) {
      count = 1;
      first = own_slot_of(p, (b * p.Hkv + h) * p.blocks_own + own / X_ROWS, 0) + own % X_ROWS;
    }
  }
};

// How a row of the tensor-core kernel ends: where it goes and which parts own keys have left of it, found by the producer
// warp while the last tiles are worked on; and what all its parts count.
struct RowTarget {
  int64_t first;    // row slot of the first part of own keys
  int64_t to;       // offset in the output, or row slot
  int64_t lse_to;
  int parts;
};
template <bool FP8, int DH>
struct PrefixCfg {
  static constexpr int SIZE = FP8 ? 1 : 2;
  static constexpr int SPANS = FP8 ? 1 : DH / 64;      // 128-byte spans of a K row
  static constexpr int V_SPANS = DH / 64;              // of a V row in 16 bits
  static constexpr int Q_SPAN = X_ROWS * 128;          // bytes
  static constexpr int KV_SPAN = X_KEYS * 128;
  static constexpr int Q_BYTES = SPANS * Q_SPAN;
  static constexpr int K_BYTES = SPANS * KV_SPAN;      // of a stage; V as loaded likewise
  static constexpr int V16_BYTES = V_SPANS * KV_SPAN;
  static constexpr int STAGES = FP8 || DH == 128 ? 2 : 4;
  static constexpr int V16S = 3;  // FP8: buffers of V in f16
  static constexpr int Q_AT = 0;
  static constexpr int K_AT = Q_BYTES;
  static constexpr int V_AT = K_AT + STAGES * K_BYTES;
  static constexpr int V16_AT = V_AT + STAGES * K_BYTES;  // FP8 only
  // row reference, then l and largest score of each group; at the end the log-sum-exp of each row
  static constexpr int X_AT = V16_AT + (FP8 ? V16S * V16_BYTES : 0);
  static constexpr int ROW_AT = X_AT + 5 * X_ROWS * 4;  // where each row of Q is
  static constexpr int TARGET_AT = ROW_AT + X_ROWS * 8;
  static constexpr int BAR_AT = TARGET_AT + X_ROWS * static_cast<int>(sizeof(RowTarget));
  static constexpr int SMEM = BAR_AT + 8 * (4 * STAGES + 7 + V16S) + 1024;
  // the exchange of a cluster takes the place of the tiles
  static constexpr int PART_BYTES = X_ROWS * (DH + X_PAD) * 4;
  static_assert(PART_BYTES <= X_AT, "");
};

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// OWN: the rows of one sequence over its own keys, one CTA for 128 rows, which leaves a part.  Else: stacked rows over the
// prefix.
template <bool FP8, int DH, bool OWN>
__global__ void __launch_bounds__(X_THREADS, 2)
attn_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ PrefixParams p) {
  using C = PrefixCfg<FP8, DH>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = smem + C::BAR_AT;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (ST + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * ST + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * ST + s); };
  const uint32_t misc = bars + 8u * 4 * ST;
  auto s_full = [&](int b) { return misc + 8u * b; };
  auto p_full = [&](int b) { return misc + 8u * (2 + b); };
  const uint32_t q_full = misc + 8u * 4, o_full = misc + 8u * 5, tmem_slot = misc + 8u * 6;
  auto v16_empty = [&](int s) { return misc + 8u * (7 + s); };
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
    for (int i = 0; i < C::V16S; ++i) mbar_init(v16_empty(i), 1);
    mbar_fence_init();
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, X_TMEM_COLS);
    tmem_relinquish();
  }
  // the unit: sequence (own keys), KV head, first row, rows, this CTA's tiles
  int b = 0, h, row0, rows, tile0, tiles, keys;
  if (OWN) {
    const int u = blockIdx.x / p.blocks_own;
    row0 = (blockIdx.x - u * p.blocks_own) * X_ROWS;
    b = u / p.Hkv, h = u - b * p.Hkv;
    rows = min(X_ROWS, p.rows_own - row0);
  } else {
    const int share = blockIdx.x % (p.cluster * p.splits), u = blockIdx.x / (p.cluster * p.splits);
    h = u / p.blocks_p, row0 = (u - h * p.blocks_p) * X_ROWS;
    rows = min(X_ROWS, p.rows_all - row0);
    keys = p.P;
    const int shares = p.cluster * p.splits, each = p.tiles_p / shares, more = p.tiles_p - each * shares;
    tile0 = share * each + min(share, more);
    tiles = each + (share < more);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  // Beside the kernel for own keys, what kernels before that one wrote is read through L2 only, by TMA behind a proxy fence.
  const bool beside = !OWN && p.S > 0;
  if (!beside) pdl_wait();
  pdl_launch_dependents();
  if (OWN) {
    keys = own_keys(p, b);
    tile0 = 0, tiles = (keys + X_KEYS - 1) / X_KEYS;
  }

  const int rank = blockIdx.x % p.cluster, members = p.cluster;
  const int mine = rank < rows ? (rows - rank + members - 1) / members : 0;  // the rows congruent to this CTA's rank
  const bool final = p.splits == 1;
  uint8_t* smem_ptr = smem_raw + (smem - smem_u32(smem_raw));
  RowTarget* targets = reinterpret_cast<RowTarget*>(smem_ptr + C::TARGET_AT);
  auto find_targets = [&]() {  // by the producer warp
    if (beside) pdl_wait();    // the parts of own keys are there
    for (int i = lane; i < mine; i += 32) {
      const int r = i * members + rank;
      RowTarget e = {};
      int own = row0 + r;
      const int seq = own / p.rows_own;
      own -= seq * p.rows_own;
      if (final) {
        const int g = own / p.Nq, n = own - g * p.Nq, head = h * p.group + g;
        e.to = seq * p.out_strides[0] + head * p.out_strides[1] + n * p.out_strides[2];
        e.lse_to = seq * p.lse_strides[0] + head * p.lse_strides[1] + n;
        if (beside) {
          const OwnParts parts(p, seq, h, own);
          e.first = parts.first, e.parts = parts.count;
        }
      } else {
        e.to = static_cast<int64_t>(blockIdx.x / p.cluster) * X_ROWS + r;
      }
      targets[i] = e;
    }
  };

  bool ok = true;  // no wait of this thread's role has given up
  float lse_row = -INFINITY, inv_row = 0.f;  // softmax threads: of their row, what its O is multiplied with
  float m_ref = -INFINITY;
  for (int pass = 0; tiles > 0; ++pass) {
    const int J = pass * tiles;  // tiles before this pass
    bool far = false;
    if (warp == 0) {
      if (lane == 0) {
        if (beside) pdl_acquire_async();
        for (int j = 0; ok && j < tiles; ++j) {
          const int st = (J + j) % ST;
          const uint32_t ph = ((J + j) / ST) & 1;
          const int key0 = (tile0 + j) * X_KEYS;
          ok = mbar_wait(k_empty(st), ph ^ 1, p.status, WK_ERR_TIMEOUT_EMPTY);
          if (!ok) break;
          mbar_expect_tx(k_full(st), C::K_BYTES);
          for (int c = 0; c < C::SPANS; ++c)
            tma_load_4d(smem + C::K_AT + st * C::K_BYTES + c * C::KV_SPAN, &map_k, k_full(st), 64 * c, key0, h, b);
          ok = mbar_wait(v_empty(st), ph ^ 1, p.status, WK_ERR_TIMEOUT_EMPTY);
          if (!ok) break;
          mbar_expect_tx(v_full(st), C::K_BYTES);
          for (int c = 0; c < C::SPANS; ++c)
            tma_load_4d(smem + C::V_AT + st * C::K_BYTES + c * C::KV_SPAN, &map_v, v_full(st), 64 * c, key0, h, b);
        }
      }
      __syncwarp();
      if (!OWN && pass == 0) find_targets();
    } else if (warp == 1) {
      const bool mine = elect_one();
      constexpr uint32_t idesc_qk = FP8 ? make_idesc(0, 0, 0, 0, X_ROWS, X_KEYS) : make_idesc(1, 1, 0, 0, X_ROWS, X_KEYS);
      constexpr uint32_t idesc_pv = make_idesc(!FP8, !FP8, 0, 1, X_ROWS, DH);
      const uint64_t q_desc = smem_desc_sw128(smem + C::Q_AT, 16, 1024);
      if (pass == 0) ok = mbar_wait_warp(q_full, 0, p.status, WK_ERR_TIMEOUT_LOAD);
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
            const uint64_t x = q_desc + (k >> 2) * (C::Q_SPAN >> 4) + 2 * (k & 3);
            const uint64_t y = k_desc + (k >> 2) * (C::KV_SPAN >> 4) + 2 * (k & 3);
            if (FP8) mma_f8_ss(d, x, y, idesc_qk, k != 0);
            else mma_f16_ss(d, x, y, idesc_qk, k != 0);
          }
          tc_commit(s_full((J + j) & 1));
          tc_commit(k_empty(st));
        }
      };
      issue_qk(0);
      if (tiles > 1) issue_qk(1);
      for (int j = 0; ok && j < tiles; ++j) {
        const int st = (J + j) % ST, buf = (J + j) & 1;
        ok = mbar_wait_warp(p_full(buf), ((J + j) >> 1) & 1, p.status, WK_ERR_TIMEOUT_P);
        if (!FP8) ok = ok && mbar_wait_warp(v_full(st), ((J + j) / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v_desc = smem_desc_sw128(
            FP8 ? smem + C::V16_AT + (J + j) % C::V16S * C::V16_BYTES : smem + C::V_AT + st * C::K_BYTES, C::KV_SPAN, 1024);
        if (mine) {
#pragma unroll
          for (int k = 0; k < X_KEYS / 16; ++k)
            mma_f16_ts(tmem + X_O_COL, tmem + buf * X_S_COLS + 8 * k, v_desc + 128 * k, idesc_pv, (j | k) != 0);
          tc_commit(FP8 ? v16_empty((J + j) % C::V16S) : v_empty(st));
          if (j == tiles - 1) tc_commit(o_full);
        }
        if (j + 2 < tiles) issue_qk(j + 2);
      }
      __syncwarp();
    } else {
      const int quad = warp & 3, grp = (warp - 2) >> 2;
      const int t = threadIdx.x - 64;
      const int r = quad * 32 + lane;  // row of the tile = lane of tensor memory
      const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
      const uint32_t s_tmem = tmem + lane_addr + grp * X_S_COLS;
      const bool live = r < rows, warp_live = quad * 32 < rows;
      int seq = b, limit = keys - 1;  // the row's sequence, the last key of the range that it sees
      int m = row0 + min(r, rows - 1);
      if (!OWN) seq = m / p.rows_own, m -= seq * p.rows_own;
      const int g = m / p.Nq, n = m - g * p.Nq;
      if (p.causal) limit = min(limit, OWN ? n + keys - p.Nq : p.P + n + own_keys(p, seq) - p.Nq);
      if (pass == 0) {
        // The unit's rows of Q, swizzled like a TMA tile, eight lanes to 128 bytes of a row.
        const int64_t from = seq * p.q_strides[0] + (h * p.group + g) * p.q_strides[1] + n * p.q_strides[2];
        if (grp == 0) asm volatile("st.shared.b64 [%0], %1;" ::"r"(smem + C::ROW_AT + r * 8), "l"(from) : "memory");
        asm volatile("bar.sync 1, 256;" ::: "memory");
        constexpr int PIECES = DH * C::SIZE / 16, LANES = PIECES < 8 ? PIECES : 8;
        const int c = t % LANES;
        for (int row = t / LANES; row < rows; row += X_SOFTMAX / LANES) {
          int64_t at;
          asm volatile("ld.shared.b64 %0, [%1];" : "=l"(at) : "r"(smem + C::ROW_AT + row * 8) : "memory");
#pragma unroll
          for (int span = 0; span < C::SPANS; ++span)
            cp_async16(smem + C::Q_AT + span * C::Q_SPAN + row * 128 + ((c ^ (row & 7)) << 4), p.q + at + span * 128 + 16 * c);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      float beta = p.scale_log2, v_scale = 1.f;
      if (FP8) {
        beta *= __ldcg(p.q_descale + seq * p.Hkv + h) * __ldcg(OWN ? p.k_descale + seq * p.Hkv + h : p.kp_descale + h);
        v_scale = __ldcg(OWN ? p.v_descale + seq * p.Hkv + h : p.vp_descale + h);
      }
      const uint32_t x_ref = smem + C::X_AT + r * 4;
      auto x_group = [&](int g) { return x_ref + (1 + 2 * g) * X_ROWS * 4; };
      const float shift = !FP8 ? 0.f : pass ? X_SHIFT_AGAIN : X_SHIFT_F16;
      float top = -INFINITY, l = 0.f;
      bool met = false;
      for (int j = (J + grp) & 1; j < tiles; j += 2) {
        const int tile = J + j;
        const int st = tile % ST, key0 = (tile0 + j) * X_KEYS;
        if (FP8) {
          // This tile of V to f16, while its scores are computed: a thread takes half a row, neighbours' stores in different
          // banks.  Rows behind the last key become zeros, whatever the cache holds there: 0 . V has to be 0.
          const int buf = tile % C::V16S;
          ok = ok && mbar_wait_warp(v_full(st), (tile / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD) &&
               mbar_wait_warp(v16_empty(buf), ((tile / C::V16S) & 1) ^ 1, p.status, WK_ERR_TIMEOUT_MMA);
          if (!ok) break;
          constexpr int HALF = DH / 32;  // 16-byte pieces of half a row
          const int row = r >> 1;
          const uint32_t src = smem + C::V_AT + st * C::K_BYTES + row * 128;
          const uint32_t dst = smem + C::V16_AT + buf * C::V16_BYTES + row * 128;
          const bool behind = key0 + row >= keys;
#pragma unroll
          for (int c = 0; c < HALF; ++c) {
            const int piece = (r & 1) * HALF + (HALF == 4 ? c ^ 2 * (r & 1) : c);
            uint32_t w[4], o[8];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(src + ((piece ^ (row & 7)) << 4)));
            if (behind) w[0] = w[1] = w[2] = w[3] = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              o[2 * x] = e4m3x2_to_f16x2(static_cast<uint16_t>(w[x]));
              o[2 * x + 1] = e4m3x2_to_f16x2(static_cast<uint16_t>(w[x] >> 16));
            }
            const uint32_t to = dst + (piece >> 2) * C::KV_SPAN;
            const int at = (2 * piece) & 7;
            sts128(to + ((at ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
            sts128(to + (((at + 1) ^ (row & 7)) << 4), o[4], o[5], o[6], o[7]);
          }
          mbar_arrive(v_empty(st));
          fence_proxy_async_smem();
        }
        ok = ok && mbar_wait_warp(s_full(grp), (tile >> 1) & 1, p.status, WK_ERR_TIMEOUT_MMA);
        if (!ok) break;
        tc_fence_after();
        const bool masked = __any_sync(0xffffffffu, key0 + X_KEYS - 1 > limit);
        const int last = limit - key0;  // columns beyond it are masked
        if (j == 0 && pass == 0) {
          float x = -INFINITY;
          if (warp_live) {
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t raw[32];
              tmem_ld32(s_tmem + c * 32, raw);
              tc_wait_ld();
              if (masked) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (c * 32 + i > last) raw[i] = 0xff800000u;
              }
              x = fmaxf(x, block_max(raw) * beta);
            }
          }
          m_ref = x;
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(x_ref), "f"(x) : "memory");
        }
        if (!met) {
          asm volatile("bar.sync 1, 256;" ::: "memory");
          met = true;
          if (j != 0 && pass == 0) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(m_ref) : "r"(x_ref) : "memory");
        }
        if (!FP8 && key0 + X_KEYS > keys) {
          ok = mbar_wait_warp(v_full(st), (tile / ST) & 1, p.status, WK_ERR_TIMEOUT_LOAD);
          if (!ok) break;
          const int row = r >> 1;
          if (key0 + row >= keys && (r & 1) < C::V_SPANS) {
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
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i > last) raw[i] = 0xff800000u;
            }
            top = fmaxf(top, block_max(raw) * beta);
            const float bias = m_ref > -INFINITY ? shift - m_ref : 0.f;
            uint32_t w[16];
            float sum;
            softmax_block<FP8>(raw, beta, bias, w, sum);
            l += sum;
            uint32_t lo[8], hi[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[i] = w[i], hi[i] = w[8 + i];
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
      ok = ok && mbar_wait_warp(o_full, pass, p.status, WK_ERR_TIMEOUT_MMA);
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(x_group(grp)), "f"(l) : "memory");
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(x_group(grp) + X_ROWS * 4), "f"(top) : "memory");
      asm volatile("bar.sync 1, 256;" ::: "memory");
      float l2, top2;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(l2) : "r"(x_group(grp ^ 1)) : "memory");
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(top2) : "r"(x_group(grp ^ 1) + X_ROWS * 4) : "memory");
      l += l2;
      top = fmaxf(top, top2);
      far = ok && live && pass == 0 && top - m_ref > (FP8 ? X_MAX_EXP_F16 : X_MAX_EXP);
      inv_row = l > 0.f ? v_scale / l : l == l ? 0.f : l;  // NaN stays
      lse_row = l == 0.f ? -INFINITY : m_ref - shift + log2f(l);
      if (pass == 0) m_ref = top;  // for the second pass
      tc_fence_after();
    }
    if (!__syncthreads_or(far) || pass) break;
  }

  // ---- this CTA's part: every tile and product has been used.  Own keys' goes to memory, the prefix's to shared memory.
  const int64_t own_slot = OWN ? own_slot_of(p, blockIdx.x, 0) : 0;
  uint8_t* part = smem_ptr;  // [row][DH + X_PAD]
  if (warp >= 2) {
    const int quad = warp & 3, grp = (warp - 2) >> 2, r = quad * 32 + lane;
    const uint32_t o_tmem = tmem + (static_cast<uint32_t>(quad * 32) << 16) + X_O_COL + grp * (DH / 2);
    if (quad * 32 < rows) {
#pragma unroll
      for (int c = 0; c < DH / 64; ++c) {
        uint32_t v[32];
        if (tiles > 0) {
          tmem_ld32(o_tmem + c * 32, v);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = grp * (DH / 8) + c * 8 + i;
          const float4 y = make_float4(__uint_as_float(v[4 * i]) * inv_row, __uint_as_float(v[4 * i + 1]) * inv_row,
                                       __uint_as_float(v[4 * i + 2]) * inv_row, __uint_as_float(v[4 * i + 3]) * inv_row);
          if (!OWN) reinterpret_cast<float4*>(part + r * (DH + X_PAD) * 4)[at] = y;
          else if (r < rows) reinterpret_cast<float4*>(p.part + (own_slot + r) * DH)[at] = y;
        }
      }
    }
    if (OWN && grp == 0 && r < rows) p.part_lse[own_slot + r] = lse_row;
    if (!OWN && grp == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(smem + C::X_AT + r * 4), "f"(lse_row) : "memory");
    tc_fence_before();
  }
  if (OWN) {
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, X_TMEM_COLS);
    }
    return;
  }

  // ---- this CTA's rows, one or several to a warp at a time: what each of their parts counts, then the sums.  The parts of
  // own keys are read ahead of their use, the first ones while the cluster meets.
  constexpr int COLS = DH / 32, WARPS = X_THREADS / 32;
  static_assert(OWN_PARTS <= 32 && X_CLUSTER <= 32, "a lane for each of a row's parts");
  const bool meet = p.cluster > 1;
  auto join = [&](auto rows_at_once, auto parts_at_once) {
    constexpr int ROWS = decltype(rows_at_once)::value, AHEAD = decltype(parts_at_once)::value;
    float own_lse[ROWS], ahead[ROWS][AHEAD][COLS];
    auto read_own = [&](const RowTarget& e, int k0, float (&to)[AHEAD][COLS]) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
#pragma unroll
        for (int x = 0; x < COLS; ++x) to[k][x] = 0.f;
        if (k0 + k >= e.parts) continue;
        const float* src = p.part + (e.first + (k0 + k) * p.own_slot) * DH + lane * COLS;
        if (COLS == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          to[k][0] = v.x, to[k][1] = v.y, to[k][COLS - 2] = v.z, to[k][COLS - 1] = v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          to[k][0] = v.x, to[k][1] = v.y;
        }
      }
    };
    auto begin = [&](int i0) {
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        const int i = i0 + q * WARPS;
        own_lse[q] = -INFINITY;
        if (i >= mine) continue;
        const RowTarget& e = targets[i];
        if (lane < e.parts) own_lse[q] = __ldcg(p.part_lse + e.first + lane * p.own_slot);
        read_own(e, 0, ahead[q]);
      }
    };
    __syncwarp();
    if (meet) cluster_arrive();
    if (beside) pdl_wait();  // nothing that comes after this kernel starts before the one for own keys has ended
    begin(warp);
    __syncwarp();
    if (meet) cluster_wait();
    else __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, X_TMEM_COLS);
    }
    for (int i0 = warp; i0 < mine; i0 += ROWS * WARPS) {
      float top[ROWS], w_own[ROWS], w[ROWS], total[ROWS], o[ROWS][COLS];
      uint32_t at[ROWS];
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        const int r = min(i0 + q * WARPS, mine - 1) * members + rank;
        const uint32_t stat = smem + C::X_AT + r * 4;
        at[q] = smem + (r * (DH + X_PAD) + lane * COLS) * 4;
        w[q] = -INFINITY;
        if (lane < members) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w[q]) : "r"(meet ? mapa(stat, lane) : stat));
        top[q] = fmaxf(own_lse[q], w[q]);
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1)
#pragma unroll
        for (int q = 0; q < ROWS; ++q) top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], x));
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        w_own[q] = own_lse[q] == -INFINITY ? 0.f : exp2f(own_lse[q] - top[q]);
        w[q] = w[q] == -INFINITY ? 0.f : exp2f(w[q] - top[q]);
        total[q] = w_own[q] + w[q];
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1)
#pragma unroll
        for (int q = 0; q < ROWS; ++q) total[q] += __shfl_xor_sync(0xffffffffu, total[q], x);
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
#pragma unroll
        for (int x = 0; x < COLS; ++x) o[q][x] = 0.f;
        if (i0 + q * WARPS >= mine) continue;
        const RowTarget& e = targets[i0 + q * WARPS];
        for (int k0 = 0; k0 < e.parts; k0 += AHEAD) {
          if (k0) read_own(e, k0, ahead[q]);
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            const float f = __shfl_sync(0xffffffffu, w_own[q], k0 + k);
#pragma unroll
            for (int x = 0; x < COLS; ++x) o[q][x] = fmaf(ahead[q][k][x], f, o[q][x]);
          }
        }
      }
      begin(i0 + ROWS * WARPS);
      for (int k0 = 0; k0 < members; k0 += AHEAD) {
        float v[ROWS][AHEAD][COLS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
#pragma unroll
            for (int x = 0; x < COLS; ++x) v[q][k][x] = 0.f;
            if (k0 + k >= members) continue;
            const uint32_t src = meet ? mapa(at[q], k0 + k) : at[q];
            if (COLS == 4)
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                           : "=f"(v[q][k][0]), "=f"(v[q][k][1]), "=f"(v[q][k][COLS - 2]), "=f"(v[q][k][COLS - 1])
                           : "r"(src));
            else
              asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[q][k][0]), "=f"(v[q][k][1]) : "r"(src));
          }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
          for (int q = 0; q < ROWS; ++q) {
            const float f = __shfl_sync(0xffffffffu, w[q], k0 + k);
#pragma unroll
            for (int x = 0; x < COLS; ++x) o[q][x] = fmaf(v[q][k][x], f, o[q][x]);
          }
      }
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        if (i0 + q * WARPS >= mine) continue;
        const RowTarget& e = targets[i0 + q * WARPS];
        const bool empty = total[q] == 0.f;
        const float inv = empty ? 0.f : 1.f / total[q], y = empty ? INFINITY : top[q] + log2f(total[q]);
#pragma unroll
        for (int x = 0; x < COLS; ++x) o[q][x] *= inv;
        if (final) {
          __nv_bfloat16* dst = p.out + e.to + lane * COLS;
          if (COLS == 4)
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[q][0], o[q][1]), pack_bf16x2(o[q][COLS - 2], o[q][COLS - 1]));
          else
            *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[q][0], o[q][1]);
          if (p.lse && lane == 0) p.lse[e.lse_to] = p.lse_natural ? y * 0.6931471805599453f : y;
        } else {
          float* dst = p.part + e.to * DH + lane * COLS;
          if (COLS == 4) *reinterpret_cast<float4*>(dst) = make_float4(o[q][0], o[q][1], o[q][COLS - 2], o[q][COLS - 1]);
          else *reinterpret_cast<float2*>(dst) = make_float2(o[q][0], o[q][1]);
          if (lane == 0) p.part_lse[e.to] = empty ? -INFINITY : y;
        }
      }
    }
  };
  // A CTA of a small cluster has many rows with few parts, one of a large cluster few with many.  Four rows at a time against
  // one, us: 79 sequences, 32 / 8 heads, 17 queries, 71 + 54 FP8 keys (one member) 60, 75; 64 sequences of 32 heads, 2048 + 300
  // FP8 keys (four members) 35, 33.5.
  if (members <= 2) join(std::integral_constant<int, 4>(), std::integral_constant<int, 1>());
  else join(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
  __syncwarp();
  if (meet) cluster_sync();  // nobody leaves while its part may still be read
}

// ---- own keys of sequences with few rows ---------------------------------------------------------------------------
// A unit is up to 16 rows of one (sequence, KV head) and its own keys, in steps of KEYS; it weighs one more than its steps,
// for its start and end.  All units form a line that is cut into as many pieces as there are warps; a warp goes through its
// piece by itself, its loads running on into the next units, and leaves a part of every unit.
//
// Keys play the 16-row side of the MMAs and the rows the 8-column side, once or twice:
//   S^T[16 keys, 8 rows] = K.Q^T     O^T[d, 8 rows] += V^T.P^T
// so that a sequence's few rows leave little of an MMA empty and the accumulators take half the registers.  Tiles of K and V
// come in turn by TMA into a ring of the warp's own (three or six times 4 KiB) and go to the MMAs by ldmatrix; P changes lanes with
// movmatrix.  FP8: ldmatrix moves pairs of codes; which index of the head dimension a pair stands for is the same for K and
// Q, and only moves O's rows for V.
//
// Bound by reading K and V once in bf16; in FP8 by a warp's instructions, about 570 for 32 keys (134 of them conversions) at
// one in five cycles, with eight warps on an SM.  (Sixteen warps with the SM to themselves, the prefix kernel behind them: 128
// sequences, 32768 and 2048 keys 197 -> 191 us FP8, 239 -> 243 bf16; 16 sequences, 8192 and 1024 keys 28.5 -> 36.  The e4m3 form
// of mma.sync: no fewer conversions.)

// Exclusive sums of the sequences' weights, by the whole CTA, and their lengths; both in shared or global memory.
template <int KEYS>
__device__ __forceinline__ void sum_weights(const PrefixParams& p, int* cum, int* lengths, int* warp_sums) {
  constexpr int THREADS = 32 * Y_WARPS;
  const int per = (p.B + THREADS - 1) / THREADS, b0 = threadIdx.x * per, b1 = min(p.B, b0 + per);
  auto weight = [](int n) { return (n + KEYS - 1) / KEYS + Y_START; };
  int sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = own_keys(p, b);
    lengths[b] = n;
    sum += weight(n);
  }
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
    at += weight(lengths[b]);
  }
  if (b1 == p.B && b0 < p.B) cum[p.B] = at;
  __syncthreads();
}

template <bool FP8, int DH, int NT>
struct OwnCfg {
  static constexpr int SIZE = FP8 ? 1 : 2;
  static constexpr int SPANS = DH * SIZE > 128 ? 2 : 1;  // 128-byte spans of a row (FP8, 64: the upper half is zeros)
  static constexpr int KEYS = 32 / SPANS;                // of a step
  static constexpr int SPAN_BYTES = KEYS * 128;
  static constexpr int SLOT_BYTES = SPANS * SPAN_BYTES;  // 4 KiB
  // Of the ring.  Units of 8 rows run in two CTAs per SM beside one of the prefix kernel, and their rings fill the shared
  // memory that it leaves; units of 16 rows in one.
  static constexpr int SLOTS = NT == 1 ? 3 : 6;
  static constexpr int K16 = DH / 16;                    // MMAs over the head dimension
  static constexpr float P_SHIFT = FP8 ? 14.f : 0.f;     // P is stored times 2^14
};

template <bool FP8, int DH>
struct OwnWalker {
  int x, x1;           // where in the line, end of the piece
  int b, h, block, u;  // sequence, KV head, 16 rows; u = h . blocks + block
  int weight, nk, step, end, base;
  const int* cum;
  const int* lengths;
  __device__ __forceinline__ void open() {
    weight = cum[b + 1] - cum[b];
    nk = lengths[b];
  }
  // Steps of the piece in the unit that starts at `at`.
  __device__ __forceinline__ void range(int at) {
    base = at;
    step = max(0, x - base - Y_START);
    end = min(weight, x1 - base) - Y_START;
  }
  __device__ __forceinline__ OwnWalker(const PrefixParams& p, const Pieces& l, const int* cum, const int* lengths, int blocks,
                                       int piece)
      : cum(cum), lengths(lengths) {
    x = x1 = 0;
    if (piece >= l.G) return;
    x = l.start(piece), x1 = l.start(piece + 1);
    const int per_seq = p.Hkv * blocks;
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (cum[mid] * per_seq <= x) lo = mid; else hi = mid - 1;
    }
    b = lo;
    open();
    const int first = cum[b] * per_seq;
    u = (x - first) / weight;
    h = u / blocks, block = u - h * blocks;
    range(first + u * weight);
    if (step >= end) next(p, blocks);
  }
  __device__ __forceinline__ bool here() const { return x < x1; }
  // To the next unit that this piece has part in.
  __device__ __forceinline__ void next(const PrefixParams& p, int blocks) {
    do {
      x = base + weight;  // where the next unit starts
      if (x >= x1) return;
      ++u;
      if (++block == blocks) block = 0, ++h;
      if (u == p.Hkv * blocks) {
        u = h = 0, ++b;
        open();
      }
      range(x);
    } while (step >= end);  // nothing of the unit but its start is in the piece, or it has no keys
  }
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// NT: groups of eight rows, 1 or 2.
template <bool FP8, int DH, int NT>
__global__ void __maxnreg__(NT == 1 ? 112 : 168)
attn_prefix_own_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ PrefixParams p) {
  using C = OwnCfg<FP8, DH, NT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int cum_mem[Y_CUM + 1], length_mem[Y_CUM], warp_sums[Y_WARPS];
  __shared__ __align__(8) uint64_t bar_mem[Y_WARPS][C::SLOTS];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + warp * C::SLOTS * C::SLOT_BYTES;
  const uint32_t bars = smem_u32(bar_mem[warp]);
  if (lane == 0) {
    for (int i = 0; i < C::SLOTS; ++i) mbar_init(bars + 8 * i, 1);
    mbar_fence_init();
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  __syncwarp();
  pdl_wait();
  // the prefix kernel runs beside this one and reads what was written before it: it may start only now
  pdl_launch_dependents();
  // every CTA writes the same counts where they do not fit shared memory; those that add the parts read them from there
  int* cum = p.B <= Y_CUM ? cum_mem : p.cum;
  int* lengths = p.B <= Y_CUM ? length_mem : p.lengths;
  sum_weights<C::KEYS>(p, cum, lengths, warp_sums);
  if (blockIdx.x == 0 && cum != p.cum)
    for (int i = threadIdx.x; i <= p.B; i += 32 * Y_WARPS) p.cum[i] = cum[i];
  const int blocks = p.blocks_own, per_seq = p.Hkv * blocks;
  const Pieces line(cum[p.B] * per_seq, p.pieces, p.least);
  const int piece = blockIdx.x * Y_WARPS + warp;

  OwnWalker<FP8, DH> now(p, line, cum, lengths, blocks, piece), ahead = now;
  // Slots are filled in turn: K of a step, V of it, K of the next.
  int to = 0;
  auto fetch = [&](bool is_v, int by) {
    if (!ahead.here()) return;
    if (lane == by) {
      const uint32_t dst = ring + to * C::SLOT_BYTES, bar = bars + 8 * to;
      mbar_expect_tx(bar, C::SLOT_BYTES);
      for (int i = 0; i < C::SPANS; ++i)
        tma_load_4d(dst + i * C::SPAN_BYTES, is_v ? &map_v : &map_k, bar, 64 * i, ahead.step * C::KEYS, ahead.h, ahead.b);
    }
    to = to + 1 == C::SLOTS ? 0 : to + 1;
    if (is_v && ++ahead.step == ahead.end) ahead.next(p, blocks);
  };
#pragma unroll
  for (int i = 0; i < C::SLOTS; ++i) fetch(i & 1, 0);

  int from = 0;
  uint32_t parity = 0;
  bool ok = true;
  auto arrive_at = [&]() {  // the slot in turn, its data there
    const uint32_t at = ring + from * C::SLOT_BYTES;
    ok = ok && mbar_wait_warp(bars + 8 * from, parity, p.status, WK_ERR_TIMEOUT_LOAD);
    if (++from == C::SLOTS) from = 0, parity ^= 1;
    return at;
  };
  for (; now.here(); now.next(p, blocks)) {
    const int row0 = now.block * Y_ROWS, sc = now.b * p.Hkv + now.h, unit = now.b * per_seq + now.u;
    // Q: row g of each group of eight, the head dimension in the order of K's fragments
    uint32_t q[NT][C::K16][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = min(row0 + 8 * i + g, p.rows_own - 1);
      const uint8_t* src = p.q + now.b * p.q_strides[0] + (now.h * p.group + r / p.Nq) * p.q_strides[1] + (r % p.Nq) * p.q_strides[2];
#pragma unroll
      for (int k = 0; k < C::K16; ++k) {
        if (FP8) {
          const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(src + 16 * k + 4 * t));
          q[i][k][0] = e4m3x2_to_f16x2(static_cast<uint16_t>(w)), q[i][k][1] = e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16));
        } else {
          q[i][k][0] = __ldcg(reinterpret_cast<const uint32_t*>(src + 32 * k + 4 * t));
          q[i][k][1] = __ldcg(reinterpret_cast<const uint32_t*>(src + 32 * k + 16 + 4 * t));
        }
      }
    }
    // this lane's rows in the accumulators are 2 t and 2 t + 1 of each group; the last keys they see
    int limit[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = min(row0 + 8 * i + 2 * t + j, p.rows_own - 1);
        limit[i][j] = p.causal ? min(now.nk - 1, r % p.Nq + now.nk - p.Nq) : now.nk - 1;
      }
    const int first_limit = p.causal ? min(now.nk - 1, now.nk - p.Nq) : now.nk - 1;  // of query 0, among them or not
    float beta = p.scale_log2, v_scale = 1.f;
    if (FP8) beta *= __ldcg(p.q_descale + sc) * __ldcg(p.k_descale + sc), v_scale = __ldcg(p.v_descale + sc);

    float o[NT][C::K16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      m[i][0] = m[i][1] = -INFINITY, l[i][0] = l[i][1] = 0.f;
#pragma unroll
      for (int k = 0; k < C::K16; ++k) o[i][k][0] = o[i][k][1] = o[i][k][2] = o[i][k][3] = 0.f;
    }
    for (int step = now.step; step < now.end; ++step) {
      constexpr int N16 = C::KEYS / 16;
      float s[NT][N16][4];  // keys g, g + 8 of each 16; rows 2 t, 2 t + 1
      {
        const uint32_t ks = arrive_at();
        // ldmatrix: lane gives the row lane % 16 of 16 keys, 16-byte piece lane / 16 of two
#pragma unroll
        for (int n = 0; n < N16; ++n) {
#pragma unroll
          for (int i = 0; i < NT; ++i) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
          const int key = 16 * n + lane % 16;
          if (FP8) {
#pragma unroll
            for (int k = 0; k < C::K16; k += 2) {  // two pieces: 32 elements
              uint32_t w[4], a[2][4];
              ldmatrix_x4(w, ks + key * 128 + (((k + lane / 16) ^ (key & 7)) << 4));
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                a[x][0] = e4m3x2_to_f16x2(static_cast<uint16_t>(w[2 * x])), a[x][2] = e4m3x2_to_f16x2(static_cast<uint16_t>(w[2 * x] >> 16));
                a[x][1] = e4m3x2_to_f16x2(static_cast<uint16_t>(w[2 * x + 1]));
                a[x][3] = e4m3x2_to_f16x2(static_cast<uint16_t>(w[2 * x + 1] >> 16));
#pragma unroll
                for (int i = 0; i < NT; ++i)
                  mma_16816<true>(s[i][n], a[x][0], a[x][1], a[x][2], a[x][3], q[i][k + x][0], q[i][k + x][1]);
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < C::K16; ++k) {
              uint32_t a[4];
              const int c = 2 * k + lane / 16;
              ldmatrix_x4(a, ks + (c >> 3) * C::SPAN_BYTES + key * 128 + (((c & 7) ^ (key & 7)) << 4));
#pragma unroll
              for (int i = 0; i < NT; ++i) mma_16816<false>(s[i][n], a[0], a[1], a[2], a[3], q[i][k][0], q[i][k][1]);
            }
          }
        }
      }
      const int key0 = step * C::KEYS;
      const bool masked = key0 + C::KEYS - 1 > first_limit;
      float mx[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int n = 0; n < N16; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (masked && key0 + 16 * n + g + 8 * (j >> 1) > limit[i][j & 1]) s[i][n][j] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx[i][j] = fmaxf(s[i][0][j], s[i][0][2 + j]);
#pragma unroll
          for (int n = 1; n < N16; ++n) mx[i][j] = max3(mx[i][j], s[i][n][j], s[i][n][2 + j]);
          mx[i][j] *= beta;
        }
      }
#pragma unroll
      for (int x = 4; x < 32; x *= 2)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) mx[i][j] = fmaxf(mx[i][j], __shfl_xor_sync(0xffffffffu, mx[i][j], x));
      bool move = false;
#pragma unroll
      for (int i = 0; i < NT; ++i) move |= mx[i][0] > m[i][0] + 1.f || mx[i][1] > m[i][1] + 1.f;
      move = __any_sync(0xffffffffu, move);
      fetch(C::SLOTS % 2, 0);  // into K's place: by now every lane has its scores, so all of K has been read
      if (move) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float f[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float to = mx[i][j] > m[i][j] + 1.f ? mx[i][j] : m[i][j];
            f[j] = to > m[i][j] ? ex2_approx(m[i][j] - to) : 1.f;
            m[i][j] = to;
            l[i][j] *= f[j];
          }
#pragma unroll
          for (int k = 0; k < C::K16; ++k) o[i][k][0] *= f[0], o[i][k][1] *= f[1], o[i][k][2] *= f[0], o[i][k][3] *= f[1];
        }
      }
      uint32_t pt[NT][N16][2];  // P^T: row g, keys 2 t and 2 t + 1 of each eight
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float bias[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) bias[j] = m[i][j] > -INFINITY ? C::P_SHIFT - m[i][j] : 0.f;
#pragma unroll
        for (int n = 0; n < N16; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][n][j] = ex2_approx(fmaf(s[i][n][j], beta, bias[j & 1]));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            l[i][j] += s[i][n][j] + s[i][n][2 + j];
            pt[i][n][j] = movmatrix(pack_16x2<FP8>(s[i][n][2 * j], s[i][n][2 * j + 1]));
          }
        }
      }

      const uint32_t vs = arrive_at();
      if (key0 + C::KEYS > now.nk) {
        // rows of V behind the last key: whatever the cache holds there, 0 . V has to be 0
        for (int x = lane; x < C::KEYS * C::SPANS * 8; x += 32) {
          const int key = x / 8 % C::KEYS;
          if (key0 + key >= now.nk) sts128(vs + x * 16, 0, 0, 0, 0);
        }
        fence_proxy_async_smem();  // before TMA writes there again
        __syncwarp();
      }
      // ldmatrix, transposed: matrices (keys 0-7, piece 0), (0-7, 1), (8-15, 0), (8-15, 1)
#pragma unroll
      for (int n = 0; n < N16; ++n) {
        const int key = 16 * n + lane % 8 + lane / 16 * 8;
        if (FP8) {
#pragma unroll
          for (int k = 0; k < C::K16; k += 2) {
            uint32_t w[4];
            ldmatrix_x4_trans(w, vs + key * 128 + (((k + lane / 8 % 2) ^ (key & 7)) << 4));
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // 16 elements: pair g of the codes becomes rows g and g + 8
              const uint32_t y = __byte_perm(w[x], 0, 0x3120), z = __byte_perm(w[2 + x], 0, 0x3120);
              const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(y)), a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(y >> 16));
              const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(z)), a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(z >> 16));
#pragma unroll
              for (int i = 0; i < NT; ++i) mma_16816<true>(o[i][k + x], a0, a1, a2, a3, pt[i][n][0], pt[i][n][1]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < C::K16; ++k) {
            uint32_t a[4];
            const int c = 2 * k + lane / 8 % 2;
            ldmatrix_x4_trans(a, vs + (c >> 3) * C::SPAN_BYTES + key * 128 + (((c & 7) ^ (key & 7)) << 4));
#pragma unroll
            for (int i = 0; i < NT; ++i) mma_16816<false>(o[i][k], a[0], a[1], a[2], a[3], pt[i][n][0], pt[i][n][1]);
          }
        }
      }
      // Into V's place, once every lane has read all of it: the vote is over bits of a sum of each fragment of V.  Which lane
      // then issues the load is all the same.
      uint32_t seen = 0;
#pragma unroll
      for (int k = 0; k < C::K16; k += FP8 ? 2 : 1) seen |= __float_as_uint(o[NT - 1][k][0]);  // FP8: one fragment for two
      fetch(C::SLOTS % 2 == 0, __any_sync(0xffffffffu, seen == 0xffffffffu) ? 1 : 0);
    }

    // ---- this warp's part: O / l and the log-sum-exp
    const int64_t slot = own_slot_of(p, unit, piece);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2) l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], x);
        const int r = 8 * i + 2 * t + j;
        if (row0 + r < p.rows_own) {
          const float inv = l[i][j] > 0.f ? v_scale / l[i][j] : l[i][j] == l[i][j] ? 0.f : l[i][j];
          float* dst = p.part + (slot + r) * DH;
#pragma unroll
          for (int k = 0; k < C::K16; ++k)
            if (FP8) {
              *reinterpret_cast<float2*>(dst + 16 * k + 2 * g) = make_float2(o[i][k][j] * inv, o[i][k][2 + j] * inv);
            } else {
              dst[16 * k + g] = o[i][k][j] * inv;
              dst[16 * k + g + 8] = o[i][k][2 + j] * inv;
            }
          if (g == 0) p.part_lse[slot + r] = l[i][j] == 0.f ? -INFINITY : m[i][j] - C::P_SHIFT + log2f(l[i][j]);
        }
        __syncwarp();
      }
  }
}

// Adds up the parts of every row: a warp for a row, as many columns to a lane as there are.
template <int DH>
__global__ void __launch_bounds__(256)
attn_prefix_combine_kernel(const __grid_constant__ PrefixParams p) {
  constexpr int COLS = DH / 32;
  struct alignas(4 * COLS) Vec {
    float x[COLS];
  };
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % 32, row = blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= p.Hkv * p.rows_all) return;
  const int h = row / p.rows_all, stacked = row - h * p.rows_all, b = stacked / p.rows_own, own = stacked - b * p.rows_own;
  const OwnParts parts(p, b, h, own);
  const int splits = p.tiles_p ? p.splits : 0, all = splits + parts.count;
  const int64_t first = static_cast<int64_t>(h * p.blocks_p + stacked / X_ROWS) * p.splits * X_ROWS + stacked % X_ROWS;
  auto slot_of = [&](int c) { return c < splits ? first + c * X_ROWS : parts.first + static_cast<int64_t>(c - splits) * parts.distance; };
  float top = -INFINITY;
  for (int c = lane; c < all; c += 32) top = fmaxf(top, __ldcg(p.part_lse + slot_of(c)));
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  float total = 0.f, o[COLS];
#pragma unroll
  for (int i = 0; i < COLS; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int c = 0; c < all; ++c) {
    const int64_t slot = slot_of(c);
    const float lse = __ldcg(p.part_lse + slot), w = lse == -INFINITY ? 0.f : exp2f(lse - top);
    Vec v;
    if (COLS == 4) {
      const float4 y = __ldcg(reinterpret_cast<const float4*>(p.part + slot * DH) + lane);
      v.x[0] = y.x, v.x[1] = y.y, v.x[COLS - 2] = y.z, v.x[COLS - 1] = y.w;
    } else {
      const float2 y = __ldcg(reinterpret_cast<const float2*>(p.part + slot * DH) + lane);
      v.x[0] = y.x, v.x[1] = y.y;
    }
    total += w;
#pragma unroll
    for (int i = 0; i < COLS; ++i) o[i] = fmaf(v.x[i], w, o[i]);
  }
  const bool empty = total == 0.f;
  const float inv = empty ? 0.f : 1.f / total;
  const int head = h * p.group + own / p.Nq, n = own % p.Nq;
  __nv_bfloat16* dst = p.out + b * p.out_strides[0] + head * p.out_strides[1] + n * p.out_strides[2] + lane * COLS;
  if (COLS == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[COLS - 2] * inv, o[COLS - 1] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[0] * inv, o[1] * inv);
  if (p.lse && lane == 0) {
    const float x = empty ? INFINITY : top + log2f(total);
    p.lse[b * p.lse_strides[0] + head * p.lse_strides[1] + n] = p.lse_natural ? x * 0.6931471805599453f : x;
  }
}

// How a call is divided.
struct Sizes {
  int rows_own, blocks_p, units_p, tiles_p, cluster, splits;
  int by_rows, blocks_own, own_slot, units_own, pieces, least;
  int64_t own_parts, row_slots, cum_bytes, bytes;
};

// CTAs of a cluster and clusters of a unit.  A CTA is taken to cost a start and end (more in a larger cluster), and its
// tiles, which go faster where it has an SM to itself; clusters of a unit beyond one cost the kernel that adds them up.  A
// cluster lies within a group of SMs, of which larger ones leave some idle: with one CTA per SM 74 clusters of 2, 33 of 4, 15
// of 8 and 7 of 16 run at once.
void divide_prefix(int sms, Sizes& z) {
  double best = 0;
  for (int cluster = 1; cluster <= X_CLUSTER; cluster *= 2)
    for (int splits = 1; splits <= 16; splits *= 2) {
      const int64_t shares = static_cast<int64_t>(cluster) * splits;
      if (shares > 1 && (shares > z.tiles_p || (splits > 1 && cluster < 8))) continue;
      const int64_t ctas = z.units_p * shares;
      const int64_t at_once = sms * (cluster <= 2 ? 148 : cluster == 4 ? 132 : cluster == 8 ? 120 : 112) / 148;
      const int64_t waves = (ctas + 2 * at_once - 1) / (2 * at_once);
      const double tiles = static_cast<double>((z.tiles_p + shares - 1) / shares);
      const double cost = waves * (4.0 + 0.15 * cluster + tiles * (ctas <= at_once ? 0.65 : 1.1)) + (splits > 1 ? 4.0 : 0.0);
      if (shares == 1 || cost < best) best = cost, z.cluster = cluster, z.splits = splits;
    }
}

// Whether own keys go to the kernel for few rows, which divides them evenly over the SMs and runs beside the prefix kernel;
// the tensor-core kernel takes a sequence's keys in one CTA and all its rows at once.  The latter wins with more than eight
// rows (two of the former's column blocks; from 17 on it reads the keys twice, from 33 on three times) where sequences fill
// the SMs and, up to 16 rows, are long enough for its start.  bf16, 4096 shared keys, own keys up to S, us of few rows and of
// tiles:
//    64 x 8 heads, S 1024: 12 rows 70, 63; 20 rows 121, 81; 32 rows 130, 88      24 x 8, S 512: 12 rows 34, 32; 32 rows 51, 42
//   300 x 8 heads, S 200: 12 rows 145, 156; 20 rows 235, 212                      8 x 8, S 1024: 12 rows 22, 27; 32 rows 30, 31
//     4 x 1 heads, S 8192: 20 rows 30, 96                              FP8, 64 x 8, S 1024: 12 rows 62, 57; 20 rows 98, 75
bool own_by_rows(int64_t rows, int64_t sequences, int S, int sms) {
  if (rows <= 8) return true;
  return sequences <= sms ? rows <= 32 : rows <= 16 && S < 512;
}

// false if the problem is beyond the kernels' 32-bit counts.
bool sizes_of(int B, int Hq, int Hkv, int Nq, int P, int S, int d, int sms, Sizes& z) {
  const int64_t rows_own = static_cast<int64_t>(Hq / Hkv) * Nq, rows_all = rows_own * B;
  if (rows_all * Hkv > INT32_MAX / 2 || static_cast<int64_t>(P) + S > INT32_MAX / 2) return false;
  z.rows_own = static_cast<int>(rows_own);
  z.blocks_p = static_cast<int>((rows_all + X_ROWS - 1) / X_ROWS);
  z.tiles_p = P / X_KEYS + (P % X_KEYS != 0);
  z.units_p = z.tiles_p ? Hkv * z.blocks_p : 0;
  z.cluster = z.splits = 1;
  if (z.units_p) divide_prefix(sms, z);
  z.by_rows = own_by_rows(rows_own, static_cast<int64_t>(B) * Hkv, S, sms);
  const int unit_rows = z.by_rows ? Y_ROWS : X_ROWS;
  z.own_slot = rows_own < unit_rows ? z.rows_own : unit_rows;
  z.blocks_own = static_cast<int>((rows_own + unit_rows - 1) / unit_rows);
  const int64_t units = S ? static_cast<int64_t>(B) * Hkv * z.blocks_own : 0, steps = units * ((S + 15ll) / 16 + Y_START);
  if (steps > INT32_MAX / 16 || static_cast<int64_t>(z.units_p) * z.cluster * z.splits > INT32_MAX / 2) return false;
  z.units_own = static_cast<int>(units);
  // every warp that runs at once has a piece, but the longest unit no more parts than those that add them have room for:
  // one for each piece that it fills, and two that it fills in part
  z.pieces = 0, z.least = 1;
  if (z.by_rows && S) {
    // of two CTAs per SM; of one where units of 16 rows leave room for no more beside a CTA of the prefix kernel
    const int64_t warps = (z.own_slot > 8 && z.units_p ? 1ll : 2ll) * sms * Y_WARPS;
    z.pieces = static_cast<int>(steps < warps ? steps : warps);
    z.least = static_cast<int>(((S + 15ll) / 16 + Y_START + OWN_PARTS - 2) / (OWN_PARTS - 1));
  }
  z.own_parts = z.splits > 1 ? static_cast<int64_t>(z.units_p) * z.splits * X_ROWS : 0;
  z.row_slots = z.own_parts + (units + z.pieces) * z.own_slot;
  z.cum_bytes = (static_cast<int64_t>(B) * 8 + 4 + 15) / 16 * 16;
  z.bytes = z.cum_bytes + z.row_slots * (d + 1) * 4;
  return true;
}

template <bool FP8, int DH>
int launch_prefix(const CUtensorMap (&maps)[4], const Sizes& z, PrefixParams& p, cudaStream_t stream) {
  using C = PrefixCfg<FP8, DH>;
  static_assert(2 * (C::SMEM + 1024) <= 228 * 1024, "two CTAs per SM");
  if (z.units_own && z.by_rows) {
    const bool narrow = z.own_slot <= 8;
    const void* fn = narrow ? reinterpret_cast<const void*>(attn_prefix_own_kernel<FP8, DH, 1>)
                            : reinterpret_cast<const void*>(attn_prefix_own_kernel<FP8, DH, 2>);
    using N1 = OwnCfg<FP8, DH, 1>;
    using N2 = OwnCfg<FP8, DH, 2>;
    const int ring = Y_WARPS * (narrow ? N1::SLOTS * N1::SLOT_BYTES : N2::SLOTS * N2::SLOT_BYTES) + 1024;
    // all of the SM's shared memory, so that a CTA of the prefix kernel fits beside
    if (allow_smem(fn, ring) || prefer_smem(fn)) return WK_E_CUDA;
    if (int bad = launch_pdl(fn, dim3((z.pieces + Y_WARPS - 1) / Y_WARPS), 32 * Y_WARPS, ring, stream, 1,
                             {const_cast<CUtensorMap*>(&maps[2]), const_cast<CUtensorMap*>(&maps[3]), &p}))
      return bad;
  } else if (z.units_own) {
    const void* fn = reinterpret_cast<const void*>(attn_prefix_kernel<FP8, DH, true>);
    if (allow_smem(fn, C::SMEM) || prefer_smem(fn)) return WK_E_CUDA;
    if (int bad = launch_pdl(fn, dim3(z.units_own), X_THREADS, C::SMEM, stream, 1,
                             {const_cast<CUtensorMap*>(&maps[2]), const_cast<CUtensorMap*>(&maps[3]), &p}))
      return bad;
  }
  if (z.units_p) {
    const void* fn = reinterpret_cast<const void*>(attn_prefix_kernel<FP8, DH, false>);
    if (allow_smem(fn, C::SMEM) || allow_large_clusters(fn) || prefer_smem(fn)) return WK_E_CUDA;
    if (int bad = launch_pdl(fn, dim3(z.units_p * z.splits * z.cluster), X_THREADS, C::SMEM, stream, z.cluster,
                             {const_cast<CUtensorMap*>(&maps[0]), const_cast<CUtensorMap*>(&maps[1]), &p}))
      return bad;
    if (z.splits == 1) return 0;
  }
  return launch_pdl(reinterpret_cast<const void*>(attn_prefix_combine_kernel<DH>), dim3((p.Hkv * p.rows_all + 7) / 8), 256, 0,
                    stream, 1, {&p});
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
  for (int i = 0; i < 4; ++i) {
    const int len = i < 2 ? a->P : a->S;
    // own keys of few rows come in steps of 4 KiB, 128 bytes of a row at a time
    const uint32_t box[4] = {fp8 ? 128u : 64u, i < 2 || !z.by_rows ? X_KEYS : !fp8 && a->d == 128 ? 16u : 32u, 1, 1};
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
  p.rows_own = z.rows_own, p.rows_all = z.rows_own * a->B;
  p.blocks_p = z.blocks_p, p.tiles_p = z.tiles_p, p.cluster = z.cluster, p.splits = z.splits;
  p.by_rows = z.by_rows, p.blocks_own = z.blocks_own, p.own_slot = z.own_slot, p.pieces = z.pieces, p.least = z.least, p.own_parts = z.own_parts;
  p.causal = a->causal, p.lse_natural = a->lse_natural;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.cum = static_cast<int*>(a->workspace), p.lengths = p.cum + a->B + 1;
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + z.cum_bytes);
  p.part_lse = p.part + z.row_slots * a->d;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp8) return a->d == 64 ? launch_prefix<true, 64>(maps, z, p, st) : launch_prefix<true, 128>(maps, z, p, st);
  return a->d == 64 ? launch_prefix<false, 64>(maps, z, p, st) : launch_prefix<false, 128>(maps, z, p, st);
}
