// What the kernels for few packed query rows share: 16 rows on mma.sync, operand fragments fetched by every thread for
// itself with cp.async (attn_rows.cu says how the head dimension is permuted for that).
#pragma once
#include "common.cuh"

namespace wk {

constexpr int R_WARPS = 4;
constexpr int R_ROWS = 16;
constexpr int R_RING_BYTES = 24 * 1024;  // per warp
constexpr float R_P_SHIFT = 14.f;        // P is stored times 2^14 (FP8 inputs)

template <bool FP8, int DH>
struct RowsCfg {
  static constexpr int SIZE = FP8 ? 1 : 2;
  static constexpr int KEYS = FP8 ? 32 : 16;              // keys per step of a warp
  static constexpr int K_PIECES = DH * SIZE / 64;         // 16-byte pieces of a K row per lane (four lanes per row)
  static constexpr int V_PIECE = DH * SIZE / 8 >= 16 ? 16 : 8;  // bytes of a V row per lane and piece (eight lanes)
  static constexpr int V_PIECES = DH * SIZE / 8 / V_PIECE;
  static constexpr int V_ELEMS = V_PIECE / SIZE;
  static constexpr int N8 = KEYS / 8;
  static constexpr int K_BYTES = N8 * K_PIECES * 16 * 32;  // per step and warp
  static constexpr int V_BYTES = (KEYS / 4) * V_PIECES * V_PIECE * 32;
  static constexpr int STAGE_BYTES = K_BYTES + V_BYTES;
  static constexpr int MAX_STAGES = R_RING_BYTES / STAGE_BYTES;
  static constexpr int NT = DH / 8;      // column tiles of O
  static constexpr int O_PITCH = DH + 4;  // fp32 values between rows of a partial O in shared memory
  static constexpr float P_SHIFT = FP8 ? R_P_SHIFT : 0.f;
  static constexpr int PART_FLOATS = R_ROWS * O_PITCH + 3 * R_ROWS;  // O, then m, l, largest score
};

__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, int bytes) {
  if (bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

#define WK_MMA16816(name, ab)                                                                                     \
  __device__ __forceinline__ void name(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {         \
    asm("mma.sync.aligned." ab " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                 \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                          \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                          \
  }
WK_MMA16816(mma_sync_f16, "m16n8k16.row.col.f32.f16.f16.f32")
WK_MMA16816(mma_sync_bf16, "m16n8k16.row.col.f32.bf16.bf16.f32")
WK_MMA16816(mma_sync_e4m3, "m16n8k32.row.col.f32.e4m3.e4m3.f32")
#undef WK_MMA16816

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// One step of a warp over KEYS keys from `key0` on, whose fragments this thread has fetched to `ks` and `vs`: scores, online
// softmax and P.V for the 16 rows.  A thread has rows g = lane / 4 and g + 8; their last visible keys are `limit`, and
// `first_limit` is the smallest one of all 16.  m: the rows' references, l: sums of this thread's keys, top: largest scores.
template <bool FP8, int DH>
__device__ __forceinline__ void rows_step(uint32_t ks, uint32_t vs, const uint4 (&q)[2][RowsCfg<FP8, DH>::K_PIECES], float beta,
                                          int key0, int first_limit, const int (&limit)[2], int t,
                                          float (&o)[RowsCfg<FP8, DH>::NT][4], float (&m)[2], float (&l)[2], float (&top)[2]) {
  using C = RowsCfg<FP8, DH>;
  constexpr float P_SHIFT = C::P_SHIFT;
  // ---- scores: s[j][0..1] row g, keys 8 j + 2 t and + 1; s[j][2..3] row g + 8
  float s[C::N8][4];
#pragma unroll
  for (int j = 0; j < C::N8; ++j) {
    s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int h = 0; h < C::K_PIECES; ++h) {
      const uint4 kk = lds128(ks + (j * C::K_PIECES + h) * 512);
      const uint32_t a0[4] = {q[0][h].x, q[1][h].x, q[0][h].y, q[1][h].y};
      const uint32_t a1[4] = {q[0][h].z, q[1][h].z, q[0][h].w, q[1][h].w};
      if (FP8) {
        mma_sync_e4m3(s[j], a0, kk.x, kk.y);
        mma_sync_e4m3(s[j], a1, kk.z, kk.w);
      } else {
        mma_sync_bf16(s[j], a0, kk.x, kk.y);
        mma_sync_bf16(s[j], a1, kk.z, kk.w);
      }
    }
  }
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < C::N8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[j][i] *= beta;
  if (key0 + C::KEYS - 1 > first_limit) {
#pragma unroll
    for (int j = 0; j < C::N8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key0 + 8 * j + 2 * t + (i & 1) > limit[i >> 1]) s[j][i] = -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < C::N8; ++j) {
    mx[0] = max3(mx[0], s[j][0], s[j][1]);
    mx[1] = max3(mx[1], s[j][2], s[j][3]);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
    top[h] = fmaxf(top[h], mx[h]);
  }
  // the reference moves when the step rises more than 1 above it (and from -inf)
  const bool move0 = mx[0] > m[0] + 1.f, move1 = mx[1] > m[1] + 1.f;
  if (__any_sync(0xffffffffu, move0 || move1)) {
    const float n0 = move0 ? mx[0] : m[0], n1 = move1 ? mx[1] : m[1];
    const float f0 = move0 ? ex2_approx(m[0] - n0) : 1.f, f1 = move1 ? ex2_approx(m[1] - n1) : 1.f;
    m[0] = n0, m[1] = n1;
    l[0] *= f0, l[1] *= f1;
#pragma unroll
    for (int j = 0; j < C::NT; ++j) {
      o[j][0] *= f0, o[j][1] *= f0;
      o[j][2] *= f1, o[j][3] *= f1;
    }
  }
  const float bias0 = m[0] > -INFINITY ? P_SHIFT - m[0] : 0.f, bias1 = m[1] > -INFINITY ? P_SHIFT - m[1] : 0.f;
#pragma unroll
  for (int j = 0; j < C::N8; ++j) {
    s[j][0] = ex2_approx(s[j][0] + bias0), s[j][1] = ex2_approx(s[j][1] + bias0);
    s[j][2] = ex2_approx(s[j][2] + bias1), s[j][3] = ex2_approx(s[j][3] + bias1);
    l[0] += s[j][0] + s[j][1];
    l[1] += s[j][2] + s[j][3];
  }

  // ---- O += P.V, 16 keys at a time
#pragma unroll
  for (int c = 0; c < C::KEYS / 16; ++c) {
    uint32_t a[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float(&x)[4] = s[2 * c + h];
      a[2 * h] = FP8 ? pack_f16x2(x[0], x[1]) : pack_bf16x2(x[0], x[1]);
      a[2 * h + 1] = FP8 ? pack_f16x2(x[2], x[3]) : pack_bf16x2(x[2], x[3]);
    }
#pragma unroll
    for (int h = 0; h < C::V_PIECES; ++h) {
      uint32_t w[4][4];  // [key 2t, 2t + 1, 2t + 8, 2t + 9][word]
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t addr = vs + ((4 * c + i) * C::V_PIECES + h) * (32 * C::V_PIECE);
        if (C::V_PIECE == 16) {
          const uint4 x = lds128(addr);
          w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
        } else {
          const uint2 x = lds64(addr);
          w[i][0] = x.x, w[i][1] = x.y;
        }
      }
#pragma unroll
      for (int x = 0; x < C::V_PIECE / 4; ++x) {
        if (FP8) {
          // bytes of key pairs side by side, then e4m3 -> f16: two columns per word, four columns per x
          const uint32_t lo0 = __byte_perm(w[0][x], w[1][x], 0x5140), hi0 = __byte_perm(w[0][x], w[1][x], 0x7362);
          const uint32_t lo1 = __byte_perm(w[2][x], w[3][x], 0x5140), hi1 = __byte_perm(w[2][x], w[3][x], 0x7362);
          float(*oo)[4] = o + h * C::V_ELEMS + 4 * x;
          mma_sync_f16(oo[0], a, e4m3x2_to_f16x2(static_cast<uint16_t>(lo0)), e4m3x2_to_f16x2(static_cast<uint16_t>(lo1)));
          mma_sync_f16(oo[1], a, e4m3x2_to_f16x2(static_cast<uint16_t>(lo0 >> 16)), e4m3x2_to_f16x2(static_cast<uint16_t>(lo1 >> 16)));
          mma_sync_f16(oo[2], a, e4m3x2_to_f16x2(static_cast<uint16_t>(hi0)), e4m3x2_to_f16x2(static_cast<uint16_t>(hi1)));
          mma_sync_f16(oo[3], a, e4m3x2_to_f16x2(static_cast<uint16_t>(hi0 >> 16)), e4m3x2_to_f16x2(static_cast<uint16_t>(hi1 >> 16)));
        } else {
          float(*oo)[4] = o + h * C::V_ELEMS + 2 * x;
          mma_sync_bf16(oo[0], a, __byte_perm(w[0][x], w[1][x], 0x5410), __byte_perm(w[2][x], w[3][x], 0x5410));
          mma_sync_bf16(oo[1], a, __byte_perm(w[0][x], w[1][x], 0x7632), __byte_perm(w[2][x], w[3][x], 0x7632));
        }
      }
    }
  }
}

}  // namespace wk
