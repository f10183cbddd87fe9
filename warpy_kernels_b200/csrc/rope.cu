// Position rotation of queries and keys, with or without the RMS norm of every head before it, in one pass; optionally
// as the e4m3 codes that the FP8 attention reads.  And the gradient of norm and rotation.
//
// One row is one head of one token, x in R^d:
//   r = (mean(x^2) + eps)^-1/2      u = x r w      y = R(theta) u        (without the norm: u = x)
// R turns the pairs (j, j + R/2), or (2 j, 2 j + 1), of the first R elements by theta_j = position[axis(j)] inv_freq[j].
// Backward, with g = R(-theta) dy, h = g w:
//   dw = sum over rows of g x r     dx = r (h - x r^2 mean(h x))
//
// A row is d / 16 lanes of a warp with 16 elements each, two 8-element pieces that hold both halves of the lane's pairs:
// the rotation needs no exchange, the norm one reduction over the lanes of a row.  A warp takes all heads of one token (of a
// few, where heads are fewer than the rows it holds; a part of the heads, where tokens are few), queries and then keys, so
// that an angle is made once for the heads of its token; its products with a side's weights stay in registers.  (Backward:
// the queries of all tokens, then the keys, so that one weight's gradient is summed at a time.)  A warp goes on to the next
// tokens by itself; every lane fetches its own pieces a few rows ahead, across tokens, with cp.async into a ring of its own,
// so that loads are under way while angles are made.
//
// Angles: position times inv_freq in turns, reduced to half a turn in fp64 (positions beyond 2^20 leave nothing of an fp32
// product's fraction), then sine and cosine in fp32.
//
// Bound by HBM: every element is read once and written once (backward: read twice).  What has to be kept small for that is
// the number of instructions, hence packed pairs of fp32: a warp's 512 elements (bf16: 2 KiB of traffic, 90 cycles at an
// SM's share of the bandwidth) take about 200.  With the 12 warps that 160 registers a thread leave an SM, what shows is the
// latency of a warp's own chain (load, reduction, rsqrt, products, store).
// Measured with inputs from HBM, bf16, 32 / 8 heads of 128: norm and rotation of 4 x 4096 tokens 60 us (5.6 TB/s, 86 % of a
// copy); its gradient 98 us (5.2 TB/s, 80 %); 32768 tokens of 64 / 8 heads to e4m3 180 us (5.0 TB/s, 78 %); rotation of
// 16385 tokens, 16 / 16 fp16 heads of 80, 38 us (4.4 TB/s: 15 of 16 lanes hold elements, and rows start on 32 bytes); one
// token 5.6 us.  Factors in shared memory instead of registers, for 16 to 20 warps on an SM: 72 to 108 us for the first.
// Streaming stores and deeper rings change nothing; four CTAs on an SM spill (gradient 176 us).  A half-rotated head takes what
// a whole one does: 4 x 8192 tokens, 16 / 4 heads of 128, 61 us, gradient 95 us.
#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "host_common.h"

namespace wk {
namespace {

constexpr int kThreads = 128;
constexpr int kCtasPerSm = 3;
constexpr int kMaxD = 256;
// Steps of a warp that are under way, two rows per lane each.
template <typename T, bool BWD>
constexpr int kStages = sizeof(T) == 2 ? (BWD ? 3 : 4) : (BWD ? 2 : 3);
constexpr int kTable = 512;  // cosines and sines of a warp's tokens: at most 32 rows / LPR . 8 LPR pairs

struct RopeParams {
  const void* x[2];  // queries, keys
  void* y[2];        // outputs; backward: dx
  const void* dy[2];
  const void* w[2];
  const float* descale[2];
  const void* positions;
  const void* inv_freq;
  float* partial;  // backward: [CTA][2][d]
  int64_t xs[2][3], ys[2][3], dys[2][3], ps[3];
  uint64_t axis_map[4];
  int heads[2];
  int N, tokens;
  int d, rot;
  int hkv;          // descale entries per batch item
  float inv_group;  // of the query heads that share one
  int hb, tb;       // heads and tokens that a warp holds at a time
  int hs;           // warps that share the heads of a token
  int w_dtype, pos64, freq64, interleaved, inverse;
  float eps;
};

// A lane's 16 elements as they lie in memory.
template <typename T>
struct Raw {
  uint4 a, b;
};
template <>
struct Raw<float> {
  float4 a0, a1, b0, b1;
};
// A warp's 512 elements in the ring: 16-byte pieces, lane after lane.
template <typename T>
constexpr int kRowBytes = 512 * sizeof(T);
template <typename T>
__device__ __forceinline__ void fetch_raw(uint32_t dst, const T* p, int between) {
  cp_async16(dst, p);
  cp_async16(dst + 512, p + between);
  if (sizeof(T) == 4) {
    cp_async16(dst + 1024, p + 4);
    cp_async16(dst + 1536, p + between + 4);
  }
}
template <typename T>
__device__ __forceinline__ void read_raw(uint32_t src, Raw<T>& r) {
  r.a = lds128(src), r.b = lds128(src + 512);
}
__device__ __forceinline__ void read_raw(uint32_t src, Raw<float>& r) {
  auto f = [](uint4 w) {
    return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
  };
  r.a0 = f(lds128(src)), r.b0 = f(lds128(src + 512)), r.a1 = f(lds128(src + 1024)), r.b1 = f(lds128(src + 1536));
}
__device__ __forceinline__ uint64_t widen(uint32_t w, __nv_bfloat16) {
  return pack_f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint64_t widen(uint32_t w, __half) {
  float lo, hi;
  f16x2_to_float2(w, lo, hi);
  return pack_f32x2(lo, hi);
}
// As eight pairs of fp32, the first piece's four first.
template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, uint64_t (&v)[8]) {
  v[0] = widen(r.a.x, T()), v[1] = widen(r.a.y, T()), v[2] = widen(r.a.z, T()), v[3] = widen(r.a.w, T());
  v[4] = widen(r.b.x, T()), v[5] = widen(r.b.y, T()), v[6] = widen(r.b.z, T()), v[7] = widen(r.b.w, T());
}
__device__ __forceinline__ void unpack(const Raw<float>& r, uint64_t (&v)[8]) {
  v[0] = pack_f32x2(r.a0.x, r.a0.y), v[1] = pack_f32x2(r.a0.z, r.a0.w);
  v[2] = pack_f32x2(r.a1.x, r.a1.y), v[3] = pack_f32x2(r.a1.z, r.a1.w);
  v[4] = pack_f32x2(r.b0.x, r.b0.y), v[5] = pack_f32x2(r.b0.z, r.b0.w);
  v[6] = pack_f32x2(r.b1.x, r.b1.y), v[7] = pack_f32x2(r.b1.z, r.b1.w);
}

__device__ __forceinline__ uint32_t narrow(uint64_t v, __nv_bfloat16) {
  float lo, hi;
  unpack_f32x2(v, lo, hi);
  return pack_bf16x2(lo, hi);
}
__device__ __forceinline__ uint32_t narrow(uint64_t v, __half) {
  float lo, hi;
  unpack_f32x2(v, lo, hi);
  uint32_t w;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}
// Four pairs to memory.
template <typename T>
__device__ __forceinline__ void store8(T* p, const uint64_t* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(narrow(v[0], T()), narrow(v[1], T()), narrow(v[2], T()), narrow(v[3], T()));
}
__device__ __forceinline__ void store8(float* p, const uint64_t* v) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack_f32x2(v[i], f[2 * i], f[2 * i + 1]);
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(uint8_t* p, const uint64_t* v) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack_f32x2(v[i], f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_e4m3x4(f[0], f[1], f[2], f[3]), pack_e4m3x4(f[4], f[5], f[6], f[7]));
}

// Eight elements of a weight, 16-byte aligned like the pieces.
__device__ __forceinline__ void weight8(const void* w, int dtype, int at, float* v) {
  if (dtype == WK_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + at);
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t y = dtype == WK_BF16 ? widen(x[i], __nv_bfloat16()) : widen(x[i], __half());
      unpack_f32x2(y, v[2 * i], v[2 * i + 1]);
    }
  }
}

// What a lane is in its warp.  LPR: lanes of a row where that is a power of two (0: any number).
template <int LPR>
struct Place {
  int lpr, in_row, hslot, tslot;
  int at_a, at_b;  // its two pieces
  bool active, turned;
  __device__ __forceinline__ explicit Place(const RopeParams& p) {
    const int lane = threadIdx.x % 32;
    lpr = LPR ? LPR : p.d / 16;
    const int slot = lane / lpr;
    in_row = lane - slot * lpr;
    tslot = slot / p.hb, hslot = slot - tslot * p.hb;
    active = tslot < p.tb;
    turned = in_row < p.rot / 16;
    // neighbouring lanes' pieces lie side by side, also where pairs are neighbours and either half would do (4 x 13020 tokens,
    // 16 / 2 heads of 160, interleaved, gradient: 273 us with each lane's pieces side by side, 186 so)
    if (turned) at_a = 8 * in_row, at_b = at_a + p.rot / 2;
    else at_a = p.rot / 2 + 8 * in_row, at_b = at_a + (p.d - p.rot) / 2;
  }
  // Two sums over the lanes of a row.
  __device__ __forceinline__ void row_sums(float (&x)[2]) const {
    if (LPR) {
#pragma unroll
      for (int i = LPR / 2; i > 0; i >>= 1) {
        const float a = __shfl_xor_sync(0xffffffffu, x[0], i), b = __shfl_xor_sync(0xffffffffu, x[1], i);
        x[0] += a, x[1] += b;
      }
      return;
    }
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int i = 8; i > 0; i >>= 1) {
      const float a = __shfl_down_sync(0xffffffffu, x[0], i), b = __shfl_down_sync(0xffffffffu, x[1], i);
      if (in_row < i && in_row + i < lpr) x[0] += a, x[1] += b;
    }
    x[0] = __shfl_sync(0xffffffffu, x[0], lane - in_row);
    x[1] = __shfl_sync(0xffffffffu, x[1], lane - in_row);
  }
};

// The lane's cosines and sines of its token.  The lanes of a token divide its pairs and exchange them in `table`
// ([token of the warp][cos, sin][pair], eight of a lane's in a row: those of both halves' elements, or four of each piece).
template <typename T, int LPR>
__device__ __forceinline__ void angles(const RopeParams& p, const Place<LPR>& at, bool live, int b, int n, float* table,
                                       float (&c)[8], float (&s)[8]) {
  const int pairs = p.rot / 2;
  float* mine = table + at.tslot * 2 * pairs;
  if (live) {
    const int every = p.hb * at.lpr;
    for (int j0 = at.hslot * at.lpr + at.in_row; j0 < pairs; j0 += 2 * every) {
      double turns[2];  // two at a time: their loads go together
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int place = min(j0 + i * every, pairs - 1);
        const int j = p.interleaved ? (place >> 3) * 4 + (place & 3) + (place & 4 ? pairs / 2 : 0) : place;
        const int axis = static_cast<int>(p.axis_map[j >> 5] >> (2 * (j & 31))) & 3;
        const int64_t from = axis * p.ps[0] + b * p.ps[1] + n * p.ps[2];
        const double pos = p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[from])
                                   : static_cast<double>(static_cast<const int32_t*>(p.positions)[from]);
        const double f = p.freq64 ? static_cast<const double*>(p.inv_freq)[j]
                                  : static_cast<double>(static_cast<const float*>(p.inv_freq)[j]);
        turns[i] = pos * (f * 0.15915494309189533577);  // 1 / (2 pi)
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = j0 + i * every;
        float sn, cs;
        const float rest = static_cast<float>(turns[i] - rint(turns[i]));
        if (sizeof(T) == 4) {
          sincospif(2.f * rest, &sn, &cs);
        } else {  // 2^-21 off within half a turn, which 16 bits of output do not see; a quarter of the instructions
          __sincosf(6.2831853071795865f * rest, &sn, &cs);
        }
        if (j < pairs) {
          mine[j] = cs;
          mine[pairs + j] = p.inverse ? -sn : sn;
        }
      }
    }
  }
  __syncwarp();
  if (live && at.turned) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 x = reinterpret_cast<const float4*>(mine + 8 * at.in_row)[i];
      const float4 y = reinterpret_cast<const float4*>(mine + pairs + 8 * at.in_row)[i];
      c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
      s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
    }
  }
  __syncwarp();  // the table may be written again
}

// Rotation of a lane's values with factors folded in: y[i] = v[i] own[i] + (the other member of each pair) other[i].
__device__ __forceinline__ uint64_t swapped(uint64_t v) {
  float lo, hi;
  unpack_f32x2(v, lo, hi);
  return pack_f32x2(hi, lo);
}
__device__ __forceinline__ void turn(const uint64_t (&v)[8], const uint64_t (&own)[8], const uint64_t (&other)[8], bool turned,
                                     bool interleaved, uint64_t (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = mul_f32x2(v[i], own[i]);
  if (turned) {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fma_f32x2(swapped(v[i]), other[i], y[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fma_f32x2(v[i ^ 4], other[i], y[i]);
    }
  }
}
// The factors, from cosines, sines and the weights of the value that is multiplied.
__device__ __forceinline__ void factors(const float (&c)[8], const float (&s)[8], const float (&w)[16], bool turned, bool interleaved,
                                        uint64_t (&own)[8], uint64_t (&other)[8]) {
  if (!turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) own[i] = pack_f32x2(w[2 * i], w[2 * i + 1]), other[i] = 0;
  } else if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      own[i] = pack_f32x2(c[i] * w[2 * i], c[i] * w[2 * i + 1]);
      other[i] = pack_f32x2(-s[i] * w[2 * i + 1], s[i] * w[2 * i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      own[i] = pack_f32x2(c[2 * i] * w[2 * i], c[2 * i + 1] * w[2 * i + 1]);
      own[4 + i] = pack_f32x2(c[2 * i] * w[8 + 2 * i], c[2 * i + 1] * w[9 + 2 * i]);
      other[i] = pack_f32x2(-s[2 * i] * w[8 + 2 * i], -s[2 * i + 1] * w[9 + 2 * i]);
      other[4 + i] = pack_f32x2(s[2 * i] * w[2 * i], s[2 * i + 1] * w[2 * i + 1]);
    }
  }
}

// The rotation alone, backwards: cosines and sines as they are, which takes half the registers.
__device__ __forceinline__ void turn_back(const uint64_t (&v)[8], const float (&c)[8], const float (&s)[8], bool turned,
                                          bool interleaved, uint64_t (&y)[8]) {
  if (!turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = v[i];
  } else if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a, b;
      unpack_f32x2(v[i], a, b);
      y[i] = pack_f32x2(a * c[i] + b * s[i], b * c[i] - a * s[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t c2 = pack_f32x2(c[2 * i], c[2 * i + 1]), s2 = pack_f32x2(s[2 * i], s[2 * i + 1]);
      y[i] = fma_f32x2(v[4 + i], s2, mul_f32x2(v[i], c2));
      y[4 + i] = fma_f32x2(mul_f32x2(v[i], s2), pack_f32x2(-1.f, -1.f), mul_f32x2(v[4 + i], c2));
    }
  }
}

__device__ __forceinline__ float sum_of(uint64_t v) {
  float lo, hi;
  unpack_f32x2(v, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ float dot(const uint64_t (&a)[8], const uint64_t (&b)[8]) {
  uint64_t x = mul_f32x2(a[0], b[0]), y = mul_f32x2(a[4], b[4]);
#pragma unroll
  for (int i = 1; i < 4; ++i) x = fma_f32x2(a[i], b[i], x), y = fma_f32x2(a[4 + i], b[4 + i], y);
  return sum_of(add_f32x2(x, y));
}

// The groups of tokens that a warp works through; it takes one of the `hs` shares of their heads.  hs divides the number of
// warps, so that neither the share nor the distance to the next group changes.
template <int LPR>
struct Walk {
  int group, groups, group_step;
  int token, b, n, token_step, b_step, n_step;  // of this lane
  __device__ __forceinline__ Walk(const RopeParams& p, const Place<LPR>& at) {
    group_step = gridDim.x * (kThreads / 32) / p.hs;
    groups = (p.tokens + p.tb - 1) / p.tb;
    token_step = group_step * p.tb;
    b_step = token_step / p.N, n_step = token_step - b_step * p.N;
    begin(p, at);
  }
  __device__ __forceinline__ void begin(const RopeParams& p, const Place<LPR>& at) {
    group = (blockIdx.x * (kThreads / 32) + threadIdx.x / 32) / p.hs;
    token = group * p.tb + at.tslot;
    b = token / p.N, n = token - b * p.N;
  }
  __device__ __forceinline__ bool here() const { return group < groups; }
  __device__ __forceinline__ void next(const RopeParams& p) {
    group += group_step, token += token_step, b += b_step, n += n_step;
    if (n >= p.N) n -= p.N, ++b;
  }
};

// The rows that a lane fetches ahead into its ring: two heads at a step, `hb` apart, of IN tensors (backward: also the
// gradients).  Forward: the queries and then the keys of a group of tokens.  Backward: the queries of all groups, then the
// keys, so that one weight's gradient is summed at a time.
template <typename T, int LPR, bool BWD>
struct Fetcher {
  static constexpr int IN = BWD ? 2 : 1, STAGES = kStages<T, BWD>, BYTES = 2 * IN * kRowBytes<T>;
  Walk<LPR> walk;
  uint32_t ring;
  int side, h, first, every, heads, between;
  bool live, more;  // the lane's token exists; something is left to fetch
  const T* from[IN];
  int64_t apart[IN], next[IN];  // of the two heads, of the steps
  __device__ __forceinline__ Fetcher(const RopeParams& p, const Place<LPR>& at, uint32_t ring, int first)
      : walk(p, at), ring(ring), side(0), first(first), every(2 * p.hs * p.hb), between(at.at_b - at.at_a), more(true) {
    start(p, at);
  }
  // The first step of the side, or of the next one that has any for this warp.
  __device__ __forceinline__ void start(const RopeParams& p, const Place<LPR>& at) {
    while (!walk.here() || first - at.hslot >= p.heads[side])
      if (!advance(p, at)) return;
    h = first, heads = p.heads[side];
    live = at.active && walk.token < p.tokens;
#pragma unroll
    for (int i = 0; i < IN; ++i) {
      const int64_t(&st)[3] = i ? p.dys[side] : p.xs[side];
      from[i] = static_cast<const T*>(i ? p.dy[side] : p.x[side]) + walk.b * st[0] + walk.n * st[2] + first * st[1] + at.at_a;
      apart[i] = p.hb * st[1], next[i] = 2 * p.hs * apart[i];
    }
  }
  __device__ __forceinline__ bool advance(const RopeParams& p, const Place<LPR>& at) {
    if (BWD) {
      if (walk.here()) walk.next(p);
      if (walk.here()) return true;
      if (side || !p.heads[1]) return more = false;
      side = 1;
      walk.begin(p, at);
      return true;
    }
    if (!walk.here()) return more = false;
    if (!side && p.heads[1]) {
      side = 1;
    } else {
      side = 0;
      walk.next(p);
    }
    return true;
  }
  __device__ __forceinline__ void operator()(const RopeParams& p, const Place<LPR>& at, int stage) {
    if (more) {
      const int there = live ? heads - h : 0;
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        const uint32_t dst = ring + stage * BYTES + 2 * i * kRowBytes<T>;
        if (there > 0) fetch_raw(dst, from[i], between);
        if (there > p.hb) fetch_raw(dst + kRowBytes<T>, from[i] + apart[i], between);
        from[i] += next[i];
      }
      h += every;
      if (h - at.hslot >= heads && advance(p, at)) start(p, at);  // the same for the whole warp
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
};

template <typename T, bool FP8, bool NORM, int LPR>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
rope_kernel(const __grid_constant__ RopeParams p) {
  using Out = typename std::conditional<FP8, uint8_t, T>::type;
  using Fetch = Fetcher<T, LPR, false>;
  constexpr int WARPS = kThreads / 32;
  extern __shared__ __align__(16) uint8_t ring_mem[];
  __shared__ __align__(16) float tables[WARPS][kTable];
  __shared__ __align__(16) float weights[NORM ? 2 * kMaxD : 4];
  const int warp = threadIdx.x / 32;
  const uint32_t ring = smem_u32(ring_mem) + warp * Fetch::STAGES * Fetch::BYTES + (threadIdx.x % 32) * 16;
  const Place<LPR> at(p);
  const float inv_d = 1.f / static_cast<float>(p.d);
  const int first = (blockIdx.x * WARPS + warp) % p.hs * 2 * p.hb + at.hslot, every = 2 * p.hs * p.hb;
  const int sides = p.heads[1] ? 2 : 1;
  pdl_launch_dependents();
  pdl_wait();

  Fetch fetch(p, at, ring, first);
  for (int i = 0; i < Fetch::STAGES; ++i) fetch(p, at, i);
  if (NORM) {
    for (int i = threadIdx.x * 8; i < sides * p.d; i += kThreads * 8) weight8(p.w[i >= p.d], p.w_dtype, i >= p.d ? i - p.d : i, weights + i);
    __syncthreads();
  }
  int stage = 0;
  Walk<LPR> now(p, at);
  for (; now.here(); now.next(p)) {
    const bool live = at.active && now.token < p.tokens;
    float c[8], s[8];
    angles<T, LPR>(p, at, live, now.b, now.n, tables[warp], c, s);
    uint64_t own[8], other[8];
    if (!NORM) {
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = 1.f;
      factors(c, s, w, at.turned, p.interleaved, own, other);
    }
    for (int side = 0; side < sides; ++side) {
      const int heads = p.heads[side];
      if (NORM && at.active) {
        float w[16];
        const float* from = weights + side * p.d;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 x = reinterpret_cast<const float4*>(from + at.at_a)[i], y = reinterpret_cast<const float4*>(from + at.at_b)[i];
          w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
          w[8 + 4 * i] = y.x, w[9 + 4 * i] = y.y, w[10 + 4 * i] = y.z, w[11 + 4 * i] = y.w;
        }
        factors(c, s, w, at.turned, p.interleaved, own, other);
      }
      const int64_t apart = p.hb * p.ys[side][1], next = 2 * p.hs * apart;
      const int between = at.at_b - at.at_a;
      Out* to = static_cast<Out*>(p.y[side]) + now.b * p.ys[side][0] + now.n * p.ys[side][2] + first * p.ys[side][1] + at.at_a;
      for (int h = first; h - at.hslot < heads; h += every, to += next) {
        const int there = live ? heads - h : 0;
        float scale[2] = {1.f, 1.f};
        if (FP8) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (there > i * p.hb)  // head / group, exact: heads are fewer than 2^20
              scale[i] = p.descale[side][now.b * p.hkv + static_cast<int>((static_cast<float>(h + i * p.hb) + 0.5f) *
                                                                          (side ? 1.f : p.inv_group))];
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(Fetch::STAGES - 1) : "memory");
        uint64_t v[2][8], y[8];
        float f[2] = {1.f, 1.f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // where there is no second head, what lies there is read for nothing
          Raw<T> raw;
          read_raw(ring + stage * Fetch::BYTES + i * kRowBytes<T>, raw);
          unpack(raw, v[i]);
        }
        if (NORM) {
          float ss[2] = {dot(v[0], v[0]), dot(v[1], v[1])};
          at.row_sums(ss);
#pragma unroll
          for (int i = 0; i < 2; ++i) f[i] = rsqrtf(ss[i] * inv_d + p.eps);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          turn(v[i], own, other, at.turned, p.interleaved, y);
          if (FP8) f[i] *= __frcp_rn(scale[i]);  // within 2^-23 of the quotient, which moves codes that close to a tie
          if (NORM || FP8) {
            const uint64_t f2 = pack_f32x2(f[i], f[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = mul_f32x2(y[j], f2);
          }
          if (there > i * p.hb) {
            Out* dst = i ? to + apart : to;
            store8(dst, y);
            store8(dst + between, y + 4);
          }
        }
        fetch(p, at, stage);  // into the place that has just been read
        if (++stage == Fetch::STAGES) stage = 0;
      }
    }
  }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
norm_rope_bwd_kernel(const __grid_constant__ RopeParams p) {
  using Fetch = Fetcher<T, LPR, true>;
  constexpr int WARPS = kThreads / 32;
  extern __shared__ __align__(16) uint8_t ring_mem[];
  __shared__ __align__(16) float tables[WARPS][kTable];
  __shared__ float sums[2][WARPS][kMaxD];
  const int warp = threadIdx.x / 32;
  const uint32_t ring = smem_u32(ring_mem) + warp * Fetch::STAGES * Fetch::BYTES + (threadIdx.x % 32) * 16;
  const Place<LPR> at(p);
  const float inv_d = 1.f / static_cast<float>(p.d);
  const int first = (blockIdx.x * WARPS + warp) % p.hs * 2 * p.hb + at.hslot, every = 2 * p.hs * p.hb;
  pdl_launch_dependents();
  pdl_wait();

  Fetch fetch(p, at, ring, first);
  for (int i = 0; i < Fetch::STAGES; ++i) fetch(p, at, i);
  int stage = 0;
  Walk<LPR> now(p, at);
  for (int side = 0; side < (p.heads[1] ? 2 : 1); ++side) {
    if (side) now.begin(p, at);
    const int heads = p.heads[side];
    uint64_t w[8], dw[8];
    {
      float v[16] = {};
      if (at.active) {
        weight8(p.w[side], p.w_dtype, at.at_a, v);
        weight8(p.w[side], p.w_dtype, at.at_b, v + 8);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = pack_f32x2(v[2 * i], v[2 * i + 1]), dw[i] = 0;
    }
    const int64_t apart = p.hb * p.ys[side][1], next = 2 * p.hs * apart;
    const int between = at.at_b - at.at_a;
    for (; now.here() && first - at.hslot < heads; now.next(p)) {
      const bool live = at.active && now.token < p.tokens;
      float c[8], s[8];
      angles<T, LPR>(p, at, live, now.b, now.n, tables[warp], c, s);
      T* to = static_cast<T*>(p.y[side]) + now.b * p.ys[side][0] + now.n * p.ys[side][2] + first * p.ys[side][1] + at.at_a;
      for (int head = first; head - at.hslot < heads; head += every, to += next) {
        const int there = live ? heads - head : 0;
        asm volatile("cp.async.wait_group %0;" ::"n"(Fetch::STAGES - 1) : "memory");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint64_t x[8], g[8], h[8];
          {
            Raw<T> raw;
            uint64_t dy[8];
            read_raw(ring + stage * Fetch::BYTES + (2 + i) * kRowBytes<T>, raw);
            unpack(raw, dy);
            turn_back(dy, c, s, at.turned, p.interleaved, g);
            read_raw(ring + stage * Fetch::BYTES + i * kRowBytes<T>, raw);
            unpack(raw, x);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] = mul_f32x2(g[j], w[j]);
          float sum[2] = {dot(x, x), dot(h, x)};
          at.row_sums(sum);
          // dx = r (h - (x r) mean(h x r)): r^3 by itself leaves fp32 where x is beyond 1e13 or below 1e-13
          const float f = rsqrtf(sum[0] * inv_d + p.eps), m = -f * (f * sum[1] * inv_d);
          const uint64_t f2 = pack_f32x2(f, f), m2 = pack_f32x2(m, m);
          if (there > i * p.hb) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              dw[j] = fma_f32x2(mul_f32x2(g[j], x[j]), f2, dw[j]);
              h[j] = mul_f32x2(fma_f32x2(x[j], m2, h[j]), f2);
            }
            T* dst = i ? to + apart : to;
            store8(dst, h);
            store8(dst + between, h + 4);
          }
        }
        fetch(p, at, stage);
        if (++stage == Fetch::STAGES) stage = 0;
      }
    }
    // the weight's gradient over the rows of the warp
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[2];
      unpack_f32x2(dw[i], v[0], v[1]);
      const int e = i < 4 ? at.at_a + 2 * i : at.at_b + 2 * (i - 4);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = v[j];
        if (LPR) {
#pragma unroll
          for (int o = 16; o >= LPR; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        } else {
          for (int o = at.lpr; o + at.lpr <= 32; o += at.lpr) {
            const float other = __shfl_down_sync(0xffffffffu, v[j], o);
            if (threadIdx.x % 32 < at.lpr) sum += other;
          }
        }
        if (threadIdx.x % 32 < at.lpr) sums[side][warp][e + j] = sum;
      }
    }
  }
  // and over the warps, always in the same order
  __syncthreads();
  for (int i = threadIdx.x; i < (p.heads[1] ? 2 : 1) * p.d; i += kThreads) {
    const int side = i >= p.d, e = side ? i - p.d : i;
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) sum += sums[side][v][e];
    p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + side) * p.d + e] = sum;
  }
}

// Sums the CTAs' parts, 32 columns to a CTA, in a fixed order.
__global__ void __launch_bounds__(1024)
dweight_kernel(const float* __restrict__ partial, int parts, int d, void* dw_q, void* dw_k, int w_dtype) {
  __shared__ float sums[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int col = blockIdx.x * 32 + threadIdx.x % 32, strip = threadIdx.x / 32, which = blockIdx.y;
  float s = 0.f;
  if (col < d)
    for (int i = strip; i < parts; i += 32) s += __ldcg(partial + (static_cast<int64_t>(i) * 2 + which) * d + col);
  sums[strip][threadIdx.x % 32] = s;
  __syncthreads();
  if (strip || col >= d) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += sums[i][threadIdx.x];
  void* out = which ? dw_k : dw_q;
  if (w_dtype == WK_F32)
    static_cast<float*>(out)[col] = s;
  else if (w_dtype == WK_BF16)
    static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(s);
  else
    static_cast<__half*>(out)[col] = __float2half_rn(s);
}

// How a warp's rows are divided into heads and tokens: the division that takes the fewest instructions per token (300 for a
// step over two rows per lane, 40 for an angle, 150 for a group of tokens), weighed with how short the pieces of memory are
// that it reads at a time: neighbouring heads of a token, or neighbouring tokens of a head, whichever lie side by side.
// (4 x 4096 tokens, 32 / 8 heads, d 128, heads side by side, bf16: 4 heads and one token at a time 60.4 us, 2 and 2 65.4,
// 1 and 4 66.2; 16385 tokens, 16 / 16 heads, d 80, fp16: 3 and 2 38.2 us, 2 and 3 41.6, 1 and 6 44.9.)
// And over how many warps the heads of a token are spread: so many (of those that divide the warps of a CTA) that the last
// round of the groups over the warps costs least.
void divide(RopeParams& p, int ctas_at_once, int size, int& ctas) {
  const int lpr = p.d / 16, rows = 32 / lpr, pairs = p.rot / 2, warps = kThreads / 32;
  auto steps = [&](int side, int hb) { return (p.heads[side] + 2 * hb - 1) / (2 * hb); };
  double best = 0, fixed = 0;
  for (int hb = 1; hb <= rows; ++hb) {
    const int tb = rows / hb;
    const double f = 150.0 + 40.0 * ((pairs + hb * lpr - 1) / (hb * lpr));
    const int side_by_side = p.xs[0][1] == p.d ? 2 * hb : p.xs[0][2] == p.d ? tb : 1;
    const double cost = (300.0 * (steps(0, hb) + steps(1, hb)) + f) / tb * (1.0 + 420.0 / (side_by_side * p.d * size));
    if (hb == 1 || cost < best) best = cost, fixed = f, p.hb = hb, p.tb = tb;
  }
  const int64_t groups = (p.tokens + p.tb - 1) / p.tb;
  for (int hs = 1; hs <= warps && hs < 2 * steps(0, p.hb); hs *= 2) {
    const double rounds = static_cast<double>(groups * hs) / (static_cast<double>(ctas_at_once) * warps);
    const double work = fixed + 300.0 * ((steps(0, p.hb) + hs - 1) / hs + (steps(1, p.hb) + hs - 1) / hs);
    const double cost = (rounds < 1 ? 1 : rounds > 4 ? rounds : ceil(rounds)) * work;
    if (hs == 1 || cost < best) best = cost, p.hs = hs;
  }
  const int64_t want = (groups * p.hs + warps - 1) / warps;
  ctas = static_cast<int>(want < ctas_at_once ? want : ctas_at_once);
}

// CTAs that fit the GPU by their shared memory (`fixed`: the static part).
int ctas_at_once(int sms, int smem, int fixed) {
  const int fit = 227 * 1024 / (smem + fixed + 1024);
  return sms * (fit < kCtasPerSm ? fit : kCtasPerSm);
}
template <typename T, bool BWD>
constexpr int kRingBytes = kThreads / 32 * Fetcher<T, 0, BWD>::STAGES * Fetcher<T, 0, BWD>::BYTES;
constexpr int kTableBytes = kThreads / 32 * kTable * 4, kSumBytes = 2 * kThreads / 32 * kMaxD * 4;

int elem_size(int dtype) { return dtype == WK_F32 ? 4 : 2; }
bool known_dtype(int t) { return t == WK_BF16 || t == WK_F32 || t == WK_F16; }

// Checks the argument block and fills the kernels' parameters.
int fill(const wk_rope_args* a, bool bwd, RopeParams& p) {
  if (!a) return WK_E_ARG;
  if (a->B <= 0 || a->N <= 0 || a->Hq <= 0 || a->Hk < 0 || !a->q || !a->q_out || !a->positions || !a->inv_freq) return WK_E_ARG;
  if (a->d < 32 || a->d > kMaxD || a->d % 16 || a->rot < 16 || a->rot > a->d || a->rot % 16) return WK_E_ARG;
  if (!known_dtype(a->dtype)) return WK_E_ARG;
  const bool keys = a->Hk > 0;
  if (keys && (!a->k || !a->k_out)) return WK_E_ARG;
  const bool norm = a->q_weight != nullptr;
  if (norm && (!aligned16(a->q_weight) || (keys && !aligned16(a->k_weight)))) return WK_E_ARG;
  if (norm && (!known_dtype(a->w_dtype) || (keys && !a->k_weight) || !(a->eps >= 0.f))) return WK_E_ARG;
  if (bwd && (!norm || !a->dq_out || (keys && !a->dk_out) || !a->dq_weight || (keys && !a->dk_weight))) return WK_E_ARG;
  const bool fp8 = a->q_descale != nullptr;
  if (fp8 && (bwd || (keys && !a->k_descale) || a->Hkv <= 0 || a->Hq % a->Hkv || (keys && a->Hk != a->Hkv))) return WK_E_ARG;
  if (!fp8 && a->k_descale) return WK_E_ARG;
  const int64_t tokens = static_cast<int64_t>(a->B) * a->N;
  if (tokens > INT32_MAX / 2 || static_cast<int64_t>(a->Hq) + a->Hk > (1 << 20)) return WK_E_ARG;
  const int size = elem_size(a->dtype), out_size = fp8 ? 1 : size;
  auto rows_ok = [](const void* base, const int64_t* s, int bytes, int unit) {
    if (reinterpret_cast<uintptr_t>(base) % unit) return false;
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0 || s[i] * bytes % unit) return false;
    return true;
  };
  auto out_ok = [&](const void* base, const int64_t* s, int heads) {  // rows of their own, too
    return rows_ok(base, s, out_size, fp8 ? 8 : 16) && (s[0] || a->B == 1) && (s[1] || heads == 1) && (s[2] || a->N == 1);
  };
  if (!rows_ok(a->q, a->q_strides, size, 16) || !out_ok(a->q_out, a->q_out_strides, a->Hq)) return WK_E_ARG;
  if (keys && (!rows_ok(a->k, a->k_strides, size, 16) || !out_ok(a->k_out, a->k_out_strides, a->Hk))) return WK_E_ARG;
  if (bwd && (!rows_ok(a->dq_out, a->dq_out_strides, size, 16) || (keys && !rows_ok(a->dk_out, a->dk_out_strides, size, 16))))
    return WK_E_ARG;
  p = {};
  p.x[0] = a->q, p.x[1] = keys ? a->k : nullptr;
  p.y[0] = a->q_out, p.y[1] = a->k_out;
  p.dy[0] = a->dq_out, p.dy[1] = a->dk_out;
  p.w[0] = a->q_weight, p.w[1] = a->k_weight;
  p.descale[0] = a->q_descale, p.descale[1] = a->k_descale;
  p.positions = a->positions, p.inv_freq = a->inv_freq;
  for (int i = 0; i < 3; ++i) {
    p.xs[0][i] = a->q_strides[i], p.xs[1][i] = a->k_strides[i];
    p.ys[0][i] = a->q_out_strides[i], p.ys[1][i] = a->k_out_strides[i];
    p.dys[0][i] = a->dq_out_strides[i], p.dys[1][i] = a->dk_out_strides[i];
    p.ps[i] = a->position_strides[i];
  }
  for (int i = 0; i < 4; ++i) p.axis_map[i] = a->axis_map[i];
  p.N = a->N, p.heads[0] = a->Hq, p.heads[1] = a->Hk;
  p.tokens = static_cast<int>(tokens);
  p.d = a->d, p.rot = a->rot;
  p.hkv = a->Hkv, p.inv_group = fp8 ? 1.f / static_cast<float>(a->Hq / a->Hkv) : 1.f;
  p.w_dtype = a->w_dtype, p.pos64 = a->position_int64, p.freq64 = a->inv_freq_f64;
  p.interleaved = a->interleaved != 0, p.inverse = a->inverse != 0;
  p.eps = a->eps;
  return 0;
}

template <typename T, bool FP8, bool NORM>
const void* forward_kernel(int d) {
  return d == 64    ? reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 4>)
         : d == 128 ? reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 8>)
                    : reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 0>);
}
template <typename T>
const void* forward_kernel(int d, bool fp8, bool norm) {
  if (fp8) return norm ? forward_kernel<T, true, true>(d) : forward_kernel<T, true, false>(d);
  return norm ? forward_kernel<T, false, true>(d) : forward_kernel<T, false, false>(d);
}
template <typename T>
const void* backward_kernel(int d) {
  return d == 64    ? reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 4>)
         : d == 128 ? reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 8>)
                    : reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 0>);
}

}  // namespace
}  // namespace wk

extern "C" int wk_rope(const wk_rope_args* a, void* stream) {
  using namespace wk;
  RopeParams p;
  if (int bad = fill(a, false, p)) return bad;
  if (int unsupported = require_sm100()) return unsupported;
  const int sms = sm_count();
  if (sms <= 0) return WK_E_CUDA;
  const bool fp8 = p.descale[0] != nullptr, norm = p.w[0] != nullptr;
  const void* kernel = a->dtype == WK_BF16 ? forward_kernel<__nv_bfloat16>(p.d, fp8, norm)
                       : a->dtype == WK_F16 ? forward_kernel<__half>(p.d, fp8, norm)
                                            : forward_kernel<float>(p.d, fp8, norm);
  const int smem = a->dtype == WK_F32 ? kRingBytes<float, false> : kRingBytes<__half, false>;
  int ctas;
  divide(p, ctas_at_once(sms, smem, kTableBytes + 2 * kMaxD * 4), elem_size(a->dtype), ctas);
  if (allow_smem(kernel, smem)) return WK_E_CUDA;
  return launch_pdl(kernel, dim3(ctas), kThreads, smem, static_cast<cudaStream_t>(stream), 1, {&p});
}

// Two rows of d sums per CTA.
extern "C" int64_t wk_qk_norm_rope_bwd_workspace_bytes(int d) {
  const int sms = wk::sm_count();
  return d > 0 && sms > 0 ? static_cast<int64_t>(wk::kCtasPerSm) * sms * 2 * d * 4 : 0;
}

extern "C" int wk_qk_norm_rope_bwd(const wk_rope_args* a, void* stream) {
  using namespace wk;
  RopeParams p;
  if (int bad = fill(a, true, p)) return bad;
  if (int unsupported = require_sm100()) return unsupported;
  const int sms = sm_count();
  if (sms <= 0) return WK_E_CUDA;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < wk_qk_norm_rope_bwd_workspace_bytes(p.d)) return WK_E_ARG;
  p.partial = static_cast<float*>(a->workspace);
  const void* kernel = a->dtype == WK_BF16 ? backward_kernel<__nv_bfloat16>(p.d)
                       : a->dtype == WK_F16 ? backward_kernel<__half>(p.d)
                                            : backward_kernel<float>(p.d);
  const int smem = a->dtype == WK_F32 ? kRingBytes<float, true> : kRingBytes<__half, true>;
  int ctas;
  divide(p, ctas_at_once(sms, smem, kTableBytes + kSumBytes), elem_size(a->dtype), ctas);
  if (allow_smem(kernel, smem)) return WK_E_CUDA;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int bad = launch_pdl(kernel, dim3(ctas), kThreads, smem, st, 1, {&p})) return bad;
  const float* partial = p.partial;
  int d = p.d, w_dtype = p.w_dtype;
  void *dq = a->dq_weight, *dk = a->dk_weight;
  return launch_pdl(reinterpret_cast<const void*>(dweight_kernel), dim3((d + 31) / 32, p.heads[1] ? 2 : 1), 1024, 0, st, 1,
                    {&partial, &ctas, &d, &dq, &dk, &w_dtype});
}
