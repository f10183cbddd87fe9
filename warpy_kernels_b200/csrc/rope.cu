// Position rotation of queries and keys, with or without the RMS norm of every head before it, in one pass; optionally
// as the e4m3 codes that the FP8 attention reads.  And the gradient of norm and rotation.
//
// One row is one head of one token, x in R^d:
//   r = (mean(x^2) + eps)^-1/2      u = x r w      y = R(theta) u        (without the norm: u = x)
// R turns the pairs (j, j + R/2), or (2 j, 2 j + 1), of the first R elements by theta_j = position[axis(j)] inv_freq[j].
// Backward, with g = R(-theta) dy, h = g w:
//   dw = sum over rows of g x r     dx = r (h - x r^2 mean(h x))
//
// A row is d / 16 lanes of a warp with 16 elements each, two 16-byte pieces (16-bit types) that hold both halves of the
// lane's pairs: the rotation needs no exchange, the norm one reduction over the lanes of a row.  A CTA takes all heads of
// a few neighbouring tokens, so that an angle is made once for all heads of its token.
//
// Angles: position times inv_freq in turns, reduced to half a turn in fp64 (positions beyond 2^20 leave nothing of an fp32
// product's fraction), then sine and cosine in fp32.
//
// Bound by HBM: every element is read once and written once (backward: read twice).
#include <cuda_fp16.h>

#include "common.cuh"
#include "host_common.h"

namespace wk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxD = 256;

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
  int B, N, Hq, H;  // H: heads of queries and keys
  int tokens, per_cta;
  int d, rot;
  int group;  // query heads per descale entry
  int hkv;
  int w_dtype, pos64, freq64, interleaved, inverse;
  float eps;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* v) {
  const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* p, float* v) {
  const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f16x2_to_float2(w[i], v[2 * i], v[2 * i + 1]);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* v) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                            pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__half* p, const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(uint8_t* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_e4m3x4(v[0], v[1], v[2], v[3]), pack_e4m3x4(v[4], v[5], v[6], v[7]));
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (dtype == WK_F32) return static_cast<const float*>(w)[i];
  if (dtype == WK_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// Cosine and sine of a CTA's tokens: cos at [token][pair], sin behind them.
__device__ __forceinline__ void make_table(const RopeParams& p, int t0, int nt, float* table) {
  const int h = p.rot / 2;
  for (int i = threadIdx.x; i < nt * h; i += kThreads) {
    const int t = i / h, j = i - t * h;
    const int axis = static_cast<int>(p.axis_map[j >> 5] >> (2 * (j & 31))) & 3;
    const int b = (t0 + t) / p.N, n = (t0 + t) - b * p.N;
    const int64_t at = axis * p.ps[0] + b * p.ps[1] + n * p.ps[2];
    const double pos = p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                               : static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
    const double f = p.freq64 ? static_cast<const double*>(p.inv_freq)[j]
                              : static_cast<double>(static_cast<const float*>(p.inv_freq)[j]);
    const double turns = pos * (f * 0.15915494309189533577);  // 1 / (2 pi)
    const float rest = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.f * rest, &s, &c);
    table[i] = c;
    table[p.per_cta * h + i] = p.inverse ? -s : s;
  }
}

// The two 8-element pieces of a lane: both members of its pairs.
__device__ __forceinline__ void pieces(const RopeParams& p, int lane, int& a, int& b) {
  const int half = p.rot / 16;
  if (p.interleaved || lane >= half) {
    a = 16 * lane, b = a + 8;
  } else {
    a = 8 * lane, b = a + p.rot / 2;
  }
}

// Turns the pairs of a lane's 16 values; sign -1 turns them back.
__device__ __forceinline__ void turn(float (&v)[16], const float* cos, const float* sin, bool interleaved, float sign) {
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 x = reinterpret_cast<const float4*>(cos)[i], y = reinterpret_cast<const float4*>(sin)[i];
    c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
    s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
  }
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = v[2 * i], y = v[2 * i + 1], sn = sign * s[i];
      v[2 * i] = x * c[i] - y * sn;
      v[2 * i + 1] = y * c[i] + x * sn;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = v[i], y = v[8 + i], sn = sign * s[i];
      v[i] = x * c[i] - y * sn;
      v[8 + i] = y * c[i] + x * sn;
    }
  }
}

// Where a row is: its token in the CTA, and whether it is a query's or a key's head.
struct Row {
  int t, which, head, b, n;
};
__device__ __forceinline__ Row row_at(const RopeParams& p, int t0, int row) {
  Row r;
  r.t = row / p.H;
  const int h = row - r.t * p.H;
  r.which = h >= p.Hq;
  r.head = r.which ? h - p.Hq : h;
  r.b = (t0 + r.t) / p.N;
  r.n = (t0 + r.t) - r.b * p.N;
  return r;
}
__device__ __forceinline__ int64_t offset(const int64_t (&s)[3], const Row& r) {
  return r.b * s[0] + r.head * s[1] + r.n * s[2];
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int i = LPR / 2; i > 0; i >>= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
  return x;
}

// LPR: lanes of a row, at least d / 16.
template <typename T, bool FP8, bool NORM, int LPR>
__global__ void __launch_bounds__(kThreads)
rope_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float smem[];
  constexpr int SLOTS = kThreads / LPR;
  float* weights = smem;  // [2][d]
  float* table = smem + (NORM ? 2 * p.d : 0);
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int t0 = blockIdx.x * p.per_cta, nt = min(p.per_cta, p.tokens - t0);
  const int rows = nt * p.H, h = p.rot / 2;
  const bool mine = lane < p.d / 16;
  const bool turned = lane < p.rot / 16;
  int at_a, at_b;
  pieces(p, lane, at_a, at_b);
  pdl_launch_dependents();
  pdl_wait();

  auto load = [&](const Row& r, float (&v)[16]) {
    const T* src = static_cast<const T*>(p.x[r.which]) + offset(p.xs[r.which], r);
    load8<T>(src + at_a, v);
    load8<T>(src + at_b, v + 8);
  };
  float v[16];
  Row r = {};
  bool live = mine && slot < rows;
  if (live) {  // under way while the angles are made
    r = row_at(p, t0, slot);
    load(r, v);
  }
  make_table(p, t0, nt, table);
  if (NORM)
    for (int i = threadIdx.x; i < 2 * p.d; i += kThreads)
      weights[i] = i < p.d ? weight_at(p.w[0], p.w_dtype, i) : p.x[1] ? weight_at(p.w[1], p.w_dtype, i - p.d) : 0.f;
  __syncthreads();

  for (int row = slot;; row += SLOTS) {
    if (NORM) {
      float ss = 0.f;
      if (live) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
      }
      ss = row_sum<LPR>(ss);
      if (live) {
        const float f = rsqrtf(ss / static_cast<float>(p.d) + p.eps);
        const float* w = weights + r.which * p.d;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] *= f * w[at_a + i];
          v[8 + i] *= f * w[at_b + i];
        }
      }
    }
    if (live) {
      if (turned) turn(v, table + r.t * h + 8 * lane, table + (p.per_cta + r.t) * h + 8 * lane, p.interleaved, 1.f);
      if (FP8) {
        const float inv = 1.f / p.descale[r.which][r.b * p.hkv + (r.which ? r.head : r.head / p.group)];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= inv;
        uint8_t* dst = static_cast<uint8_t*>(p.y[r.which]) + offset(p.ys[r.which], r);
        store8(dst + at_a, v);
        store8(dst + at_b, v + 8);
      } else {
        T* dst = static_cast<T*>(p.y[r.which]) + offset(p.ys[r.which], r);
        store8(dst + at_a, v);
        store8(dst + at_b, v + 8);
      }
    }
    if ((row - slot) + SLOTS >= rows) break;  // the same for the whole CTA: the reduction above takes whole warps
    live = mine && row + SLOTS < rows;
    if (live) {
      r = row_at(p, t0, row + SLOTS);
      load(r, v);
    }
  }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads)
norm_rope_bwd_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float smem[];
  constexpr int SLOTS = kThreads / LPR, WARPS = kThreads / 32;
  float* weights = smem;  // [2][d]
  float* table = smem + 2 * p.d;
  const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const int h = p.rot / 2;
  const bool mine = lane < p.d / 16;
  const bool turned = lane < p.rot / 16;
  int at_a, at_b;
  pieces(p, lane, at_a, at_b);
  pdl_launch_dependents();
  pdl_wait();
  for (int i = threadIdx.x; i < 2 * p.d; i += kThreads)
    weights[i] = i < p.d ? weight_at(p.w[0], p.w_dtype, i) : p.x[1] ? weight_at(p.w[1], p.w_dtype, i - p.d) : 0.f;

  float dw[2][16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[0][i] = dw[1][i] = 0.f;

  for (int t0 = blockIdx.x * p.per_cta; t0 < p.tokens; t0 += gridDim.x * p.per_cta) {
    const int nt = min(p.per_cta, p.tokens - t0), rows = nt * p.H;
    __syncthreads();  // the table of the tokens before has been read
    make_table(p, t0, nt, table);
    __syncthreads();
    for (int row0 = 0; row0 < rows; row0 += SLOTS) {
      const bool live = mine && row0 + slot < rows;
      Row r = {};
      float x[16], g[16];
      float ss = 0.f, hx = 0.f;
      if (live) {
        r = row_at(p, t0, row0 + slot);
        const T* xp = static_cast<const T*>(p.x[r.which]) + offset(p.xs[r.which], r);
        const T* gp = static_cast<const T*>(p.dy[r.which]) + offset(p.dys[r.which], r);
        load8<T>(xp + at_a, x);
        load8<T>(xp + at_b, x + 8);
        load8<T>(gp + at_a, g);
        load8<T>(gp + at_b, g + 8);
        if (turned) turn(g, table + r.t * h + 8 * lane, table + (p.per_cta + r.t) * h + 8 * lane, p.interleaved, -1.f);
        const float* w = weights + r.which * p.d;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ss = fmaf(x[i], x[i], ss);
          hx = fmaf(g[i] * w[i < 8 ? at_a + i : at_b + i - 8], x[i], hx);
        }
      }
      ss = row_sum<LPR>(ss);
      hx = row_sum<LPR>(hx);
      if (live) {
        const float inv_d = 1.f / static_cast<float>(p.d);
        const float f = rsqrtf(ss * inv_d + p.eps);
        const float m = f * f * hx * inv_d;
        const float* w = weights + r.which * p.d;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float gx = g[i] * x[i] * f;
          dw[0][i] += r.which ? 0.f : gx;
          dw[1][i] += r.which ? gx : 0.f;
          x[i] = f * (g[i] * w[i < 8 ? at_a + i : at_b + i - 8] - x[i] * m);
        }
        T* dst = static_cast<T*>(p.y[r.which]) + offset(p.ys[r.which], r);
        store8(dst + at_a, x);
        store8(dst + at_b, x + 8);
      }
    }
  }

  // the weights' gradients of this CTA: over the rows of a warp, then over the warps, always in the same order
  __syncthreads();
  float* sums = smem;  // [WARPS][d], for queries and then for keys
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int o = 16; o >= LPR; o >>= 1) dw[q][i] += __shfl_xor_sync(0xffffffffu, dw[q][i], o);
      if (threadIdx.x % 32 < LPR && mine) sums[(threadIdx.x / 32) * p.d + (i < 8 ? at_a + i : at_b + i - 8)] = dw[q][i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.d; i += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += sums[w * p.d + i];
      p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + q) * p.d + i] = s;
    }
    __syncthreads();
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

int lanes_of(int d) { return d <= 32 ? 2 : d <= 64 ? 4 : d <= 128 ? 8 : 16; }

// Tokens of a CTA: four passes over its rows, fewer where the tokens would not fill the SMs.
int tokens_per_cta(int64_t tokens, int heads, int d, int sms) {
  const int slots = kThreads / lanes_of(d);
  int n = 4 * slots / heads;
  const int64_t share = (tokens + 4 * sms - 1) / (4 * sms);
  if (n > share) n = static_cast<int>(share);
  return n < 1 ? 1 : n > 16 ? 16 : n;
}

int bwd_ctas(int64_t tokens, int per_cta, int sms) {
  const int64_t groups = (tokens + per_cta - 1) / per_cta, most = 3ll * sms;
  return static_cast<int>(groups < most ? groups : most);
}

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
  p.B = a->B, p.N = a->N, p.Hq = a->Hq, p.H = a->Hq + a->Hk;
  p.tokens = static_cast<int>(tokens);
  p.d = a->d, p.rot = a->rot;
  p.hkv = a->Hkv, p.group = fp8 ? a->Hq / a->Hkv : 1;
  p.w_dtype = a->w_dtype, p.pos64 = a->position_int64, p.freq64 = a->inv_freq_f64;
  p.interleaved = a->interleaved != 0, p.inverse = a->inverse != 0;
  p.eps = a->eps;
  return 0;
}

template <typename T, bool FP8, bool NORM>
const void* forward_kernel(int lanes) {
  switch (lanes) {
    case 2: return reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 2>);
    case 4: return reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 4>);
    case 8: return reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 8>);
    default: return reinterpret_cast<const void*>(rope_kernel<T, FP8, NORM, 16>);
  }
}
template <typename T>
const void* forward_kernel(int lanes, bool fp8, bool norm) {
  if (fp8) return norm ? forward_kernel<T, true, true>(lanes) : forward_kernel<T, true, false>(lanes);
  return norm ? forward_kernel<T, false, true>(lanes) : forward_kernel<T, false, false>(lanes);
}
template <typename T>
const void* backward_kernel(int lanes) {
  switch (lanes) {
    case 2: return reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 2>);
    case 4: return reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 4>);
    case 8: return reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 8>);
    default: return reinterpret_cast<const void*>(norm_rope_bwd_kernel<T, 16>);
  }
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
  const int lanes = lanes_of(p.d);
  const bool fp8 = p.descale[0] != nullptr, norm = p.w[0] != nullptr;
  p.per_cta = tokens_per_cta(p.tokens, p.H, p.d, sms);
  const void* kernel = a->dtype == WK_BF16 ? forward_kernel<__nv_bfloat16>(lanes, fp8, norm)
                       : a->dtype == WK_F16 ? forward_kernel<__half>(lanes, fp8, norm)
                                            : forward_kernel<float>(lanes, fp8, norm);
  const int smem = (p.per_cta * p.rot + (norm ? 2 * p.d : 0)) * 4;
  const unsigned grid = static_cast<unsigned>((p.tokens + p.per_cta - 1) / p.per_cta);
  return launch_pdl(kernel, dim3(grid), kThreads, smem, static_cast<cudaStream_t>(stream), 1, {&p});
}

extern "C" int64_t wk_qk_norm_rope_bwd_workspace_bytes(int B, int N, int heads, int d) {
  const int sms = wk::sm_count();
  if (B <= 0 || N <= 0 || heads <= 0 || d <= 0 || sms <= 0) return 0;
  const int64_t tokens = static_cast<int64_t>(B) * N;
  return static_cast<int64_t>(wk::bwd_ctas(tokens, wk::tokens_per_cta(tokens, heads, d, sms), sms)) * 2 * d * 4;
}

extern "C" int wk_qk_norm_rope_bwd(const wk_rope_args* a, void* stream) {
  using namespace wk;
  RopeParams p;
  if (int bad = fill(a, true, p)) return bad;
  if (int unsupported = require_sm100()) return unsupported;
  const int sms = sm_count();
  if (sms <= 0) return WK_E_CUDA;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
      a->workspace_bytes < wk_qk_norm_rope_bwd_workspace_bytes(p.B, p.N, p.H, p.d))
    return WK_E_ARG;
  p.partial = static_cast<float*>(a->workspace);
  const int lanes = lanes_of(p.d);
  p.per_cta = tokens_per_cta(p.tokens, p.H, p.d, sms);
  const int ctas = bwd_ctas(p.tokens, p.per_cta, sms);
  const void* kernel = a->dtype == WK_BF16 ? backward_kernel<__nv_bfloat16>(lanes)
                       : a->dtype == WK_F16 ? backward_kernel<__half>(lanes)
                                            : backward_kernel<float>(lanes);
  const int tables = (p.per_cta * p.rot + 2 * p.d) * 4, sums = kThreads / 32 * p.d * 4;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int bad = launch_pdl(kernel, dim3(ctas), kThreads, tables > sums ? tables : sums, st, 1, {&p})) return bad;
  const float* partial = p.partial;
  int parts = ctas, d = p.d, w_dtype = p.w_dtype;
  void *dq = a->dq_weight, *dk = a->dk_weight;
  return launch_pdl(reinterpret_cast<const void*>(dweight_kernel), dim3((d + 31) / 32, p.x[1] ? 2 : 1), 1024, 0, st, 1,
                    {&partial, &parts, &d, &dq, &dk, &w_dtype});
}
