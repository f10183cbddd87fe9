// Softmax of one row's scores as the kernels with 16-bit probabilities take them out of tensor memory: blocks of 32 keys in
// one thread.
#pragma once
#include "common.cuh"

namespace wk {

template <bool F16>
__device__ __forceinline__ uint32_t pack_16x2(float lo, float hi) {
  if (!F16) return pack_bf16x2(lo, hi);
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// One block of 32 keys of one row: P as 16 pairs of bf16 (or f16) and the sum of the unrounded values.
template <bool F16 = false>
__device__ __forceinline__ void softmax_block(const uint32_t (&sraw)[32], float beta, float bias, uint32_t (&w)[16],
                                              float& sum_exact) {
  const uint64_t beta2 = pack_f32x2(beta, beta), bias2 = pack_f32x2(bias, bias);
  uint64_t acc01 = 0, acc23 = 0;  // packed fp32 partial sums
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float p0, p1, p2, p3;
    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sraw[4 * i + 0]), __uint_as_float(sraw[4 * i + 1])), beta2, bias2),
                 p0, p1);
    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sraw[4 * i + 2]), __uint_as_float(sraw[4 * i + 3])), beta2, bias2),
                 p2, p3);
    p0 = ex2_approx(p0);
    p1 = ex2_approx(p1);
    p2 = ex2_approx(p2);
    p3 = ex2_approx(p3);
    acc01 = add_f32x2(acc01, pack_f32x2(p0, p1));
    acc23 = add_f32x2(acc23, pack_f32x2(p2, p3));
    w[2 * i] = pack_16x2<F16>(p0, p1);
    w[2 * i + 1] = pack_16x2<F16>(p2, p3);
  }
  {
    float a0, a1, a2, a3;
    unpack_f32x2(acc01, a0, a1);
    unpack_f32x2(acc23, a2, a3);
    sum_exact = (a0 + a1) + (a2 + a3);
  }
}

__device__ __forceinline__ float block_max(const uint32_t (&s)[32]) {
  float a0 = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  float a1 = fmaxf(__uint_as_float(s[2]), __uint_as_float(s[3]));
  float a2 = fmaxf(__uint_as_float(s[4]), __uint_as_float(s[5]));
  float a3 = fmaxf(__uint_as_float(s[6]), __uint_as_float(s[7]));
#pragma unroll
  for (int i = 8; i < 32; i += 8) {
    a0 = max3(a0, __uint_as_float(s[i + 0]), __uint_as_float(s[i + 1]));
    a1 = max3(a1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
    a2 = max3(a2, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
    a3 = max3(a3, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
  }
  return fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
}

}  // namespace wk
