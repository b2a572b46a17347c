// Shared definitions for the b200moe kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200moe.h"

namespace b200moe {

// Device error word bits (the word lives in caller memory).
constexpr int32_t ERR_DEV_BAD_EXPERT = B200MOE_DEVERR_BAD_EXPERT_ID;
constexpr int32_t ERR_DEV_TIMEOUT = B200MOE_DEVERR_TIMEOUT;
constexpr int32_t ERR_DEV_CAPACITY = B200MOE_DEVERR_CAPACITY;

// FP8 E4M3 quantisation of one value with a per-group fp32 scale, following
// the torch expression (x / s).clamp(-448, 448).to(float8_e4m3fn)
// (phase5_orchestrator.py:26-32): IEEE division, clamp, round-to-nearest-even.
__device__ __forceinline__ uint8_t quant_e4m3(float x, float scale) {
  float v = __fdiv_rn(x, scale);
  v = fminf(fmaxf(v, -448.0f), 448.0f);
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3));
}

// The same bits with the division replaced by a product and two fmas on two values
// at a time, for callers that quantise many values with one scale. By Markstein's
// theorem q + (x - q * scale) * rcp is the correctly rounded quotient when rcp is the
// correctly rounded reciprocal, q is within an ulp and nothing underflows: scale is at
// least 1e-12, so where the remainder could underflow (x below 2^-102) the quotient is
// far below the smallest code and rounds to zero either way. It is computed negated,
// qn = -q with nrcp = -rcp, which gives a zero the quotient's sign, and the codes'
// signs are turned over. An infinite scale (nrcp = -0, its place taken by 0) gives
// x * 0 as the division does. The conversion saturates at 448 by itself and gives NaN its
// own code; CLAMP: NaN becomes -448. 8,192 x 6,144 bf16 values quantised 1x128:
// 47.7 us with the division, 39.4 with scalar fmas, sign and range put right for each
// value, 32.1 like this.
struct CodeScale {
  float nrcp, scale;
};
__device__ __forceinline__ CodeScale code_scale(float scale) {
  return CodeScale{-__frcp_rn(scale), scale < INFINITY ? scale : 0.0f};
}
// Negated codes of two values, the first in the low byte.
template <bool CLAMP>
__device__ __forceinline__ uint32_t negated_codes(float x0, float x1, CodeScale c) {
  uint64_t x, s, n, q, r;
  float q0, q1;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(x0), "f"(x1));
  asm("mov.b64 %0, {%1, %1};" : "=l"(s) : "f"(c.scale));
  asm("mov.b64 %0, {%1, %1};" : "=l"(n) : "f"(c.nrcp));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(x), "l"(n));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q), "l"(s), "l"(x));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(q) : "l"(r), "l"(n));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(q0), "=f"(q1) : "l"(q));
  if (CLAMP) {
    q0 = fminf(q0, 448.0f);
    q1 = fminf(q1, 448.0f);
  }
  return __nv_cvt_float2_to_fp8x2(make_float2(q0, q1), __NV_SATFINITE, __NV_E4M3);
}
template <bool CLAMP>
__device__ __forceinline__ uint16_t quant_e4m3x2(float x0, float x1, CodeScale c) {
  return (uint16_t)(negated_codes<CLAMP>(x0, x1, c) ^ 0x8080u);
}
template <bool CLAMP>
__device__ __forceinline__ uint32_t quant_e4m3x4(float x0, float x1, float x2, float x3, CodeScale c) {
  return (negated_codes<CLAMP>(x0, x1, c) | negated_codes<CLAMP>(x2, x3, c) << 16) ^ 0x80808080u;
}

// Group scale: max(amax / 448, 1e-12) in fp32 (phase5_orchestrator.py:29-30).
__device__ __forceinline__ float group_scale(float amax) { return fmaxf(__fdiv_rn(amax, 448.0f), 1e-12f); }

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The same scale where a NaN among the magnitudes has to reach it, as it does through
// torch's amax and clamp: with an unclamped code_scale conversion all codes of the group
// become NaN, and an infinity (scale infinite) leaves zeros and NaN in its own place.
__device__ __forceinline__ float group_scale_nan(float amax) { return max_nan(__fdiv_rn(amax, 448.0f), 1e-12f); }

// Work-unit order of the grouped GEMMs. A unit is (chunk, weight tile nt).
// Chunks are taken in groups of `group` consecutive chunks, and inside a group
// weight-tile-major: (c0, 0), (c1, 0), ..., (c0, 1), (c1, 1), ... CTAs running
// at the same time then share the weight tile of an expert that has several
// chunks (one HBM read, the rest from L2) and reuse the group's activation rows
// from L2. group = 1 is plain chunk-major order. A bijection of
// [0, n_chunks * NT) for every group >= 1.
__device__ __forceinline__ void unit_coords(int u, int n_chunks, int NT, int group, int& chunk, int& nt) {
  const int span = group * NT;
  const int g = u / span;
  const int r = u - g * span;
  const int first = g * group;
  const int gc = n_chunks - first < group ? n_chunks - first : group;
  nt = r / gc;
  chunk = first + (r - nt * gc);
}

}  // namespace b200moe
