// Parts shared by the dense FP8 block-scaled product kernels.
//
// Rows, scales and residuals are read with plain loads, not through the read-only path
// (__ldg): under programmatic launch the kernel that writes them can still be running
// when this one has started, and that path is for memory that nobody writes while the
// kernel lives.
#pragma once

#include "common.cuh"
#include "dense.h"
#include "moe_gemm.cuh"
#include "moe_gemm_tok.cuh"
#include "ptx.cuh"

namespace b200moe {

// acc += sc * (this warp's 32 TMEM lanes x NC columns from taddr on), LB 16-column
// loads to a wait. Loads in flight behind the fmas, and releasing the buffer
// before the last fmas, measured 1-5% slower.
template <int NC, int LB>
__device__ __forceinline__ void promote(float (&acc)[NC], uint32_t taddr, float sc) {
#pragma unroll
  for (int c0 = 0; c0 < NC / 16; c0 += LB) {
    uint32_t v[LB][16];
#pragma unroll
    for (int b = 0; b < LB; ++b) tmem_ld16(taddr + (c0 + b) * 16, v[b]);
    tmem_wait_ld();
#pragma unroll
    for (int b = 0; b < LB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) tmem_reg_fence(v[b][i]);
#pragma unroll
    for (int b = 0; b < LB; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 2)
        ffma2(acc[(c0 + b) * 16 + i], acc[(c0 + b) * 16 + i + 1], __uint_as_float(v[b][i]),
              __uint_as_float(v[b][i + 1]), sc);
  }
}

// silu_f32 with a NaN kept (there d < 1e30 fails for it and gives -0).
__device__ __forceinline__ float silu_nan(float g) {
#if B200MOE_FAST_SILU
  const float d = 1.0f + __expf(-g);
  return d >= 1e30f ? -0.0f : __fdividef(g, d);
#else
  return silu_f32(g);
#endif
}

// silu(gate) * up of a token's NC / 2 (gate, up) pairs into acc[0 .. NC/2 - 1];
// returns their largest magnitude, NaN if one is. (A reciprocal shared by four values, for half the
// load of the special-function unit, needs a branch for large gates and measured 4-12%
// slower: 62 us to 70 for 5772 x 768 x 3584.)
template <int NC>
__device__ __forceinline__ float silu_pairs(float (&acc)[NC]) {
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < NC / 2; ++i) {
    acc[i] = silu_nan(acc[2 * i]) * acc[2 * i + 1];
    mx = max_nan(mx, fabsf(acc[i]));
  }
  return mx;
}

// acc[0 .. NC/2 - 1] quantised with `scale` to consecutive codes (16-byte aligned).
template <int NC>
__device__ __forceinline__ void store_codes(const float (&acc)[NC], float scale, uint8_t* q) {
  const CodeScale cs = code_scale(scale);
#pragma unroll
  for (int k = 0; k < NC / 32; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* v = acc + k * 16 + i * 4;
      w[i] = quant_e4m3x4<false>(v[0], v[1], v[2], v[3], cs);
    }
    reinterpret_cast<uint4*>(q)[k] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The residual (four bf16) of four consecutive outputs n.. of token m, where rows are
// vector aligned (p.vec).
__device__ __forceinline__ uint2 dense_residual4(const DenseParams& p, int64_t m, int n) {
  if (!p.residual || n >= p.N) return make_uint2(0, 0);
  return *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.residual) + m * p.ld_res + n);
}

// Four consecutive outputs n..n+3 of token m (p.vec); res: dense_residual4 of them.
__device__ __forceinline__ void dense_store4(const DenseParams& p, int64_t m, int n, float4 v, uint2 res) {
  if (n >= p.N) return;
  if (p.residual) {
    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&res.x));
    const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&res.y));
    v.x += lo.x;
    v.y += lo.y;
    v.z += hi.x;
    v.w += hi.y;
  }
  if (p.out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + m * p.ld_out + n) = v;
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    uint2 pk;
    pk.x = *reinterpret_cast<const uint32_t*>(&lo);
    pk.y = *reinterpret_cast<const uint32_t*>(&hi);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + m * p.ld_out + n) = pk;
  }
}

// Element (row r, column c) of 32 rows x 64 fp32 columns in shared memory, 16-byte
// pieces swizzled by row.
__device__ __forceinline__ float* staged(uint8_t* st, int r, int c) {
  return reinterpret_cast<float*>(st + r * 256 + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4);
}

// Columns n1 .. n1 + nc - 1 (nc <= 64) of staged rows m0 ..: whole aligned 16-byte
// pieces, and the elements before and behind them one by one.
template <bool F32>
__device__ __forceinline__ void store_staged(const DenseParams& p, int m0, int n1, int nc, int rows, uint8_t* st,
                                             int lane) {
  constexpr int ES = F32 ? 4 : 2, EP = 16 / ES, L = 64 / EP;  // bytes; elements and lanes: of a piece, of a row
  for (int r = lane / L; r < rows; r += 32 / L) {
    uint8_t* row = static_cast<uint8_t*>(p.out) + ((int64_t)(m0 + r) * p.ld_out + n1) * ES;
    const int ahead = (int)((0 - reinterpret_cast<uintptr_t>(row)) & 15) / ES;
    const int lead = ahead < nc ? ahead : nc, pieces = (nc - lead) / EP, tail = lead + pieces * EP;
    const int j = lane % L;
    if (j < pieces) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = lead + j * EP + i * (EP / 4);
        if (F32) {
          w[i] = __float_as_uint(*staged(st, r, c));
        } else {
          const __nv_bfloat162 v = __floats2bfloat162_rn(*staged(st, r, c), *staged(st, r, c + 1));
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      *reinterpret_cast<uint4*>(row + (lead + j * EP) * ES) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    for (int e = j; e < lead + nc - tail; e += L) {
      const int c = e < lead ? e : tail + e - lead;
      if (F32) reinterpret_cast<float*>(row)[c] = *staged(st, r, c);
      else reinterpret_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16_rn(*staged(st, r, c));
    }
  }
}

// Stores 32 rows (m0.., one per lane) x NC columns (n0..) of fp32 results where rows
// are not vector aligned (!p.vec), 64 columns at a time through st (8 KB of this
// warp). The residuals of all of them are asked for together: a load between stores,
// which may alias it, waits for the one before. (1349 x 1467 x 1024: 13.3 us, 15.6 with
// 32 columns of a row to a store of 2 bytes a lane; 9.5 for 1464 columns.)
template <int NC>
__device__ __forceinline__ void dense_store_tile(const DenseParams& p, int m0, int n0, const float (&acc)[NC],
                                                 uint8_t* st, int lane) {
  const int rows = p.M - m0 < 32 ? p.M - m0 : 32;
#pragma unroll
  for (int cb = 0; cb < NC / 64; ++cb) {
    const int n1 = n0 + cb * 64, nc = p.N - n1 < 64 ? p.N - n1 : 64;
    if (nc > 0) {  // warp-uniform
#pragma unroll
      for (int c = 0; c < 16; ++c)
        *reinterpret_cast<float4*>(staged(st, lane, 4 * c)) =
            make_float4(acc[cb * 64 + 4 * c], acc[cb * 64 + 4 * c + 1], acc[cb * 64 + 4 * c + 2],
                        acc[cb * 64 + 4 * c + 3]);
      __syncwarp();
      if (p.residual) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = h * 32 + lane;
          const __nv_bfloat16* src =
              static_cast<const __nv_bfloat16*>(p.residual) + (int64_t)m0 * p.ld_res + n1 + c;
          __nv_bfloat16 res[32];
#pragma unroll
          for (int r = 0; r < 32; ++r) res[r] = c < nc && r < rows ? src[r * p.ld_res] : __nv_bfloat16();
#pragma unroll
          for (int r = 0; r < 32; ++r)
            if (c < nc && r < rows) *staged(st, r, c) += __bfloat162float(res[r]);
        }
        __syncwarp();
      }
      if (p.out_f32) store_staged<true>(p, m0, n1, nc, rows, st, lane);
      else store_staged<false>(p, m0, n1, nc, rows, st, lane);
      __syncwarp();
    }
  }
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// A lane's columns 4 * lane .. of 128 -> columns lane, lane + 32, lane + 64, lane + 96.
__device__ __forceinline__ float4 spread_cols(float4 v, int lane) {
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int src = (lane >> 2) + 8 * i;
    const float x = __shfl_sync(0xffffffffu, v.x, src), y = __shfl_sync(0xffffffffu, v.y, src);
    const float z = __shfl_sync(0xffffffffu, v.z, src), w = __shfl_sync(0xffffffffu, v.w, src);
    o[i] = (lane & 2) ? ((lane & 1) ? w : z) : ((lane & 1) ? y : x);
  }
  return make_float4(o[0], o[1], o[2], o[3]);
}

// Rows that are not vector aligned: outputs n, n + 32, n + 64, n + 96 of token m,
// so that a store instruction of the warp covers 32 consecutive ones, and the
// residual of them (four bf16).
__device__ __forceinline__ uint2 dense_residual_cols(const DenseParams& p, int64_t m, int n) {
  if (!p.residual) return make_uint2(0, 0);
  const uint16_t* src = static_cast<const uint16_t*>(p.residual) + m * p.ld_res + n;
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = n + 32 * i < p.N ? src[32 * i] : 0;
  return make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
}
__device__ __forceinline__ void dense_store_cols(const DenseParams& p, int64_t m, int n, float4 v, uint2 res) {
  const float a[4] = {v.x, v.y, v.z, v.w};
  const uint32_t r[4] = {res.x << 16, res.x & 0xffff0000u, res.y << 16, res.y & 0xffff0000u};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + 32 * i < p.N) {
      float y = a[i];
      if (p.residual) y += __uint_as_float(r[i]);
      if (p.out_f32) static_cast<float*>(p.out)[m * p.ld_out + n + 32 * i] = y;
      else static_cast<__nv_bfloat16*>(p.out)[m * p.ld_out + n + 32 * i] = __float2bfloat16_rn(y);
    }
}

// One warp: the tokens first, first + step, .. < live of a tile (global token
// m0 + t) from the sums of the S <= MAXS CTAs of a cluster that share K, and their
// epilogue. at(t, s, h): cluster address of CTA s's sums of this lane's four
// columns (4 * lane ..) of token t, 128-column half h. Added in the order of s. B
// tokens at a time: their loads go out together, as each takes most of a
// microsecond (the shared expert on 200 tokens with a residual, 6144 x 2048: 41.1
// us with one token at a time, 35.1 like this).
// DENSE_SILU (HALVES = 2): the 256 columns are one 1x128 group of gate/up pairs,
// output columns 128 * (n0 / 256) ..; DENSE_OUT: columns n0 + 128 * h + 4 * lane ..
template <int EPI, int HALVES, int MAXS, int B, typename F>
__device__ __forceinline__ void finish_tokens_of(const DenseParams& p, int64_t m0, int n0, int splits, int lane,
                                                 int first, int step, int live, F at) {
  for (int t0 = first; t0 < live; t0 += B * step) {
    float4 v[B][HALVES][MAXS];
    uint2 res[B][HALVES];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int t = t0 + b * step;
      if (t < live) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
#pragma unroll
          for (int s = 0; s < MAXS; ++s)
            if (s < splits) v[b][h][s] = ld_cluster_f4(at(t, s, h));
          if (EPI == DENSE_OUT)
            res[b][h] = p.vec ? dense_residual4(p, m0 + t, n0 + 128 * h + lane * 4)
                              : dense_residual_cols(p, m0 + t, n0 + 128 * h + lane);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int t = t0 + b * step;
      if (t >= live) break;
      const int64_t m = m0 + t;
      float4 sum[HALVES];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        sum[h] = v[b][h][0];
#pragma unroll
        for (int s = 1; s < MAXS; ++s)
          if (s < splits) {
            sum[h].x += v[b][h][s].x;
            sum[h].y += v[b][h][s].y;
            sum[h].z += v[b][h][s].z;
            sum[h].w += v[b][h][s].w;
          }
      }
      if constexpr (EPI == DENSE_SILU) {
        static_assert(HALVES == 2, "a group of gate/up pairs is 256 columns");
        // lane: inter columns 2 * lane, 2 * lane + 1 of each 64-column half
        float y[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          y[2 * h] = silu_nan(sum[h].x) * sum[h].y;
          y[2 * h + 1] = silu_nan(sum[h].z) * sum[h].w;
        }
        float mx = max_nan(max_nan(fabsf(y[0]), fabsf(y[1])), max_nan(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float scale = group_scale_nan(mx);
        const CodeScale cs = code_scale(scale);
        const int unit = n0 >> 8;
        uint8_t* dst = p.q + m * p.ld_q + unit * 128 + lane * 2;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint16_t*>(dst + h * 64) = quant_e4m3x2<false>(y[2 * h], y[2 * h + 1], cs);
        if (lane == 0) p.s[m * p.ld_s + unit] = scale;
      } else {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          if (p.vec) dense_store4(p, m, n0 + 128 * h + lane * 4, sum[h], res[b][h]);
          else dense_store_cols(p, m, n0 + 128 * h + lane, spread_cols(sum[h], lane), res[b][h]);
        }
      }
    }
  }
}

template <int EPI, int HALVES, typename F>
__device__ __forceinline__ void finish_tokens(const DenseParams& p, int64_t m0, int n0, int splits, int lane, int first,
                                              int step, int live, F at) {
  if (splits <= 2) finish_tokens_of<EPI, HALVES, 2, 4>(p, m0, n0, splits, lane, first, step, live, at);
  else if (splits <= 4) finish_tokens_of<EPI, HALVES, 4, 2>(p, m0, n0, splits, lane, first, step, live, at);
  else finish_tokens_of<EPI, HALVES, 8, 1>(p, m0, n0, splits, lane, first, step, live, at);
}

}  // namespace b200moe
