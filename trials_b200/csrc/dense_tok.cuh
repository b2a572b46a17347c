// Dense FP8 block-scaled product, token-major (sm_100a):
//   y[m, n] = sum_kb xs[m, kb] * ws[n/128, kb] * sum_{k in kb} x[m, k] * w[n, k]
// The tensor core sums one 128-wide K block unscaled. The two f32 scales are not the power-of-two scales it could apply, so each block's
// partial is read back from TMEM, multiplied by xs * ws and added to an fp32
// accumulator in registers ("promotion").
//
// Tile: MMA M = 128 tokens (x), MMA N = 256 weight rows (w), one 128x256x32
// MMA per K step. An epilogue thread owns one token and 128 weight rows of one
// scale block, so its factor is one scalar per K block; gate/up pairs
// (interleaved rows 2j, 2j+1) meet in one thread.
// Warps: 0 TMA producer, 1 MMA issuer and TMEM owner, 4..11 epilogue (two
// warpgroups, which take over the first one's registers: 168 a thread at launch
// spilled the accumulators' neighbours).
// Rows past M and weight rows past N are zero-filled by TMA and not stored.
#pragma once

#include "common.cuh"
#include "dense.h"
#include "launch.h"
#include "moe_gemm_tok.cuh"
#include "ptx.cuh"

namespace b200moe {

struct DenseTokCfg {
  static constexpr int TM = 128;
  static constexpr int TN = 256;
  static constexpr int EW = 8;     // epilogue warps: 4 lane quarters x 2 column halves
  static constexpr int COLS = 128; // columns per epilogue thread
  static constexpr int THREADS = 128 + 32 * EW;
  // 384 threads x 168 registers at launch = 128 x (40 + 232 + 232).
  static constexpr int REGS_LOAD = 40, REGS_EPI = 232;
  static constexpr int X_BYTES = TM * 128;
  static constexpr int W_BYTES = TN * 128;
  static constexpr int TILE_BYTES = X_BYTES + W_BYTES;
  static constexpr int NBUF = 2;
  static constexpr int TMEM_COLS = 512;
  static constexpr int NSTAGE = 4;
  // DENSE_SILU: amax exchange, double-buffered by unit parity. DENSE_OUT: 32
  // rows x 32 columns of fp32 per epilogue warp on their way out.
  static constexpr int RED = 2 * 2 * TM * 4;
  static constexpr int STAGING = EW * 32 * 128;
  static constexpr int SMEM_BYTES = 1024 + NSTAGE * TILE_BYTES + (STAGING > RED ? STAGING : RED) + 256;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// Stores 32 rows (m0.., one per lane) x 128 columns (n0..) of fp32 results. They
// pass through st (4 KB of this warp, rows of 32 columns, 16-byte pieces
// swizzled by row), so that a store instruction covers whole 64-byte (bf16) or
// 128-byte (f32) runs of 4 rows, or 32 consecutive columns of one row where
// rows are not aligned.
__device__ __forceinline__ void dense_store_tile(const DenseParams& p, int m0, int n0, const float (&acc)[128],
                                                 uint8_t* st, int lane) {
  const int rows = p.M - m0 < 32 ? p.M - m0 : 32;
#pragma unroll
  for (int cb = 0; cb < 4; ++cb) {
    const int n1 = n0 + cb * 32;
    if (n1 < p.N) {  // warp-uniform
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<float4*>(st + lane * 128 + ((c ^ (lane & 7)) << 4)) =
            make_float4(acc[cb * 32 + 4 * c], acc[cb * 32 + 4 * c + 1], acc[cb * 32 + 4 * c + 2],
                        acc[cb * 32 + 4 * c + 3]);
      __syncwarp();
      if (p.vec) {  // N is a multiple of 8: a piece of 4 columns exists or does not
        const int c = lane & 7, n = n1 + 4 * c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3);
          if (r < rows && n < p.N) {
            float4 v = *reinterpret_cast<const float4*>(st + r * 128 + ((c ^ (r & 7)) << 4));
            const int64_t m = m0 + r;
            if (p.residual) {
              const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.residual) +
                                                                m * p.ld_res + n);
              const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
              const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
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
        }
      } else if (n1 + lane < p.N) {
        for (int r = 0; r < rows; ++r) {
          float v = *reinterpret_cast<const float*>(st + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
          const int64_t m = m0 + r;
          const int n = n1 + lane;
          if (p.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(p.residual)[m * p.ld_res + n]);
          if (p.out_f32) static_cast<float*>(p.out)[m * p.ld_out + n] = v;
          else static_cast<__nv_bfloat16*>(p.out)[m * p.ld_out + n] = __float2bfloat16_rn(v);
        }
      }
      __syncwarp();
    }
  }
}

template <int EPI>
__global__ void __launch_bounds__(DenseTokCfg::THREADS, 1)
    dense_tok_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const DenseParams p, int n_mt, int n_nt, int group) {
  using C = DenseTokCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tiles = smem;
  uint8_t* scratch = tiles + C::NSTAGE * C::TILE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(scratch + (EPI == DENSE_SILU ? C::RED : C::STAGING));
  uint64_t* empty = full + C::NSTAGE;
  uint64_t* tfull = empty + C::NSTAGE;
  uint64_t* tempty = tfull + C::NBUF;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + C::NBUF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int NKB = p.K >> 7;
  const int n_units = n_mt * n_nt;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NSTAGE; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < C::NBUF; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], C::EW);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();  // the kernel ahead of it wrote x (programmatic launch)
  griddep_launch_dependents();

  if (warp < 4) {
    regs_dec<C::REGS_LOAD>();
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        long issued = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < n_units && ok; u += gridDim.x) {
          int mt, nt;
          unit_coords(u, n_mt, n_nt, group, mt, nt);
          for (int kb = 0; kb < NKB; ++kb) {
            if (*abort_flag || !mbar_wait_bounded(&empty[stage], phase ^ 1, p.timeout_ns)) {
              ok = false;
              break;
            }
            uint8_t* tile = tiles + stage * C::TILE_BYTES;
            mbar_arrive_expect_tx(&full[stage], C::TILE_BYTES);
            tma_load_2d(tile, &tm_x, &full[stage], kb * 128, mt * C::TM);
            tma_load_2d(tile + C::X_BYTES, &tm_w, &full[stage], kb * 128, nt * C::TN);
            ++issued;
            if (++stage == C::NSTAGE) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
        if (!ok) {
          atomicOr(p.err, ERR_DEV_TIMEOUT);
          *abort_flag = 1;
          const long first = issued > C::NSTAGE ? issued - C::NSTAGE : 0;
          for (long g = first; g < issued; ++g)
            mbar_wait_bounded(&full[g % C::NSTAGE], (uint32_t)((g / C::NSTAGE) & 1), p.timeout_ns);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      if (lane == 0) {
        const uint32_t idesc = idesc_e4m3_f32(C::TM, C::TN);
        int stage = 0, buf = 0, last_buf = 0;
        uint32_t phase = 0, bphase = 0, last_bphase = 0;
        bool ok = true, any = false;
        for (int u = blockIdx.x; u < n_units && ok; u += gridDim.x) {
          for (int kb = 0; kb < NKB; ++kb) {
            if (*abort_flag || !mbar_wait_bounded(&tempty[buf], bphase ^ 1, p.timeout_ns) ||
                !mbar_wait_bounded(&full[stage], phase, p.timeout_ns)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t x_addr = smem_u32(tiles + stage * C::TILE_BYTES);
            const uint32_t w_addr = x_addr + C::X_BYTES;
            const uint32_t d = tmem_base + (uint32_t)(buf * C::TN);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma_f8(d, sdesc_kmajor_sw128(x_addr + ks * 32), sdesc_kmajor_sw128(w_addr + ks * 32), idesc,
                      ks > 0 ? 1u : 0u);
            umma_commit(&empty[stage]);
            umma_commit(&tfull[buf]);
            any = true;
            last_buf = buf;
            last_bphase = bphase;
            if (++stage == C::NSTAGE) {
              stage = 0;
              phase ^= 1;
            }
            if (++buf == C::NBUF) {
              buf = 0;
              bphase ^= 1;
            }
          }
        }
        if (!ok) {
          atomicOr(p.err, ERR_DEV_TIMEOUT);
          *abort_flag = 1;
        }
        // The tensor core must be done with TMEM before it is released.
        if (any) mbar_wait_bounded(&tfull[last_buf], last_bphase, p.timeout_ns);
      }
    }
  } else {
    regs_inc<C::REGS_EPI>();
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 4;
    const int q = warp & 3;       // TMEM lane quarter
    const int h = ew >> 2;        // column half = one weight scale block
    const int r = q * 32 + lane;  // token of the tile
    const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * C::COLS);
    int buf = 0, parity = 0;
    uint32_t bphase = 0;
    bool ok = true;
    // A warp whose wait gave up still walks all units (without waiting or
    // storing), so that the named barriers below keep their full count.
    for (int u = blockIdx.x; u < n_units; u += gridDim.x, parity ^= 1) {
      int mt, nt;
      unit_coords(u, n_mt, n_nt, group, mt, nt);
      const int64_t m = (int64_t)mt * C::TM + r;
      const int n0 = nt * C::TN + h * C::COLS;
      const bool live = mt * C::TM + q * 32 < p.M && n0 < p.N;  // warp-uniform
      const float* xsr = p.xs + (m < p.M ? m : p.M - 1) * p.ld_xs;
      const float* wsr = p.ws + (int64_t)(n0 < p.N ? (n0 >> 7) : 0) * NKB;
      float acc[C::COLS];
#pragma unroll
      for (int j = 0; j < C::COLS; ++j) acc[j] = 0.f;
      float sc_next = __ldg(xsr) * __ldg(wsr);
      for (int kb = 0; kb < NKB && ok; ++kb) {
        const float sc = sc_next;
        float xs_n = 0.f, ws_n = 0.f;
        if (kb + 1 < NKB) {
          xs_n = __ldg(xsr + kb + 1);
          ws_n = __ldg(wsr + kb + 1);
        }
        if (*abort_flag || !mbar_wait_bounded(&tfull[buf], bphase, p.timeout_ns)) {
          ok = false;
          atomicOr(p.err, ERR_DEV_TIMEOUT);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        if (live) {
          const uint32_t taddr = taddr0 + (uint32_t)(buf * C::TN);
#pragma unroll
          for (int c0 = 0; c0 < C::COLS / 16; c0 += 2) {
            uint32_t v[2][16];
            tmem_ld16(taddr + c0 * 16, v[0]);
            tmem_ld16(taddr + c0 * 16 + 16, v[1]);
            tmem_wait_ld();
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int i = 0; i < 16; ++i) tmem_reg_fence(v[b][i]);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                ffma2(acc[(c0 + b) * 16 + i], acc[(c0 + b) * 16 + i + 1], __uint_as_float(v[b][i]),
                      __uint_as_float(v[b][i + 1]), sc);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[buf]);
        if (++buf == C::NBUF) {
          buf = 0;
          bphase ^= 1;
        }
        sc_next = xs_n * ws_n;
      }
      if constexpr (EPI == DENSE_SILU) {
        // The thread's 64 (gate, up) pairs; the 1x128 group is both halves.
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          acc[i] = silu_f32(acc[2 * i]) * acc[2 * i + 1];
          mx = fmaxf(mx, fabsf(acc[i]));
        }
        float* rb = reinterpret_cast<float*>(scratch) + parity * 2 * C::TM;
        rb[h * C::TM + r] = mx;
        // One barrier per unit: the exchange buffer alternates, and a warp
        // reaches the write two units on only after every warp has passed the
        // next unit's barrier, so after it has read this one.
        named_bar_sync(1, C::EW * 32);
        const float scale = group_scale(fmaxf(rb[r], rb[C::TM + r]));
        if (ok && m < p.M) {
          uint4* dst = reinterpret_cast<uint4*>(p.q + m * p.ld_q + nt * 128 + h * 64);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i] = 0;
#pragma unroll
              for (int t = 0; t < 4; ++t)
                w[i] |= (uint32_t)quant_e4m3(acc[k * 16 + i * 4 + t], scale) << (8 * t);
            }
            dst[k] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (h == 0) p.s[m * p.ld_s + nt] = scale;
        }
      } else {
        if (ok && live) dense_store_tile(p, mt * C::TM + q * 32, n0, acc, scratch + ew * 4096, lane);
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

}  // namespace b200moe
