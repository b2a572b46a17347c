// Dense FP8 block-scaled product for few tokens (sm_100a): the time is that of
// streaming the weights once, so the work is split over every SM.
//   y[m, n] = sum_kb xs[m, kb] * ws[n/128, kb] * sum_{k in kb} x[m, k] * w[n, k]
//
// One CTA takes 128 weight rows (MMA M), a tile of `tt` <= T tokens (MMA N) and a
// share of the K blocks; a cluster of S CTAs covers K (DENSE_SILU: 2 x S, the two
// 128-row halves of one 1x128 group of gate/up pairs). Each K block's partial
// goes to a fresh TMEM buffer and is promoted with xs * ws into fp32 registers,
// as in dense_tok.cuh (here the factor changes along a thread's columns, so it
// comes from shared memory in pairs for the packed fma). The CTAs' fp32 sums
// then meet in distributed shared memory: token t is finished by one warp of CTA
// t % R, which adds the S sums in split order (the result does not depend on
// timing) and stores 128 consecutive outputs, or quantises the token's 128
// silu(gate) * up values.
//
// QX: x comes in bf16 and every CTA quantises its K blocks of it itself (the
// arithmetic of b200moe_quant_1x128, NaN kept), straight into the swizzled operand tiles:
// for a few tokens that is cheaper than a launch.
//
// With `early_w` the kernel ahead of it in the stream is one of this call's own
// (it writes x, never w, and starts this one only after everything before it is
// complete), so the weight tiles are requested before waiting for it.
// Warps: 0 TMA producer, 1 MMA issuer and TMEM owner, 2.. epilogue (4 TMEM lane
// quarters x CG column groups).
#pragma once

#include "common.cuh"
#include "dense_common.cuh"
#include "launch.h"

namespace b200moe {

// Most (token, K block) groups a CTA quantises itself (QX): up to 48 it is faster than the
// launch that quantises every row once (us inside a graph, here and with the launch: one
// token of 6144 x 2048 6.5 and 8.0; 36 and 48 groups, 3 and 4 tokens of 4096 x 6144, 10.2
// and 10.7, 10.5 and 10.7; 32, 8 of 4096 x 2048, 6.8 and 7.3; 48, 12 of 6144 x 2048, 8.0
// and 8.2; 32, 16 of 1024 x 2048, 5.1 and 5.9; gate/up, 36, 3 of 6144 x 2048 10.7 and 11.3;
// an eager call of 4 x 4096 x 6144 10.2 and 14.2). At 64 (16 of 6144 x 2048) it was 9.8
// against 8.4.
constexpr int kQuantGroups = 48;

template <int T_>
struct DenseSplitCfg {
  static constexpr int T = T_;                      // most tokens of a tile
  static constexpr int CG = T <= 32 ? 1 : 2;        // column groups of the epilogue
  static constexpr int TC = T / CG;                 // columns per epilogue thread
  static constexpr int EW = 4 * CG;
  static constexpr int THREADS = 64 + 32 * EW;
  static constexpr int TMEM_COLS = 256;             // half of it: two CTAs share an SM
  static constexpr int NBUF = TMEM_COLS / T > 8 ? 8 : TMEM_COLS / T;
  static_assert(T == 16 || T == 32 || T == 64, "tokens per tile");
  static constexpr int W_BYTES = 128 * 128;
  static constexpr int MAX_STAGE = 12;
  static constexpr int BAR_BYTES = (2 * MAX_STAGE + 2 * NBUF + 1) * 8 + 16;
  static constexpr int tile_bytes(int tt, bool qx) { return W_BYTES + (qx ? 0 : tt * 128); }
  // Shared memory of nstage stages and nkb K blocks a CTA.
  static int smem_bytes(int nstage, int nkb, int tt, bool qx) {
    return 1024 + nstage * tile_bytes(tt, qx) + (qx ? nkb * tt * 128 : 0) + nkb * tt * 4 + BAR_BYTES;
  }
};

// (d0, d1) += (a0, a1) * (s0, s1), each an IEEE fma; s: two floats of shared memory.
__device__ __forceinline__ void ffma2_pair(float& d0, float& d1, uint32_t a0, uint32_t a1, uint64_t s) {
  uint64_t rd, ra;
  asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "r"(a0), "r"(a1));
  asm("mov.b64 %0, {%1, %2};" : "=l"(rd) : "f"(d0), "f"(d1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(rd) : "l"(ra), "l"(s));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d0), "=f"(d1) : "l"(rd));
}

template <int EPI, int T, bool QX>
__global__ void __launch_bounds__(DenseSplitCfg<T>::THREADS, 2)
    dense_split_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                       const DenseParams p, int splits, int tt, int nstage, int early_w) {
  using C = DenseSplitCfg<T>;
  constexpr int HALVES = EPI == DENSE_SILU ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int NKB = p.K >> 7;
  const int R = HALVES * splits;
  const int rank = (int)cluster_ctarank();
  const int half = rank % HALVES, split = rank / HALVES;
  const int unit = blockIdx.x / R;
  const int row0 = (unit * HALVES + half) * 128;  // first weight row
  const int t0 = blockIdx.y * tt;
  const int live = p.M - t0 < tt ? p.M - t0 : tt;  // tokens of this tile
  const int kb0 = (int)((int64_t)NKB * split / splits);
  const int nkb = (int)((int64_t)NKB * (split + 1) / splits) - kb0;
  const int nkb_max = (NKB + splits - 1) / splits;
  const int tile_bytes = C::tile_bytes(tt, QX);

  uint8_t* tiles = smem;
  uint8_t* xq = tiles + nstage * tile_bytes;  // QX: [nkb][tt][128] operand tiles
  float* sx = reinterpret_cast<float*>(xq + (QX ? nkb_max * tt * 128 : 0));  // [nkb][tt]: xs * ws
  uint64_t* full = reinterpret_cast<uint64_t*>(sx + nkb_max * tt);
  uint64_t* empty = full + C::MAX_STAGE;
  uint64_t* tfull = empty + C::MAX_STAGE;
  uint64_t* tempty = tfull + C::NBUF;
  uint64_t* xfull = tempty + C::NBUF;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(xfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_w);
    if (!QX) prefetch_tmap(&tm_x);
    for (int s = 0; s < nstage; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < C::NBUF; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], C::EW);
    }
    mbar_init(xfull, C::EW);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const int ahead = early_w ? (nkb < nstage ? nkb : nstage) : 0;
      for (int i = 0; i < ahead; ++i) {
        mbar_arrive_expect_tx(&full[i], tile_bytes);
        tma_load_2d(tiles + i * tile_bytes, &tm_w, &full[i], (kb0 + i) * 128, row0);
      }
      griddep_wait();
      griddep_launch_dependents();
      if (!QX)
        for (int i = 0; i < ahead; ++i)
          tma_load_2d(tiles + i * tile_bytes + C::W_BYTES, &tm_x, &full[i], (kb0 + i) * 128, t0);
      int stage = ahead == nstage ? 0 : ahead;
      uint32_t phase = ahead == nstage ? 1 : 0;
      int issued = ahead;
      bool ok = true;
      for (; issued < nkb; ++issued) {
        if (*abort_flag || !mbar_wait_bounded(&empty[stage], phase ^ 1, p.timeout_ns)) {
          ok = false;
          break;
        }
        uint8_t* tile = tiles + stage * tile_bytes;
        mbar_arrive_expect_tx(&full[stage], tile_bytes);
        tma_load_2d(tile, &tm_w, &full[stage], (kb0 + issued) * 128, row0);
        if (!QX) tma_load_2d(tile + C::W_BYTES, &tm_x, &full[stage], (kb0 + issued) * 128, t0);
        if (++stage == nstage) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) {
        atomicOr(p.err, ERR_DEV_TIMEOUT);
        *abort_flag = 1;
        // Let every copy already issued land before the CTA exits.
        for (int g = issued > nstage ? issued - nstage : 0; g < issued; ++g)
          mbar_wait_bounded(&full[g % nstage], (uint32_t)((g / nstage) & 1), p.timeout_ns);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc = idesc_e4m3_f32(128, tt);
      int stage = 0, buf = 0;
      uint32_t phase = 0, bphase = 0;
      int done = 0;
      const bool go = !QX || mbar_wait_bounded(xfull, 0, p.timeout_ns);
      for (; done < nkb; ++done) {
        if (!go || *abort_flag || !mbar_wait_bounded(&tempty[buf], bphase ^ 1, p.timeout_ns) ||
            !mbar_wait_bounded(&full[stage], phase, p.timeout_ns)) {
          atomicOr(p.err, ERR_DEV_TIMEOUT);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t w_addr = smem_u32(tiles + stage * tile_bytes);
        const uint32_t x_addr = QX ? smem_u32(xq + done * tt * 128) : w_addr + C::W_BYTES;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_f8(tmem_base + (uint32_t)(buf * T), sdesc_kmajor_sw128(w_addr + ks * 32),
                  sdesc_kmajor_sw128(x_addr + ks * 32), idesc, ks > 0 ? 1u : 0u);
        umma_commit(&empty[stage]);
        umma_commit(&tfull[buf]);
        if (++stage == nstage) {
          stage = 0;
          phase ^= 1;
        }
        if (++buf == C::NBUF) {
          buf = 0;
          bphase ^= 1;
        }
      }
      // The tensor core must be done with TMEM before it is released.
      if (done > 0)
        mbar_wait_bounded(&tfull[(done - 1) % C::NBUF], (uint32_t)(((done - 1) / C::NBUF) & 1), p.timeout_ns);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lane quarter
    const int tid = threadIdx.x - 64;
    // This warp's columns: the tile's 16-column groups split over the column groups.
    const int groups = tt >> 4;
    const int per = (groups + C::CG - 1) / C::CG;
    const int col0 = ((warp - 2) >> 2) * per * 16;
    const int cols = live - col0;  // live columns from col0 on (may be <= 0)
    griddep_wait();
    const float* wsr = p.ws + (int64_t)(row0 < p.N ? (row0 >> 7) : 0) * NKB + kb0;
    if (QX) {
      // One half-warp per (token, K block): 16 lanes x 8 columns. The plan sees to
      // at most kQuantGroups of them a CTA, so all loads go out first.
      constexpr int U = kQuantGroups / (C::EW * 2);
      const int hw = tid >> 4, sub = tid & 15;
      const int total = live * nkb;
      uint4 raw[U];
      float wv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int g = u * C::EW * 2 + hw;
        const int t = g / nkb, kb = g - t * nkb;
        raw[u] = make_uint4(0, 0, 0, 0);
        wv[u] = g < total ? wsr[kb] : 0.f;
        if (g < total)
          raw[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.xb) +
                                                   (int64_t)(t0 + t) * p.ld_xb + (kb0 + kb) * 128 + sub * 8);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u * C::EW * 2 + (hw & ~1) >= total) break;  // warp-uniform
        const int g = u * C::EW * 2 + hw;
        const int t = g / nkb, kb = g - t * nkb;
        const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&raw[u]);
        float v[8];
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __bfloat1622float2(h2[i]);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
          mx = max_nan(mx, max_nan(fabsf(f.x), fabsf(f.y)));
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float scale = group_scale_nan(mx);
        const CodeScale cs = code_scale(scale);
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = quant_e4m3x4<false>(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], cs);
        if (g < total) {
          *reinterpret_cast<uint2*>(xq + kb * tt * 128 + t * 128 + (((sub >> 1) ^ (t & 7)) << 4) + (sub & 1) * 8) =
              make_uint2(w[0], w[1]);
          if (sub == 0) sx[kb * tt + t] = scale * wv[u];
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(xfull);
    } else {
      // Consecutive threads: consecutive K blocks of one token; the loads of eight products
      // go out together, as none passes a store that may alias it.
      constexpr int U = 8, STEP = C::EW * 32;
      // tid / nkb and STEP / nkb: (n + 0.5) / nkb is 0.5 / nkb away from every integer, far
      // more than the rounding of so small a number.
      const float inv = __fdividef(1.0f, (float)nkb);
      const int dt = (int)(((float)STEP + 0.5f) * inv), dk = STEP - dt * nkb;
      int t = (int)(((float)tid + 0.5f) * inv), kb = tid - t * nkb;
      for (int i0 = 0; i0 < nkb * live; i0 += U * STEP) {
        float a[U], b[U];
        int at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          at[u] = -1;
          if (i0 + u * STEP < nkb * live) {  // uniform
            if (t < live) {
              at[u] = kb * tt + t;
              a[u] = p.xs[(int64_t)(t0 + t) * p.ld_xs + kb0 + kb];
              b[u] = wsr[kb];
            }
            t += dt;
            kb += dk;
            if (kb >= nkb) {
              kb -= nkb;
              ++t;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at[u] >= 0) sx[at[u]] = a[u] * b[u];
      }
    }
    named_bar_sync(1, C::EW * 32);
    float acc[C::TC];
#pragma unroll
    for (int j = 0; j < C::TC; ++j) acc[j] = 0.f;
    int buf = 0;
    uint32_t bphase = 0;
    for (int kb = 0; kb < nkb; ++kb) {
      if (*abort_flag || !mbar_wait_bounded(&tfull[buf], bphase, p.timeout_ns)) {
        atomicOr(p.err, ERR_DEV_TIMEOUT);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * T + col0);
      const float* ss = sx + kb * tt + col0;
      constexpr int LB = C::TC >= 32 ? 2 : 1;  // 16-column loads per wait
#pragma unroll
      for (int c = 0; c < C::TC / 16; c += LB) {
        if (c * 16 < cols && c < per) {  // warp-uniform
          uint32_t v[LB][16];
#pragma unroll
          for (int b = 0; b < LB; ++b)
            if ((c + b) * 16 < cols && c + b < per) tmem_ld16(taddr + (c + b) * 16, v[b]);
          tmem_wait_ld();
#pragma unroll
          for (int b = 0; b < LB; ++b)
            if ((c + b) * 16 < cols && c + b < per) {
#pragma unroll
              for (int i = 0; i < 16; ++i) tmem_reg_fence(v[b][i]);
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(ss + (c + b) * 16 + i);
                float* a = acc + (c + b) * 16 + i;
                ffma2_pair(a[0], a[1], v[b][i], v[b][i + 1], s4.x);
                ffma2_pair(a[2], a[3], v[b][i + 2], v[b][i + 3], s4.y);
              }
            }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
      if (++buf == C::NBUF) {
        buf = 0;
        bphase ^= 1;
      }
    }
    // The last partial is out of the tensor core, so the tiles are free: this
    // CTA's sums, [token][weight row].
    float* part = reinterpret_cast<float*>(tiles);
#pragma unroll
    for (int j = 0; j < C::TC; ++j)
      if (j < cols && j < per * 16) part[(col0 + j) * 128 + q * 32 + lane] = acc[j];
  }

  __syncwarp();
  cluster_sync_all();
  if (warp >= 2) {
    const uint32_t part = smem_u32(tiles);
    finish_tokens<EPI, HALVES>(p, t0, unit * HALVES * 128, splits, lane, rank + R * (warp - 2), R * C::EW, live,
                               [&](int t, int s, int h) {
                                 return mapa_shared(part + (uint32_t)((t * 128 + lane * 4) * 4), s * HALVES + h);
                               });
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while another reads its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

}  // namespace b200moe
