// Dense FP8 block-scaled product, token-major (sm_100a):
//   y[m, n] = sum_kb xs[m, kb] * ws[n/128, kb] * sum_{k in kb} x[m, k] * w[n, k]
// The tensor core sums one 128-wide K block unscaled. The two f32 scales are not
// the power-of-two scales it could apply, so each block's partial is read back
// from TMEM, multiplied by xs * ws and added to an fp32 accumulator in registers
// ("promotion").
//
// Tile: MMA M = 128 tokens (x), MMA N = TN = 256 or 128 weight rows (w), one MMA
// per K step. An epilogue thread owns one token and TN / 2 weight rows of one
// scale block, so its factor is one scalar per K block. A K block takes about 0.6
// us with TN = 256 and 0.44 with 128 whatever its surroundings: the hand-off of a
// partial (commit, wake-up, promotion, release) against the TMEM buffers bounds
// it, not the operands. So where tiles are fewer than SMs, a cluster of S CTAs
// shares a tile's K blocks; their fp32 sums meet in distributed shared memory,
// where CTA c finishes the tokens c, c + S, .. (added in CTA order: the result
// does not depend on timing). That exchange moves each CTA's sums once, 128 KB
// with TN = 256 in 2 to 4 us: TN = 128 halves it.
// Warps: 0 TMA producer, 1 MMA issuer and TMEM owner, 4..11 epilogue (two
// warpgroups, which take over the first one's registers: 168 a thread at launch
// spilled the accumulators' neighbours).
// Rows past M and weight rows past N are zero-filled by TMA and not stored.
// early_w: as in dense_split.cuh.
#pragma once

#include "dense_common.cuh"
#include "launch.h"

namespace b200moe {

template <int TN_>
struct DenseTokCfg {
  static constexpr int TM = 128;
  static constexpr int TN = TN_;
  static constexpr int EW = 8;          // epilogue warps: 4 lane quarters x 2 column halves
  static constexpr int COLS = TN / 2;   // columns per epilogue thread
  static constexpr int THREADS = 128 + 32 * EW;
  // 384 threads x 168 registers at launch = 128 x (40 + 232 + 232).
  static constexpr int REGS_LOAD = 40, REGS_EPI = 232;
  static constexpr int X_BYTES = TM * 128;
  static constexpr int W_BYTES = TN * 128;
  static constexpr int TILE_BYTES = X_BYTES + W_BYTES;
  static constexpr int TMEM_COLS = 512;
  static constexpr int NBUF = TMEM_COLS / TN;
  static constexpr int NSTAGE = 192 * 1024 / TILE_BYTES;
  static constexpr int SUM_BYTES = TM * TN * 4;  // a CTA's sums, in the tiles' place
  static constexpr int SMEM_BYTES = 1024 + NSTAGE * TILE_BYTES + 256;
  static_assert(SUM_BYTES <= NSTAGE * TILE_BYTES, "sums reuse the tiles");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

template <int EPI, int TN>
__global__ void __launch_bounds__(DenseTokCfg<TN>::THREADS, 1)
    dense_tok_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const DenseParams p, int splits, int n_mt, int n_nt, int group, int early_w) {
  using C = DenseTokCfg<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tiles = smem;
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + C::NSTAGE * C::TILE_BYTES);
  uint64_t* empty = full + C::NSTAGE;
  uint64_t* tfull = empty + C::NSTAGE;
  uint64_t* tempty = tfull + C::NBUF;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + C::NBUF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int NKB = p.K >> 7;
  const int rank = (int)cluster_ctarank();  // this CTA's share of K
  int mt, nt;
  unit_coords(blockIdx.x / splits, n_mt, n_nt, group, mt, nt);
  const int m0 = mt * C::TM, w0 = nt * TN;
  const int kb0 = (int)((int64_t)NKB * rank / splits);
  const int nkb = (int)((int64_t)NKB * (rank + 1) / splits) - kb0;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < 4) {
    regs_dec<C::REGS_LOAD>();
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        const int ahead = early_w ? (nkb < C::NSTAGE ? nkb : C::NSTAGE) : 0;
        for (int i = 0; i < ahead; ++i) {
          mbar_arrive_expect_tx(&full[i], C::TILE_BYTES);
          tma_load_2d(tiles + i * C::TILE_BYTES + C::X_BYTES, &tm_w, &full[i], (kb0 + i) * 128, w0);
        }
        griddep_wait();
        griddep_launch_dependents();
        for (int i = 0; i < ahead; ++i)
          tma_load_2d(tiles + i * C::TILE_BYTES, &tm_x, &full[i], (kb0 + i) * 128, m0);
        int stage = ahead == C::NSTAGE ? 0 : ahead;
        uint32_t phase = ahead == C::NSTAGE ? 1 : 0;
        int issued = ahead;
        bool ok = true;
        for (; issued < nkb; ++issued) {
          if (*abort_flag || !mbar_wait_bounded(&empty[stage], phase ^ 1, p.timeout_ns)) {
            ok = false;
            break;
          }
          uint8_t* tile = tiles + stage * C::TILE_BYTES;
          mbar_arrive_expect_tx(&full[stage], C::TILE_BYTES);
          tma_load_2d(tile, &tm_x, &full[stage], (kb0 + issued) * 128, m0);
          tma_load_2d(tile + C::X_BYTES, &tm_w, &full[stage], (kb0 + issued) * 128, w0);
          if (++stage == C::NSTAGE) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) {
          atomicOr(p.err, ERR_DEV_TIMEOUT);
          *abort_flag = 1;
          // Let every copy already issued land before the CTA exits.
          for (int g = issued > C::NSTAGE ? issued - C::NSTAGE : 0; g < issued; ++g)
            mbar_wait_bounded(&full[g % C::NSTAGE], (uint32_t)((g / C::NSTAGE) & 1), p.timeout_ns);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      if (lane == 0) {
        const uint32_t idesc = idesc_e4m3_f32(C::TM, C::TN);
        int stage = 0, buf = 0;
        uint32_t phase = 0, bphase = 0;
        int done = 0;
        for (; done < nkb; ++done) {
          if (*abort_flag || !mbar_wait_bounded(&tempty[buf], bphase ^ 1, p.timeout_ns) ||
              !mbar_wait_bounded(&full[stage], phase, p.timeout_ns)) {
            atomicOr(p.err, ERR_DEV_TIMEOUT);
            *abort_flag = 1;
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
          if (++stage == C::NSTAGE) {
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
    }
    __syncwarp();
    cluster_sync_all();
  } else {
    regs_inc<C::REGS_EPI>();
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 4;
    const int q = warp & 3;       // TMEM lane quarter
    const int h = ew >> 2;        // column half = one weight scale block
    const int r = q * 32 + lane;  // token of the tile
    const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * C::COLS);
    const int n0 = w0 + h * C::COLS;
    const bool live = m0 + q * 32 < p.M && n0 < p.N;  // warp-uniform
    griddep_wait();
    const float* xsr = p.xs + (int64_t)(m0 + r < p.M ? m0 + r : p.M - 1) * p.ld_xs + kb0;
    const float* wsr = p.ws + (int64_t)(n0 < p.N ? (n0 >> 7) : 0) * NKB + kb0;
    float acc[C::COLS];
#pragma unroll
    for (int j = 0; j < C::COLS; ++j) acc[j] = 0.f;
    int buf = 0;
    uint32_t bphase = 0;
    float sc_next = *xsr * *wsr;
    for (int kb = 0; kb < nkb; ++kb) {
      const float sc = sc_next;
      float xs_n = 0.f, ws_n = 0.f;
      if (kb + 1 < nkb) {
        xs_n = xsr[kb + 1];
        ws_n = wsr[kb + 1];
      }
      if (*abort_flag || !mbar_wait_bounded(&tfull[buf], bphase, p.timeout_ns)) {
        atomicOr(p.err, ERR_DEV_TIMEOUT);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      if (live) promote<C::COLS, 4>(acc, taddr0 + (uint32_t)(buf * C::TN), sc);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
      if (++buf == C::NBUF) {
        buf = 0;
        bphase ^= 1;
      }
      sc_next = xs_n * ws_n;
    }
    // The last partial is out of the tensor core, so the tiles are free: this
    // CTA's sums, rows of TN columns in 16-byte pieces swizzled by row.
    if (live) {
#pragma unroll
      for (int c = 0; c < C::COLS / 4; ++c)
        *reinterpret_cast<float4*>(tiles + r * (TN * 4) + (((h * (C::COLS / 4) + c) ^ (r & 7)) << 4)) =
            make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    }
    __syncwarp();
    cluster_sync_all();
    const uint32_t sums = smem_u32(tiles);
    const int rows = p.M - m0 < C::TM ? p.M - m0 : C::TM;
    finish_tokens<EPI, TN / 128>(
        p, m0, w0, splits, lane, rank + splits * ew, splits * C::EW, rows, [&](int t, int s, int hh) {
          return mapa_shared(sums + (uint32_t)(t * (TN * 4) + (((hh * 32 + lane) ^ (t & 7)) << 4)), s);
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
