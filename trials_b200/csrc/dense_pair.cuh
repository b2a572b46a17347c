// Dense FP8 block-scaled product on CTA pairs (tcgen05 cta_group::2), for many
// tokens: persistent, the mathematics of dense_tok.cuh.
//
// A pair computes 256 tokens x 256 weight rows with one MMA over both SMs: each
// CTA holds 128 tokens and 128 of the weight rows (32 KB per K block instead of
// the 48 KB of a one-CTA 128x256 tile) and gets its own 128 tokens x 256 columns
// of the result in TMEM.
//
// Synchronisation: both CTAs' loads complete on the leader's `full` barrier (no
// multicast); the leader's MMA thread commits to `empty` / `tfull` of both CTAs;
// both CTAs' epilogue warps release a TMEM buffer on the leader's `tempty`.
// Warps: 0 TMA producer, 1 MMA issuer (leader) and TMEM owner, 4..11 epilogue.
//
// The promotion of partials is what a K block waits for, so the epilogue warps leave
// the output to TMA: they put a tile's rounded results into swizzled staging and go on
// with the next tile; its residual was brought there the same way while its K blocks
// were multiplied. Plain stores by the same warps took 4 us a tile and a residual read
// beside them 12 more, one latency after another: 5772 x 7424 x 768 took 82.5 us and 202
// with a residual, like this 49 and 63; 2048 x 6144 x 2048 41.8 and 78.1, now 34 and
// 38; 8192 x 6144 x 6144 323 and 458, now 321 and 332. Five stages carry this as well as
// six with half the staging, stored in two steps (52 and 61 to 54 and 65).
#pragma once

#include "dense_common.cuh"
#include "launch.h"

namespace b200moe {

template <int EPI>
struct DensePairCfg {
  static constexpr int TM = 128;   // tokens per CTA
  static constexpr int TN = 256;   // weight rows per pair
  static constexpr int WR = 128;   // weight rows per CTA
  static constexpr int EW = 8;     // 16 (64 columns a thread) measured 40% slower
  static constexpr int COLS = 128; // columns per epilogue thread
  static constexpr int THREADS = 128 + 32 * EW;
  static constexpr int REGS_LOAD = 40, REGS_EPI = 232;  // as DenseTokCfg
  static constexpr int X_BYTES = TM * 128;
  static constexpr int W_BYTES = WR * 128;
  static constexpr int TILE_BYTES = X_BYTES + W_BYTES;
  static constexpr int NBUF = 2;
  static constexpr int TMEM_COLS = 512;
  static constexpr int NSTAGE = EPI == DENSE_SILU ? 6 : 5;
  static constexpr int STAGING = 32 * COLS * 2;  // of a warp: its 32 x 128 results in bf16
  // DENSE_SILU: two buffers of row maxima; DENSE_OUT: staging.
  static constexpr int SCRATCH = EPI == DENSE_SILU ? 2 * 2 * TM * 4 : EW * STAGING;
  static constexpr int SMEM_BYTES = 1024 + NSTAGE * TILE_BYTES + SCRATCH + 256;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// The epilogue of a warp's 32 tokens (m0 ..) x 128 columns (n0 ..) of DENSE_OUT. tm_o:
// boxes of 32 rows x 128 bytes of the output; st: 8 KB in swizzled rows of 128 bytes,
// holding the residual in two boxes of 64 columns (if any) and then the results.
__device__ __forceinline__ void pair_store_tile(const DenseParams& p, const CUtensorMap& tm_o, int m0, int n0,
                                                float (&acc)[128], uint8_t* st, int lane) {
  uint8_t* row = st + lane * 128;
  const int sw = lane & 7;
  if (p.residual) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint4 raw = *reinterpret_cast<const uint4*>(row + (j >> 3) * 4096 + (((j & 7) ^ sw) << 4));
      const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v[e]));
        acc[j * 8 + 2 * e] += f.x;
        acc[j * 8 + 2 * e + 1] += f.y;
      }
    }
  } else {
    if (lane == 0) bulk_wait_read_all();  // the tile before has left the staging
  }
  __syncwarp();
  if (p.out_f32) {
    // Four boxes of 32 columns, two at a time.
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half) {
        if (lane == 0) bulk_wait_read_all();
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float* a = acc + half * 64 + j * 4;
        *reinterpret_cast<float4*>(row + (j >> 3) * 4096 + (((j & 7) ^ sw) << 4)) = make_float4(a[0], a[1], a[2], a[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        for (int b = 0; b < 2; ++b)
          if (n0 + half * 64 + b * 32 < p.N) tma_store_2d(&tm_o, st + b * 4096, n0 + half * 64 + b * 32, m0);
        bulk_commit_group();
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 c = __floats2bfloat162_rn(acc[j * 8 + 2 * e], acc[j * 8 + 2 * e + 1]);
        v[e] = *reinterpret_cast<const uint32_t*>(&c);
      }
      *reinterpret_cast<uint4*>(row + (j >> 3) * 4096 + (((j & 7) ^ sw) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      for (int b = 0; b < 2; ++b)
        if (n0 + b * 64 < p.N) tma_store_2d(&tm_o, st + b * 4096, n0 + b * 64, m0);
      bulk_commit_group();
    }
  }
}

// tm_o, tm_r (DENSE_OUT with p.vec): the output and, if any, the residual.
template <int EPI>
__global__ void __launch_bounds__(DensePairCfg<EPI>::THREADS, 1)
    dense_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ CUtensorMap tm_r,
                      const DenseParams p, int n_mt, int n_nt, int group) {
  using C = DensePairCfg<EPI>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tiles = smem;
  uint8_t* scratch = tiles + C::NSTAGE * C::TILE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(scratch + C::SCRATCH);
  uint64_t* empty = full + C::NSTAGE;
  uint64_t* tfull = empty + C::NSTAGE;
  uint64_t* tempty = tfull + C::NBUF;
  uint64_t* res_full = tempty + C::NBUF;  // of each epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + C::EW);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();  // 0 = leader
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int NKB = p.K >> 7;
  const int n_units = n_mt * n_nt;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NSTAGE; ++s) {
      mbar_init(&full[s], 1);   // leader: its producer's arrive; the bytes of both CTAs
      mbar_init(&empty[s], 1);  // the pair MMA's commit
    }
    for (int b = 0; b < C::NBUF; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * C::EW);  // leader: the epilogue warps of both CTAs
    }
    for (int e = 0; e < C::EW; ++e) mbar_init(&res_full[e], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    if (EPI == DENSE_OUT && p.vec) prefetch_tmap(&tm_o);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers initialised and TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();  // the kernel ahead of it wrote x (programmatic launch)
  griddep_launch_dependents();

  if (warp < 4) {
    regs_dec<C::REGS_LOAD>();
    if (warp == 0) {
      // ------------------------------------------------------------ producer (both CTAs)
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        long issued = 0;
        bool ok = true;
        for (int u = pair; u < n_units && ok; u += n_pairs) {
          int mt, nt;
          unit_coords(u, n_mt, n_nt, group, mt, nt);
          const int m0 = (mt * 2 + rank) * C::TM, w0 = nt * C::TN + rank * C::WR;
          for (int kb = 0; kb < NKB; ++kb) {
            if (*abort_flag || !mbar_wait_bounded(&empty[stage], phase ^ 1, p.timeout_ns)) {
              ok = false;
              break;
            }
            uint8_t* tile = tiles + stage * C::TILE_BYTES;
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::TILE_BYTES);
            const uint32_t leader_full = mapa_shared(smem_u32(&full[stage]), 0);
            tma_load_2d_pair(tile, &tm_x, leader_full, kb * 128, m0);
            tma_load_2d_pair(tile + C::X_BYTES, &tm_w, leader_full, kb * 128, w0);
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
          // Both CTAs' copies complete on the leader's barriers; the cluster
          // barrier at the end holds the other CTA until this wait is over.
          if (rank == 0) {
            const long first = issued > C::NSTAGE ? issued - C::NSTAGE : 0;
            for (long g = first; g < issued; ++g)
              mbar_wait_bounded(&full[g % C::NSTAGE], (uint32_t)((g / C::NSTAGE) & 1), p.timeout_ns);
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ pair MMA issuer (leader)
      if (lane == 0 && rank == 0) {
        const uint32_t idesc = idesc_e4m3_f32(2 * C::TM, C::TN);
        int stage = 0, buf = 0, last_buf = 0;
        uint32_t phase = 0, bphase = 0, last_bphase = 0;
        bool ok = true, any = false;
        for (int u = pair; u < n_units && ok; u += n_pairs) {
          for (int kb = 0; kb < NKB; ++kb) {
            if (*abort_flag || !mbar_wait_cluster_bounded(&tempty[buf], bphase ^ 1, p.timeout_ns) ||
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
              umma_f8_pair(d, sdesc_kmajor_sw128(x_addr + ks * 32), sdesc_kmajor_sw128(w_addr + ks * 32), idesc,
                           ks > 0 ? 1u : 0u);
            umma_commit_pair(&empty[stage], 0x3);
            umma_commit_pair(&tfull[buf], 0x3);
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
        // The tensor cores must be done with TMEM before it is released.
        if (any) mbar_wait_bounded(&tfull[last_buf], last_bphase, p.timeout_ns);
      }
    }
  } else {
    regs_inc<C::REGS_EPI>();
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int ew = warp - 4;
    const int q = warp & 3;       // TMEM lane quarter
    const int h = ew >> 2;        // column half = one weight scale block
    const int r = q * 32 + lane;  // token of this CTA's half tile
    const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * C::COLS);
    int buf = 0, parity = 0;
    uint32_t bphase = 0, rphase = 0;
    bool ok = true;
    uint8_t* st = scratch + ew * C::STAGING;
    const bool residual = EPI == DENSE_OUT && p.vec && p.residual;
    // A warp whose wait gave up still walks all tiles (without waiting or
    // storing), so that the named barriers below keep their full count.
    for (int u = pair; u < n_units; u += n_pairs) {
      int mt, nt;
      unit_coords(u, n_mt, n_nt, group, mt, nt);
      const int m0 = (mt * 2 + rank) * C::TM;
      const int64_t m = (int64_t)m0 + r;
      const int n0 = nt * C::TN + h * C::COLS;
      const bool live = m0 + q * 32 < p.M && n0 < p.N;  // warp-uniform
      const float* xsr = p.xs + (m < p.M ? m : p.M - 1) * p.ld_xs;
      const float* wsr = p.ws + (int64_t)(n0 < p.N ? (n0 >> 7) : 0) * NKB;
      float acc[C::COLS];
#pragma unroll
      for (int j = 0; j < C::COLS; ++j) acc[j] = 0.f;
      float sc_next = *xsr * *wsr;
      // The residual is asked for here although the tile before has just been stored: a
      // branch for it in the loop, after the first K block, slowed every K block (2048 x
      // 7168 x 18432: 337 us against 316; 5772 x 7424 x 768 with its six: 60.5, here 63).
      const bool asked = residual && live;
      if (asked && lane == 0) {
        bulk_wait_read_all();  // the tile before has left the staging
        const int boxes = n0 + 64 < p.N ? 2 : 1;
        mbar_arrive_expect_tx(&res_full[ew], boxes * 4096);
        for (int b = 0; b < boxes; ++b)
          tma_load_2d(st + b * 4096, &tm_r, &res_full[ew], n0 + b * 64, m0 + q * 32);
      }
      __syncwarp();
      for (int kb = 0; kb < NKB && ok; ++kb) {
        const float sc = sc_next;
        float xs_n = 0.f, ws_n = 0.f;
        if (kb + 1 < NKB) {
          xs_n = xsr[kb + 1];
          ws_n = wsr[kb + 1];
        }
        if (*abort_flag || !mbar_wait_bounded(&tfull[buf], bphase, p.timeout_ns)) {
          ok = false;
          atomicOr(p.err, ERR_DEV_TIMEOUT);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        if (live) promote<C::COLS, 4>(acc, taddr0 + (uint32_t)(buf * C::TN), sc);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[buf]), 0));
        if (++buf == C::NBUF) {
          buf = 0;
          bphase ^= 1;
        }
        sc_next = xs_n * ws_n;
      }
      if constexpr (EPI == DENSE_SILU) {
        // The 1x128 group is both column halves. One barrier per tile: the
        // exchange buffer alternates, and a warp reaches the write two tiles on
        // only after every warp has passed the next tile's barrier, so after it
        // has read this one.
        float* rb = reinterpret_cast<float*>(scratch) + parity * 2 * C::TM;
        parity ^= 1;
        rb[h * C::TM + r] = silu_pairs(acc);
        named_bar_sync(1, C::EW * 32);
        const float scale = group_scale_nan(max_nan(rb[r], rb[C::TM + r]));
        if (ok && m < p.M) {
          store_codes(acc, scale, p.q + m * p.ld_q + nt * 128 + h * 64);
          if (h == 0) p.s[m * p.ld_s + nt] = scale;
        }
      } else {
        if (asked) {  // waited for even when the tile is given up
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(&res_full[ew], rphase, p.timeout_ns))) {
            ok = false;
            atomicOr(p.err, ERR_DEV_TIMEOUT);
            *abort_flag = 1;
          }
          rphase ^= 1;
        }
        if (ok && live) {
          if (p.vec) pair_store_tile(p, tm_o, m0 + q * 32, n0, acc, st, lane);
          else dense_store_tile(p, m0 + q * 32, n0, acc, st, lane);
        }
      }
    }
    if (EPI == DENSE_OUT && lane == 0) bulk_wait_all();  // the output has arrived
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // commits, arrivals and copies of the other CTA have landed
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
  }
}

}  // namespace b200moe
