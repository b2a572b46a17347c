// Dense FP8 block-scaled products: choice and launch of the kernels.
#include "dense.h"

#include <atomic>

#include "dense_pair.cuh"
#include "dense_split.cuh"
#include "dense_tok.cuh"
#include "moe_gemm_tok2.cuh"
#include "launch.h"

namespace b200moe {

namespace {

constexpr int kMaxDevices = 64;

int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}

int sm_count_of(int dev) {
  static std::atomic<int> cache[kMaxDevices];
  if (dev >= 0 && dev < kMaxDevices && cache[dev].load() > 0) return cache[dev].load();
  int n = 0;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (n <= 0) n = 1;
  if (dev >= 0 && dev < kMaxDevices) cache[dev].store(n);
  return n;
}

// Raises the kernel's shared memory limit once per device, to a size that is the same in
// every call of a kernel: a limit that went by the call could be lowered again by another
// host thread between here and the launch.
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, int dev, std::atomic<int> (&done)[kMaxDevices]) {
  if (dev >= 0 && dev < kMaxDevices && done[dev].load() >= bytes) return cudaSuccess;
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess && dev >= 0 && dev < kMaxDevices) done[dev].store(bytes);
  return err;
}

// Launch attributes of every kernel here: a cluster of R CTAs, programmatic
// order behind the kernel ahead of it.
void cluster_launch(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int R, dim3 grid, int threads, int smem,
                    cudaStream_t stream) {
  cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = R;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = B200MOE_PDL ? 2 : 1;
}

// Tiles are taken in groups of this many token tiles: CTAs that run at the same
// time then share weight tiles and activations through L2.
constexpr int kTileGroup = 8;

template <int EPI, int TN>
cudaError_t launch_tok_dense(const DensePlan& pl, const CUtensorMap& tm_x, const CUtensorMap& tm_w,
                             const DenseParams& p, bool early_w, cudaStream_t stream) {
  using C = DenseTokCfg<TN>;
  static std::atomic<int> done[kMaxDevices];
  auto kernel = dense_tok_kernel<EPI, TN>;
  const cudaError_t err = allow_smem(kernel, C::SMEM_BYTES, current_device(), done);
  if (err != cudaSuccess) return err;
  const int n_mt = (p.M + C::TM - 1) / C::TM, n_nt = (p.N + TN - 1) / TN;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  cluster_launch(cfg, attr, pl.splits, dim3((unsigned)n_mt * n_nt * pl.splits), C::THREADS, C::SMEM_BYTES, stream);
  return cudaLaunchKernelEx(&cfg, kernel, tm_x, tm_w, p, pl.splits, n_mt, n_nt, kTileGroup,
                            early_w && B200MOE_PDL ? 1 : 0);
}

// Shared memory of a CTA of the split kernel, whatever it needs of it. A CTA that waits
// for TMEM holds its place in its cluster, and two clusters that wait for each other's
// TMEM never end: so the CTAs that fit on an SM together (of one launch or of several
// streams) must also have TMEM enough. The size sees to it: two CTAs of this kernel,
// with half of the TMEM each, fill the SM (2 x 114 KB = 228, 1 KB of each the system's),
// and none stands beside a CTA that takes all of it, as the token-major, pair and expert
// kernels do with 194 KB and more. That is said of this library's kernels: a clustered
// kernel of another one that takes more than half of the TMEM with 113 KB at most can
// meet a split CTA on an SM, and neither the allocation nor a cluster barrier has a time
// limit. (78 KB where that is enough, which leaves other kernels 148, measured no faster.)
constexpr int kSplitSmem = 113 * 1024;
constexpr bool alone(int smem) { return smem + kSplitSmem + 2 * 1024 > 228 * 1024; }
static_assert(2 * (kSplitSmem + 1024) <= 228 * 1024 && alone(kSplitSmem + 1), "two split CTAs fill an SM");
static_assert(alone(DenseTokCfg<256>::SMEM_BYTES) && alone(DenseTokCfg<128>::SMEM_BYTES) &&
                  alone(DensePairCfg<DENSE_OUT>::SMEM_BYTES) && alone(DensePairCfg<DENSE_SILU>::SMEM_BYTES) &&
                  alone(GemmCfg<32, 1>::SMEM_BYTES) && alone(GemmCfg<64, 1>::SMEM_BYTES) &&
                  alone(GemmCfg<64, 2>::SMEM_BYTES) && alone(TokCfgE<EPI_SILU>::SMEM_BYTES) &&
                  alone(TokCfgE<EPI_COMBINE>::SMEM_BYTES) && alone(Tok2Cfg::SMEM_BYTES),
              "no split CTA beside one that takes all of the TMEM");

// Stages that fit next to the scales (and quantised rows) of nkb K blocks, or 0.
template <int T>
int split_stages(int nkb, int tt, bool qx) {
  using C = DenseSplitCfg<T>;
  int n = nkb < C::MAX_STAGE ? nkb : C::MAX_STAGE;
  while (n * C::tile_bytes(tt, qx) < tt * 512) ++n;  // the CTA's sums reuse the tiles
  while (n > 1 && C::smem_bytes(n, nkb, tt, qx) > kSplitSmem) --n;
  const bool fits = C::smem_bytes(n, nkb, tt, qx) <= kSplitSmem && n * C::tile_bytes(tt, qx) >= tt * 512 &&
                    (n >= 2 || nkb == 1);
  return fits ? n : 0;
}

template <int EPI, int T, bool QX>
cudaError_t launch_split_dense(const DensePlan& pl, const CUtensorMap& tm_x, const CUtensorMap& tm_w,
                               const DenseParams& p, bool early_w, cudaStream_t stream) {
  using C = DenseSplitCfg<T>;
  constexpr int HALVES = EPI == DENSE_SILU ? 2 : 1;
  static std::atomic<int> done[kMaxDevices];
  auto kernel = dense_split_kernel<EPI, T, QX>;
  const int nkb = ((p.K >> 7) + pl.splits - 1) / pl.splits;
  const int nstage = split_stages<T>(nkb, pl.tokens, QX);
  if (nstage == 0) return cudaErrorInvalidValue;
  cudaError_t err = allow_smem(kernel, kSplitSmem, current_device(), done);
  if (err != cudaSuccess) return err;
  const int R = HALVES * pl.splits;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  cluster_launch(cfg, attr, R,
                 dim3((unsigned)((p.N + 128 * HALVES - 1) / (128 * HALVES) * R),
                      (unsigned)((p.M + pl.tokens - 1) / pl.tokens), 1),
                 C::THREADS, kSplitSmem, stream);
  return cudaLaunchKernelEx(&cfg, kernel, tm_x, tm_w, p, pl.splits, pl.tokens, nstage,
                            early_w && B200MOE_PDL ? 1 : 0);
}

// Clusters of R CTAs of a kernel that are resident at once on the current device.
template <typename K>
int resident_clusters(K kernel, int R, int threads, int smem, std::atomic<int> (&cache)[kMaxDevices][9]) {
  const int dev = current_device();
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (known && cache[dev][R].load() > 0) return cache[dev][R].load();
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  cluster_launch(cfg, attr, R, dim3(R), threads, smem, nullptr);
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = sm_count_of(dev) / R > 0 ? sm_count_of(dev) / R : 1;  // no such device: any plan will do
  }
  if (known) cache[dev][R].store(n);
  return n;
}
int resident_tok(int R) {
  static std::atomic<int> cache[kMaxDevices][9];
  using C = DenseTokCfg<256>;  // 128 columns take the same threads and shared memory
  static_assert(C::THREADS == DenseTokCfg<128>::THREADS && C::SMEM_BYTES == DenseTokCfg<128>::SMEM_BYTES, "");
  return resident_clusters(dense_tok_kernel<DENSE_OUT, 256>, R, C::THREADS, C::SMEM_BYTES, cache);
}
int resident_pairs() {
  static std::atomic<int> cache[kMaxDevices][9];
  using C = DensePairCfg<DENSE_OUT>;
  return resident_clusters(dense_pair_kernel<DENSE_OUT>, 2, C::THREADS, C::SMEM_BYTES, cache);
}

template <int EPI>
cudaError_t launch_pair_dense(const CUtensorMap& tm_x, const CUtensorMap& tm_w, const CUtensorMap& tm_o,
                              const CUtensorMap& tm_r, const DenseParams& p, cudaStream_t stream) {
  using C = DensePairCfg<EPI>;
  static std::atomic<int> done[kMaxDevices];
  auto kernel = dense_pair_kernel<EPI>;
  cudaError_t err = allow_smem(kernel, C::SMEM_BYTES, current_device(), done);
  if (err != cudaSuccess) return err;
  const int n_mt = (p.M + 2 * C::TM - 1) / (2 * C::TM), n_nt = (p.N + C::TN - 1) / C::TN;
  const int64_t units = (int64_t)n_mt * n_nt;
  const int pairs = units < resident_pairs() ? (int)units : resident_pairs();
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  cluster_launch(cfg, attr, 2, dim3(2 * pairs), C::THREADS, C::SMEM_BYTES, stream);
  return cudaLaunchKernelEx(&cfg, kernel, tm_x, tm_w, tm_o, tm_r, p, n_mt, n_nt, kTileGroup);
}

template <int EPI>
cudaError_t launch_epi_dense(const DensePlan& pl, const CUtensorMap& tm_x, const CUtensorMap& tm_w,
                             const CUtensorMap& tm_o, const CUtensorMap& tm_r, const DenseParams& p, bool early_w, cudaStream_t stream) {
  switch (pl.cfg) {
    case 16:
      return pl.quantise_x ? launch_split_dense<EPI, 16, true>(pl, tm_x, tm_w, p, early_w, stream)
                           : launch_split_dense<EPI, 16, false>(pl, tm_x, tm_w, p, early_w, stream);
    case 32:
      return launch_split_dense<EPI, 32, false>(pl, tm_x, tm_w, p, early_w, stream);
    case 64:
      return launch_split_dense<EPI, 64, false>(pl, tm_x, tm_w, p, early_w, stream);
    case kDensePair:
      return launch_pair_dense<EPI>(tm_x, tm_w, tm_o, tm_r, p, stream);
    default:
      // (DENSE_SILU: a tile holds 128 gate and their 128 up rows.)
      if constexpr (EPI == DENSE_OUT)
        if (pl.w_box_rows == 128) return launch_tok_dense<EPI, 128>(pl, tm_x, tm_w, p, early_w, stream);
      return launch_tok_dense<EPI, 256>(pl, tm_x, tm_w, p, early_w, stream);
  }
}

}  // namespace

namespace {

// The split kernel for these sizes, or cfg = kDenseTok when it does not suit.
DensePlan split_plan(int epi, int64_t M, int64_t N, int nkb, bool x_bf16) {
  DensePlan pl{};
  pl.cfg = kDenseTok;
  const int halves = epi == DENSE_SILU ? 2 : 1;
  const int64_t n_tt = (M + 63) / 64;
  const int tt = (int)((M + n_tt - 1) / n_tt + 15) / 16 * 16;
  const int T = tt <= 16 ? 16 : (tt <= 32 ? 32 : 64);
  const int64_t units = (N + 128 * halves - 1) / (128 * halves) * n_tt;
  const int sms = sm_count_of(current_device());
  // CTAs along K, at least two K blocks each. Where 8 would exchange the sums of more than
  // 32 tokens they have an SM each, or at least four: two of them on an SM measured slower
  // than 4 with twice the K blocks (64 tokens of K = 2048, 8 and 4 CTAs along it: N = 512
  // 5.1 us and 5.8, 1536 5.6 and 6.0, 1920 6.0 and 6.3, then 2048 7.0 and 6.4, 2304 7.7
  // and 6.6; of K = 3584: 1536 6.9 and 7.5, 1920 7.1 and 7.6, 2048 8.5
  // and 7.7; 40 tokens of 1920 x 2048 5.3 and 5.8, of 2048 x 2048 6.0 and 5.8).
  int s = 8 / halves;
  auto fewest = [&](int k) { return T == 64 && M <= 64 && k == 8 && units > resident_tok(8) ? 4 : 2; };
  while (s > 1 && s * fewest(s) > nkb) s /= 2;
  if (M > 64) {
    // More than 64 tokens read the weights more than once, which pays while the tiles'
    // clusters run in one wave, two CTAs an SM less what clusters cannot use (gate/up of
    // 200 x 2048 x 256 5.9 us, token-major 8.7; 1500 x 1024 x 256 6.2 and 7.8), with one
    // CTA an SM where K is long: token-major clusters then wait less for their operands
    // (gate/up of 128 x 6144 x 2048, 256 CTAs of 12 K blocks: 14.7 and 13.9; 128 x 4096 x
    // 2048, of 8: 12.3 and 12.9), with DENSE_OUT, whose tiles of 128 columns exchange
    // little, from 4 CTAs along K on (500 x 1000 x 1024, 256 CTAs: 7.2 and 6.6; 200 x 576
    // x 7168, 160: 10.0 and 8.5; 300 x 100 x 6144, 40: 6.7 and 7.5).
    const bool two_an_sm = epi == DENSE_SILU ? nkb <= 8 * s : s <= 2;
    const int64_t most = two_an_sm ? (int64_t)sms * 7 / 4 : sms;
    if (units * halves * s > most) return pl;
  } else {
    // Two CTAs an SM where that leaves more than 8 K blocks to each (one token of 8192 x
    // 8192 14.6 us, 16.4 with half of them; 64 tokens of 7168 x 18432 28.8 and 38.4), else
    // up to 4/3 of the SMs: one token of 6144 x 2048 (48 tiles) takes 6.2 us with 4 CTAs
    // along K, 6.8 with 2 and, in two waves, 10.8 with 6; 64 tokens of 4096 x 6144 (32
    // tiles) 10.8 with 4, 11.5 with 8. One an SM where more than 32 tokens would leave
    // fewer than 8 K blocks (64 of 6144 x 2048: 8.1 with 2, 9.2 with 4).
    auto fits = [&](int k) {
      const int64_t ctas = units * halves * k;
      if (nkb > 8 * k) return ctas <= (int64_t)sms * 2;
      return ctas <= (T == 64 && nkb < 8 * k ? sms : (int64_t)sms * 4 / 3);
    };
    while (s > 1 && !fits(s)) s /= 2;
  }
  const int per = (nkb + s - 1) / s;
  // A few tokens: a CTA can quantise its own K blocks of bf16 rows.
  const bool qx = x_bf16 && T == 16 && M * per <= kQuantGroups && split_stages<16>(per, tt, true) > 0;
  const int stages = qx ? 1
                        : (T == 16 ? split_stages<16>(per, tt, false)
                                   : (T == 32 ? split_stages<32>(per, tt, false) : split_stages<64>(per, tt, false)));
  if (stages == 0) return pl;
  pl.cfg = T;
  pl.tokens = tt;
  pl.splits = s;
  pl.quantise_x = qx;
  pl.x_box_rows = tt;
  pl.w_box_rows = 128;
  return pl;
}

}  // namespace

DensePlan dense_plan(int epi, int64_t M, int64_t N, int64_t K, bool x_bf16) {
  const int nkb = (int)(K / 128);
  DensePlan pl = split_plan(epi, M, N, nkb, x_bf16);
  if (pl.cfg != kDenseTok) return pl;
  // The largest cluster, one wave of them, that shares `tiles` output tiles' K blocks.
  auto most_splits = [nkb](int64_t tiles) {
    int s = 8;
    while (s > 1 && (s * 2 > nkb || tiles > resident_tok(s))) --s;
    return s;
  };
  const int64_t m_tiles = (M + 127) / 128;
  // Tiles of 128 columns where they still leave three CTAs to each, since a CTA then
  // has few K blocks and half the sums to exchange (300 x 1000 x 4096: 8.7 us against
  // 11.3; 100 x 4096 x 6144: 11.1 against 13.1), or where 256 would be half empty and
  // two rounds do (7796 x 11 x 3584: 14.4 against 21.5, 30000 x 128 x 4096: 39 against
  // 44; in the six of 100000 x 100 x 2048 persistent pairs hide the start of each: 80
  // against 90). With two CTAs each or one the longer tile's K block, 0.6 us against
  // 2 x 0.44, decides (200 x 4096 x 6144: 15.0 against 15.6 with two, 200 x 6144 x
  // 2048: 11.8 against 13.5 with one).
  if (epi == DENSE_OUT) {
    const int s = most_splits(m_tiles * ((N + 127) / 128));
    if (s >= 3 || (N <= 128 && m_tiles <= 2 * resident_tok(1))) {
      pl.splits = s;
      pl.x_box_rows = 128;
      pl.w_box_rows = 128;
      return pl;
    }
  }
  // Token-major tiles of 256 columns while a cluster of two or more CTAs can share each
  // (512 x 4096 x 6144: 20.9 us against 30.7 with pairs), unless two of them share so
  // few K blocks that their exchange costs more (gate/up 300 x 1024 x 2048, 8 K blocks:
  // 11.5 against 10.0 with pairs; 300 x 2048 x 2048, 16: 13.4 and 13.8). Then pairs unless
  // they take more rounds (1024 x 4096 x 6144: 31.5 and token-major 32.9; 2048: 59.5 and
  // 64.3), and with more rounds, as an odd number of 128-token tiles leaves half of a
  // pair's tile empty, whichever takes less time. A token-major round, whose start and end
  // nothing hides, measured 8.7 us and 0.48 a K block, one of the persistent pairs 2.0 and
  // 0.52 and 1.6 more a launch, for products and gate/up alike, 2.5 here as rows that are
  // not aligned cost pairs more (us token-major and with pairs; x N, K blocks, rounds:
  //   300 x 12544, 32, 1 and 2: 25.5, 39.7    1100 x 8192, 32, 2 and 3: 49, 57
  //   600 x 15104, 16, 2 and 3: 34.2, 33.1    600 x 15101, 16: 42.9, 46.6
  //   1100 x 16384, 32, 4 and 5: 98, 94       1100 x 16381, 32: 115.5, 115.8
  //   1100 x 32768, 16, 8 and 9: 136, 94      2100 x 36864, 56, 17 and 18: 643, 598
  //   gate/up 4160 x 36864, 56, 33 and 34: 1400, 1195
  //   4200 x 129280, 8, 113 and 117: 1447, 752). The bits are the same either way.
  using T = DenseTokCfg<256>;
  const int64_t n_nt = (N + T::TN - 1) / T::TN;
  const int64_t units = m_tiles * n_nt, pair_units = (M + 2 * T::TM - 1) / (2 * T::TM) * n_nt;
  const int s = most_splits(units);
  const int64_t rounds = (units + resident_tok(1) - 1) / resident_tok(1);
  const int64_t pair_rounds = (pair_units + resident_pairs() - 1) / resident_pairs();
  const int64_t ns_tok = rounds * (8700 + 480 * (int64_t)nkb);
  const int64_t ns_pair = 2500 + pair_rounds * (2000 + 520 * (int64_t)nkb);
  if ((s == 1 || (s == 2 && nkb <= 8)) && (rounds >= pair_rounds || ns_pair <= ns_tok)) {
    pl.cfg = kDensePair;
    pl.splits = 1;
    pl.x_box_rows = DensePairCfg<DENSE_OUT>::TM;
    pl.w_box_rows = DensePairCfg<DENSE_OUT>::WR;
    pl.out_box_rows = 32;
    return pl;
  }
  pl.splits = s;
  pl.x_box_rows = T::TM;
  pl.w_box_rows = T::TN;
  return pl;
}

cudaError_t launch_dense(int epi, const DensePlan& pl, const CUtensorMap& tm_x, const CUtensorMap& tm_w,
                         const CUtensorMap& tm_o, const CUtensorMap& tm_r, const DenseParams& p, bool early_w,
                         cudaStream_t stream) {
  return epi == DENSE_SILU ? launch_epi_dense<DENSE_SILU>(pl, tm_x, tm_w, tm_o, tm_r, p, early_w, stream)
                           : launch_epi_dense<DENSE_OUT>(pl, tm_x, tm_w, tm_o, tm_r, p, early_w, stream);
}

}  // namespace b200moe
