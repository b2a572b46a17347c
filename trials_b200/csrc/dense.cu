// Dense FP8 block-scaled products: launch of the token-major kernel.
#include "dense.h"

#include "dense_tok.cuh"
#include "launch.h"

namespace b200moe {

namespace {

int sm_count_of_current() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 1;
}

template <int EPI>
cudaError_t launch_tok_dense(const CUtensorMap& tm_x, const CUtensorMap& tm_w, const DenseParams& p,
                             cudaStream_t stream) {
  using C = DenseTokCfg;
  auto kernel = dense_tok_kernel<EPI>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
  if (err != cudaSuccess) return err;
  const int n_mt = (p.M + C::TM - 1) / C::TM, n_nt = (p.N + C::TN - 1) / C::TN;
  const int64_t units = (int64_t)n_mt * n_nt;
  const int sms = sm_count_of_current();
  const int grid = units < sms ? (int)units : sms;
  return launch_pdl(kernel, dim3(grid), dim3(C::THREADS), C::SMEM_BYTES, stream, tm_x, tm_w, p, n_mt, n_nt, 8);
}

}  // namespace

DensePlan dense_plan(int epi, int64_t M, int64_t N, int64_t K) {
  (void)epi;
  (void)M;
  (void)N;
  (void)K;
  return DensePlan{DenseTokCfg::TM, DenseTokCfg::TN};
}

cudaError_t launch_dense(int epi, const DensePlan& pl, const CUtensorMap& tm_x, const CUtensorMap& tm_w,
                         const DenseParams& p, cudaStream_t stream) {
  (void)pl;
  return epi == DENSE_SILU ? launch_tok_dense<DENSE_SILU>(tm_x, tm_w, p, stream)
                           : launch_tok_dense<DENSE_OUT>(tm_x, tm_w, p, stream);
}

}  // namespace b200moe
