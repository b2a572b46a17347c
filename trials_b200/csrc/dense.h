// Internal interface of the dense (not expert-grouped) FP8 block-scaled
// products: fp8_block_linear and fp8_gate_up (dense.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200moe {

struct DenseParams {
  const float* xs;  // activation scales: row m, K block kb at xs[m * ld_xs + kb]
  int64_t ld_xs;
  const void* xb;   // bf16 rows instead (plan.quantise_x): row m at xb + m * ld_xb
  int64_t ld_xb;
  const float* ws;  // weight scales (ceil(N/128), K/128)
  int M, N, K;
  // DENSE_OUT: out[m * ld_out + n] = y (+ residual[m * ld_res + n])
  void* out;
  int64_t ld_out;
  int out_f32;
  const void* residual;  // bf16, nullable
  int64_t ld_res;
  int vec;  // rows of out (and residual) start 16-byte aligned and N is a multiple of 8
  // DENSE_SILU: q[m * ld_q + j] / s[m * ld_s + j/128], j < N/2
  uint8_t* q;
  int64_t ld_q;
  float* s;
  int64_t ld_s;
  int32_t* err;
  uint64_t timeout_ns;
};

enum { DENSE_OUT = 0, DENSE_SILU = 1 };

// How a product is cut up, and the boxes its tensor maps need.
constexpr int kDenseTok = 0, kDensePair = 1;
struct DensePlan {
  int cfg;     // kDenseTok, kDensePair, or the split kernel's T (dense_split.cuh)
  int tokens;  // split kernel: tokens of a tile, a multiple of 16 up to T
  int splits;  // split and token-major kernel: CTAs that share K
  int quantise_x;  // bf16 rows are quantised inside the kernel
  int x_box_rows;
  int w_box_rows;
  int out_box_rows;  // DENSE_OUT of vector-aligned rows (p.vec) through TMA; 0: plain stores
};
// x_bf16: the rows come in bf16 (quantise_x can only be set then).
DensePlan dense_plan(int epi, int64_t M, int64_t N, int64_t K, bool x_bf16);
// early_w: the kernel ahead of this one in the stream belongs to the same call
// and does not write w. tm_o, tm_r: output and residual in boxes of 128 bytes x
// out_box_rows; any map where they are not used.
cudaError_t launch_dense(int epi, const DensePlan& pl, const CUtensorMap& tm_x, const CUtensorMap& tm_w,
                         const CUtensorMap& tm_o, const CUtensorMap& tm_r, const DenseParams& p, bool early_w, cudaStream_t stream);

}  // namespace b200moe
