// Router: scores -> top-k expert ids and weights, one warp per token (the
// arithmetic is route_token_warp / route_token_grouped in router.cuh, shared
// with routing's first launch when routing starts from logits).
#include "common.cuh"
#include "launch.h"
#include "router.cuh"

namespace b200moe {

namespace {

constexpr int kRouterWarps = 4;

template <int PER, bool GROUPED>
__global__ void __launch_bounds__(kRouterWarps * 32) router_topk_kernel(const RouterArgs r, int64_t M) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kRouterWarps + (threadIdx.x >> 5);
  if (t >= M) return;
  route_token<PER, GROUPED>(r, t, lane);
}

template <bool GROUPED>
cudaError_t launch_router_per(const RouterArgs& r, int64_t M, cudaStream_t stream) {
  const unsigned blocks = (unsigned)((M + kRouterWarps - 1) / kRouterWarps);
  switch (GROUPED ? grouped_per_lane(r) : router_per_lane(r.E)) {
    case 8:
      router_topk_kernel<8, GROUPED><<<blocks, kRouterWarps * 32, 0, stream>>>(r, M);
      break;
    case 16:
      router_topk_kernel<16, GROUPED><<<blocks, kRouterWarps * 32, 0, stream>>>(r, M);
      break;
    default:
      router_topk_kernel<32, GROUPED><<<blocks, kRouterWarps * 32, 0, stream>>>(r, M);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_router_topk(const RouterArgs& r, int64_t M, cudaStream_t stream) {
  if (M <= 0) return cudaSuccess;
  return r.groups > 0 ? launch_router_per<true>(r, M, stream) : launch_router_per<false>(r, M, stream);
}

}  // namespace b200moe
