// Router top-k of one token by one warp: scores -> k expert ids and weights.
//
// The router in front of the reference's MoE call (aiter's topksoftmax kernel
// in its runs, MBR/micro/glm52_fp8_moe.log; GLM's sigmoid "noaux_tc" routing,
// measure_xcd_imbalance.py:50-55 and phase1_xcd_imbalance_and_proof.md:37-39):
//   softmax: p = softmax(logits); select the k largest p (= largest logits);
//   sigmoid: s = 1 / (1 + exp(-logits)); select the k largest s + bias
//            (bias = per-expert correction, optional);
//   weights = unbiased p or s of the selected experts, optionally divided by
//   their sum, times scaling (routed_scaling_factor).
// Output order: descending selection value; equal values -> lower id first.
// Used by the standalone router kernel (router.cu) and by routing's first
// launch when routing starts from logits (route.cu): the same arithmetic, so
// the two give the same bits.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace b200moe {

constexpr int kRouterMaxTopk = 16;  // E <= 1024 (32 values per lane)

struct RouterArgs {
  const void* logits;  // (M, E) f32, or bf16 when bf16 != 0
  int bf16;
  int E, topk, scoring, renormalize;
  const float* bias;   // nullable (sigmoid only)
  float scaling;
  float* out_w;        // (M, topk)
  int32_t* out_ids;    // (M, topk)
  int groups;          // group-limited routing (route_token_grouped); 0 = ungrouped
  int topk_groups;     // groups whose experts may be selected
};

__device__ __forceinline__ float router_logit(const RouterArgs& r, int64_t t, int e) {
  if (r.bf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(r.logits)[t * r.E + e]);
  return __ldg(reinterpret_cast<const float*>(r.logits) + t * r.E + e);
}

// Warp-wide: routes token t; lane j < topk returns the j-th id and weight and
// also stores them to r.out_ids / r.out_w. All 32 lanes must call it. PER =
// values per lane (expert e = lane + 32 i, i < PER): 8 for E <= 256, 16 for
// E <= 512, 32 for E <= 1024 (router_per_lane), so the logits stay in
// registers; the selected id and weight of round k stay in lane k.
template <int PER>
__device__ __forceinline__ void route_token_warp(const RouterArgs& r, int64_t t, int lane, int& id_out,
                                                 float& w_out) {
  const int E = r.E, topk = r.topk;
  float x[PER], sel[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    x[i] = e < E ? router_logit(r, t, e) : -INFINITY;
  }
  float denom = 1.f, xmax = 0.f;
  if (r.scoring == 0) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmaxf(m, x[i]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < E) sum += expf(x[i] - m);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    denom = sum;
    xmax = m;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    if (e < E) {
      if (r.scoring == 0) {
        sel[i] = x[i];  // softmax is monotone in the logit
      } else {
        const float s = 1.0f / (1.0f + expf(-x[i]));
        x[i] = s;
        sel[i] = r.bias ? s + __ldg(&r.bias[e]) : s;
      }
    } else {
      sel[i] = -INFINITY;
    }
  }
  float wsum = 0.f, my_w = 0.f;
  int my_id = 0;
  for (int k = 0; k < topk; ++k) {
    // lane-local best, then warp argmax (larger value, then lower id)
    float bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 32 * i;
      if (sel[i] > bv || (sel[i] == bv && e < bi && sel[i] != -INFINITY)) {
        bv = sel[i];
        bi = e;
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (ov > bv || (ov == bv && oi < bi)) {
        bv = ov;
        bi = oi;
      }
    }
    // owner lane marks it and publishes the weight
    float w = 0.f;
    if ((bi & 31) == lane) {
      const int i = bi >> 5;
#pragma unroll
      for (int ii = 0; ii < PER; ++ii)
        if (ii == i) {
          w = r.scoring == 0 ? expf(x[ii] - xmax) / denom : x[ii];
          sel[ii] = -INFINITY;
        }
    }
    w = __shfl_sync(0xffffffffu, w, bi & 31);
    if (lane == k) {
      my_w = w;
      my_id = bi;
    }
    wsum += w;
  }
  id_out = 0;
  w_out = 0.f;
  if (lane < topk) {
    w_out = my_w;
    id_out = my_id;
    if (r.renormalize) w_out = w_out / wsum;
    w_out *= r.scaling;
    r.out_w[t * topk + lane] = w_out;
    r.out_ids[t * topk + lane] = id_out;
  }
}

// ---------------------------------------------------------------------------
// Group-limited routing. The E experts form `groups` equal runs of consecutive
// ids; only the experts of the topk_groups best groups can be selected.
//   s = softmax(x) or sigmoid(x);  c = s + bias (sigmoid only) or s
//   group score: without a bias the largest c, with one the sum of the two
//   largest; best groups, then best experts, equal values lower index first.
// The selection is the one exact arithmetic on the given f32 (bf16) values
// makes. Without a bias s is monotone in x, so x itself is compared. With one,
// c is computed in fp32 and is off by at most ~4e-7 + 6e-8 |c|; when two values
// whose order matters are closer than kGroupedEps + kGroupedEpsRel * |c| (about
// one token in a thousand) the token's selection is redone in fp64.
// NaN logits count as -inf (score 0), NaN c as -inf; a row whose selected
// scores sum to 0 has weights 0 when renormalised.
//
// One warp per token; lane l owns the experts [l * per, (l + 1) * per), so the
// lowest lane holding a value also holds its lowest id and the warp's argmax is
// one redux of order-preserving integer keys and one ballot.
// ---------------------------------------------------------------------------
constexpr int kRouterMaxGroups = 32;
constexpr float kGroupedEps = 2e-6f;
constexpr float kGroupedEpsRel = 5e-7f;

// Integers in the order of the floats (-0 = +0); 0 is below every float.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

template <typename T>
__device__ __forceinline__ void merge_top2(T& a1, T& a2, T b1, T b2) {
  const T lo = a1 < b1 ? a1 : b1;
  a1 = a1 < b1 ? b1 : a1;
  a2 = a2 < b2 ? b2 : a2;
  a2 = a2 < lo ? lo : a2;
}

// Scores of the groups, group g's in lane g (-inf in the lanes past the last),
// from this lane's per values c.
template <typename T, int PER>
__device__ __forceinline__ T group_scores(const T (&c)[PER], int E, int groups, int per, bool two, int lane) {
  const T ninf = -INFINITY;
  const int gs = E / groups;
  const int span = gs / per;  // lanes of a group, if its experts fill whole lanes
  T score = ninf;
  if (gs % per == 0 && (span & (span - 1)) == 0) {
    T a1 = ninf, a2 = ninf;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < per) merge_top2(a1, a2, c[i], ninf);
    for (int o = 1; o < span; o <<= 1) {
      const T b1 = __shfl_xor_sync(0xffffffffu, a1, o), b2 = __shfl_xor_sync(0xffffffffu, a2, o);
      merge_top2(a1, a2, b1, b2);
    }
    const T v = two && gs > 1 ? a1 + a2 : a1;
    score = __shfl_sync(0xffffffffu, v, (lane * span) & 31);
  } else {
    for (int g = 0; g < groups; ++g) {
      T a1 = ninf, a2 = ninf;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane * per + i;
        if (i < per && e >= g * gs && e < (g + 1) * gs) merge_top2(a1, a2, c[i], ninf);
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const T b1 = __shfl_xor_sync(0xffffffffu, a1, o), b2 = __shfl_xor_sync(0xffffffffu, a2, o);
        merge_top2(a1, a2, b1, b2);
      }
      const T v = two && gs > 1 ? a1 + a2 : a1;
      if (lane == g) score = v;
    }
  }
  if (lane >= groups || score != score) score = ninf;
  return score;
}

// Rank of lane g's group among the groups (lane < groups).
template <typename T>
__device__ __forceinline__ int group_rank(T score, int groups, int lane) {
  int rank = 0;
  for (int h = 0; h < groups; ++h) {
    const T other = __shfl_sync(0xffffffffu, score, h);
    rank += (other > score || (other == score && h < lane)) ? 1 : 0;
  }
  return rank;
}

// The selection of one token with a bias in fp64; lane j < topk returns the
// j-th id.
template <int PER>
__device__ __noinline__ int grouped_select_f64(const RouterArgs r, int64_t t, int lane) {
  const int per = (r.E + 31) >> 5, gs = r.E / r.groups;
  double c[PER];
  uint32_t open = 0;  // bit i: expert lane * per + i may still be selected
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * per + i;
    c[i] = -INFINITY;
    if (i < per && e < r.E) {
      const double x = router_logit(r, t, e);
      const double s = x == x ? 1.0 / (1.0 + exp(-x)) : 0.0;
      const double v = s + (double)__ldg(&r.bias[e]);
      if (v == v) c[i] = v;
      open |= 1u << i;
    }
  }
  const double score = group_scores<double, PER>(c, r.E, r.groups, per, true, lane);
  const int rank = group_rank(score, r.groups, lane);
  const uint32_t taken = __ballot_sync(0xffffffffu, lane < r.groups && rank < r.topk_groups);
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (((open >> i) & 1u) && !((taken >> ((lane * per + i) / gs)) & 1u)) open &= ~(1u << i);
  int id = 0;
  for (int k = 0; k < r.topk; ++k) {
    double bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (((open >> i) & 1u) && (bi == 0x7fffffff || c[i] > bv)) {
        bv = c[i];
        bi = lane * per + i;
      }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      // a lane with nothing left (0x7fffffff, -inf) never beats one that has something
      if (oi != 0x7fffffff && (bi == 0x7fffffff || ov > bv || (ov == bv && oi < bi))) {
        bv = ov;
        bi = oi;
      }
    }
    if (bi / per == lane) open &= ~(1u << (bi - lane * per));
    if (lane == k) id = bi;
  }
  return id;
}

// As route_token_warp, with groups.
template <int PER>
__device__ __forceinline__ void route_token_grouped(const RouterArgs& r, int64_t t, int lane, int& id_out,
                                                    float& w_out) {
  const int E = r.E, topk = r.topk, groups = r.groups;
  const int per = (E + 31) >> 5, gs = E / groups;
  const bool biased = r.bias != nullptr;
  const int e0 = lane * per;
  float x[PER];  // logits, then the values that are compared
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = i < per && e0 + i < E ? router_logit(r, t, e0 + i) : -INFINITY;
  float xmax = -INFINITY, denom = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
  if (r.scoring == 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) xmax = fmaxf(xmax, x[i]);
    xmax = order_value(__reduce_max_sync(0xffffffffu, order_key(xmax)));
    if (!r.renormalize) {  // renormalised weights do not depend on it
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (x[i] != -INFINITY) denom += x[i] == xmax ? 1.0f : expf(x[i] - xmax);
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) denom += __shfl_xor_sync(0xffffffffu, denom, o);
    }
  }
  if (biased) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i < per && e0 + i < E) {
        const float d = 1.0f + __expf(-x[i]);
        const float c = (d < 1e30f ? __fdividef(1.0f, d) : 0.0f) + __ldg(&r.bias[e0 + i]);
        x[i] = c == c ? c : -INFINITY;
      }
  }
  // The groups whose experts may be selected, and whether fp32 could tell.
  const float score = group_scores<float, PER>(x, E, groups, per, biased, lane);
  const int rank = group_rank(score, groups, lane);
  const uint32_t taken = __ballot_sync(0xffffffffu, lane < groups && rank < r.topk_groups);
  bool close = false;
  if (biased && r.topk_groups < groups) {
    // A score is the sum of two values of any size: its error goes by the largest.
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) big = fabsf(x[i]) < INFINITY ? fmaxf(big, fabsf(x[i])) : big;
    big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
    const int in = __ffs(__ballot_sync(0xffffffffu, lane < groups && rank == r.topk_groups - 1)) - 1;
    const int out = __ffs(__ballot_sync(0xffffffffu, lane < groups && rank == r.topk_groups)) - 1;
    const float a = __shfl_sync(0xffffffffu, score, in), b = __shfl_sync(0xffffffffu, score, out);
    close = !(a - b > 2.0f * (kGroupedEps + kGroupedEpsRel * big));
  }
  // Keys of this lane's experts; 0 = cannot be selected (any more).
  uint32_t key[PER];
  uint32_t best = 0;
  int at = 0;
  {
    int g = e0 / gs, left = (g + 1) * gs - e0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = i < per && e0 + i < E && ((taken >> (g & 31)) & 1u) ? order_key(x[i]) : 0u;
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
      if (--left == 0) {
        ++g;
        left = gs;
      }
    }
  }
  int my_id = 0;
  // With a bias one round more: is the last one taken clearly ahead of the next?
  const int rounds = biased && topk < r.topk_groups * gs ? topk + 1 : topk;
  float prev = 0.f;
  for (int k = 0; k < rounds; ++k) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    const int src = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
    const int id = __shfl_sync(0xffffffffu, e0 + at, src);
    if (lane == k) my_id = id;
    if (biased) {
      const float v = order_value(m);
      if (k > 0 && !(prev - v > kGroupedEps + kGroupedEpsRel * fabsf(prev))) close = true;
      prev = v;
    }
    if (lane == src) {
      best = 0;
      int next = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (i == at) key[i] = 0;
        if (key[i] > best) {
          best = key[i];
          next = i;
        }
      }
      at = next;
    }
  }
  if (biased && close) my_id = grouped_select_f64<PER>(r, t, lane);  // warp-uniform
  float w = 0.f;
  if (lane < topk) {
    const float v = router_logit(r, t, my_id);
    if (r.scoring == 1) w = v == v ? 1.0f / (1.0f + expf(-v)) : 0.f;
    else if (v == v && v != -INFINITY) w = v == xmax ? 1.0f : expf(v - xmax);
  }
  float sum = w;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (r.renormalize) w = sum > 0.f ? w / sum : 0.f;
  else if (r.scoring == 0) w = denom > 0.f ? w / denom : 0.f;
  id_out = my_id;
  w_out = 0.f;
  if (lane < topk) {
    w_out = w * r.scaling;
    r.out_w[t * topk + lane] = w_out;
    r.out_ids[t * topk + lane] = my_id;
  }
}

template <int PER, bool GROUPED>
__device__ __forceinline__ void route_token(const RouterArgs& r, int64_t t, int lane, int& id, float& w) {
  if constexpr (GROUPED) route_token_grouped<PER>(r, t, lane, id, w);
  else route_token_warp<PER>(r, t, lane, id, w);
}

// Values per lane for E experts (see route_token_warp).
__host__ __device__ __forceinline__ int router_per_lane(int E) { return E <= 256 ? 8 : (E <= 512 ? 16 : 32); }

}  // namespace b200moe
