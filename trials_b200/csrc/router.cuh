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
  int vec;             // rows of logits start 16-byte aligned (E * element size too)
  int vec_bias;        // bias 16-byte aligned
  int per;             // with groups: most experts a lane owns (grouped_lanes)
  int gs;              // experts of a group
  int span_log2;       // log2 of the lanes of a group, -1: lanes own experts of several groups
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
// NaN logits count as -inf (score 0), NaN c as -inf; a row whose selected
// scores are all 0 has weights 0 when renormalised.
//
// The selection is the one exact arithmetic on the given f32 (bf16) values
// makes. Without a bias s is monotone in x, so x itself is compared. With one, c
// is computed in fp32 and is off by at most 4.5e-7 + 7e-8 |c|. Experts are
// compared by integer keys in the order of the values whose low bits hold the
// expert's place in its lane, so the value in a key is off by up to 32 units in
// the last place (none for bf16 logits, whose low bits are zero). Where two
// neighbours in the order are closer than the errors (one token in a few
// hundred), every expert not clearly behind the last one taken joins the
// candidates, which are put in order by their exact values in fp64; where groups
// are that close, their scores are computed again in fp64.
//
// One warp per token; a lane owns up to `per` consecutive experts, ascending with
// the lanes, so the lowest lane holding a value also holds its lowest id. A group
// has a power of two of lanes to itself, the last of them not always full, wherever
// that leaves no lane more than 32 (5,580 tokens of 312 experts in 4 groups with a
// bias: 15.9 us, 23.5 with lanes across groups). What bounds it is the number of
// instructions a warp issues, 889 with a bias (issue slots 69% busy, the integer
// pipe 80%; fewer registers for more warps measured 0-8% slower): a round of the
// selection is one redux and one ballot on the lanes' best keys, the lists behind
// them sorted once. 8,192 tokens of 256 experts in 8 groups: 11.2 us with a bias
// (25.7 with every value compared in turn and each close token redone in fp64),
// 8.9 without.
// ---------------------------------------------------------------------------
constexpr int kRouterMaxGroups = 32;
// Bound of the error of two values c together: the sigmoid's (exp 6e-8 where its
// slope lets it through, 1 + e 6e-8, the 2-ulp division 2.4e-7) and the addition's
// half step, twice.
constexpr float kValueEps = 9e-7f, kValueEpsRel = 1.5e-7f;

// Integers in the order of the floats (-0 = +0); 0 is below every float.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// The experts of a lane: n from e0 on.
__device__ __forceinline__ void lane_experts(const RouterArgs& r, int lane, int& e0, int& n) {
  int left;
  if (r.span_log2 >= 0) {
    const int g = lane >> r.span_log2, first = (lane & ((1 << r.span_log2) - 1)) * r.per;
    e0 = g * r.gs + first;
    left = g < r.groups ? r.gs - first : 0;
  } else {
    e0 = lane * r.per;
    left = r.E - e0;
  }
  n = left < 0 ? 0 : (left < r.per ? left : r.per);
}

template <typename T>
__device__ __forceinline__ void merge_top2(T& a1, T& a2, T b1, T b2) {
  const T lo = a1 < b1 ? a1 : b1;
  a1 = a1 < b1 ? b1 : a1;
  a2 = a2 < b2 ? b2 : a2;
  a2 = a2 < lo ? lo : a2;
}

// Scores of the groups, group g's in lane g (-inf in the lanes past the last),
// from this lane's n values c (experts e0 ..; -inf past them). size: the magnitudes
// added in the score.
template <typename T, int PER>
__device__ __forceinline__ T group_scores(const RouterArgs& r, const T (&c)[PER], bool two, int lane, int e0, int n,
                                          T& size) {
  const T ninf = -INFINITY;
  const int groups = r.groups, gs = r.gs;
  two = two && gs > 1;
  T s1 = ninf, s2 = ninf;
  if (r.span_log2 >= 0) {
    const int span = 1 << r.span_log2;
    T a1 = c[0], a2 = ninf;
#pragma unroll
    for (int i = 1; i < PER; ++i) {
      const T lo = a1 < c[i] ? a1 : c[i];
      a1 = a1 < c[i] ? c[i] : a1;
      a2 = a2 < lo ? lo : a2;
    }
    for (int o = 1; o < span; o <<= 1) {
      const T b1 = __shfl_xor_sync(0xffffffffu, a1, o), b2 = __shfl_xor_sync(0xffffffffu, a2, o);
      merge_top2(a1, a2, b1, b2);
    }
    s1 = __shfl_sync(0xffffffffu, a1, (lane << r.span_log2) & 31);
    s2 = __shfl_sync(0xffffffffu, a2, (lane << r.span_log2) & 31);
  } else {
    for (int g = 0; g < groups; ++g) {
      T a1 = ninf, a2 = ninf;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = e0 + i;
        if (i < n && e >= g * gs && e < (g + 1) * gs) merge_top2(a1, a2, c[i], ninf);
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const T b1 = __shfl_xor_sync(0xffffffffu, a1, o), b2 = __shfl_xor_sync(0xffffffffu, a2, o);
        merge_top2(a1, a2, b1, b2);
      }
      if (lane == g) {
        s1 = a1;
        s2 = a2;
      }
    }
  }
  const T score = two ? s1 + s2 : s1;
  if (lane >= groups || score != score) {
    size = 0;
    return ninf;
  }
  size = (s1 < 0 ? -s1 : s1) + (two ? (s2 < 0 ? -s2 : s2) : T(0));
  return score;
}

// Expert e's value c in fp64 (-inf for a NaN).
__device__ __forceinline__ double grouped_value_f64(const RouterArgs& r, int64_t t, int e) {
  const double x = router_logit(r, t, e);
  double v = x;
  if (r.bias) v = (x == x ? 1.0 / (1.0 + exp(-x)) : 0.0) + (double)__ldg(&r.bias[e]);
  return v == v ? v : -INFINITY;
}

// The groups that may be selected from (bit g), in fp64.
template <int PER>
__device__ __noinline__ uint32_t grouped_taken_f64(const RouterArgs r, int64_t t, int lane) {
  double c[PER];
  int e0, n;
  lane_experts(r, lane, e0, n);
#pragma unroll
  for (int i = 0; i < PER; ++i) c[i] = i < n ? grouped_value_f64(r, t, e0 + i) : -INFINITY;
  double size;
  const double score = group_scores<double, PER>(r, c, r.bias != nullptr, lane, e0, n, size);
  int rank = 0;
  for (int h = 0; h < r.groups; ++h) {
    const double other = __shfl_sync(0xffffffffu, score, h);
    rank += (other > score || (other == score && h < lane)) ? 1 : 0;
  }
  return __ballot_sync(0xffffffffu, lane < r.groups && rank < r.topk_groups);
}

// The selection from the groups `taken` in fp64, for a token with more experts
// near its border than lanes; lane j < topk returns the j-th id.
template <int PER>
__device__ __noinline__ int grouped_select_f64(const RouterArgs r, int64_t t, uint32_t taken, int lane) {
  double c[PER];
  uint32_t open = 0;  // bit i: expert e0 + i may still be selected
  int e0, n;
  lane_experts(r, lane, e0, n);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = -INFINITY;
    if (i < n && ((taken >> ((e0 + i) / r.gs)) & 1u)) {
      c[i] = grouped_value_f64(r, t, e0 + i);
      open |= 1u << i;
    }
  }
  int id = 0;
  for (int k = 0; k < r.topk; ++k) {
    double bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (((open >> i) & 1u) && (bi == 0x7fffffff || c[i] > bv)) {
        bv = c[i];
        bi = e0 + i;
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
    if (bi >= e0 && bi < e0 + n) open &= ~(1u << (bi - e0));
    if (lane == k) id = bi;
  }
  return id;
}

// n candidates in descending order of approximate values, lane j < n holding the
// j-th one's id, among them every expert that can be one of the topk best: the
// place of this lane's candidate among them in exact order (fp64; lower id first).
static __device__ __noinline__ int grouped_order_f64(const RouterArgs r, int64_t t, int id, int n, int lane) {
  const double c = lane < n ? grouped_value_f64(r, t, id) : -INFINITY;
  int rank = 0;
  for (int j = 0; j < n; ++j) {
    const double other = __shfl_sync(0xffffffffu, c, j);
    const int oid = __shfl_sync(0xffffffffu, id, j);
    rank += (other > c || (other == c && oid < id)) ? 1 : 0;
  }
  return rank;
}

// This lane's sigmoid over the sum of those of the lanes that are `mine`, in fp64; 0 if
// they are all 0 there.
static __device__ __noinline__ float grouped_ratio_f64(float v, bool mine) {
  const double s = mine && v == v ? 1.0 / (1.0 + exp(-(double)v)) : 0.0;
  double sum = s;
  for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum > 0.0 ? (float)(s / sum) : 0.f;
}

// Descending order of N keys (N = 8: a 19-exchange network; else halves, merged).
__device__ __forceinline__ void key_exchange(uint32_t& a, uint32_t& b) {
  const uint32_t hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi;
  b = lo;
}
template <int N>
__device__ __forceinline__ void merge_keys(uint32_t* k) {  // a bitonic sequence
  if constexpr (N > 1) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) key_exchange(k[i], k[i + N / 2]);
    merge_keys<N / 2>(k);
    merge_keys<N / 2>(k + N / 2);
  }
}
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t* k) {
  if constexpr (N == 8) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) key_exchange(k[i], k[i + 1]);
    key_exchange(k[0], k[2]), key_exchange(k[1], k[3]), key_exchange(k[4], k[6]), key_exchange(k[5], k[7]);
    key_exchange(k[1], k[2]), key_exchange(k[5], k[6]), key_exchange(k[0], k[4]), key_exchange(k[3], k[7]);
    key_exchange(k[1], k[5]), key_exchange(k[2], k[6]);
    key_exchange(k[1], k[4]), key_exchange(k[3], k[6]);
    key_exchange(k[2], k[4]), key_exchange(k[3], k[5]);
    key_exchange(k[3], k[4]);
  } else {
    sort_keys<N / 2>(k);
    sort_keys<N / 2>(k + N / 2);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) key_exchange(k[i], k[N - 1 - i]);
    merge_keys<N / 2>(k);
    merge_keys<N / 2>(k + N / 2);
  }
}

// Routes token t with groups (all 32 lanes call it): ids and weights go to
// r.out_ids / r.out_w.
template <int PER, bool BIASED>
__device__ __forceinline__ void route_token_grouped(const RouterArgs& r, int64_t t, int lane) {
  constexpr uint32_t kPlace = PER - 1;  // low bits of a key: kPlace - place in the lane
  // How far apart two neighbours must be to be sure of their order: without a
  // bias only equal values say nothing (dropping low bits keeps the order); with
  // one, the errors of both, and the dropped bits.
  constexpr float kEps = BIASED ? kValueEps : 0.f;
  constexpr float kEpsRel = BIASED ? kValueEpsRel + PER * 1.2e-7f : 0.f;
  const int E = r.E, topk = r.topk, groups = r.groups;
  const int gs = r.gs;
  int e0, own;  // this lane's experts
  lane_experts(r, lane, e0, own);
  const bool whole = r.per == PER && E == 32 * PER && r.vec;  // every lane full, rows aligned for vector loads
  float x[PER];  // logits, then the values that are compared
  if (whole && !r.bf16) {
    const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(r.logits) + t * E + e0);
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
      const float4 v = __ldg(src + i);
      x[4 * i] = v.x;
      x[4 * i + 1] = v.y;
      x[4 * i + 2] = v.z;
      x[4 * i + 3] = v.w;
    }
  } else if (whole) {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(r.logits) + t * E + e0);
#pragma unroll
    for (int i = 0; i < PER / 8; ++i) {
      const uint4 v = __ldg(src + i);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
        x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = i < own ? router_logit(r, t, e0 + i) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
  float xmax = -INFINITY, denom = 0.f;
  if (!BIASED && r.scoring == 0) {
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
  if (BIASED) {
    float b[PER];
    if (whole && r.vec_bias) {
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(r.bias + e0 + i));
        b[i] = v.x;
        b[i + 1] = v.y;
        b[i + 2] = v.z;
        b[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) b[i] = i < own ? __ldg(&r.bias[e0 + i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (whole || i < own) {
        const float d = 1.0f + __expf(-x[i]);
        const float c = (d < 1e30f ? __fdividef(1.0f, d) : 0.0f) + b[i];
        x[i] = c == c ? c : -INFINITY;
      }
  }
  // The groups whose experts may be selected: best ones first; again in fp64 if
  // the last of them is not clearly ahead of the first that is left out.
  uint32_t taken = 0xffffffffu;
  if (r.topk_groups < groups) {
    taken = 0;
    float size;
    const float score = group_scores<float, PER>(r, x, BIASED, lane, e0, own, size);
    uint32_t sk = lane < groups ? order_key(score) : 0u;
    uint32_t m = 0;
    for (int k = 0; k < r.topk_groups; ++k) {
      m = __reduce_max_sync(0xffffffffu, sk);
      const uint32_t who = __ballot_sync(0xffffffffu, sk == m);
      const uint32_t first = who & (0u - who);
      taken |= first;
      if ((first >> lane) & 1u) sk = 0;
    }
    if (BIASED) {
      const float a = order_value(m), b = order_value(__reduce_max_sync(0xffffffffu, sk));
      // a sum of two values of any size: its error goes by the largest
      const float big = __uint_as_float(__reduce_max_sync(0xffffffffu, size < INFINITY ? __float_as_uint(size) : 0u));
      if (!(a - b > 2.0f * (kValueEps + kValueEpsRel * big))) taken = grouped_taken_f64<PER>(r, t, lane);
    }
  }
  // Keys of this lane's experts; 0 = cannot be selected (any more).
  uint32_t key[PER];
  if (r.span_log2 >= 0) {
    const bool in = (taken >> (lane >> r.span_log2)) & 1u;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      key[i] = in && (whole || i < own) ? ((order_key(x[i]) & ~kPlace) | (kPlace - i)) : 0u;
  } else {
    int g = e0 / gs, left = (g + 1) * gs - e0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = i < own && ((taken >> (g & 31)) & 1u) ? ((order_key(x[i]) & ~kPlace) | (kPlace - i)) : 0u;
      if (--left == 0) {
        ++g;
        left = gs;
      }
    }
  }
  sort_keys<PER>(key);
  // Rounds: lane n keeps the n-th best key (there are topk experts at least), and
  // the lane it came from.
  const uint32_t cut = ~kPlace;
  uint32_t my_key = 0;
  int my_src = 0, n = 0;
  auto take = [&](uint32_t m) {
    // the lowest lane with the largest value; its place is its key's own
    const int src = __ffs(__ballot_sync(0xffffffffu, (key[0] & cut) == m)) - 1;
    const uint32_t won = __shfl_sync(0xffffffffu, key[0], src);
    if (lane == n) {
      my_key = won;
      my_src = src;
    }
    ++n;
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = lane == src ? (i + 1 < PER ? key[i + 1] : 0u) : key[i];
  };
  while (n < topk) take(__reduce_max_sync(0xffffffffu, key[0] & cut));
  // Where values can be off, the ones not clearly behind the last of them join.
  bool order = false;  // two candidates too close to tell which comes first
  bool many = false;   // more of them than lanes
  if (BIASED || !r.bf16) {
    const float last = order_value(__shfl_sync(0xffffffffu, my_key, topk - 1) & cut);
    while (true) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, key[0] & cut);
      if (m == 0 || last - order_value(m) > kEps + kEpsRel * fabsf(last)) break;
      if (n == 32) {
        many = true;
        break;
      }
      take(m);
    }
    const float v = order_value(my_key & cut);
    const float next = __shfl_down_sync(0xffffffffu, v, 1);
    order = __any_sync(0xffffffffu, lane + 1 < n && !(v - next > kEps + kEpsRel * fabsf(v)));
  }
  int src_e0, src_n;
  lane_experts(r, my_src, src_e0, src_n);
  int my_id = src_e0 + (int)(kPlace - (my_key & kPlace));
  int place = lane;  // of this lane's expert in the output (topk and more: none)
  if (many) my_id = grouped_select_f64<PER>(r, t, taken, lane);  // warp-uniform
  else if (order) place = grouped_order_f64(r, t, my_id, n, lane);
  const bool mine = place < topk && (many || lane < n);
  float w = 0.f, v = 0.f;
  if (mine) {
    v = router_logit(r, t, my_id);
    if (r.scoring == 1) w = v == v ? 1.0f / (1.0f + expf(-v)) : 0.f;
    else if (v == v && v != -INFINITY) w = v == xmax ? 1.0f : expf(v - xmax);
  }
  // Sigmoids that fp32 does not hold although fp64 does still have a ratio.
  if (r.scoring == 1 && r.renormalize && __any_sync(0xffffffffu, v < -87.0f && v > -710.0f)) {
    w = grouped_ratio_f64(v, mine);
  } else if (r.renormalize) {
    float sum = w;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w = sum > 0.f ? w / sum : 0.f;
  } else if (r.scoring == 0) {
    w = denom > 0.f ? w / denom : 0.f;
  }
  if (mine) {
    r.out_w[t * topk + place] = w * r.scaling;
    r.out_ids[t * topk + place] = my_id;
  }
}

template <int PER, bool GROUPED>
__device__ __forceinline__ void route_token(const RouterArgs& r, int64_t t, int lane) {
  if constexpr (GROUPED) {
    if (r.bias) route_token_grouped<PER, true>(r, t, lane);
    else route_token_grouped<PER, false>(r, t, lane);
  } else {
    int id;
    float w;
    route_token_warp<PER>(r, t, lane, id, w);
  }
}

// Values per lane for E experts (see route_token_warp).
__host__ __device__ __forceinline__ int router_per_lane(int E) { return E <= 256 ? 8 : (E <= 512 ? 16 : 32); }

// Values per lane in group-limited routing (r.per of them used).
inline int grouped_per_lane(const RouterArgs& r) { return r.per <= 8 ? 8 : (r.per <= 16 ? 16 : 32); }

// How the experts of r.groups groups are dealt to the lanes (lane_experts).
inline void grouped_lanes(RouterArgs& r) {
  r.gs = r.E / r.groups;
  int log2 = 0;
  while (r.groups << (log2 + 1) <= 32) ++log2;
  r.span_log2 = log2;
  r.per = (r.gs + (1 << log2) - 1) >> log2;
  if (r.per > 32) {  // more than 512 experts in groups that are no power of two
    r.span_log2 = -1;
    r.per = (r.E + 31) / 32;
  }
}

}  // namespace b200moe
