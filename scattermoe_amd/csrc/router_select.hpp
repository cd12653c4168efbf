// The routing of one token by one wave: softmax over its expert logits, selection of the k most probable experts,
// optional renormalisation of the selected probabilities.  Lane l holds logits l, l + 64, ... (at most
// ROUTER_MAX_PER_LANE per lane, i.e. E <= 512).
//
// Selection is k rounds of a wave-wide maximum and a search for its first holder; among equal values the lowest expert
// id wins.  All arithmetic in fp32.  The rounds follow one another, so what bounds it is the latency of one: row shifts
// and broadcasts between lanes (probabilities are never negative, so they order as their bits do) and ballots, no
// shuffles through LDS.
// Every id emitted is a valid expert id whatever the logits hold: a NaN logit counts as -inf, and a row without
// any usable logit is routed as if all its logits were equal.
#pragma once
#include "common.hpp"

namespace smoe {

static constexpr int ROUTER_MAX_PER_LANE = 8;

// `logit(e)`: the logit of expert e < E; `exp_of(x)`: the exponential; `expert(j, e)` is called by lane 0 with the j-th
// selection.  Returns in lane j < k (k <= 64) the weight of the j-th selection.
template <class Logit, class Exp, class Expert>
__device__ __forceinline__ float select_experts(int E, int k, bool renorm, Logit logit, Exp exp_of, Expert expert) {
  const int lane = lane_id();
  float v[ROUTER_MAX_PER_LANE];
  float mx = -INFINITY;
#pragma unroll
  for (int q = 0; q < ROUTER_MAX_PER_LANE; ++q) {
    const int e = q * 64 + lane;
    v[q] = e < E ? logit(e) : -INFINITY;
    if (v[q] != v[q]) v[q] = -INFINITY;                        // a NaN logit never wins: its expert gets probability 0
    mx = fmaxf(mx, v[q]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  const bool none = !(mx > -INFINITY);                         // no usable logit in the row: uniform probabilities
  float sum = 0.0f;
#pragma unroll
  for (int q = 0; q < ROUTER_MAX_PER_LANE; ++q) {
    float p = none ? 1.0f : exp_of(v[q] - mx);
    if (p != p) p = 1.0f;                                      // +inf - +inf: the logit is the maximum
    v[q] = q * 64 + lane < E ? p : -1.0f;                      // -1: not a candidate (probabilities are >= 0)
    sum += fmaxf(v[q], 0.0f);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  const float inv = 1.0f / sum;
  float picked = 0.0f;          // lane j keeps the j-th selected probability (k <= 64)
  float sel_sum = 0.0f;
  for (int j = 0; j < k; ++j) {
    int most = __float_as_int(v[0]);                            // (-1, no candidate, is a negative integer as well)
#pragma unroll
    for (int q = 1; q < ROUTER_MAX_PER_LANE; ++q) most = max(most, __float_as_int(v[q]));
    most = wave_max(most);
    int be = 0;
    unsigned long long holders = 0;
#pragma unroll
    for (int q = 0; q < ROUTER_MAX_PER_LANE; ++q) {
      if (holders == 0 && q * 64 < E) {
        holders = __ballot(__float_as_int(v[q]) == most);
        be = q * 64 + __ffsll((long long)holders) - 1;
      }
    }
    const float best = __int_as_float(most);
    const float pr = best * inv;
    if (lane == j) picked = pr;
    sel_sum += pr;
    if (lane == 0) expert(j, be);
    if ((be & 63) == lane) {
#pragma unroll
      for (int q = 0; q < ROUTER_MAX_PER_LANE; ++q)
        if (q == (be >> 6)) v[q] = -1.0f;                       // taken
    }
  }
  return renorm ? picked / sel_sum : picked;
}

}  // namespace smoe
