// Expert routing beyond the plain softmax top-k of alut_route.cuh: softmax or sigmoid
// scores, a bias that takes part in the choice but not in the weights (load balance without
// an auxiliary loss), groups of experts of which only the best few may be chosen from,
// renormalised and scaled weights, and the same keep mask.
//
// Per token, with scores p = softmax(l) or 1 / (1 + exp(-l)):
//   key_j   = p_j + b_j; without a bias, and when groups go by their largest key, the logit
//             itself: the order is the same and rounding makes no ties. -inf (an expert masked
//             out) and NaN rank below every other key.
//   group   = its largest key, or the sum of its two largest; the topk_group best groups stay.
//   chosen  = the top_k largest keys in the groups that stay, lowest expert id first on ties.
//   weights = p[chosen], divided by max(their sum, 1e-20) if asked, times scale. A row with
//             every logit -inf has weights 0.
// The softmax denominator is summed in 64 bits and rounded once: the sum's order then does
// not show in the result, so a biased choice is reproducible to the last bit.
//
// One warp per token, experts lane-strided (expert lane + 32 v in register v). A round of the
// top-k is a local arg-max over NV registers and two warp reductions (redux.sync: largest
// ordered key, then lowest expert id among equal keys). Latency-bound: a token's logits are
// one or a few coalesced loads, the rest is the dependent chain of top_k + topk_group rounds.
// Measured: 1 token of 128 experts, top 8: 3.0 us; 4096 of 256 in 8 groups (sigmoid, bias, two largest):
// 12.8 us; 20011 of 72, biased softmax, top 6: 13.8 us (0.7 us of memory traffic each).
#pragma once

#include "alut_common.cuh"
#include "alut_route.cuh"

namespace alut {

constexpr int kRouteMaxGroups = 32;  // one lane per group, one bit per group

struct RouteExpertsArgs {
  RouteArgs r;
  const float* bias;  // [E] or NULL
  int sigmoid;
  int n_group, topk_group, top2;
  float scale;
};

// Keys in ascending unsigned order; -0 and +0 are one key.
__device__ __forceinline__ uint32_t route_key(float v) { return order_f32(v + 0.0f); }

// NV > 0: E <= 32 NV, keys in registers. NV == 0: any E, keys in shared memory.
template <int NV>
__global__ void __launch_bounds__(kRouteWarps * 32) k_route_experts(RouteExpertsArgs a) {
  extern __shared__ float rx_smem[];  // [kRouteWarps][scores E | ordered keys E]
  constexpr unsigned kAll = 0xffffffffu;
  if (a.r.mode != ALUT_KEEP_FIXED) pdl_launch_dependents();  // (a call's last kernel lets nobody ahead)
  const int E = a.r.e;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (t >= a.r.q) return;
  float* p = rx_smem + static_cast<size_t>(warp) * 2 * E;
  uint32_t* ks = reinterpret_cast<uint32_t*>(p + E);
  const int nv = NV > 0 ? NV : (E + 31) / 32;
  constexpr int NR = NV > 0 ? NV : 1;
  float x[NR];
  uint32_t key[NR];
  float mx = -INFINITY;
#pragma unroll
  for (int v = 0; v < nv; ++v) {
    const int j = lane + 32 * v;
    const float xv = j < E ? logit_at(a.r, t, j) : -INFINITY;
    if constexpr (NV > 0) x[v] = xv;
    else if (j < E) p[j] = xv;
    mx = fmaxf(mx, xv);
  }
  float total = 0.f, shift = 0.f;
  if (!a.sigmoid) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
    shift = mx == -INFINITY ? 0.f : mx;
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < nv; ++v) {
      const int j = lane + 32 * v;
      if (j < E) sum += expf((NV > 0 ? x[NV > 0 ? v : 0] : p[j]) - shift);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    total = static_cast<float>(sum);
  }
  const bool by_logit = !a.bias && !a.top2;
#pragma unroll
  for (int v = 0; v < nv; ++v) {
    const int j = lane + 32 * v;
    uint32_t k = 0;  // below every real key: no such expert
    if (j < E) {
      const float xv = NV > 0 ? x[NV > 0 ? v : 0] : p[j];
      float score;
      if (a.sigmoid) score = 1.0f / (1.0f + expf(-xv));
      else score = total == 0.f ? 0.f : expf(xv - shift) / total;
      float kf = by_logit ? xv : a.bias ? score + a.bias[j] : score;
      if (xv == -INFINITY || isnan(kf)) kf = -INFINITY;
      k = route_key(kf);
      p[j] = score;
      if (NV == 0 || a.n_group > 1) ks[j] = k;
    }
    if constexpr (NV > 0) key[v] = k;
  }
  __syncwarp();
  if (a.n_group > 1) {
    // Group scores, one group at a time: the warp's two largest keys of the group.
    const int per = E / a.n_group;
    uint32_t mine = 0;
    for (int g = 0; g < a.n_group; ++g) {
      uint32_t m1 = 0, m2 = 0;
      for (int i = lane; i < per; i += 32) {
        const uint32_t k = ks[g * per + i];
        m2 = max(m2, min(m1, k));
        m1 = max(m1, k);
      }
      const uint32_t best = __reduce_max_sync(kAll, m1);
      uint32_t gk = best;
      if (a.top2 && per > 1) {
        const int owner = __ffs(__ballot_sync(kAll, m1 == best)) - 1;
        const uint32_t second = __reduce_max_sync(kAll, lane == owner ? m2 : m1);
        const float sum = unorder_f32(best) + unorder_f32(second);
        gk = route_key(isnan(sum) ? -INFINITY : sum);
      }
      if (lane == g) mine = gk;
    }
    unsigned allowed = 0;
    for (int r = 0; r < a.topk_group; ++r) {
      const uint32_t best = __reduce_max_sync(kAll, mine);
      const int g = __ffs(__ballot_sync(kAll, mine == best)) - 1;
      allowed |= 1u << g;
      if (lane == g) mine = 0;
    }
#pragma unroll
    for (int v = 0; v < nv; ++v) {
      const int j = lane + 32 * v;
      if (j < E && !(allowed >> (j / per) & 1u)) {
        if constexpr (NV > 0) key[v] = 0;
        else ks[j] = 0;
      }
    }
    __syncwarp();
  }
  int sel0 = 0, sel1 = 0;  // slots lane and lane + 32
  for (int s = 0; s < a.r.k; ++s) {
    uint32_t best = 0;
    int bv = 0;
#pragma unroll
    for (int v = 0; v < nv; ++v) {
      const uint32_t k = NV > 0 ? key[NV > 0 ? v : 0] : (lane + 32 * v < E ? ks[lane + 32 * v] : 0u);
      if (k > best) {  // ascending experts per lane: the first of equal keys stays
        best = k;
        bv = v;
      }
    }
    const uint32_t m = __reduce_max_sync(kAll, best);
    const unsigned j = __reduce_min_sync(kAll, best == m ? static_cast<unsigned>(lane + 32 * bv) : 0x7fffffffu);
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < nv; ++v)
        if (static_cast<unsigned>(lane + 32 * v) == j) key[v] = 0;
    } else {
      if (lane == 0) ks[j] = 0;
      __syncwarp();
    }
    if ((s & 31) == lane) (s < 32 ? sel0 : sel1) = static_cast<int>(j);
  }
  float w0 = lane < a.r.k ? p[sel0] : 0.f, w1 = lane + 32 < a.r.k ? p[sel1] : 0.f;
  if (a.r.normalize) {
    float tot = w0 + w1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tot += __shfl_xor_sync(kAll, tot, o);
    tot = tot < 1e-20f ? 1e-20f : tot;  // a NaN stays one
    w0 /= tot;
    w1 /= tot;
  }
  if (a.r.mode != ALUT_KEEP_FIXED) pdl_wait();  // the sums are clear
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int s = lane + 32 * h;
    if (s >= a.r.k) break;
    const float wv = (h ? w1 : w0) * a.scale;
    const int e = h ? sel1 : sel0;
    const int64_t o = t * a.r.out_stride + s;
    a.r.w[o] = wv;
    a.r.sel[o] = e;
    if (a.r.mode == ALUT_KEEP_FIXED) {
      const bool comp = s < a.r.keep_k;
      a.r.compute[o] = comp ? 1 : 0;
      a.r.reuse[o] = comp ? 0 : 1;
    } else {  // the importance sums of alut_route
      add_score(a.r, e, a.r.attn ? a.r.attn[t] * wv : wv / static_cast<float>(max(a.r.q, 1)));
    }
  }
}

}  // namespace alut
