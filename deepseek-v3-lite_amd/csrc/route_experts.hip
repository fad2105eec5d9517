// Routing to experts from logits, and its gradient: the scores, choice and weights of
// models/moe.py:32-36 with softmax scores, groups of experts and weights left as they are.
//
//   s = sigmoid(l) or softmax(l), evaluated in double and rounded to fp32 once
//   c = s + bias; a group's score is the sum of its two largest c, or its largest; the
//   topk_groups best groups stay (equal scores: the lower group); of their experts the
//   k with the largest c are taken in descending order (equal c: the lower id; NaN last)
//   w_j = s_j / max(sum_j s_j, 1e-10) route_scale, or s_j route_scale
//
// and with g_j = dw_j route_scale (over the sum S where the weights are normalised, less
// sum_j g_j s_j / S where S is not held up by 1e-10):
//   sigmoid   dl = g s (1 - s) at the experts taken, 0 elsewhere
//   softmax   dl_i = s_i (g_i - sum_j g_j s_j), every expert
//
// LPT lanes hold one token, EPL experts each (a wave holds 64 / LPT tokens).  With VEC a
// lane's experts come in fours, 4 (c + LPT i) .. + 3, so that a row is read in whole
// 16-byte loads of consecutive lanes; else c + LPT i.
#include "common.h"
#include "route.h"

namespace dsmoe {

struct RouteArgs {
  const float* logits;   // (T, E)
  const float* bias;     // (E) or null
  float* weights;        // (T, k)
  int32_t* idx;          // (T, k)
  int32_t* counts;       // (E) or null
  // backward
  const float* dweights; // (T, k)
  float* dlogits;        // (T, E)
  int T, E, k;
  int G, gs, keep;       // groups, experts of one, groups that stay
  int gs_inv;            // e / gs = e gs_inv >> 20 for e < 512 (off by less than e 2^-20 < 1 / 512)
  int top2;              // a group's score: its two largest, else its largest
  int normalise;
  float scale;
  int blocks_add;        // counts are added up by several blocks (else written)
};

constexpr int ROUTE_WAVES = 4;

template <int LPT>
__device__ __forceinline__ int32_t part_max(int32_t v) {
  if constexpr (LPT == 16) return row_max_i32(v);
  return wave_max_i32(v);
}
template <int LPT>
__device__ __forceinline__ int32_t part_min(int32_t v) {
  if constexpr (LPT == 16) return row_min_i32(v);
  return ~wave_max_i32(~v);
}
template <int LPT>
__device__ __forceinline__ double part_sum(double v) {
#pragma unroll
  for (int d = 1; d < LPT; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
template <int LPT>
__device__ __forceinline__ float part_sum(float v) {
#pragma unroll
  for (int d = 1; d < LPT; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
template <int LPT>
__device__ __forceinline__ float part_fmax(float v) {
#pragma unroll
  for (int d = 1; d < LPT; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

template <int LPT, bool VEC>
__device__ __forceinline__ int route_expert(int c, int q) {
  return VEC ? 4 * (c + LPT * (q >> 2)) + (q & 3) : c + LPT * q;
}

// The lane's logits of a token (-infinity past E).
template <int LPT, int EPL, bool VEC>
__device__ __forceinline__ void route_load(const float* row, int c, int E, bool live, float (&x)[EPL]) {
#pragma unroll
  for (int q = 0; q < EPL; q += VEC ? 4 : 1) {
    const int e = route_expert<LPT, VEC>(c, q);
    const bool on = live && e < E;
    if constexpr (VEC) {
      const float4 v = *reinterpret_cast<const float4*>(row + (on ? e : 0));
      x[q] = on ? v.x : -INFINITY;
      x[q + 1] = on ? v.y : -INFINITY;
      x[q + 2] = on ? v.z : -INFINITY;
      x[q + 3] = on ? v.w : -INFINITY;
    } else {
      const float v = row[on ? e : 0];
      x[q] = on ? v : -INFINITY;
    }
  }
}

// NaN below every number, as the choice orders it.
__device__ __forceinline__ bool route_before(float a, float b) { return route_key(a) > route_key(b); }

template <int LPT, int EPL, bool VEC, bool SOFTMAX>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_experts_kernel(const RouteArgs a) {
  extern __shared__ __attribute__((aligned(16))) float route_sm[];
  constexpr int TOK = 64 / LPT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane % LPT, r = lane / LPT;
  int* hist = reinterpret_cast<int*>(route_sm);
  float* cs = route_sm + a.E + (wave * TOK + r) * (a.E + 64);   // this token's c, then its group scores
  float* gsc = cs + a.E;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  float bias[EPL];
#pragma unroll
  for (int q = 0; q < EPL; ++q) {
    const int e = route_expert<LPT, VEC>(c, q);
    bias[q] = a.bias && e < a.E ? a.bias[e] : 0.0f;
  }
  const int step = gridDim.x * ROUTE_WAVES * TOK;
  for (int t0 = (blockIdx.x * ROUTE_WAVES + wave) * TOK; t0 < a.T; t0 += step) {
    const int t = t0 + r;
    const bool live = t < a.T;
    const float* row = a.logits + (int64_t)min(t, a.T - 1) * a.E;
    float x[EPL], s[EPL];
    route_load<LPT, EPL, VEC>(row, c, a.E, live, x);
    double den = 1.0;
    float top = 0.0f;
    if constexpr (SOFTMAX) {
      top = x[0];
#pragma unroll
      for (int q = 1; q < EPL; ++q) top = fmaxf(top, x[q]);
      top = part_fmax<LPT>(top);
      double sum = 0.0;
      double ex[EPL];
#pragma unroll
      for (int q = 0; q < EPL; ++q) {
        const bool on = route_expert<LPT, VEC>(c, q) < a.E;
        ex[q] = on ? exp((double)x[q] - (double)top) : 0.0;
        sum += ex[q];
      }
      den = part_sum<LPT>(sum);
#pragma unroll
      for (int q = 0; q < EPL; ++q) s[q] = (float)(ex[q] / den);
    } else {
#pragma unroll
      for (int q = 0; q < EPL; ++q) s[q] = route_sigmoid(x[q]);
    }
    int32_t key[EPL];
#pragma unroll
    for (int q = 0; q < EPL; ++q)
      key[q] = live && route_expert<LPT, VEC>(c, q) < a.E ? route_key(s[q] + bias[q]) : INT32_MIN;
    if (a.G > 1) {
#pragma unroll
      for (int q = 0; q < EPL; ++q) {
        const int e = route_expert<LPT, VEC>(c, q);
        if (e < a.E) cs[e] = s[q] + bias[q];
      }
      __builtin_amdgcn_wave_barrier();
      for (int g = c; g < a.G; g += LPT) {
        float m1 = cs[g * a.gs], m2 = -INFINITY;
        for (int i = 1; i < a.gs; ++i) {
          const float v = cs[g * a.gs + i];
          const bool b1 = route_before(v, m1);
          m2 = b1 ? m1 : i == 1 || route_before(v, m2) ? v : m2;
          m1 = b1 ? v : m1;
        }
        gsc[g] = a.top2 && a.gs > 1 ? m1 + m2 : m1;
      }
      __builtin_amdgcn_wave_barrier();
      // group g stays where fewer than `keep` come before it
      uint64_t stays = 0;
      for (int g0 = 0; g0 < a.G; g0 += LPT) {
        const int g = min(g0 + c, a.G - 1);
        const int32_t kg = route_key(gsc[g]);
        int before = 0;
        for (int j = 0; j < a.G; ++j) {
          const int32_t kj = route_key(gsc[j]);
          before += kj > kg || (kj == kg && j < g);
        }
        uint64_t b = __builtin_amdgcn_ballot_w64(before < a.keep && g0 + c < a.G) >> (LPT * r);
        if (LPT < 64) b &= (1ull << (LPT & 63)) - 1;
        stays |= b << g0;
      }
#pragma unroll
      for (int q = 0; q < EPL; ++q)
        if (!((stays >> (route_expert<LPT, VEC>(c, q) * a.gs_inv >> 20 & 63)) & 1)) key[q] = INT32_MIN;
    }
    // k rounds of the largest key, the lowest expert that holds it; lane j keeps slot j
    int mine = 0;
    for (int j = 0; j < a.k; ++j) {
      int32_t best = key[0];
#pragma unroll
      for (int q = 1; q < EPL; ++q) best = max(best, key[q]);
      const int32_t m = part_max<LPT>(best);
      int32_t cand = INT32_MAX;
#pragma unroll
      for (int q = EPL - 1; q >= 0; --q)
        if (key[q] == m) cand = route_expert<LPT, VEC>(c, q);
      const int32_t win = part_min<LPT>(cand);
      if (c == j) mine = win;
#pragma unroll
      for (int q = 0; q < EPL; ++q)
        if (route_expert<LPT, VEC>(c, q) == win) key[q] = INT32_MIN;
    }
    // the scores of the experts taken, one per lane, as above
    const bool slot = live && c < a.k;
    mine = min(max(mine, 0), a.E - 1);
    const float xs = row[mine];
    const float sv = SOFTMAX ? (float)(exp((double)xs - (double)top) / den) : route_sigmoid(xs);
    float total = 0.0f;
    for (int j = 0; j < a.k; ++j) total += __shfl(sv, r * LPT + j);
    if (slot) {
      const float w = (a.normalise ? sv / (total < 1e-10f ? 1e-10f : total) : sv) * a.scale;
      const int64_t at = (int64_t)t * a.k + c;
      a.weights[at] = w;
      a.idx[at] = mine;
      if (a.counts) atomicAdd(&hist[mine], 1);
    }
  }
  if (!a.counts) return;
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    if (!a.blocks_add)
      a.counts[e] = hist[e];
    else if (hist[e])
      atomicAdd(&a.counts[e], hist[e]);
  }
}

// exp(x - top) in fp32 with what the difference's rounding took away (for far logits
// |x - top| 2^-24 of the result) put back: exp(d + e) = exp(d) (1 + e) to e^2.
__device__ __forceinline__ float route_exp(float x, float top) {
  const float d = x - top, b = d - x;
  const float e = (x - (d - b)) - (top + b);
  const float p = expf(d);
  return d > -120.0f ? fmaf(p, e, p) : p;   // (under that p is 0, and of an infinite d there is no e)
}

template <int LPT, int EPL, bool VEC, bool SOFTMAX>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_experts_bwd_kernel(const RouteArgs a) {
  constexpr int TOK = 64 / LPT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane % LPT, r = lane / LPT;
  const int t = (blockIdx.x * ROUTE_WAVES + wave) * TOK + r;
  const bool live = t < a.T;
  const int64_t tc = min(t, a.T - 1);
  const float* row = a.logits + tc * a.E;
  const bool slot = c < a.k;
  const int mine = slot ? min(max(a.idx[tc * a.k + c], 0), a.E - 1) : -1;
  const float g0 = slot ? a.dweights[tc * a.k + c] * a.scale : 0.0f;
  float x[EPL];
  float sv, top = 0.0f, inv = 1.0f;
  if constexpr (SOFTMAX) {
    route_load<LPT, EPL, VEC>(row, c, a.E, live, x);
    top = x[0];
#pragma unroll
    for (int q = 1; q < EPL; ++q) top = fmaxf(top, x[q]);
    top = part_fmax<LPT>(top);
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < EPL; ++q) {
      x[q] = route_expert<LPT, VEC>(c, q) < a.E ? route_exp(x[q], top) : 0.0f;
      sum += x[q];
    }
    inv = 1.0f / part_sum<LPT>(sum);
    sv = slot ? route_exp(row[mine], top) * inv : 0.0f;
  } else {
    sv = slot ? route_sigmoid(row[mine]) : 0.0f;
  }
  float g = g0;
  if (a.normalise) {
    const float total = part_sum<LPT>(sv), S = total < 1e-10f ? 1e-10f : total;
    const float dot = part_sum<LPT>(g0 * sv);
    g = g0 / S - (total < 1e-10f ? 0.0f : dot / S / S);
    if (!slot) g = 0.0f;
  }
  const float all = SOFTMAX ? part_sum<LPT>(g * sv) : 0.0f;
  const float d = g * sv * (1.0f - sv);   // sigmoid: the slot's own
  float out[EPL];
#pragma unroll
  for (int q = 0; q < EPL; ++q) out[q] = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    const int e = __shfl(mine, r * LPT + j);
    const float v = __shfl(SOFTMAX ? g : d, r * LPT + j);
#pragma unroll
    for (int q = 0; q < EPL; ++q)
      if (route_expert<LPT, VEC>(c, q) == e) out[q] += v;
  }
  if (!live) return;
  float* dst = a.dlogits + tc * a.E;
#pragma unroll
  for (int q = 0; q < EPL; q += VEC ? 4 : 1) {
    const int e = route_expert<LPT, VEC>(c, q);
    if (e >= a.E) continue;
    if constexpr (VEC) {
      float4 v = make_float4(out[q], out[q + 1], out[q + 2], out[q + 3]);
      if (SOFTMAX)
        v = make_float4(x[q] * inv * (v.x - all), x[q + 1] * inv * (v.y - all), x[q + 2] * inv * (v.z - all),
                        x[q + 3] * inv * (v.w - all));
      *reinterpret_cast<float4*>(dst + e) = v;
    } else {
      dst[e] = SOFTMAX ? x[q] * inv * (out[q] - all) : out[q];
    }
  }
}

// ------------------------------------------------------------------ host
static int route_validate(const dsmoe_route_dims* d) {
  DSMOE_REQUIRE(d, DSMOE_ERR_INVALID, "route_experts: NULL dims");
  DSMOE_REQUIRE(d->T >= 0 && d->E > 0, DSMOE_ERR_INVALID, "route_experts: T must not be negative and E positive");
  DSMOE_REQUIRE(d->E <= DSMOE_ROUTE_MAX_EXPERTS, DSMOE_ERR_UNSUPPORTED, "route_experts: more than 512 experts");
  DSMOE_REQUIRE(d->score == DSMOE_SCORE_SIGMOID || d->score == DSMOE_SCORE_SOFTMAX, DSMOE_ERR_INVALID,
                "route_experts: unknown score");
  DSMOE_REQUIRE(d->n_groups >= 1 && d->n_groups <= 64 && d->E % d->n_groups == 0, DSMOE_ERR_INVALID,
                "route_experts: n_groups must be in 1 .. 64 and divide the experts");
  DSMOE_REQUIRE(d->topk_groups >= 1 && d->topk_groups <= d->n_groups, DSMOE_ERR_INVALID,
                "route_experts: topk_groups must be in 1 .. n_groups");
  DSMOE_REQUIRE(d->k >= 1 && d->k <= d->E / d->n_groups * d->topk_groups, DSMOE_ERR_INVALID,
                "route_experts: k must be in 1 .. the experts of topk_groups groups");
  DSMOE_REQUIRE(d->k <= MAX_TOPK, DSMOE_ERR_UNSUPPORTED, "route_experts: k > 16 is not supported");
  return DSMOE_OK;
}

static RouteArgs route_args(const dsmoe_route_dims* d) {
  RouteArgs a{};
  a.T = d->T; a.E = d->E; a.k = d->k;
  a.G = d->n_groups; a.gs = d->E / d->n_groups; a.keep = d->topk_groups;
  a.gs_inv = ((1 << 20) + a.gs - 1) / a.gs;
  a.top2 = d->group_top2; a.normalise = d->normalise; a.scale = d->route_scale;
  return a;
}

template <int LPT, int EPL, bool VEC, bool SOFTMAX>
static void route_launch(const RouteArgs& a, bool bwd, hipStream_t st) {
  const int per = ROUTE_WAVES * (64 / LPT);
  const int64_t blocks = cdiv(a.T, per);
  if (bwd) {
    hipLaunchKernelGGL((route_experts_bwd_kernel<LPT, EPL, VEC, SOFTMAX>), dim3((unsigned)blocks),
                       dim3(64 * ROUTE_WAVES), 0, st, a);
    return;
  }
  RouteArgs b = a;
  b.blocks_add = blocks > 1;
  if (b.blocks_add && b.counts) launch_fill_i32(b.counts, b.E, 0, st);
  const size_t lds = sizeof(float) * (a.E + (size_t)per * (a.E + 64));
  hipLaunchKernelGGL((route_experts_kernel<LPT, EPL, VEC, SOFTMAX>), dim3((unsigned)blocks), dim3(64 * ROUTE_WAVES),
                     lds, st, b);
}

template <int LPT, int EPL>
static void route_pick(const RouteArgs& a, bool vec, bool softmax, bool bwd, hipStream_t st) {
  if constexpr (EPL % 4 == 0) {
    if (vec) {
      softmax ? route_launch<LPT, EPL, true, true>(a, bwd, st) : route_launch<LPT, EPL, true, false>(a, bwd, st);
      return;
    }
  }
  softmax ? route_launch<LPT, EPL, false, true>(a, bwd, st) : route_launch<LPT, EPL, false, false>(a, bwd, st);
}

static int route_run(const RouteArgs& a, int score, bool bwd, hipStream_t st) {
  const auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.E % 4 == 0 && al(a.logits) && al(a.dlogits);
  const bool sm = score == DSMOE_SCORE_SOFTMAX;
  if (a.E <= 16)
    route_pick<16, 1>(a, false, sm, bwd, st);
  else if (a.E <= 32)
    route_pick<16, 2>(a, false, sm, bwd, st);
  else if (a.E <= 64)
    route_pick<16, 4>(a, vec, sm, bwd, st);
  else if (a.E <= 128)
    route_pick<16, 8>(a, vec, sm, bwd, st);
  else if (a.E <= 256)
    route_pick<16, 16>(a, vec, sm, bwd, st);
  else
    route_pick<64, 8>(a, vec, sm, bwd, st);
  return check_launch(bwd ? "route_experts_bwd" : "route_experts");
}

}  // namespace dsmoe

using namespace dsmoe;

extern "C" int dsmoe_route_experts(const float* logits, const float* bias, const dsmoe_route_dims* dims, float* weights,
                                   int32_t* idx, int32_t* counts, void* stream) {
  const int rc = route_validate(dims);
  if (rc) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dims->T == 0) {
    if (counts) launch_fill_i32(counts, dims->E, 0, st);
    return check_launch("route_experts");
  }
  DSMOE_REQUIRE(logits && weights && idx, DSMOE_ERR_INVALID, "route_experts: NULL pointer");
  RouteArgs a = route_args(dims);
  a.logits = logits; a.bias = bias; a.weights = weights; a.idx = idx; a.counts = counts;
  return route_run(a, dims->score, false, st);
}

extern "C" int dsmoe_route_experts_bwd(const float* logits, const int32_t* idx, const float* dweights,
                                       const dsmoe_route_dims* dims, float* dlogits, void* stream) {
  const int rc = route_validate(dims);
  if (rc) return rc;
  if (dims->T == 0) return DSMOE_OK;
  DSMOE_REQUIRE(logits && idx && dweights && dlogits, DSMOE_ERR_INVALID, "route_experts_bwd: NULL pointer");
  RouteArgs a = route_args(dims);
  a.logits = logits; a.idx = const_cast<int32_t*>(idx); a.dweights = dweights; a.dlogits = dlogits;
  return route_run(a, dims->score, true, static_cast<hipStream_t>(stream));
}
