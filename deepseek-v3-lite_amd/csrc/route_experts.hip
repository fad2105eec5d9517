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
// LPT lanes hold one token (16 or 64; a wave holds 64 / LPT tokens), lane c of them experts
// c EPL .. c EPL + EPL - 1: a lower lane holds lower ids, so that of equal keys the first
// lane's wins, and a group of gs = P EPL experts is P whole lanes.
//
// What bounds the forward is not its bytes but the double-precision score of every expert (a
// sigmoid is about 65 instructions of half the rate), the rounds of the choice and the
// groups' scores.  So the choice runs on single-precision estimates first (route_margin), and
// on the scores themselves only where two estimates that were compared stand closer than
// their errors; only the experts taken get the double score then.  Measured at T 8192, E 256,
// 8 groups, k 8: 24 us with every score in double and group scores through LDS, 19 us so.
#include <algorithm>
#include <type_traits>

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
  int lanes_of_group;    // of a group of whole lanes, 0: none
  int gs_inv;            // e / gs = e gs_inv >> 20 for e < 512 (off by less than e 2^-20 < 1 / 512)
  int top2;              // a group's score: its two largest, else its largest
  int normalise;
  float scale;
  int32_t* part;         // (blocks, E) counts of each block's tokens, null: one block, which writes counts
  int per;               // tokens of a block
};

constexpr int ROUTE_WAVES = 4;   // of a block of the backward

template <int LPT>
__device__ __forceinline__ int32_t part_max(int32_t v) {
  if constexpr (LPT == 16) return row_max_i32(v);
  return wave_max_i32(v);
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

// The lane's logits of a token (-infinity past E): whole vectors of W, which divides E and EPL.
template <int EPL, int W>
__device__ __forceinline__ void route_load(const float* row, int c, int E, bool live, float (&x)[EPL]) {
#pragma unroll
  for (int q = 0; q < EPL; q += W) {
    const int e = c * EPL + q;
    const bool on = live && e < E;
    float v[W];
    if constexpr (W == 4)
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(row + (on ? e : 0));
    else if constexpr (W == 2)
      *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(row + (on ? e : 0));
    else
      v[0] = row[on ? e : 0];
#pragma unroll
    for (int u = 0; u < W; ++u) x[q + u] = on ? v[u] : -INFINITY;
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

__device__ __forceinline__ float route_val(int32_t key) {
  return key == INT32_MIN + 1 ? __builtin_nanf("") : __int_as_float(key >= 0 ? key : key ^ 0x7fffffff);
}

// Estimates and their errors.  Sigmoid: rcp(1 + exp2(-x log2 e)) is within 2^-22 of the
// score (route.h, route_batch_fast).  Softmax: e / sum of e with e within 1.5 2^-23 of
// exp(x - top) (route_exp) and their sum in double, so within 3 2^-23 and two roundings of
// itself: 2^-21 of the row's largest score covers every one.  Two biased values are apart
// beyond doubt where their distance is more than twice the error, twice over, and an ulp each.
__device__ __forceinline__ bool route_apart(float a, float b, float err) {
  return fabsf(a - b) > 4.0f * err + 4.0f * ROUTE_ULP * fmaxf(fabsf(a), fabsf(b));   // (false for a NaN)
}

template <int LPT, int EPL, int W, bool SOFTMAX, int THREADS>
__global__ __launch_bounds__(THREADS) void route_experts_kernel(const RouteArgs a) {
  extern __shared__ __attribute__((aligned(16))) float route_sm[];
  constexpr int TOK = 64 / LPT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane % LPT, r = lane / LPT;
  int* hist = reinterpret_cast<int*>(route_sm);
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  float bias[EPL];
#pragma unroll
  for (int q = 0; q < EPL; ++q) bias[q] = 0.0f;
  if (a.bias) route_load<EPL, W>(a.bias, c, a.E, true, bias);   // (-infinity past E: no expert there)
  const int tend = (int)min((int64_t)a.T, (int64_t)(blockIdx.x + 1) * a.per);
  for (int t0 = blockIdx.x * a.per + wave * TOK; t0 < tend; t0 += (blockDim.x >> 6) * TOK) {
    const int t = t0 + r;
    const bool live = t < tend;
    const float* row = a.logits + (int64_t)min(t, a.T - 1) * a.E;
    float x[EPL];
    route_load<EPL, W>(row, c, a.E, live, x);
    float top = 0.0f, inv = 1.0f, err = 2.384185791015625e-7f;   // 2^-22
    double den = 1.0;
    if constexpr (SOFTMAX) {
      top = x[0];
#pragma unroll
      for (int q = 1; q < EPL; ++q) top = fmaxf(top, x[q]);
      top = part_fmax<LPT>(top);
      double sum = 0.0;
#pragma unroll
      for (int q = 0; q < EPL; ++q)
        if (c * EPL + q < a.E) sum += (double)route_exp(x[q], top);
      den = part_sum<LPT>(sum);
      inv = (float)(1.0 / den);
      err = 4.76837158203125e-7f * inv;   // the largest score is 1 / den
    }
    const int P = a.lanes_of_group;   // lanes of a group, 0: through LDS
    int mine = 0;
    // pass 0 on estimates; pass 1, for the waves with a token in doubt, on the scores
    for (int pass = 0; pass < 2; ++pass) {
      int32_t key[EPL];
      if (pass == 0) {
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
          const float s = SOFTMAX ? route_exp(x[q], top) * inv
                                  : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[q] * -1.4426950408889634f));
          // (a NaN's key says nothing, but it is among those taken or compared, or changes nothing)
          key[q] = live && c * EPL + q < a.E ? max(mono_key(s + bias[q]), INT32_MIN + 1) : INT32_MIN;
        }
      } else {
        if constexpr (SOFTMAX) {   // (the estimate's sum serves the weights alone)
          double sum = 0.0;
#pragma unroll
          for (int q = 0; q < EPL; ++q)
            if (c * EPL + q < a.E) sum += exp((double)x[q] - (double)top);
          den = part_sum<LPT>(sum);
        }
#pragma unroll
        for (int q = 0; q < EPL; ++q) {
          const float s = SOFTMAX ? (float)(exp((double)x[q] - (double)top) / den) : route_sigmoid(x[q]);
          key[q] = live && c * EPL + q < a.E ? route_key(s + bias[q]) : INT32_MIN;
        }
      }
      bool sure = true;
      if (a.G > 1) {
        // the two largest keys of a group, m1 >= m2
        if (P > 0) {
          int32_t m1 = key[0], m2 = INT32_MIN;
#pragma unroll
          for (int q = 1; q < EPL; ++q) {
            m2 = max(m2, min(m1, key[q]));
            m1 = max(m1, key[q]);
          }
          const int g = c / P;
          if ((P & (P - 1)) == 0) {
            for (int d = 1; d < P; d <<= 1) {
              const int32_t p1 = __shfl_xor(m1, d), p2 = __shfl_xor(m2, d);
              m2 = max(min(m1, p1), max(m2, p2));
              m1 = max(m1, p1);
            }
          } else {
            const int32_t l1 = m1, l2 = m2;
            for (int d = 1, at = c - g * P; d < P; ++d) {
              at = at + 1 == P ? 0 : at + 1;
              const int32_t p1 = __shfl(l1, r * LPT + g * P + at), p2 = __shfl(l2, r * LPT + g * P + at);
              m2 = max(min(m1, p1), max(m2, p2));
              m1 = max(m1, p1);
            }
          }
          const float gs = a.top2 && m2 != INT32_MIN ? route_val(m1) + route_val(m2) : route_val(m1);
          const int32_t kg = route_key(gs);
          int before = 0;
          for (int j = 0; j < a.G; ++j) {
            const float oj = __shfl(gs, r * LPT + j * P);
            const int32_t kj = route_key(oj);
            before += kj > kg || (kj == kg && j < g);
            if (j != g && g < a.G) sure = sure && route_apart(gs, oj, 2.0f * err);
          }
          if (before >= a.keep || g >= a.G)
#pragma unroll
            for (int q = 0; q < EPL; ++q) key[q] = INT32_MIN;
        } else {
          int32_t* ks = reinterpret_cast<int32_t*>(route_sm) + a.E + (wave * TOK + r) * (a.E + 64);   // this token's keys
          float* gsc = reinterpret_cast<float*>(ks + a.E);                                               // and group scores
#pragma unroll
          for (int q = 0; q < EPL; ++q)
            if (c * EPL + q < a.E) ks[c * EPL + q] = key[q];
          __builtin_amdgcn_wave_barrier();
          for (int g = c; g < a.G; g += LPT) {
            int32_t m1 = ks[g * a.gs], m2 = INT32_MIN;
            for (int i = 1; i < a.gs; ++i) {
              const int32_t v = ks[g * a.gs + i];
              m2 = max(m2, min(m1, v));
              m1 = max(m1, v);
            }
            gsc[g] = a.top2 && m2 != INT32_MIN ? route_val(m1) + route_val(m2) : route_val(m1);
          }
          __builtin_amdgcn_wave_barrier();
          // group g stays where fewer than `keep` come before it
          uint64_t stays = 0;
          for (int g0 = 0; g0 < a.G; g0 += LPT) {
            const int g = min(g0 + c, a.G - 1);
            const float gs = gsc[g];
            const int32_t kg = route_key(gs);
            int before = 0;
            for (int j = 0; j < a.G; ++j) {
              const float oj = gsc[j];
              const int32_t kj = route_key(oj);
              before += kj > kg || (kj == kg && j < g);
              if (j != g) sure = sure && route_apart(gs, oj, 2.0f * err);
            }
            uint64_t b = __builtin_amdgcn_ballot_w64(before < a.keep && g0 + c < a.G) >> (LPT * r);
            if (LPT < 64) b &= (1ull << (LPT & 63)) - 1;
            stays |= b << g0;
          }
#pragma unroll
          for (int q = 0; q < EPL; ++q)
            if (!((stays >> ((c * EPL + q) * a.gs_inv >> 20 & 63)) & 1)) key[q] = INT32_MIN;
        }
      }
      // rounds of the largest key, the lowest expert that holds it; lane j keeps slot j.  On
      // estimates one round more, and every round's key well above the next one's
      float last = INFINITY;
      for (int j = 0; j < a.k + (pass == 0 ? 1 : 0); ++j) {
        int32_t best = key[0];
#pragma unroll
        for (int q = 1; q < EPL; ++q) best = max(best, key[q]);
        const int32_t m = part_max<LPT>(best);
        int32_t wq = INT32_MAX;
#pragma unroll
        for (int q = EPL - 1; q >= 0; --q)
          if (key[q] == m) wq = c * EPL + q;
        int win;
        if constexpr (LPT == 64)   // the first lane that holds it
          win = __builtin_amdgcn_readlane(wq, __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(best == m)) - 1);
        else
          win = row_min_i32(wq);
        if (m != INT32_MIN) {   // (the round more may find no one left)
          const float v = route_val(m);
          if (j > 0) sure = sure && route_apart(last, v, err);
          sure = sure && fabsf(v) < INFINITY;
          last = v;
        }
        if (c == j && j < a.k) mine = win;
        const int own = win - c * EPL;
#pragma unroll
        for (int q = 0; q < EPL; ++q)
          if (q == own) key[q] = INT32_MIN;
      }
      if (__builtin_amdgcn_ballot_w64(live && !sure) == 0) break;
    }
    // the scores of the experts taken, one per lane, as in pass 1
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
      atomicAdd(&hist[mine], 1);
    }
  }
  __syncthreads();
  int32_t* counts = a.part ? a.part + (int64_t)blockIdx.x * a.E : a.counts;
  if (counts)
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) counts[e] = hist[e];
}

// The blocks' counts added: 64 experts a block, 16 waves over the rows.  (Added by atomics
// instead, 512 blocks' took 6 us of 16 at E 64, T 8192, and the clearing before a launch.)  3.9 us of
// the 24 that E 256, T 8192 takes.
__global__ __launch_bounds__(1024) void route_counts_kernel(const int32_t* part, int rows, int E, int32_t* counts) {
  __shared__ int32_t sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = blockIdx.x * 64 + lane;
  int32_t n = 0;
  for (int i0 = wave; i0 < rows; i0 += 16 * 16) {
    int32_t v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) v[u] = part[(int64_t)min(i0 + 16 * u, rows - 1) * E + min(e, E - 1)];
#pragma unroll
    for (int u = 0; u < 16; ++u) n += i0 + 16 * u < rows ? v[u] : 0;
  }
  sums[wave][lane] = n;
  __syncthreads();
  if (wave != 0 || e >= E) return;
  n = 0;
  for (int w = 0; w < 16; ++w) n += sums[w][lane];
  counts[e] = n;
}

// The backward reads the logits again (softmax) or the chosen ones alone (sigmoid) and writes every
// dlogit: 9.0 us at T 16384, E 160, softmax (2.3 TB/s of logits and dlogits).  Its lanes: with VEC
// a lane's experts come in fours, 4 (c + LPT i) .. + 3, so that consecutive lanes write whole lines;
// else c + LPT i.
template <int LPT, bool VEC>
__device__ __forceinline__ int route_expert(int c, int q) {
  return VEC ? 4 * (c + LPT * (q >> 2)) + (q & 3) : c + LPT * q;
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
#pragma unroll
    for (int q = 0; q < EPL; q += VEC ? 4 : 1) {
      const int e = route_expert<LPT, VEC>(c, q);
      const bool on = live && e < a.E;
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
  DSMOE_REQUIRE(d->T <= INT32_MAX - 4096, DSMOE_ERR_UNSUPPORTED, "route_experts: too many tokens");
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

// Blocks: one of up to 16 waves where that holds all tokens (it writes the counts itself),
// else of four waves, up to 1024 of them.
static int route_blocks(int T, int E) {
  const int tok = E <= 256 ? 4 : 1;   // tokens of a wave
  return T <= 16 * tok ? 1 : (int)std::min<int64_t>(1024, cdiv(T, 4 * tok));
}

template <int LPT, int EPL, int W, bool SOFTMAX>
static void route_launch(RouteArgs a, hipStream_t st) {
  a.lanes_of_group = a.gs % EPL == 0 ? a.gs / EPL : 0;
  constexpr int TOK = 64 / LPT;
  const int waves = a.T <= 16 * TOK ? (int)cdiv(a.T, TOK) : 4;
  const int blocks = route_blocks(a.T, a.E);
  a.per = (int)cdiv(a.T, blocks);
  if (blocks == 1 || !a.counts) a.part = nullptr;
  const size_t lds = sizeof(float) * (a.E + (a.G > 1 && a.lanes_of_group == 0 ? (size_t)waves * TOK * (a.E + 64) : 0));
  // (a block of 16 waves has half of the registers that the widest lanes would use)
  auto kern = waves > 4 ? route_experts_kernel<LPT, EPL, W, SOFTMAX, 1024> : route_experts_kernel<LPT, EPL, W, SOFTMAX, 256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(64 * waves), lds, st, a);
  if (a.part)
    hipLaunchKernelGGL(route_counts_kernel, dim3((unsigned)cdiv(a.E, 64)), dim3(1024), 0, st, a.part, blocks, a.E, a.counts);
}

template <int LPT, int EPL>
static void route_pick(const RouteArgs& a, bool softmax, hipStream_t st) {
  const auto by_score = [&](auto w) {
    constexpr int W = decltype(w)::value;
    softmax ? route_launch<LPT, EPL, W, true>(a, st) : route_launch<LPT, EPL, W, false>(a, st);
  };
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.bias);
  if constexpr (EPL % 4 == 0)
    if (a.E % 4 == 0 && at % 16 == 0) return by_score(std::integral_constant<int, 4>{});
  if constexpr (EPL % 2 == 0 && EPL % 4 != 0)
    if (a.E % 2 == 0 && at % 8 == 0) return by_score(std::integral_constant<int, 2>{});
  by_score(std::integral_constant<int, 1>{});
}

static int route_fwd(const RouteArgs& a, int score, hipStream_t st) {
  const bool sm = score == DSMOE_SCORE_SOFTMAX;
  // 16 lanes a token up to 256 experts.  (A wave a token above 64 experts, as many waves again to
  // hide what the 16 lanes wait for, took 21 us against 22 at E 256, T 8192, but 34 against 20 at
  // E 160, softmax, T 16384: its rounds serve one token where these serve four.)
  const int need = (a.E + 15) / 16;
  if (need <= 1) route_pick<16, 1>(a, sm, st);
  else if (need <= 2) route_pick<16, 2>(a, sm, st);
  else if (need <= 4) route_pick<16, 4>(a, sm, st);
  else if (need <= 6) route_pick<16, 6>(a, sm, st);
  else if (need <= 8) route_pick<16, 8>(a, sm, st);
  else if (need <= 10) route_pick<16, 10>(a, sm, st);
  else if (need <= 12) route_pick<16, 12>(a, sm, st);
  else if (need <= 16) route_pick<16, 16>(a, sm, st);
  else route_pick<64, 8>(a, sm, st);
  return check_launch("route_experts");
}

template <int LPT, int EPL>
static void route_bwd_pick(const RouteArgs& a, bool vec, bool softmax, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(a.T, ROUTE_WAVES * (64 / LPT)));
  const auto run = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(64 * ROUTE_WAVES), 0, st, a); };
  if constexpr (EPL % 4 == 0)
    if (vec) return softmax ? run(route_experts_bwd_kernel<LPT, EPL, true, true>) : run(route_experts_bwd_kernel<LPT, EPL, true, false>);
  softmax ? run(route_experts_bwd_kernel<LPT, EPL, false, true>) : run(route_experts_bwd_kernel<LPT, EPL, false, false>);
}

static int route_bwd(const RouteArgs& a, int score, hipStream_t st) {
  const auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.E % 4 == 0 && al(a.logits) && al(a.dlogits);
  const bool sm = score == DSMOE_SCORE_SOFTMAX;
  if (a.E <= 16) route_bwd_pick<16, 1>(a, false, sm, st);
  else if (a.E <= 32) route_bwd_pick<16, 2>(a, false, sm, st);
  else if (a.E <= 64) route_bwd_pick<16, 4>(a, vec, sm, st);
  else if (a.E <= 128) route_bwd_pick<16, 8>(a, vec, sm, st);
  else if (a.E <= 192) route_bwd_pick<16, 12>(a, vec, sm, st);
  else if (a.E <= 256) route_bwd_pick<16, 16>(a, vec, sm, st);
  else route_bwd_pick<64, 8>(a, vec, sm, st);
  return check_launch("route_experts_bwd");
}

}  // namespace dsmoe

using namespace dsmoe;

extern "C" size_t dsmoe_route_experts_workspace_size(const dsmoe_route_dims* dims) {
  if (route_validate(dims)) return 0;
  const int blocks = route_blocks(dims->T, dims->E);
  return std::max<size_t>(256, blocks > 1 ? sizeof(int32_t) * blocks * dims->E : 0);
}

extern "C" int dsmoe_route_experts(const float* logits, const float* bias, const dsmoe_route_dims* dims, float* weights,
                                   int32_t* idx, int32_t* counts, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const int rc = route_validate(dims);
  if (rc) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dims->T == 0) {
    if (!counts) return DSMOE_OK;
    launch_fill_i32(counts, dims->E, 0, st);
    return check_launch("route_experts");
  }
  DSMOE_REQUIRE(logits && weights && idx, DSMOE_ERR_INVALID, "route_experts: NULL pointer");
  DSMOE_REQUIRE(!counts || (workspace && workspace_bytes >= dsmoe_route_experts_workspace_size(dims)),
                DSMOE_ERR_WORKSPACE, "route_experts: workspace too small");
  RouteArgs a = route_args(dims);
  a.logits = logits; a.bias = bias; a.weights = weights; a.idx = idx; a.counts = counts;
  a.part = static_cast<int32_t*>(workspace);
  return route_fwd(a, dims->score, st);
}

extern "C" int dsmoe_route_experts_bwd(const float* logits, const int32_t* idx, const float* dweights,
                                       const dsmoe_route_dims* dims, float* dlogits, void* stream) {
  const int rc = route_validate(dims);
  if (rc) return rc;
  if (dims->T == 0) return DSMOE_OK;
  DSMOE_REQUIRE(logits && idx && dweights && dlogits, DSMOE_ERR_INVALID, "route_experts_bwd: NULL pointer");
  RouteArgs a = route_args(dims);
  a.logits = logits; a.idx = const_cast<int32_t*>(idx); a.dweights = dweights; a.dlogits = dlogits;
  return route_bwd(a, dims->score, static_cast<hipStream_t>(stream));
}
