// MLA attention of the new tokens of many sequences over a paged latent cache, on
// the latent rows: the causal attention of models/mla_triton.py:73-183 with pages, ragged
// lengths and decoded tokens beside chunks of prompts, and no K and V built.
//
// With k_nope = c W_k^T and v = c W_v^T for a latent row c, a query's score is
// (q_nope W_k) . c + q_pe . pe and its output (sum_j p_j c_j) W_v^T, so a pass reads
// each visible latent row once for up to 32 (token, head) rows.  A sequence's rows are
// (new token, head) pairs, head fastest, n H of them in tiles of 32; tile numbers start
// at floor(offset H / 32) + b for sequence b, which leaves every sequence enough of them
// whatever the lengths, so the grid needs no lengths on the host.
//
//   paged_absorb_kernel  q_abs = q_nope W_k in fp32, kept as an exact pair of bf16 parts
//                        (hi, lo: about 16 significant bits), followed by q_pe.
//   paged_few_kernel     flash attention of 32 rows over one range of keys per wave.
//   paged_out_kernel     the ranges added by their weights, times W_v^T in fp32.
//
// Masked places: positions behind a sequence's length are never read (a lane past the
// last visible key reads that key again), a page outside the pool reads page 0 and is
// masked, and where the rows of a tile see different keys a latent row with a NaN or an
// infinity is taken as zeros for p c, with the score NaN for the rows that do see it: it
// reaches those and no other.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cstring>

#include "mla_paged.h"
#include "mla_tile.h"

namespace dsmoe {

constexpr int PG_MAX_SPLITS = 128;

// 8 bf16 at p (16 bytes), or those of p[0 .. n) one by one and zeros.
__device__ __forceinline__ bf16x8_t pg_ld8(const bf16_t* p, int n, bool vec) {
  mla_u32x4 v;
  if (vec) {
    v = *reinterpret_cast<const mla_u32x4*>(p);
  } else {
    bf16_t e8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) e8[e] = e < n ? p[e] : bf16_t(0);
    v = *reinterpret_cast<const mla_u32x4*>(e8);
  }
  return __builtin_bit_cast(bf16x8_t, v);
}

// The first position that no row of tile mt sees (0: nothing to see).
__device__ __forceinline__ int pg_kend(const PagedSeq& s, int H, int mt) {
  return max(0, min(s.kv, s.first + (min(s.m * H, 32 * mt + 32) - 1) / H + 1));
}

// Key ranges that hold keys, of a tile that sees kend of them.
__device__ __forceinline__ int pg_ranges(const PagedAttn& a, int kend) {
  return min(a.nsplit, (kend + 32 * a.cpw - 1) / (32 * a.cpw));
}

__device__ __forceinline__ void paged_absorb_row(const PagedAttn& a, int rt, int h) {
  extern __shared__ __attribute__((aligned(16))) float pg_sm[];
  const int tid = threadIdx.x;
  int t = rt;
  if (a.p.rows != a.p.offsets) {
    const PagedSeq s = paged_seq(a.p, paged_find(a.p, a.p.rows, rt, 1, 1, 0));
    t = s.t0 + rt - s.r0;
  }
  const bf16_t* qn = a.q_nope + t * a.qn_ts + h * a.qn_hs;
  const bf16_t* qp = a.q_pe + t * a.qp_ts + h * a.qp_hs;
  bf16_t* dst = a.qabs + ((int64_t)rt * a.H + h) * (2 * a.Rq + a.Drp);
  const int cols = a.Rq / 8, groups = 256 / cols;
  const int g = tid / cols, c = tid - g * cols;
  if (g < groups) {
    float acc[8] = {};
    const int n = min(8, a.R - 8 * c);
    const bf16_t* w = a.w_k + h * a.wk_hs + 8 * c;
    if (n > 0) {
#pragma unroll 4
      for (int d = g; d < a.Dn; d += groups) {
        const bf16x8_t v = pg_ld8(w + (int64_t)d * a.R, n, a.wvec != 0);
        const float qd = bf2f(qn[d]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(qd, (float)v[e], acc[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) pg_sm[g * a.Rq + 8 * c + e] = acc[e];
  }
  __syncthreads();
  for (int r = tid; r < a.Rq; r += 256) {
    float v = pg_sm[r];
    for (int i = 1; i < groups; ++i) v += pg_sm[i * a.Rq + r];
    if (a.neg) v = -v;
    const bf16_t hi = f2bf(v);
    dst[r] = hi;
    dst[a.Rq + r] = f2bf(v - bf2f(hi));
  }
  for (int d = tid; d < a.Drp; d += 256)
    dst[2 * a.Rq + d] = d < a.Dr ? (bf16_t)(qp[d] ^ (a.neg ? 0x8000 : 0)) : bf16_t(0);
  __syncthreads();   // the LDS is the next row's
}

// Tokens on the latent rows (at most).
__device__ __forceinline__ int pg_tokens(const PagedAttn& a) {
  return a.p.rows == a.p.offsets ? a.p.T : paged_clamp(a.p.rows[a.p.B], 0, a.p.T);
}

// A block takes (token, head) rows blockIdx.x, + gridDim.x, ..., head by head.  Thread
// (g, c): columns 8 c .. 8 c + 7 over the D_nope rows g, g + groups, ..., the groups added
// through LDS.
__global__ __launch_bounds__(256) void paged_absorb_kernel(const PagedAttn a) {
  const int tokens = pg_tokens(a);
  for (int i = blockIdx.x; i < tokens * a.H; i += gridDim.x) {
    const int h = i / tokens;
    paged_absorb_row(a, i - h * tokens, h);
  }
}
// One wave per (tile, key range), range fastest.  A range without keys writes nothing
// (paged_out_kernel does not read it).  NS = Rq / 16; VEC: 16-byte loads of latent and
// rope rows.
template <int NS, bool VEC>
__global__ __launch_bounds__(256) void paged_few_kernel(const PagedAttn a) {
  constexpr int NV = NS / 2;                             // 32-column tiles of the latent row
  constexpr int RB = (NS * 16 + 127) / 128 * 256;        // LDS tile row bytes
  extern __shared__ __attribute__((aligned(16))) char pg_tile[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hi = lane >> 5, l32 = lane & 31;
  const int units = ((int)((int64_t)pg_tokens(a) * a.H / 32) + a.p.B) * a.nsplit;
  for (int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wave); unit < units; unit += 4 * gridDim.x) {
  const int tnum = unit / a.nsplit, split = unit - tnum * a.nsplit;
  const PagedSeq s = paged_seq(a.p, paged_find(a.p, a.p.rows, tnum, a.H, 32, 1));
  if (s.b < 0) continue;
  const int M = s.m * a.H;
  const int mt = tnum - (int)((int64_t)s.r0 * a.H / 32) - s.b;
  if (32 * mt >= M) continue;
  const int kend = pg_kend(s, a.H, mt);
  const int kb = split * a.cpw * 32;
  const int ke = split == a.nsplit - 1 ? kend : min(kend, kb + a.cpw * 32);
  if (kb >= ke) continue;
  const int row = 32 * mt + l32, rowc = min(row, M - 1);
  const int qpos = s.first + rowc / a.H;
  const int64_t grow = (int64_t)s.r0 * a.H + rowc;
  char* tile = pg_tile + wave * 32 * RB;
  const MlbLane<RB> lk(lane);
  const bf16_t* qrow = a.qabs + grow * (2 * a.Rq + a.Drp) + 8 * hi;
  bf16x8_t qh[NS], ql[NS];
#pragma unroll
  for (int st = 0; st < NS; ++st) {
    qh[st] = *reinterpret_cast<const bf16x8_t*>(qrow + 16 * st);
    ql[st] = *reinterpret_cast<const bf16x8_t*>(qrow + a.Rq + 16 * st);
  }
  mla_f32x16 o[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[v][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  // the lane's latent and rope row of a chunk, clamped to the last visible key; columns
  // past R: whole-chunk loads repeat the row's last ones (q_abs is zero there)
  bf16x8_t cf[NS];
  const bf16_t* pr = a.pe_pages;
  bool there = true;
  const auto load = [&](int k0) {
    int in_page;
    const int page = paged_page(a.p, s.b, min(k0 + l32, ke - 1), in_page);
    there = page >= 0 && k0 + l32 < ke;
    const int64_t pg = max(page, 0);
    const bf16_t* cr = a.kv_pages + pg * a.p.kv_ps + in_page * a.p.kv_rs;
    pr = a.pe_pages + pg * a.p.pe_ps + in_page * a.p.pe_rs;
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      const int col = 16 * st + 8 * hi;
      cf[st] = VEC ? pg_ld8(cr + min(col, a.R - 8), 8, true) : pg_ld8(cr + col, a.R - col, false);
    }
  };
  load(kb);
  for (int k0 = kb; k0 < ke; k0 += 32) {
    // bit j: key k0 + j is one of the range's; the chunk is an edge where a row of the
    // tile (they stand at first .. kend - 1 or before) may not see all of them
    const uint32_t keys = (uint32_t)__builtin_amdgcn_ballot_w64(there);
    const bool edge = keys != 0xffffffffu || k0 + 31 > s.first + 32 * mt / a.H;
    uint32_t bad = 0;
    if (edge) {
      uint32_t mx = 0;
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const mla_u32x4 w = __builtin_bit_cast(mla_u32x4, cf[st]);
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = max(mx, max((w[i] << 16) & 0x7fff0000u, w[i] & 0x7fff0000u));
      }
      const bool nf = mx >= 0x7f800000u;
      const uint64_t bl = __builtin_amdgcn_ballot_w64(nf);
      bad = (uint32_t)bl | (uint32_t)(bl >> 32);
      if ((bad >> l32) & 1)
#pragma unroll
        for (int st = 0; st < NS; ++st) cf[st] = __builtin_bit_cast(bf16x8_t, mla_u32x4{0u, 0u, 0u, 0u});
    }
#pragma unroll
    for (int st = 0; st < NS; ++st)
      *reinterpret_cast<bf16x8_t*>(tile + lk.f[st & 7] + 256 * (st >> 3)) = cf[st];
    // scores: register i -> key k0 + 8 (i / 4) + 4 hi + i % 4
    mla_f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    for (int d = 8 * hi; d < a.Drp; d += 16) {
      const bf16x8_t pf = VEC ? pg_ld8(pr + min(d, a.Dr - 8), 8, true) : pg_ld8(pr + d, a.Dr - d, false);
      z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          pf, *reinterpret_cast<const bf16x8_t*>(qrow + 2 * a.Rq + d - 8 * hi), z, 0, 0, 0);
    }
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cf[st], ql[st], z, 0, 0, 0);
      z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cf[st], qh[st], z, 0, 0, 0);
    }
    if (k0 + 32 < ke) load(k0 + 32);
    if (edge) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = 8 * (i >> 2) + 4 * hi + (i & 3);
        if ((bad >> j) & 1) z[i] = __builtin_nanf("");
        if (!((keys >> j) & 1) || k0 + j > qpos) z[i] = -INFINITY;
      }
    }
    float mb = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mb = fmaxf(mb, z[i]);
    mb = mla_pair_max(mb);
    const float mn = fmaxf(m, mb);
    const float mc = mn == -INFINITY ? 0.0f : mn * a.c;
    const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(m, a.c, -mc));
    const bool moved = m != mn;
    m = mn;
    float ls = 0.0f;
    bf16x8_t pf[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      bf16x2_t w[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(fmaf(z[8 * half + e], a.c, -mc));
        ls += p;
        w[e >> 1][e & 1] = (__bf16)p;   // as mla.hip rounds it; l takes the unrounded p
      }
      pf[half] = __builtin_bit_cast(bf16x8_t, w);
    }
    l = l * alpha + ls;
    if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[v][i] *= alpha;
    }
    // the tile's writes (this wave's own, completed in order) before its transposed reads
    wait_lgkm0();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int ps = 0; ps < 2; ++ps)
#pragma unroll
      for (int v = 0; v < NV; ++v)
        o[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lk.tfrag(tile, 16 * ps, v), pf[ps], o[v], 0, 0, 0);
    wait_lgkm0();
    asm volatile("" ::: "memory");
  }
  l = mla_pair_sum(l);
  if (row >= M) continue;
  const int64_t part = (int64_t)split * a.p.T * a.H + grow;
  if (hi == 0) a.ml[part] = make_float2(m, l);
  float* po = a.po + part * a.Rq;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(po + 32 * v + 8 * g + 4 * hi) =
          make_float4(o[v][4 * g], o[v][4 * g + 1], o[v][4 * g + 2], o[v][4 * g + 3]);
  }
}

// The ranges of a row added by their weights.  Every range that paged_few_kernel wrote
// takes part, so a NaN in its sums reaches the output also through a weight of 0.  A
// row that saw no key gives zeros.
// Rows as paged_absorb_kernel takes them.  LDS (floats): weights of the ranges [PG_MAX_SPLITS] | group sums
// [groups][Rq] (the first row then holds the normalised sum).
__device__ __forceinline__ void paged_out_row(const PagedAttn& a, int rt, int h) {
  extern __shared__ __attribute__((aligned(16))) float pg_sm[];
  float* wt = pg_sm;
  float* sum = pg_sm + PG_MAX_SPLITS;
  const int tid = threadIdx.x;
  const PagedSeq s = paged_seq(a.p, paged_find(a.p, a.p.rows, rt, 1, 1, 0));
  const int i0 = rt - s.r0;
  if (s.b < 0 || i0 >= s.m) return;
  const int64_t rows = (int64_t)a.p.T * a.H, p0 = (int64_t)rt * a.H + h;
  const int nr = pg_ranges(a, pg_kend(s, a.H, (i0 * a.H + h) / 32));
  bf16_t* orow = a.out + ((int64_t)(s.t0 + i0) * a.H + h) * a.Dv;
  if (nr == 0) {
    for (int dv = tid; dv < a.Dv; dv += 256) orow[dv] = bf16_t(0);
    return;
  }
  // every wave reduces the ranges' maxima and normalisers, two ranges per lane
  const int lane = tid & 63;
  static_assert(PG_MAX_SPLITS == 128, "two ranges per lane");
  float2 r2[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 64 * u;
    r2[u] = a.ml[p0 + min(i, nr - 1) * rows];
    if (i >= nr) r2[u] = make_float2(-INFINITY, 0.0f);
  }
  float m = fmaxf(r2[0].x, r2[1].x);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  float lt = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    // a range whose scores are all NaN has no maximum, and a NaN for its sum
    const float w = r2[u].x != -INFINITY ? __builtin_amdgcn_exp2f((r2[u].x - m) * a.c) : 0.0f;
    lt = fmaf(w, r2[u].y, lt);
    if (tid < 64) wt[lane + 64 * u] = w;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) lt += __shfl_xor(lt, d);
  __syncthreads();
  const int cols = a.Rq / 4, groups = 256 / cols;
  const int g = tid / cols, c = tid - g * cols;
  if (g < groups) {
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float* po = a.po + p0 * a.Rq + 4 * c;
    const int64_t step = rows * a.Rq;
    constexpr int U = 6;   // loads in flight
    for (int i = g; i < nr; i += U * groups) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = *reinterpret_cast<const float4*>(po + min(i + u * groups, nr - 1) * step);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = i + u * groups < nr;
        const float w = wt[min(i + u * groups, PG_MAX_SPLITS - 1)];
        acc.x = fmaf(w, on ? v[u].x : 0.0f, acc.x);
        acc.y = fmaf(w, on ? v[u].y : 0.0f, acc.y);
        acc.z = fmaf(w, on ? v[u].z : 0.0f, acc.z);
        acc.w = fmaf(w, on ? v[u].w : 0.0f, acc.w);
      }
    }
    *reinterpret_cast<float4*>(sum + g * a.Rq + 4 * c) = acc;
  }
  __syncthreads();
  const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;   // (a NaN stays one)
  for (int r = tid; r < a.Rq; r += 256) {
    float v = sum[r];
    for (int i = 1; i < groups; ++i) v += sum[i * a.Rq + r];
    sum[r] = v * inv;
  }
  __syncthreads();
  // four lanes per output column, every fourth chunk of 8 latent columns each
  const int q4 = tid & 3;
  for (int dv = tid >> 2; dv < a.Dv; dv += 64) {
    const bf16_t* w = a.w_v + h * a.wv_hs + (int64_t)dv * a.R;
    float acc = 0.0f;
#pragma unroll 4
    for (int r = 8 * q4; r < a.R; r += 32) {
      const bf16x8_t v = pg_ld8(w + r, a.R - r, a.wvec != 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc = fmaf(sum[min(r + e, a.Rq - 1)], (float)v[e], acc);
    }
    acc += __shfl_xor(acc, 1);
    acc += __shfl_xor(acc, 2);
    if (q4 == 0) orow[dv] = f2bf(acc);
  }
}

__global__ __launch_bounds__(256) void paged_out_kernel(const PagedAttn a) {
  const int tokens = pg_tokens(a);   // rows behind the last sequence stay as they were
  for (int i = blockIdx.x; i < tokens * a.H; i += gridDim.x) {
    const int h = i / tokens;
    if (i >= (int)gridDim.x) __syncthreads();   // the LDS is the last row's
    paged_out_row(a, i - h * tokens, h);
  }
}

// ------------------------------------------------------------------ host
static int pg_validate(const dsmoe_mla_paged_dims* d) {
  const int rc = paged_validate(d);
  if (rc) return rc;
  DSMOE_REQUIRE(d->H > 0 && d->D_nope > 0 && d->D_v > 0 && d->D_nope <= 256 && d->D_v <= 256, DSMOE_ERR_INVALID,
                "mla_paged: H must be positive, D_nope and D_v in 1 .. 256");
  DSMOE_REQUIRE(d->D_nope + d->D_rope <= 256, DSMOE_ERR_UNSUPPORTED, "mla_paged: D_nope + D_rope > 256 is not supported");
  DSMOE_REQUIRE(d->H <= 65535, DSMOE_ERR_UNSUPPORTED, "mla_paged: more than 65535 heads");
  DSMOE_REQUIRE((int64_t)d->T * d->H < (int64_t(1) << 24) && d->B < (1 << 24), DSMOE_ERR_UNSUPPORTED,
                "mla_paged: T H and B must stay below 2^24");
  DSMOE_REQUIRE(d->max_kv >= 0 && d->max_q >= 0, DSMOE_ERR_INVALID, "mla_paged: negative max_q or max_kv");
  return DSMOE_OK;
}

// More new tokens of a sequence than this have its K and V built (mla_paged_kv.hip):
// for one (head, key) the latent rows cost 6 R + 2 D_rope operations a token (the two
// parts of q_abs among them) against 2 (D_nope + D_rope + D_v), and K and V 2 R (D_nope + D_v) once.
static int pg_threshold(const dsmoe_mla_paged_dims* d) {
  const int64_t build = (int64_t)2 * d->R * (d->D_nope + d->D_v);
  const int64_t more = 6 * d->R + 2 * d->D_rope - 2 * (d->D_nope + d->D_rope + d->D_v);
  return more <= 0 ? INT_MAX : (int)std::max<int64_t>(16, build / more);
}

static PagedAttn pg_args(const dsmoe_mla_paged_dims* d, size_t* bytes, void* ws) {
  PagedAttn a;
  std::memset(static_cast<void*>(&a), 0, sizeof(a));
  a.p = paged_batch(d, nullptr, nullptr, nullptr);
  a.H = d->H; a.R = d->R; a.Dn = d->D_nope; a.Dr = d->D_rope; a.Dv = d->D_v;
  for (int ns : {2, 4, 8, 12, 16})
    if (a.Rq == 0 && d->R <= 16 * ns) a.Rq = 16 * ns;
  a.Drp = (int)align_up(d->D_rope, 16);
  a.neg = d->softmax_scale < 0.0f ? 1 : 0;
  // not below the smallest normal number: a masked score, -infinity, stays one for a scale of 0
  a.c = std::max((d->softmax_scale < 0.0f ? -d->softmax_scale : d->softmax_scale) * MLA_LOG2E, FLT_MIN);
  Carver c(ws);
  a.thr = pg_threshold(d);
  // with longer chunks about, most of the tokens are theirs: as many row tiles here as
  // every sequence has for one token
  const size_t rows = (size_t)a.p.T * a.H;
  const bool both = d->max_q > a.thr && paged_kv_carve(a, d, c) > 0;
  if (!both) a.slots = 0;
  const int64_t tiles = std::max<int64_t>(1, cdiv(both ? (int64_t)d->B * d->H : (int64_t)rows, 32));
  // about 1024 waves (four for each CU) if every sequence were as long as the longest
  const int64_t chunks = std::max<int64_t>(1, cdiv(d->max_kv, 32));
  a.cpw = (int)std::max<int64_t>(std::max<int64_t>(1, tiles * chunks / 1024), cdiv(chunks, PG_MAX_SPLITS));
  // the partial sums of all rows in 256 MB, or one range
  const int64_t most = std::max<int64_t>(1, (int64_t(256) << 20) / std::max<int64_t>(1, (int64_t)rows * a.Rq * 4));
  a.cpw = (int)std::max<int64_t>(a.cpw, cdiv(chunks, most));
  a.nsplit = (int)cdiv(chunks, a.cpw);
  a.qabs = c.take<bf16_t>(rows * (2 * a.Rq + a.Drp));
  a.ml = c.take<float2>(rows * a.nsplit);
  a.po = c.take<float>(rows * a.nsplit * a.Rq);
  *bytes = c.used();
  return a;
}

template <int NS>
static int launch_paged_few(const PagedAttn& a, hipStream_t st) {
  constexpr size_t lds = 4 * 32 * ((NS * 16 + 127) / 128 * 256);
  auto kern = a.kvvec ? paged_few_kernel<NS, true> : paged_few_kernel<NS, false>;
  int64_t blocks = cdiv(((int64_t)a.p.T * a.H / 32 + a.p.B) * a.nsplit, 4);
  if (a.slots) blocks = std::min<int64_t>(blocks, 2048);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, a);
  return check_launch("mla_paged_few");
}

}  // namespace dsmoe

using namespace dsmoe;

extern "C" size_t dsmoe_mla_attn_paged_workspace_size(const dsmoe_mla_paged_dims* dims) {
  if (pg_validate(dims)) return 0;
  size_t need = 0;
  pg_args(dims, &need, nullptr);
  return std::max<size_t>(need, 256);
}

extern "C" int dsmoe_mla_attn_paged(const void* q_nope, const void* q_pe, const void* kv_pages, const void* pe_pages,
                                    const int32_t* block_table, const int32_t* kv_lens, const int32_t* q_offsets,
                                    const void* wkv_b_k, int64_t wk_head_stride, const void* wkv_b_v,
                                    int64_t wv_head_stride, const dsmoe_mla_paged_dims* dims, void* out,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  int rc = pg_validate(dims);
  if (rc) return rc;
  if (dims->T == 0 || dims->B == 0) return DSMOE_OK;
  DSMOE_REQUIRE(q_nope && q_pe && kv_pages && pe_pages && kv_lens && q_offsets && wkv_b_k && wkv_b_v && out &&
                    (block_table || dims->table_width == 0), DSMOE_ERR_INVALID, "mla_paged: NULL tensor pointer");
  DSMOE_REQUIRE(wk_head_stride >= 0 && wv_head_stride >= 0 && dims->qn_token_stride >= 0 && dims->qn_head_stride >= 0 &&
                    dims->qp_token_stride >= 0 && dims->qp_head_stride >= 0, DSMOE_ERR_INVALID,
                "mla_paged: negative stride");
  size_t need = 0;
  PagedAttn a = pg_args(dims, &need, workspace);
  DSMOE_REQUIRE(workspace && workspace_bytes >= need, DSMOE_ERR_WORKSPACE, "mla_paged: workspace too small");
  const auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  DSMOE_REQUIRE(al(workspace), DSMOE_ERR_INVALID, "mla_paged: workspace must be 16-byte aligned");
  a.p = paged_batch(dims, block_table, kv_lens, q_offsets);
  a.q_nope = static_cast<const bf16_t*>(q_nope);
  a.q_pe = static_cast<const bf16_t*>(q_pe);
  a.qn_ts = dims->qn_token_stride; a.qn_hs = dims->qn_head_stride;
  a.qp_ts = dims->qp_token_stride; a.qp_hs = dims->qp_head_stride;
  a.kv_pages = static_cast<const bf16_t*>(kv_pages);
  a.pe_pages = static_cast<const bf16_t*>(pe_pages);
  a.w_k = static_cast<const bf16_t*>(wkv_b_k);
  a.w_v = static_cast<const bf16_t*>(wkv_b_v);
  a.wk_hs = wk_head_stride;
  a.wv_hs = wv_head_stride;
  a.out = static_cast<bf16_t*>(out);
  a.wvec = (a.R % 8 == 0 && wk_head_stride % 8 == 0 && wv_head_stride % 8 == 0 && al(wkv_b_k) && al(wkv_b_v)) ? 1 : 0;
  a.kvvec = (a.R % 8 == 0 && a.Dr % 8 == 0 && a.p.kv_ps % 8 == 0 && a.p.kv_rs % 8 == 0 && a.p.pe_ps % 8 == 0 &&
             a.p.pe_rs % 8 == 0 && al(kv_pages) && al(pe_pages)) ? 1 : 0;
  a.qvec = (a.Dn % 8 == 0 && a.Dr % 8 == 0 && a.qn_ts % 8 == 0 && a.qn_hs % 8 == 0 && a.qp_ts % 8 == 0 &&
            a.qp_hs % 8 == 0 && al(q_nope) && al(q_pe)) ? 1 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int64_t blocks = (int64_t)a.p.T * a.H;
  if (a.slots) {
    rc = launch_paged_plan(a, st);
    if (rc) return rc;
    rc = launch_paged_kv(a, st);
    if (rc) return rc;
    a.p.rows = a.plan_rows;
    // most of the tokens are not the latent rows': blocks that take several
    blocks = std::min<int64_t>(blocks, 4096);
  }
  hipLaunchKernelGGL(paged_absorb_kernel, dim3((unsigned)blocks), dim3(256), sizeof(float) * (256 / (a.Rq / 8)) * a.Rq, st, a);
  rc = check_launch("mla_paged_absorb");
  if (rc) return rc;
  switch (a.Rq / 16) {
    case 2: rc = launch_paged_few<2>(a, st); break;
    case 4: rc = launch_paged_few<4>(a, st); break;
    case 8: rc = launch_paged_few<8>(a, st); break;
    case 12: rc = launch_paged_few<12>(a, st); break;
    default: rc = launch_paged_few<16>(a, st); break;
  }
  if (rc) return rc;
  hipLaunchKernelGGL(paged_out_kernel, dim3((unsigned)blocks), dim3(256),
                     sizeof(float) * (PG_MAX_SPLITS + (size_t)(256 / (a.Rq / 4)) * a.Rq), st, a);
  return check_launch("mla_paged_out");
}
