// MLA attention of the new tokens of many sequences over a paged latent cache, on
// the latent rows: the causal attention of models/mla_triton.py:73-183 with pages, ragged
// lengths and decoded tokens beside chunks of prompts, and no K and V built.
//
// With k_nope = c W_k^T and v = c W_v^T for a latent row c, a query's score is
// (q_nope W_k) . c + q_pe . pe and its output (sum_j p_j c_j) W_v^T, so a pass reads
// each visible latent row once for up to 32 (token, head) rows.  A sequence's rows are
// (new token, head) pairs, head fastest, n H of them in tiles of 16 or 32 (16 rt); tile numbers
// start at floor(offset H / (16 rt)) + b for sequence b, which leaves every sequence enough of
// them whatever the lengths, so no grid needs lengths on the host.
//
//   paged_absorb_kernel  q_abs = q_nope W_k in fp32, kept as an exact pair of bf16 parts
//                        (hi, lo: about 16 significant bits), followed by q_pe.
//   paged_few_kernel     flash attention: even shares of all tiles' keys per block.
//   paged_out_kernel     a tile's parts added by their weights, times W_v^T in fp32.
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

// Row tiles: rows of one, a sequence's first one, and the first position that no row of
// its tile mt sees (0: nothing to see).
__device__ __forceinline__ int pg_tile0(const PagedAttn& a, const PagedSeq& s) {
  return (int)((int64_t)s.r0 * a.H / (16 * a.rt)) + s.b;
}
__device__ __forceinline__ int pg_kend(const PagedAttn& a, const PagedSeq& s, int mt) {
  return max(0, min(s.kv, s.first + (min(s.m * a.H, 16 * a.rt * (mt + 1)) - 1) / a.H + 1));
}

// Tokens on the latent rows (at most).
__device__ __forceinline__ int pg_tokens(const PagedAttn& a) {
  return a.p.rows == a.p.offsets ? a.p.T : paged_clamp(a.p.rows[a.p.B], 0, a.p.T);
}

// A block takes (token, head) rows blockIdx.x, + gridDim.x, ..., head by head.  Thread
// (g, c): columns 8 c .. 8 c + 7 over the D_nope rows g, g + groups, ..., the groups added
// through LDS.  The first weight rows are on their way while the token is looked up.  What
// bounds it is that chain (token, query, LDS, stores), not its bytes: 5 us for one token of 12
// heads (D_nope 48, R 192), 6.7 for 64, 8.0 for 12 tokens of 32 heads (128, 256).
template <bool WVEC>
__global__ __launch_bounds__(256, 4) void paged_absorb_kernel(const PagedAttn a) {
  extern __shared__ __attribute__((aligned(16))) float pg_sm[];
  const int tid = threadIdx.x;
  const int cols = a.Rq / 8, groups = 256 / cols;
  const int g = tid / cols, c = tid - g * cols;
  const int n = min(8, a.R - 8 * c);
  const bool on = g < groups && n > 0;
  if (a.p.rows == a.p.offsets && blockIdx.x == gridDim.x - 1 && tid < 64) {   // (else paged_plan_kernel's)
    PagedUnits units;
    for (int b0 = 0; b0 < a.p.B; b0 += 64) {
      const PagedSeq s = paged_seq(a.p, min(b0 + tid, a.p.B - 1));
      paged_unit_step(a, b0 + tid, s.m, s.kv, units);
    }
    paged_unit_end(a, units);
  }
  const int tokens = pg_tokens(a);
  for (int i = blockIdx.x; i < tokens * a.H; i += gridDim.x) {
    const int h = i / tokens, rt = i - h * tokens;
    constexpr int U = 5;
    const bf16_t* w = a.w_k + h * a.wk_hs + 8 * c;
    bf16x8_t v0[U];
    if (on)
#pragma unroll
      for (int u = 0; u < U; ++u) v0[u] = pg_ld8(w + (int64_t)min(g + u * groups, a.Dn - 1) * a.R, n, WVEC);
    const PagedSeq s = paged_at<PAGED_ROWS>(a.p, rt, 1, 1, 0);
    const int i0 = rt - s.r0;   // (below 0: offsets that decrease)
    if (s.b < 0 || i0 < 0 || i0 >= s.m) continue;
    const int t = s.t0 + i0, row = i0 * a.H + h;
    const bf16_t* qn = a.q_nope + t * a.qn_ts + h * a.qn_hs;
    const bf16_t* qp = a.q_pe + t * a.qp_ts + h * a.qp_hs;
    // column d of part (0: hi, 1: lo, 2: pe) of the row, as paged_few_kernel's lanes take it
    bf16_t* base = a.qabs + ((int64_t)pg_tile0(a, s) * a.rt + row / 16) * 16 * (2 * a.Rq + a.Drp) + 8 * (row & 15);
    const auto dst = [&](int part, int d) -> bf16_t& {
      return base[512 * (part * (a.Rq / 32) + d / 32) + 128 * (d % 32 / 8) + d % 8];
    };
    if (g < groups) {
      float acc[8] = {};
      if (on) {
        float q0[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float q = bf2f(qn[min(g + u * groups, a.Dn - 1)]);
          q0[u] = g + u * groups < a.Dn ? q : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (g + u * groups < a.Dn) acc[e] = fmaf(q0[u], (float)v0[u][e], acc[e]);
#pragma unroll 4
        for (int d = g + U * groups; d < a.Dn; d += groups) {
          const bf16x8_t v = pg_ld8(w + (int64_t)d * a.R, n, WVEC);
          const float qd = bf2f(qn[d]);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = fmaf(qd, (float)v[e], acc[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) pg_sm[g * a.Rq + 8 * c + e] = acc[e];
    }
    for (int d = tid; d < a.Drp; d += 256)
      dst(2, d) = d < a.Dr ? (bf16_t)(qp[d] ^ (a.neg ? 0x8000 : 0)) : bf16_t(0);
    __syncthreads();
    for (int r = tid; r < a.Rq; r += 256) {
      float v = pg_sm[r];
      for (int u = 1; u < groups; ++u) v += pg_sm[u * a.Rq + r];
      if (a.neg) v = -v;
      const bf16_t hi = f2bf(v);
      dst(0, r) = hi;
      dst(1, r) = f2bf(v - bf2f(hi));
    }
    __syncthreads();   // the LDS is the next row's
  }
}

// Maximum and sum over the four lanes that hold a row's keys (l, l + 16, l + 32, l + 48).
__device__ __forceinline__ float pg_quad_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  return mla_pair_max(fmaxf(__int_as_float(r[0]), __int_as_float(r[1])));
}
__device__ __forceinline__ float pg_quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  return mla_pair_sum(__int_as_float(r[0]) + __int_as_float(r[1]));
}

// A block takes its share of the units (paged_unit_step), cut where a tile of 16 RT rows
// ends.  Of its four waves, wave w takes 16 rows and every (4 / RT)-th chunk of 16 G keys, and
// their sums meet in LDS at the end, so that a block leaves one partial row a tile however
// many waves it takes.  A part without visible keys writes nothing (paged_out_kernel does not
// read it).
//
// v_mfma_f32_16x16x32_bf16, keys first, rows second: a lane holds row l % 16 and keys
// 4 (l / 16) + i of either half of the chunk, which is the order in which the PV product
// takes its keys (ds_read_b64_tr_b16 of four rows gives a lane the same ones).  16 rows
// take half of the registers of 32: two waves on a SIMD, one of which computes while the
// other waits.  A chunk's latent and rope rows are loaded while the one before is
// computed, its page numbers one chunk earlier still: three loads in a row would cost their
// latencies one after another.  NS = Rq / 32; NP: 32-column steps of the rope rows held in
// registers (0: any number, loaded where they are used); VEC: 16-byte loads of latent and
// rope rows; FULL: R = 32 NS, no column to clamp.
//
// Measured: 58 us for 12 sequences of 228345 positions together, H 32, R 256, D_rope 64 (146 MB of
// cache: 2.5 TB/s over the launch, 4.2 in the chunks' loop; the start, a lookup, a page and a row
// one after another, and the join are the rest), 19 us for 64 of 82206, H 12, R 192, D_rope 24
// (36 MB), 8 us for one of 300, which is the start.
constexpr float PG_LAZY = 8.0f;   // sums are rescaled once a maximum grew by 2^8: p stays under it

// Groups of 16 keys of a chunk: with the widest rows 64 keys at a time and one wave on a
// SIMD, which has room for them, else 32 and two waves.
constexpr int pg_groups(int ns) { return ns == 8 ? 4 : 2; }

template <int NS, int NP, bool VEC, bool FULL, int RT>
__global__ __launch_bounds__(256, pg_groups(NS) > 2 ? 1 : 2) void paged_few_kernel(const PagedAttn a) {
  constexpr int NC = 2 * NS;                             // 16-column tiles of the latent row
  constexpr int RB = (NS * 32 + 127) / 128 * 256;        // LDS tile row bytes
  constexpr int G = pg_groups(NS);
  constexpr int STEP = 16 * G * 4 / RT;                  // keys from one chunk of a wave to its next
  extern __shared__ __attribute__((aligned(16))) char pg_tile[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int sub = wave % RT, kw = wave / RT;
  const int l16 = lane & 15, kg = lane >> 4;
  char* tile = pg_tile + wave * 16 * G * RB;
  // behind the tiles the lo part of q_abs, [sub][step][lane], in the registers' stead; after the
  // chunks the waves' maxima and sums, [4][16]
  char* slo = pg_tile + 4 * 16 * G * RB;
  const char* qls = slo + sub * NS * 1024 + 16 * lane;
  float2* sml = reinterpret_cast<float2*>(slo);
  // LDS offsets in the mlb_off layout: row l16 (and + 16, by 16 RB) at 16-byte chunk kg, chunk
  // kg + 4 st at fo ^ 64 st; for the transposed reads row 4 kg + l16 / 4 at 8-byte unit l16 % 4,
  // unit l16 % 4 + 4 ct at to ^ 32 ct (within 256 bytes, the swizzle being an exclusive or)
  const int fo = mlb_off(l16, kg, RB);
  const int to = mlb_off(4 * kg + (l16 >> 2), (l16 & 3) >> 1, RB) + ((l16 & 1) << 3);
  const int all = a.p.units[a.p.B], share = a.p.units[a.p.B + 1];
  const int uend = (int)min((int64_t)all, (int64_t)(blockIdx.x + 1) * share);
  for (int64_t u = (int64_t)blockIdx.x * share; u < uend;) {
    const PagedSeq s = paged_at<PAGED_UNITS>(a.p, u, 1, 1, 0);
    if (s.b < 0) return;   // (u lies within the work: never)
    const int per = (s.kv + STEP - 1) / STEP;
    const int mt = (int)(u - s.u0) / per, it0 = (int)(u - s.u0) - mt * per;
    const int its = min(per - it0, (int)(uend - u));
    u += its;
    const int M = s.m * a.H, tnum = pg_tile0(a, s) + mt;
    const int kend = pg_kend(a, s, mt);
    const int kb = it0 * STEP, ke = min(kend, (it0 + its) * STEP);
    if (kb >= ke) continue;
    const int64_t part = (int64_t)(blockIdx.x + tnum) * 16 * RT;   // (numbers of blocks and tiles grow together)
    const int row0 = 16 * (RT * mt + sub), row = row0 + l16;
    const int qpos = s.first + min(row, M - 1) / a.H;
    const int qfirst = s.first + min(row0, M - 1) / a.H;   // the wave's first row's
    // the lane's latent and rope rows of a chunk, clamped to the last visible key; columns
    // past R: whole-chunk loads repeat the row's last ones (q_abs is zero there)
    bf16x8_t cf[G][NS], pf[G][NP > 0 ? NP : 1];
    const bf16_t* pr[G];
    uint64_t keys = 0;   // bit j: key j of the chunk is one of the range's
    // page numbers, one chunk further on than the rows.  Loads return in order: a wait for
    // these must not be one for rows asked for before them, so they are asked for first
    int page[G], in_page[G], npage[G], nin_page[G];
    const auto lookup = [&](int k0) {
#pragma unroll
      for (int g = 0; g < G; ++g) npage[g] = paged_page(a.p, s.b, min(k0 + 16 * g + l16, ke - 1), nin_page[g]);
      __builtin_amdgcn_sched_barrier(0);
    };
    const auto looked_up = [&]() {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        page[g] = npage[g];
        in_page[g] = nin_page[g];
      }
    };
    const auto load = [&](int k0) {
      keys = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const bool there = page[g] >= 0 && k0 + 16 * g + l16 < ke;
        keys |= (__builtin_amdgcn_ballot_w64(there) & 0xffffu) << (16 * g);
        const int64_t pg = max(page[g], 0);
        const bf16_t* cr = a.kv_pages + pg * a.p.kv_ps + in_page[g] * a.p.kv_rs;
        pr[g] = a.pe_pages + pg * a.p.pe_ps + in_page[g] * a.p.pe_rs;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const int col = 32 * st + 8 * kg;
          cf[g][st] = VEC ? pg_ld8(cr + (FULL ? col : min(col, a.R - 8)), 8, true) : pg_ld8(cr + col, a.R - col, false);
        }
#pragma unroll
        for (int st = 0; st < NP; ++st) pf[g][st] = pg_ld8(pr[g] + min(32 * st + 8 * kg, a.Dr - 8), 8, true);
      }
    };
    const int k1 = kb + 16 * G * kw;
    // (chunks behind the range read its last key: nothing of them is used)
    lookup(k1);
    looked_up();
    lookup(k1 + STEP);
    load(k1);
    looked_up();
    const bf16_t* qfrag = a.qabs + (int64_t)(tnum * RT + sub) * 16 * (2 * a.Rq + a.Drp) + 8 * lane;
    bf16x8_t qh[NS], qp[NP > 0 ? NP : 1];
#pragma unroll
    for (int st = 0; st < NS; ++st) qh[st] = *reinterpret_cast<const bf16x8_t*>(qfrag + 512 * st);
#pragma unroll
    for (int st = 0; st < NS; ++st)
      if (st % (4 / RT) == kw)
        *reinterpret_cast<bf16x8_t*>(slo + (sub * NS + st) * 1024 + 16 * lane) =
            *reinterpret_cast<const bf16x8_t*>(qfrag + 512 * (NS + st));
#pragma unroll
    for (int st = 0; st < NP; ++st) {
      qp[st] = *reinterpret_cast<const bf16x8_t*>(qfrag + 512 * (2 * NS + min(st, a.Drp / 32 - 1)));
      if (32 * st >= a.Drp) qp[st] = __builtin_bit_cast(bf16x8_t, mla_u32x4{0u, 0u, 0u, 0u});
    }
    mla_f32x4 o[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = mla_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    __syncthreads();   // the lo parts are there
    for (int k0 = k1; k0 < ke; k0 += STEP) {
      // an edge: some row of the wave may not see all of the chunk's keys
      const uint64_t seen = keys;
      const bool edge = seen != (G == 4 ? ~0ull : (1ull << (16 * G & 63)) - 1) || k0 + 16 * G - 1 > qfirst;
      uint64_t bad = 0;
      if (edge) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t mx = 0;
#pragma unroll
          for (int st = 0; st < NS; ++st) {
            const mla_u32x4 w = __builtin_bit_cast(mla_u32x4, cf[g][st]);
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = max(mx, max((w[i] << 16) & 0x7fff0000u, w[i] & 0x7fff0000u));
          }
          uint64_t bl = __builtin_amdgcn_ballot_w64(mx >= 0x7f800000u);
          bl |= bl >> 32;
          const uint32_t rows = ((uint32_t)bl | (uint32_t)(bl >> 16)) & 0xffffu;
          bad |= (uint64_t)rows << (16 * g);
          if ((rows >> l16) & 1)
#pragma unroll
            for (int st = 0; st < NS; ++st) cf[g][st] = __builtin_bit_cast(bf16x8_t, mla_u32x4{0u, 0u, 0u, 0u});
        }
      }
      // scores: z[g][i] -> key k0 + 16 g + 4 kg + i
      mla_f32x4 z[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        z[g] = mla_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < NS; ++st)
          *reinterpret_cast<bf16x8_t*>(tile + 16 * RB * g + (fo ^ 64 * (st & 3)) + 256 * (st >> 2)) = cf[g][st];
      }
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const bf16x8_t ql = *reinterpret_cast<const bf16x8_t*>(qls + 1024 * st);
#pragma unroll
        for (int g = 0; g < G; ++g) z[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cf[g][st], ql, z[g], 0, 0, 0);
      }
#pragma unroll
      for (int st = 0; st < NS; ++st)
#pragma unroll
        for (int g = 0; g < G; ++g) z[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cf[g][st], qh[st], z[g], 0, 0, 0);
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int st = 0; st < NP; ++st) z[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[g][st], qp[st], z[g], 0, 0, 0);
        if (NP == 0)
          for (int st = 0; 32 * st < a.Drp; ++st) {
            const int d = 32 * st + 8 * kg;
            const bf16x8_t pv = VEC ? pg_ld8(pr[g] + min(d, a.Dr - 8), 8, true) : pg_ld8(pr[g] + d, a.Dr - d, false);
            z[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                pv, *reinterpret_cast<const bf16x8_t*>(qfrag + 512 * (2 * NS + st)), z[g], 0, 0, 0);
          }
      }
      if (k0 + STEP < ke) {
        lookup(k0 + 2 * STEP);
        load(k0 + STEP);
        looked_up();
      }
      if (edge) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 16 * g + 4 * kg + i;
            if ((bad >> j) & 1) z[g][i] = __builtin_nanf("");
            if (!((seen >> j) & 1) || k0 + j > qpos) z[g][i] = -INFINITY;
          }
      }
      float mb = -INFINITY;
#pragma unroll
      for (int g = 0; g < G; ++g) mb = fmaxf(mb, fmaxf(fmaxf(z[g][0], z[g][1]), fmaxf(z[g][2], z[g][3])));
      mb = pg_quad_max(mb);
      // the sums stay under an older maximum until some row's grew by 2^8
      if (__builtin_amdgcn_ballot_w64(mb > m && !((mb - m) * a.c <= PG_LAZY))) {
        const float mn = fmaxf(m, mb);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * a.c);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] *= alpha;
      }
      const float mc = m == -INFINITY ? 0.0f : m * a.c;
      bf16x8_t pv[G / 2];
#pragma unroll
      for (int k = 0; k < G / 2; ++k) {
        bf16x2_t w[4];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(z[2 * k + g][i], a.c, -mc));
            l += p;
            w[2 * g + (i >> 1)][i & 1] = (__bf16)p;   // as mla.hip rounds it; l takes the unrounded p
          }
        pv[k] = __builtin_bit_cast(bf16x8_t, w);
      }
      // the tile's writes (this wave's own, completed in order) before its transposed reads
      wait_lgkm0();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int k = 0; k < G / 2; ++k) {
          const char* at = tile + 32 * RB * k + (to ^ 32 * (c & 7)) + 256 * (c >> 3);
          const mla_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mla_v4s*)(at));
          const mla_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mla_v4s*)(at + 16 * RB));
          typedef short v8s __attribute__((ext_vector_type(8)));
          const v8s v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), pv[k], o[c], 0, 0, 0);
        }
      wait_lgkm0();
      asm volatile("" ::: "memory");
    }
    // the waves' sums under one maximum; a wave without keys has m = -infinity and zeros
    l = pg_quad_sum(l);
    __syncthreads();   // no wave reads the lo parts any more
    if (kg == 0) sml[wave * 16 + l16] = make_float2(m, l);
    __syncthreads();
    float mt4 = -INFINITY, lt = 0.0f;
#pragma unroll
    for (int w = sub; w < 4; w += RT) mt4 = fmaxf(mt4, sml[w * 16 + l16].x);
#pragma unroll
    for (int w = sub; w < 4; w += RT) {
      const float2 v = sml[w * 16 + l16];
      // (scores that are all NaN have no maximum, and a NaN for their sum)
      lt = fmaf(v.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((v.x - mt4) * a.c), v.y, lt);
    }
    const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mt4) * a.c);
    // 16-byte column pieces [tile][lane], each in its wave's own part of the LDS
    float4* own = reinterpret_cast<float4*>(tile);
#pragma unroll
    for (int c = 0; c < NC; ++c) own[c * 64 + lane] = make_float4(o[c][0] * f, o[c][1] * f, o[c][2] * f, o[c][3] * f);
    const int64_t prow = part + 16 * sub + l16;
    if (kw == 0 && kg == 0 && row < M) a.ml[prow] = make_float2(mt4, lt);
    __syncthreads();
    if (row < M) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (c % (4 / RT) != kw) continue;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = sub; w < 4; w += RT) {
          const float4 x = reinterpret_cast<const float4*>(pg_tile + w * 16 * G * RB)[c * 64 + lane];
          v.x += x.x;
          v.y += x.y;
          v.z += x.z;
          v.w += x.w;
        }
        *reinterpret_cast<float4*>(a.po + prow * a.Rq + 16 * c + 4 * kg) = v;
      }
    }
    __syncthreads();   // the LDS is the next tile's
  }
}

// The partial sums of a row added by their weights.  All that paged_few_kernel wrote
// take part, so a NaN in its sums reaches the output also through a weight of 0.  A
// row that saw no key gives zeros.
// Rows as paged_absorb_kernel takes them.  LDS (floats): weights of the parts [PG_MAX_SPLITS] | group sums
// [groups][Rq] (the first row then holds the normalised sum).  Bound by its chain of loads as that
// is: 5.9 us for one token of 12 heads, 7.5 for 64, 9.9 for 12 of 32 heads with up to 37 parts each.
template <bool WVEC>
__global__ __launch_bounds__(256, 4) void paged_out_kernel(const PagedAttn a) {
  extern __shared__ __attribute__((aligned(16))) float pg_sm[];
  float* wt = pg_sm;
  float* sum = pg_sm + PG_MAX_SPLITS;
  const int tid = threadIdx.x, lane = tid & 63;
  const int cols = a.Rq / 4, groups = 256 / cols;
  const int g = tid / cols, c = tid - g * cols;
  const int q4 = tid & 3;
  const int tokens = pg_tokens(a);   // rows behind the last sequence stay as they were
  for (int i = blockIdx.x; i < tokens * a.H; i += gridDim.x) {
    const int h = i / tokens, rt = i - h * tokens;
    // the first weight rows are on their way while the rest is looked up
    const bf16_t* w = a.w_v + h * a.wv_hs;
    constexpr int U = WVEC ? 8 : 1;   // R <= 256: eight chunks of every fourth 8 columns
    bf16x8_t wv[U];
    const auto wload = [&](int dv) {
      if (WVEC)
#pragma unroll
        for (int u = 0; u < U; ++u)
          wv[u] = pg_ld8(w + (int64_t)min(dv, a.Dv - 1) * a.R + min(8 * q4 + 32 * u, a.R - 8), 8, true);
    };
    wload(tid >> 2);
    const int share = max(a.p.units[a.p.B + 1], 1);
    const PagedSeq s = paged_at<PAGED_ROWS, true>(a.p, rt, 1, 1, 0);
    const int i0 = rt - s.r0;
    if (s.b < 0 || i0 < 0 || i0 >= s.m) continue;
    const int row = i0 * a.H + h, mt = row / (16 * a.rt);
    // the units of the row's tile that hold keys it sees, and the blocks that took them
    const int its = (pg_kend(a, s, mt) + a.keys - 1) / a.keys, per = (s.kv + a.keys - 1) / a.keys;
    const int64_t first = s.u0 + (int64_t)mt * per;
    const int b0 = (int)min(first / share, (int64_t)a.blocks - 1);   // (more than 2^31 units: not beyond the buffers)
    const int nr = its > 0 ? (int)min((first + its - 1) / share, (int64_t)a.blocks - 1) - b0 + 1 : 0;
    const int64_t rows = 16 * a.rt;
    const int64_t p0 = (int64_t)(b0 + pg_tile0(a, s) + mt) * rows + (row - mt * 16 * a.rt);
    bf16_t* orow = a.out + ((int64_t)(s.t0 + i0) * a.H + h) * a.Dv;
    if (nr == 0) {
      for (int dv = tid; dv < a.Dv; dv += 256) orow[dv] = bf16_t(0);
      continue;
    }
    // every wave reduces the ranges' maxima and normalisers, two ranges per lane
    static_assert(PG_MAX_SPLITS == 128, "two ranges per lane");
    float2 r2[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = lane + 64 * u;
      r2[u] = a.ml[p0 + min(k, nr - 1) * rows];
      if (k >= nr) r2[u] = make_float2(-INFINITY, 0.0f);
    }
    constexpr int V = 4;   // partial sums in flight
    float4 v[V];
    const float* po = a.po + p0 * a.Rq + 4 * c;
    const int64_t step = rows * a.Rq;
#pragma unroll
    for (int u = 0; u < V; ++u) v[u] = *reinterpret_cast<const float4*>(po + min(g + u * groups, nr - 1) * step);
    float m = fmaxf(r2[0].x, r2[1].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    float lt = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // a range whose scores are all NaN has no maximum, and a NaN for its sum
      const float x = r2[u].x != -INFINITY ? __builtin_amdgcn_exp2f((r2[u].x - m) * a.c) : 0.0f;
      lt = fmaf(x, r2[u].y, lt);
      if (tid < 64) wt[lane + 64 * u] = x;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) lt += __shfl_xor(lt, d);
    __syncthreads();
    if (g < groups) {
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = g; k < nr; k += V * groups) {
        if (k != g) {
#pragma unroll
          for (int u = 0; u < V; ++u) v[u] = *reinterpret_cast<const float4*>(po + min(k + u * groups, nr - 1) * step);
        }
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const bool on = k + u * groups < nr;
          const float x = wt[min(k + u * groups, PG_MAX_SPLITS - 1)];
          acc.x = fmaf(x, on ? v[u].x : 0.0f, acc.x);
          acc.y = fmaf(x, on ? v[u].y : 0.0f, acc.y);
          acc.z = fmaf(x, on ? v[u].z : 0.0f, acc.z);
          acc.w = fmaf(x, on ? v[u].w : 0.0f, acc.w);
        }
      }
      *reinterpret_cast<float4*>(sum + g * a.Rq + 4 * c) = acc;
    }
    __syncthreads();
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;   // (a NaN stays one)
    for (int r = tid; r < a.Rq; r += 256) {
      float x = sum[r];
      for (int k = 1; k < groups; ++k) x += sum[k * a.Rq + r];
      sum[r] = x * inv;
    }
    __syncthreads();
    // four lanes per output column, every fourth chunk of 8 latent columns each
    for (int dv = tid >> 2; dv < a.Dv; dv += 64) {
      float acc = 0.0f;
      if constexpr (WVEC) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = 8 * q4 + 32 * u;
          if (r < a.R)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc = fmaf(sum[r + e], (float)wv[u][e], acc);
        }
        if (dv + 64 < a.Dv) wload(dv + 64);
      } else {
        for (int r = q4; r < a.R; r += 4) acc = fmaf(sum[r], bf2f(w[(int64_t)dv * a.R + r]), acc);
      }
      acc += __shfl_xor(acc, 1);
      acc += __shfl_xor(acc, 2);
      if (q4 == 0) orow[dv] = f2bf(acc);
    }
    __syncthreads();   // the LDS is the next row's
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
  DSMOE_REQUIRE((int64_t)d->T * d->H < (int64_t(1) << 24), DSMOE_ERR_UNSUPPORTED, "mla_paged: T H must stay below 2^24");
  DSMOE_REQUIRE(d->max_kv >= 0 && d->max_q >= 0, DSMOE_ERR_INVALID, "mla_paged: negative max_q or max_kv");
  return DSMOE_OK;
}

// Rows whose two 16-row halves share a block's chunks (more than 16 heads) where the
// registers have room for their rope steps.
static int pg_rt(const PagedAttn& a) { return a.H > 16 && a.Drp <= 64 ? 2 : 1; }

// Whether K and V may be built at all: of fewer rows (token, head) the three launches of the latent rows
// take 24 to 32 us, and those of both kinds 32 to 36, most of it the host's time (a fresh prompt of 32
// tokens at H 32: 32 / 32, of 96 at H 12: 27 / 33).
static bool pg_both(const dsmoe_mla_paged_dims* d) {
  return d->max_q > PAGED_FEW && (int64_t)d->T * d->H >= 1280;
}

static PagedAttn pg_args(const dsmoe_mla_paged_dims* d, size_t* bytes, void* ws) {
  PagedAttn a;
  std::memset(static_cast<void*>(&a), 0, sizeof(a));
  a.p = paged_batch(d, nullptr, nullptr, nullptr);
  a.H = d->H; a.R = d->R; a.Dn = d->D_nope; a.Dr = d->D_rope; a.Dv = d->D_v;
  for (int ns : {2, 4, 8, 12, 16})
    if (a.Rq == 0 && d->R <= 16 * ns) a.Rq = 16 * ns;
  a.Drp = (int)align_up(d->D_rope, 32);
  a.neg = d->softmax_scale < 0.0f ? 1 : 0;
  // not below the smallest normal number: a masked score, -infinity, stays one for a scale of 0
  a.c = std::max((d->softmax_scale < 0.0f ? -d->softmax_scale : d->softmax_scale) * MLA_LOG2E, FLT_MIN);
  Carver c(ws);
  const size_t rows = (size_t)a.p.T * a.H;
  const bool both = pg_both(d) && paged_kv_carve(a, d, c) > 0;
  if (!both) a.slots = 0;
  a.rt = pg_rt(a);
  a.keys = 16 * pg_groups(a.Rq / 32) * 4 / a.rt;
  a.blocks = pg_groups(a.Rq / 32) > 2 ? 256 : 512;   // what the CUs hold at a time
  const size_t tile = 16 * (size_t)a.rt, tiles = rows / tile + a.p.B + 1;
  a.units = c.take<int32_t>(a.p.B + 2);
  a.qabs = c.take<bf16_t>(tiles * tile * (2 * a.Rq + a.Drp));
  a.ml = c.take<float2>((a.blocks + tiles) * tile);
  a.po = c.take<float>((a.blocks + tiles) * tile * a.Rq);
  *bytes = c.used();
  return a;
}

template <int NS, int NP, bool VEC, bool FULL, int RT>
static int launch_paged_few(const PagedAttn& a, hipStream_t st) {
  constexpr size_t lds = 4 * 16 * pg_groups(NS) * ((NS * 32 + 127) / 128 * 256) + RT * NS * 1024;
  static_assert(lds <= 160 * 1024 && (pg_groups(NS) > 2 || lds <= 80 * 1024), "one block or two on a CU");
  auto kern = paged_few_kernel<NS, NP, VEC, FULL, RT>;
  if (lds > 64 * 1024) {
    static const hipError_t attr =
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (attr != hipSuccess) return fail(DSMOE_ERR_HIP, "mla_paged: cannot raise LDS limit");
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)a.blocks), dim3(256), lds, st, a);
  return check_launch("mla_paged_few");
}

template <int NS, int NP>
static int launch_paged_few(const PagedAttn& a, hipStream_t st) {
  if (a.R == 32 * NS)
    return a.rt == 2 ? launch_paged_few<NS, NP, true, true, 2>(a, st) : launch_paged_few<NS, NP, true, true, 1>(a, st);
  return a.rt == 2 ? launch_paged_few<NS, NP, true, false, 2>(a, st) : launch_paged_few<NS, NP, true, false, 1>(a, st);
}

template <int NS>
static int launch_paged_few(const PagedAttn& a, hipStream_t st) {
  if (!a.kvvec)
    return a.rt == 2 ? launch_paged_few<NS, 0, false, false, 2>(a, st) : launch_paged_few<NS, 0, false, false, 1>(a, st);
  if (a.Drp <= 32) return launch_paged_few<NS, 1>(a, st);
  if (a.Drp <= 64) return launch_paged_few<NS, 2>(a, st);
  return launch_paged_few<NS, 0, true, false, 1>(a, st);
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
  a.p.units = a.units;
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
  hipLaunchKernelGGL((a.wvec ? paged_absorb_kernel<true> : paged_absorb_kernel<false>), dim3((unsigned)blocks), dim3(256),
                     sizeof(float) * (256 / (a.Rq / 8)) * a.Rq, st, a);
  rc = check_launch("mla_paged_absorb");
  if (rc) return rc;
  switch (a.Rq / 32) {
    case 1: rc = launch_paged_few<1>(a, st); break;
    case 2: rc = launch_paged_few<2>(a, st); break;
    case 4: rc = launch_paged_few<4>(a, st); break;
    case 6: rc = launch_paged_few<6>(a, st); break;
    default: rc = launch_paged_few<8>(a, st); break;
  }
  if (rc) return rc;
  hipLaunchKernelGGL((a.wvec ? paged_out_kernel<true> : paged_out_kernel<false>), dim3((unsigned)blocks), dim3(256),
                     sizeof(float) * (PG_MAX_SPLITS + (size_t)(256 / (a.Rq / 4)) * a.Rq), st, a);
  return check_launch("mla_paged_out");
}
