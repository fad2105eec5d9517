// What the kernels of the paged latent cache share (mla_cache.hip, mla_paged.hip,
// mla_paged_kv.hip): the batch of sequences with new tokens, and its keys' addresses.
#pragma once

#include "common.h"

namespace dsmoe {

// Sequence b's new tokens are the rows offsets[b] .. offsets[b + 1] - 1 of the packed
// tensors; it holds kv_lens[b] positions with them, so new token i stands at position
// kv_lens[b] - (its new tokens) + i.  Position p lies on page table[b][p / page_size].
// Nothing here trusts the device values: offsets are clamped into [0, T], positions
// into the table, and a page outside the pool holds no key.
struct PagedBatch {
  const int32_t* table;     // (B, width), rows table_stride apart
  const int32_t* kv_lens;   // (B)
  const int32_t* offsets;   // (B + 1)
  const int32_t* rows;      // (B + 1): where the new tokens that the latent rows serve stand among themselves
                            // (offsets, or the plan's where other sequences have K and V built)
  const int32_t* units;     // (B + 2): where their work starts (paged_unit_step), then all of it, then a block's share
  int64_t table_stride;
  int64_t kv_ps, kv_rs;     // page and row strides of the latent pool, in elements
  int64_t pe_ps, pe_rs;     // and of the rope pool
  int T, B, pages, page_size, width;
  int page_shift;           // log2 of page_size, -1 where it is no power of two
};

struct PagedSeq {
  int b;         // -1: no sequence
  int t0, n;     // rows of its new tokens
  int r0, m;     // of them on the latent rows: their first one's number, and how many
  int first;     // position of its first new token (may be negative)
  int kv;        // positions that the table can hold
  int u0;        // units before its work
};

__device__ __forceinline__ int paged_clamp(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Of the raw values of sequence b: its offsets, its length and, where not the offsets, its
// numbers among the tokens on the latent rows.
__device__ __forceinline__ PagedSeq paged_make(const PagedBatch& p, int b, int o0, int o1, int len, int r0, int r1,
                                               int u0) {
  PagedSeq s;
  s.b = b;
  s.t0 = paged_clamp(o0, 0, p.T);
  s.n = max(paged_clamp(o1, 0, p.T) - s.t0, 0);
  const bool same = p.rows == p.offsets;
  s.r0 = same ? s.t0 : r0;
  s.m = same ? s.n : r1 - r0;
  len = max(len, 0);
  s.first = len - s.n;
  s.kv = (int)min((int64_t)len, (int64_t)p.width * p.page_size);
  s.u0 = u0;
  return s;
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
  if (b < 0) return PagedSeq{-1, 0, 0, 0, 0, 0, 0, 0};
  const bool same = p.rows == p.offsets;
  return paged_make(p, b, p.offsets[b], p.offsets[b + 1], p.kv_lens[b], same ? 0 : p.rows[b], same ? 0 : p.rows[b + 1], 0);
}

// The last sequence that starts at or before u, where sequence b starts at
// floor(at[b] num / den) + step b, at: p.offsets, p.rows or (UNITS) p.units; b = -1 if there is
// none.  Uniform over the wave.  Of up to 64 sequences every lane loads one with all that is
// to be known of it: the loads are independent, where looking up the number first and then
// the rest would cost two trips to memory.  Of more, every 64th first (every 4096th, ...).
// UNITS_TOO: u0 is wanted as well.
enum PagedBy { PAGED_OFFSETS, PAGED_ROWS, PAGED_UNITS };
template <PagedBy BY, bool UNITS_TOO = BY == PAGED_UNITS>
__device__ __forceinline__ PagedSeq paged_at(const PagedBatch& p, int64_t u, int num, int den, int step) {
  const int lane = threadIdx.x & 63;
  const bool same = p.rows == p.offsets;
  const int32_t* arr = BY == PAGED_UNITS ? p.units : BY == PAGED_ROWS ? p.rows : p.offsets;
  const auto starts = [&](int v, int b) {
    if (BY == PAGED_UNITS) return (int64_t)v <= u;
    return (int64_t)paged_clamp(v, 0, p.T) * num / den + (int64_t)step * b <= u;
  };
  int base = 0, stride = 1;
  while ((p.B + stride - 1) / stride > 64) stride *= 64;
  for (; stride > 1; stride /= 64) {
    const int b = base + lane * stride;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(b < p.B && starts(arr[min(b, p.B - 1)], b)));
    base += max(n - 1, 0) * stride;
  }
  const int b = base + lane, bc = min(b, p.B - 1);
  const int o0 = p.offsets[bc], o1 = p.offsets[bc + 1], len = p.kv_lens[bc];
  const int r0 = same ? 0 : p.rows[bc], r1 = same ? 0 : p.rows[bc + 1];
  const int u0 = UNITS_TOO ? p.units[bc] : 0;
  const int v = BY == PAGED_UNITS ? u0 : BY == PAGED_ROWS && !same ? r0 : o0;
  const int n = __popcll(__builtin_amdgcn_ballot_w64(b < p.B && starts(v, b)));
  if (n == 0) return PagedSeq{-1, 0, 0, 0, 0, 0, 0, 0};
  const auto pick = [&](int x) { return __builtin_amdgcn_readlane(x, n - 1); };
  return paged_make(p, base + n - 1, pick(o0), pick(o1), pick(len), pick(r0), pick(r1), pick(u0));
}

// The page of position pos (0 <= pos < the sequence's kv), or -1 outside the pool.
__device__ __forceinline__ int paged_page(const PagedBatch& p, int b, int pos, int& in_page) {
  const int e = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
  in_page = pos - e * p.page_size;
  const int page = p.table[b * p.table_stride + e];
  return page >= 0 && page < p.pages ? page : -1;
}

// What building K and V saves a sequence of n new tokens and kv positions, up to a factor: the latent rows cost
// n tokens' way in and out (q W_k, times W_v) and more for every pair, K and V are built for every
// key, and they meet at n (1 / 72 + 7 / kv) = 1.  Measured with eight sequences of up to n new tokens, H 12,
// 16, 32 with R 192, 256, 256, us on the latent rows / with K and V: behind 4000 positions n 32 takes
// 67 / 100, 104 / 180, 199 / 454 and n 128 200 / 110, 353 / 177, 727 / 410 (they meet at 64, 64, 78);
// behind 500 n 16 takes 30 / 42, 39 / 51, 76 / 90 and n 64 70 / 47, 102 / 57, 209 / 101; fresh
// prompts of n 32 38 / 32, 53 / 33, 100 / 37.  A batch of both kinds pays for both (behind 500, n up to 32:
// 45 on the latent rows, 43 with K and V, 66 by each sequence's own gain), so sequences that
// lie near the line (paged_open) go one way together, by the sum of their gains.
constexpr int PAGED_FEW = 16;   // K and V are never built for as few tokens
__host__ __device__ inline int64_t paged_gain(int n, int kv) { return (int64_t)n * ((int64_t)kv + 512) - 72 * (int64_t)kv; }
__host__ __device__ inline bool paged_open(int n, int kv) { return n > PAGED_FEW && paged_gain(n, kv) > -48 * (int64_t)kv; }

struct PagedAttn {
  PagedBatch p;
  const bf16_t* q_nope;   // row of token t, head h at t qn_ts + h qn_hs
  const bf16_t* q_pe;
  int64_t qn_ts, qn_hs, qp_ts, qp_hs;
  const bf16_t* kv_pages;
  const bf16_t* pe_pages;
  const bf16_t* w_k;      // head h's (Dn, R) rows at h wk_hs
  const bf16_t* w_v;      // head h's (Dv, R) rows at h wv_hs
  int64_t wk_hs, wv_hs;
  bf16_t* out;            // (T, H, Dv)
  int H, R, Dn, Dr, Dv;
  int Rq, Drp;            // R and Dr in whole steps of 32
  int neg;                // softmax_scale < 0: q is negated, c = |scale| log2(e)
  int kvvec;              // 16-byte loads of latent and rope rows
  int wvec;               // of weight rows
  int qvec;               // of query rows
  float c;
  // on the latent rows (mla_paged.hip)
  int rt;                 // a row tile is 16 rt rows
  bf16_t* qabs;           // (tiles rt, 2 Rq + Drp columns / 32, 64 lanes, 8): [hi | lo | pe] of 16 rows as the
                          // lanes of paged_few_kernel take them, zeros in the columns' padding
  float* po;              // (partials, 16 rt rows, Rq) sums of p c
  float2* ml;             // (partials, 16 rt rows) {max of the scores, sum of p}
  int32_t* units;         // p.units
  int blocks, keys;       // blocks of paged_few_kernel, and keys of a unit
  // on K and V (mla_paged_kv.hip)
  int slots, cap;         // sequences at most, and positions of each (a multiple of 128)
  int kvt;                // tiles of 128 positions of a block that builds them
  int slot0, pass;        // the slots of this pass: slot0 .. slot0 + pass - 1
  int32_t* slot_of;       // (B) slot of a sequence, -1: on the latent rows
  int32_t* seq_of;        // (slots) sequence of a slot, -1: none
  int32_t* plan_rows;     // (B + 1) p.rows of such a call
  int DQp, DVp;           // K and V columns (multiples of 16 and 32)
  _Float16* kbuf;         // (pass, H, cap, DQp): 2^-kx times [k_nope | pe | 0]
  _Float16* vbuf;         // (pass, H, cap, DVp): 2^-vx times v
  float* kx;              // (pass, H, cap / 32): 2^kx of 32 keys
  float* vx;              // (pass, H, cap / 32): vx
  uint32_t* gone;         // (pass, H, cap / 32): bit j, the key is on no page
  int nsp;                // key ranges
  float* po2;             // nsp > 1: (nsp, T H, DVp)
  float2* ml2;            // nsp > 1: (nsp, T H)
};

// Units of work on the latent rows: `keys` keys of one row tile.  They are numbered
// sequence by sequence, tile by tile, and block i takes those from i times its share on,
// so that every block has as many whatever the lengths.  One wave, 64 sequences at a time, run the
// units so far; m, kv of the lane's sequence b.
struct PagedUnits {
  int64_t run = 0;
  int most = 1;   // the longest tile's
};
__device__ __forceinline__ void paged_unit_step(const PagedAttn& a, int b, int m, int kv, PagedUnits& w) {
  const int lane = threadIdx.x & 63;
  const int per = (kv + a.keys - 1) / a.keys;   // kv < 2^31 - keys: see paged_make and pg_validate
  const int64_t own = b < a.p.B && m > 0 ? (int64_t)((m * a.H + 16 * a.rt - 1) / (16 * a.rt)) * per : 0;
  int64_t sum = own;
  int most = own > 0 ? per : 1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
    most = max(most, __shfl_xor(most, d));
  }
  if (b < a.p.B) a.units[b] = (int)min(w.run + sum - own, (int64_t)INT32_MAX);
  w.run += __shfl(sum, 63);
  w.most = max(w.most, most);
}
constexpr int PG_MAX_SPLITS = 128;
__device__ __forceinline__ void paged_unit_end(const PagedAttn& a, const PagedUnits& w) {
  if ((threadIdx.x & 63) != 0) return;
  const int64_t all = min(w.run, (int64_t)INT32_MAX);
  a.units[a.p.B] = (int)all;
  // a tile is cut by at most PG_MAX_SPLITS blocks
  a.units[a.p.B + 1] = (int)max((all + a.blocks - 1) / a.blocks, (int64_t)(w.most + PG_MAX_SPLITS - 2) / (PG_MAX_SPLITS - 1));
}

// The plan, K and V and the attention on them, of the sequences with many new tokens.
size_t paged_kv_carve(PagedAttn& a, const dsmoe_mla_paged_dims* d, Carver& c);
int launch_paged_plan(const PagedAttn& a, hipStream_t st);
int launch_paged_kv(PagedAttn a, hipStream_t st);

int paged_validate(const dsmoe_mla_paged_dims* d);
PagedBatch paged_batch(const dsmoe_mla_paged_dims* d, const int32_t* table, const int32_t* kv_lens,
                       const int32_t* offsets);

}  // namespace dsmoe
