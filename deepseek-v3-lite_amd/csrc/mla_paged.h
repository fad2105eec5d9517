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
  int64_t table_stride;
  int64_t kv_ps, kv_rs;     // page and row strides of the latent pool, in elements
  int64_t pe_ps, pe_rs;     // and of the rope pool
  int T, B, pages, page_size, width;
};

struct PagedSeq {
  int b;         // -1: no sequence
  int t0, n;     // rows of its new tokens
  int r0, m;     // of them on the latent rows: their first one's number, and how many
  int first;     // position of its first new token (may be negative)
  int kv;        // positions that the table can hold
};

__device__ __forceinline__ int paged_clamp(int v, int lo, int hi) { return min(max(v, lo), hi); }

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
  PagedSeq s;
  s.b = b;
  s.t0 = s.n = s.r0 = s.m = s.first = s.kv = 0;
  if (b < 0) return s;
  s.t0 = paged_clamp(p.offsets[b], 0, p.T);
  s.n = max(paged_clamp(p.offsets[b + 1], 0, p.T) - s.t0, 0);
  s.r0 = s.t0;
  s.m = s.n;
  if (p.rows != p.offsets) {
    s.r0 = p.rows[b];
    s.m = p.rows[b + 1] - s.r0;
  }
  const int len = max(p.kv_lens[b], 0);
  s.first = len - s.n;
  s.kv = (int)min((int64_t)len, (int64_t)p.width * p.page_size);
  return s;
}

// The last sequence b whose work starts at or before unit u, where sequence b's starts
// at unit at[b] * num / den + step * b (at: p.offsets or p.rows); -1 if there is none.
// Uniform over the wave: 64 sequences at a time, one per lane, all loads independent.
__device__ __forceinline__ int paged_find(const PagedBatch& p, const int32_t* at, int64_t u, int num, int den, int step) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    const int off = paged_clamp(at[min(b, p.B - 1)], 0, p.T);
    const bool le = b < p.B && (int64_t)off * num / den + (int64_t)step * b <= u;
    n += __popcll(__builtin_amdgcn_ballot_w64(le));
  }
  return __builtin_amdgcn_readfirstlane(n) - 1;
}

// The page of position pos (0 <= pos < the sequence's kv), or -1 outside the pool.
__device__ __forceinline__ int paged_page(const PagedBatch& p, int b, int pos, int& in_page) {
  const int e = pos / p.page_size;
  in_page = pos - e * p.page_size;
  const int page = p.table[b * p.table_stride + e];
  return page >= 0 && page < p.pages ? page : -1;
}

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
  int Rq, Drp;            // R and Dr in whole MFMA steps
  int neg;                // softmax_scale < 0: q is negated, c = |scale| log2(e)
  int kvvec;              // 16-byte loads of latent and rope rows
  int wvec;               // of weight rows
  int qvec;               // of query rows
  float c;
  // on the latent rows (mla_paged.hip)
  bf16_t* qabs;           // (rows, 2 Rq + Drp): [hi | lo | pe], zeros in the padding
  float* po;              // (nsplit, rows, Rq) partial sums of p c
  float2* ml;             // (nsplit, rows) {max of the scores, sum of p}
  int nsplit, cpw;        // key ranges, and 32-key chunks of each but the last
  // on K and V (mla_paged_kv.hip)
  int thr;                // sequences with more new tokens take them
  int slots, cap;         // sequences at most, and positions of each (a multiple of 128)
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

// The plan, K and V and the attention on them, of the sequences with many new tokens.
size_t paged_kv_carve(PagedAttn& a, const dsmoe_mla_paged_dims* d, Carver& c);
int launch_paged_plan(const PagedAttn& a, hipStream_t st);
int launch_paged_kv(PagedAttn a, hipStream_t st);

int paged_validate(const dsmoe_mla_paged_dims* d);
PagedBatch paged_batch(const dsmoe_mla_paged_dims* d, const int32_t* table, const int32_t* kv_lens,
                       const int32_t* offsets);

}  // namespace dsmoe
