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
  int64_t table_stride;
  int64_t kv_ps, kv_rs;     // page and row strides of the latent pool, in elements
  int64_t pe_ps, pe_rs;     // and of the rope pool
  int T, B, pages, page_size, width;
};

struct PagedSeq {
  int b;         // -1: no sequence
  int t0, n;     // rows of its new tokens
  int first;     // position of its first new token (may be negative)
  int kv;        // positions that the table can hold
};

__device__ __forceinline__ int paged_clamp(int v, int lo, int hi) { return min(max(v, lo), hi); }

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
  PagedSeq s;
  s.b = b;
  s.t0 = s.n = s.first = s.kv = 0;
  if (b < 0) return s;
  s.t0 = paged_clamp(p.offsets[b], 0, p.T);
  s.n = max(paged_clamp(p.offsets[b + 1], 0, p.T) - s.t0, 0);
  const int len = max(p.kv_lens[b], 0);
  s.first = len - s.n;
  s.kv = (int)min((int64_t)len, (int64_t)p.width * p.page_size);
  return s;
}

// The last sequence b whose work starts at or before unit u, where sequence b's starts
// at unit offsets[b] * num / den + step * b; -1 if there is none.  Uniform over the
// wave: 64 sequences at a time, one per lane, all of a lane's loads independent.
__device__ __forceinline__ int paged_find(const PagedBatch& p, int64_t u, int num, int den, int step) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    const int off = paged_clamp(p.offsets[min(b, p.B - 1)], 0, p.T);
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

int paged_validate(const dsmoe_mla_paged_dims* d);
PagedBatch paged_batch(const dsmoe_mla_paged_dims* d, const int32_t* table, const int32_t* kv_lens,
                       const int32_t* offsets);

}  // namespace dsmoe
