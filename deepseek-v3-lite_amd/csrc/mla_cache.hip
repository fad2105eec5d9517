// New latent rows into the pages of a latent cache: the writes before the attention of
// mla_paged.hip (the reference keeps one contiguous cache per batch row and assigns
// slices of it, models/mla.py:95-125).
//
//   c'[r] = c[r] rsqrt(mean(c^2) + eps) w[r]   (or c as it is), rounded to bf16 once
//   kv_pages[page, in_page] = c',  pe_pages[page, in_page] = pe
//
// One wave per token.  A row is at most 32 chunks of 8 columns, so lanes 0-31 hold the
// latent row and lanes 32-63 the rope row, one load and one 16-byte store each; the
// squares are added over the wave in fp32.  Rows of other widths, strides or alignment
// go element by element.
//
// Bound by a chain of three loads (offsets, page, row) where there are few rows, by its bytes
// where there are many: 3.6 us for 48 rows with the norm (R 192, D_rope 24), 9.4 us for 23075
// without (R 256, D_rope 64; 3.1 TB/s).
#include "mla_paged.h"
#include "mfma.h"

namespace dsmoe {

struct CacheArgs {
  PagedBatch p;
  const void* ctx_kv;      // (T, R) rows ckv_rs apart, bf16 or fp32
  const void* ctx_pe;      // (T, Dr) rows cpe_rs apart
  const float* norm_w;     // (R) or null
  bf16_t* kv_pages;
  bf16_t* pe_pages;
  int64_t ckv_rs, cpe_rs;
  int R, Dr;
  float eps;
};

template <typename T>
__device__ __forceinline__ void cache_ld8(const void* base, int64_t at, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(static_cast<const bf16_t*>(base) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = f[0], b = f[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mla_cache_append_kernel(const CacheArgs a) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.p.T) return;
  const bool pe_side = lane >= 32;
  const int c8 = 8 * (lane & 31);
  float v[8] = {}, w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.0f;
  const bool live = c8 < (pe_side ? a.Dr : a.R);
  if (VEC && live) {   // issued before the sequence is known
    if (pe_side)
      cache_ld8<T>(a.ctx_pe, t * a.cpe_rs + c8, v);
    else
      cache_ld8<T>(a.ctx_kv, t * a.ckv_rs + c8, v);
    if (a.norm_w && !pe_side) cache_ld8<float>(a.norm_w, c8, w);
  }
  const PagedSeq s = paged_at<PAGED_OFFSETS>(a.p, t, 1, 1, 0);
  const int pos = s.first + t - s.t0;
  // rows behind the last sequence, and positions without a place, are left alone
  if (s.b < 0 || t < s.t0 || t - s.t0 >= s.n || pos < 0 || pos >= s.kv) return;
  int in_page;
  const int page = paged_page(a.p, s.b, pos, in_page);
  if (page < 0) return;
  bf16_t* kd = a.kv_pages + page * a.p.kv_ps + in_page * a.p.kv_rs;
  bf16_t* pd = a.pe_pages + page * a.p.pe_ps + in_page * a.p.pe_rs;
  const T* ck = static_cast<const T*>(a.ctx_kv) + t * a.ckv_rs;
  const T* cp = static_cast<const T*>(a.ctx_pe) + t * a.cpe_rs;
  float r = 1.0f;
  if (a.norm_w) {
    float q = 0.0f;
    if (VEC) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q = fmaf(v[i], pe_side ? 0.0f : v[i], q);
    } else {
      for (int c = lane; c < a.R; c += 64) {
        const float x = to_f(ck[c]);
        q = fmaf(x, x, q);
      }
    }
    if (VEC && pe_side) q = 0.0f;   // (a NaN or infinity of the rope row is not the norm's)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) q += __shfl_xor(q, d);
    r = 1.0f / sqrtf(q / (float)a.R + a.eps);
  }
  if (VEC) {
    if (!live) return;
    if (pe_side) r = 1.0f;
    u32x4_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(v[2 * i] * r * w[2 * i], v[2 * i + 1] * r * w[2 * i + 1]);
    *reinterpret_cast<u32x4_t*>((pe_side ? pd : kd) + c8) = o;
  } else {
    for (int c = lane; c < a.R; c += 64) kd[c] = f2bf(to_f(ck[c]) * r * (a.norm_w ? a.norm_w[c] : 1.0f));
    for (int c = lane; c < a.Dr; c += 64) pd[c] = f2bf(to_f(cp[c]));
  }
}

int paged_validate(const dsmoe_mla_paged_dims* d) {
  DSMOE_REQUIRE(d, DSMOE_ERR_INVALID, "mla_paged: NULL dims");
  DSMOE_REQUIRE(d->T >= 0 && d->B >= 0, DSMOE_ERR_INVALID, "mla_paged: T and B must not be negative");
  DSMOE_REQUIRE(d->B < (1 << 24), DSMOE_ERR_UNSUPPORTED, "mla_paged: 2^24 sequences or more");
  DSMOE_REQUIRE(d->R > 0 && d->D_rope > 0 && d->R <= 256 && d->D_rope <= 256, DSMOE_ERR_INVALID,
                "mla_paged: R and D_rope must be in 1 .. 256");
  DSMOE_REQUIRE(d->pages > 0 && d->page_size > 0 && d->table_width >= 0, DSMOE_ERR_INVALID,
                "mla_paged: pages and page_size must be positive");
  DSMOE_REQUIRE((int64_t)d->table_width * d->page_size < (int64_t(1) << 31) - (1 << 16), DSMOE_ERR_UNSUPPORTED,
                "mla_paged: a row of the table has room for 2^31 positions");
  DSMOE_REQUIRE(d->table_stride >= 0 && d->kv_page_stride >= 0 && d->kv_row_stride >= 0 && d->pe_page_stride >= 0 &&
                    d->pe_row_stride >= 0, DSMOE_ERR_INVALID, "mla_paged: negative stride");
  return DSMOE_OK;
}

PagedBatch paged_batch(const dsmoe_mla_paged_dims* d, const int32_t* table, const int32_t* kv_lens,
                       const int32_t* offsets) {
  PagedBatch p;
  p.table = table; p.kv_lens = kv_lens; p.offsets = p.rows = offsets;
  p.units = nullptr;
  p.table_stride = d->table_stride;
  p.kv_ps = d->kv_page_stride; p.kv_rs = d->kv_row_stride;
  p.pe_ps = d->pe_page_stride; p.pe_rs = d->pe_row_stride;
  p.T = d->T; p.B = d->B; p.pages = d->pages; p.page_size = d->page_size; p.width = d->table_width;
  p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
  return p;
}

}  // namespace dsmoe

using namespace dsmoe;

extern "C" int dsmoe_mla_cache_append(const void* ctx_kv, int64_t ctx_kv_stride, const void* ctx_pe,
                                      int64_t ctx_pe_stride, int dtype, const float* norm_weight, float norm_eps,
                                      void* kv_pages, void* pe_pages, const int32_t* block_table,
                                      const int32_t* kv_lens, const int32_t* q_offsets,
                                      const dsmoe_mla_paged_dims* dims, void* stream) {
  const int rc = paged_validate(dims);
  if (rc) return rc;
  DSMOE_REQUIRE(dtype == DSMOE_F32 || dtype == DSMOE_BF16, DSMOE_ERR_UNSUPPORTED, "mla_cache_append: unsupported dtype");
  DSMOE_REQUIRE(ctx_kv_stride >= 0 && ctx_pe_stride >= 0, DSMOE_ERR_INVALID, "mla_cache_append: negative stride");
  if (dims->T == 0 || dims->B == 0 || dims->table_width == 0) return DSMOE_OK;
  DSMOE_REQUIRE(ctx_kv && ctx_pe && kv_pages && pe_pages && block_table && kv_lens && q_offsets, DSMOE_ERR_INVALID,
                "mla_cache_append: NULL pointer");
  CacheArgs a;
  a.p = paged_batch(dims, block_table, kv_lens, q_offsets);
  a.ctx_kv = ctx_kv; a.ctx_pe = ctx_pe; a.norm_w = norm_weight;
  a.kv_pages = static_cast<bf16_t*>(kv_pages); a.pe_pages = static_cast<bf16_t*>(pe_pages);
  a.ckv_rs = ctx_kv_stride; a.cpe_rs = ctx_pe_stride;
  a.R = dims->R; a.Dr = dims->D_rope; a.eps = norm_eps;
  const auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  const bool vec = a.R % 8 == 0 && a.Dr % 8 == 0 && a.ckv_rs % 8 == 0 && a.cpe_rs % 8 == 0 && a.p.kv_ps % 8 == 0 &&
                   a.p.kv_rs % 8 == 0 && a.p.pe_ps % 8 == 0 && a.p.pe_rs % 8 == 0 && al(ctx_kv) && al(ctx_pe) &&
                   al(kv_pages) && al(pe_pages) && al(norm_weight);
  const dim3 grid((unsigned)cdiv(a.p.T, 4));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == DSMOE_BF16)
    hipLaunchKernelGGL((vec ? mla_cache_append_kernel<bf16_t, true> : mla_cache_append_kernel<bf16_t, false>), grid,
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((vec ? mla_cache_append_kernel<float, true> : mla_cache_append_kernel<float, false>), grid,
                       dim3(256), 0, st, a);
  return check_launch("mla_cache_append");
}
