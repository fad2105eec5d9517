// The sequences of a paged call (mla_paged.hip) that have many new tokens: K and V of
// their positions built per head, and the causal flash attention of the chunk on them.
//
//   paged_plan_kernel   which sequences those are (paged_open, at most `cap` positions,
//                       while there are slots), and how the other sequences' tokens are
//                       numbered.  One wave.
//   paged_kv_kernel     K = [c W_k^T | pe | 0] and V = c W_v^T of 128 positions of a (slot,
//                       head), 32 a wave: an MFMA product with the weight rows as first and
//                       the latent rows as second operand, so a lane holds four consecutive
//                       columns of its key.
//   paged_fa_kernel     flash attention of 32 NW queries of a (slot, head), 32 a wave, over
//                       blocks of 64 keys through LDS (tiles, operand order and softmax as
//                       mla_fa_kernel of mla.hip).
//   paged_merge_kernel  key ranges added, where few query blocks were cut along the keys.
//
// K, V, q and p are held in fp16 (11 significant bits; bf16's 8 would double the error
// of the output: k, v and p each cost as much as its own rounding), under powers of two
// that fit its range whatever the input's: 2^-kx for the K rows of 32 keys, 2^-vx for
// their V rows, the row's own for q.  They return where a scalar costs nothing: kx and
// q's in the factor of the scores, vx as weight 2^vx in the softmax,
//   out = sum_j 2^(s_j + vx_j - m) (2^-vx_j v_j) / sum_j 2^(s_j + vx_j - m) 2^-vx_j,
// m the running maximum of s_j + vx_j, or one up to 2^8 behind it.  A row keeps its 11 bits
// down to 2^-27 of the largest value of its 32 keys.
//
// Masked places: a key on no page has its bit in `gone` (and zero rows); a latent row
// with a NaN or an infinity has K all NaN and V zero, so that it reaches the queries that
// see it, through their normaliser, and no other.
#include <algorithm>
#include <type_traits>

#include "mla_paged.h"
#include "mla_tile.h"

namespace dsmoe {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int PKV_ROWS = 128;   // positions of a block of paged_kv_kernel
constexpr int PKV_KB = 64;      // keys of a block of the attention

// ---------------------------------------------------------------- plan
__global__ __launch_bounds__(64) void paged_plan_kernel(const PagedAttn a) {
  const int lane = threadIdx.x;
  int slot0 = 0, row0 = 0;
  PagedUnits units;
  int64_t gain = 0;
  for (int b = lane; b < a.p.B; b += 64) {
    const PagedSeq s = paged_seq(a.p, b);
    if (paged_open(s.n, s.kv)) gain += paged_gain(s.n, s.kv);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) gain += __shfl_xor(gain, d);
  for (int b0 = 0; b0 < a.p.B; b0 += 64) {
    const int b = b0 + lane;
    PagedSeq s = paged_seq(a.p, min(b, a.p.B - 1));
    if (b >= a.p.B) s.n = 0;
    const bool many = gain > 0 && paged_open(s.n, s.kv) && s.kv <= a.cap;
    const uint64_t mask = __builtin_amdgcn_ballot_w64(many);
    const int slot = slot0 + __popcll(mask & ((1ull << lane) - 1));
    const bool has = many && slot < a.slots;
    slot0 += __popcll(mask);
    // rows of the sequences before this one (lane's n stays under 2^24)
    int64_t sum = has ? 0 : s.n;
    const int64_t own = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (b < a.p.B) {
      a.slot_of[b] = has ? slot : -1;
      if (has) a.seq_of[slot] = b;
      a.plan_rows[b] = (int)min((int64_t)a.p.T, row0 + sum - own);
    }
    // (of sane offsets the sum stays under T; others' tokens behind it are left out)
    const int m = (int)(min((int64_t)a.p.T, row0 + sum) - min((int64_t)a.p.T, row0 + sum - own));
    paged_unit_step(a, b, m, s.kv, units);
    row0 = (int)min((int64_t)a.p.T, row0 + __shfl(sum, 63));
  }
  if (lane == 0) a.plan_rows[a.p.B] = row0;
  paged_unit_end(a, units);
  for (int i = min(slot0, a.slots) + lane; i < a.slots; i += 64) a.seq_of[i] = -1;
}

// ---------------------------------------------------------------- K, V
__device__ __forceinline__ mla_u32x4 pkv_ld8(const bf16_t* p, int n, bool vec) {
  if (vec) return *reinterpret_cast<const mla_u32x4*>(p);
  bf16_t e8[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) e8[e] = e < n ? p[e] : bf16_t(0);
  return *reinterpret_cast<const mla_u32x4*>(e8);
}

// The larger of mx and the magnitudes of eight bf16, as fp32 bits.
__device__ __forceinline__ uint32_t pkv_absmax(mla_u32x4 w, uint32_t mx) {
#pragma unroll
  for (int i = 0; i < 4; ++i) mx = max(mx, max((w[i] << 16) & 0x7fff0000u, w[i] & 0x7fff0000u));
  return mx;
}

__device__ __forceinline__ float pkv_pow2(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }   // -126 .. 127

__device__ __forceinline__ uint32_t pkv_pack(float a, float b) {
  f16x2_t v;
  v[0] = (_Float16)a;
  v[1] = (_Float16)b;
  return __builtin_bit_cast(uint32_t, v);
}

// Grid (tiles of 128 positions / a.kvt, H, slots of the pass).  A block keeps its head's weight
// rows in LDS (mlb_off layout) for a.kvt tiles, whose latent rows are asked for one tile
// ahead: read by every wave from memory they took 232 us for prompts of 6144 and 3973 positions (H
// 32, R 256, D_nope and D_v 128, D_rope 64), this way 120 us: 207 MB of K and V written, which
// alone take 44, and 42 GFLOP.  Without its stores the kernel takes 84, without its products 78: the
// two blocks of a CU overlap little of either.  Rope rows held in registers so that no load waits
// behind a store: 122, and 37 against 33 where they cost a block its place on the CU (R 192).
// part: K, V, or 2: by the block's parity.  NT: 32-column tiles, all computed (LDS rows past the last weight row repeat it and are not stored).  VEC:
// 16-byte loads of latent, rope and weight rows, every load of a batch issued from a valid
// address before it is used.
template <int NS, int NT, bool VEC>
__global__ __launch_bounds__(256) void paged_kv_kernel(const PagedAttn a, int part) {
  constexpr int RB = (NS * 16 + 127) / 128 * 256;
  extern __shared__ __attribute__((aligned(16))) char pkv_smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, l32 = lane & 31;
  const int h = blockIdx.y, slot = part == 2 ? blockIdx.z >> 1 : blockIdx.z;
  const bool vpart = part == 2 ? blockIdx.z & 1 : part;
  const PagedSeq s = paged_seq(a.p, a.seq_of[a.slot0 + slot]);
  const int tile0 = blockIdx.x * a.kvt, tiles = min(tile0 + a.kvt, (s.kv + PKV_ROWS - 1) / PKV_ROWS);
  if (s.b < 0 || tile0 >= tiles) return;
  const int ncols = vpart ? a.Dv : a.Dn;
  const int64_t sh = (int64_t)slot * a.H + h;
  const bf16_t* w = vpart ? a.w_v + h * a.wv_hs : a.w_k + h * a.wk_hs;
  // the lane's latent and rope row of a tile; positions behind the last one read that
  bf16x8_t fx[NS];
  const bf16_t* pr;
  int page, in_page, npage, nin_page;
  bool live, gone1;
  const auto key_of = [&](int t) { return t * PKV_ROWS + 32 * wave + l32; };
  const auto lookup = [&](int t) { npage = paged_page(a.p, s.b, min(key_of(t), s.kv - 1), nin_page); };
  const auto load = [&](int t) {
    live = key_of(t) < s.kv && page >= 0;
    gone1 = key_of(t) < s.kv && page < 0;
    const int64_t pg = max(page, 0);
    const bf16_t* cr = a.kv_pages + pg * a.p.kv_ps + in_page * a.p.kv_rs;
    pr = a.pe_pages + pg * a.p.pe_ps + in_page * a.p.pe_rs;
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      const int col = 16 * st + 8 * hi;
      fx[st] = __builtin_bit_cast(bf16x8_t, pkv_ld8(cr + (VEC ? min(col, a.R - 8) : col), a.R - col, VEC));
    }
  };
  lookup(tile0);
  page = npage;
  in_page = nin_page;
  // the weight rows, each thread's pieces in a batch
  {
    constexpr int PER = (NT * 32 * NS * 2 + 255) / 256;
    mla_u32x4 v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + 256 * u, r = i / (2 * NS), c = i - r * (2 * NS);
      v[u] = pkv_ld8(w + (int64_t)min(r, ncols - 1) * a.R + (VEC ? min(8 * c, a.R - 8) : 8 * c), a.R - 8 * c, VEC);
    }
    load(tile0);
    lookup(tile0 + 1);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + 256 * u, r = i / (2 * NS), c = i - r * (2 * NS);
      // (columns past R: zeros against whatever the latent rows' loads repeat)
      if (i < NT * 32 * NS * 2)
        *reinterpret_cast<mla_u32x4*>(pkv_smem + mlb_off(r, c, RB)) = 8 * c < a.R ? v[u] : mla_u32x4{0u, 0u, 0u, 0u};
    }
  }
  __syncthreads();
  const MlbLane<RB> lk(lane);
  for (int t = tile0; t < tiles; ++t) {
    const int key = key_of(t);
    mla_f32x16 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
#pragma unroll
      for (int st = 0; st < NS; ++st)
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lk.frag(pkv_smem, 32 * j, st), fx[st], acc[j], 0, 0, 0);
    }
    // a NaN or an infinity in a latent row makes every column one
    const uint64_t bl = __builtin_amdgcn_ballot_w64(!(fabsf(acc[0][0]) < INFINITY));
    const bool bad = (((uint32_t)bl | (uint32_t)(bl >> 32)) >> l32) & 1;
    const bool alive = live;
    const uint32_t gone = (uint32_t)__builtin_amdgcn_ballot_w64(gone1);
    const bf16_t* prow = pr;
    if (t + 1 < tiles) {
      page = npage;
      in_page = nin_page;
      lookup(t + 2);
      __builtin_amdgcn_sched_barrier(0);   // (asked for before the rows: see paged_few_kernel)
      load(t + 1);
    }
    // the largest finite magnitude of the wave's keys goes to [2^13, 2^14)
    float mx = 0.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(acc[j][i]));
    if (!vpart)
      for (int d = 8 * hi; d < a.Dr; d += 16) {
        const mla_u32x4 v = pkv_ld8(prow + d, a.Dr - d, VEC);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = fabsf(__uint_as_float(v[i] << 16)), y = fabsf(__uint_as_float(v[i] & 0xffff0000u));
          mx = fmaxf(mx, x < INFINITY ? x : 0.0f);
          mx = fmaxf(mx, y < INFINITY ? y : 0.0f);
        }
      }
    if (!alive || bad) mx = 0.0f;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    // (V's at most 2^96: keys' weights are under it in the normaliser, beside those of ordinary
    // values, and neither the sum of 2^24 of them may pass the range nor one of 2^-24 vanish)
    const int n = mx > 0.0f ? min(max(13 - ((int)(__float_as_uint(mx) >> 23) - 127), -126), vpart ? 96 : 126) : 0;
    if (lane == 0) {
      const int64_t meta = sh * (a.cap / 32) + t * (PKV_ROWS / 32) + wave;
      if (vpart) {
        a.vx[meta] = (float)-n;
      } else {
        a.kx[meta] = pkv_pow2(-n);
        a.gone[meta] = gone;
      }
    }
    // dead rows: zeros (a select: their values may be anything), NaN for K rows that hold one
    const float f = pkv_pow2(n), nan = __builtin_nanf("");
    const bool zero = !alive || (vpart && bad);
    _Float16* row = vpart ? a.vbuf + (sh * a.cap + key) * a.DVp : a.kbuf + (sh * a.cap + key) * a.DQp;
    const auto store = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      const auto put = [&](float v) { return WHOLE ? v * f : zero ? 0.0f : (!vpart && bad) ? nan : v * f; };
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int gp = 0; gp < 2; ++gp) {
          // columns 32 j + 16 gp + 8 hi .. + 7 of the lane's key: the halves of a register
          // pair (four columns each of lanes l and l + 32) change places
          uint32_t u[2][2];
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int d = 0; d < 2; ++d)
              u[g][d] = pkv_pack(put(acc[j][8 * gp + 4 * g + 2 * d]), put(acc[j][8 * gp + 4 * g + 2 * d + 1]));
          const auto r0 = __builtin_amdgcn_permlane32_swap(u[0][0], u[1][0], false, false);
          const auto r1 = __builtin_amdgcn_permlane32_swap(u[0][1], u[1][1], false, false);
          const int col = 32 * j + 16 * gp + 8 * hi;
          const mla_u32x4 o = {(uint32_t)r0[0], (uint32_t)r1[0], (uint32_t)r0[1], (uint32_t)r1[1]};
          if (WHOLE || col + 8 <= ncols) {
            *reinterpret_cast<mla_u32x4*>(row + col) = o;
          } else {
            const f16x8_t e8 = __builtin_bit_cast(f16x8_t, o);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col + e < ncols) row[col + e] = e8[e];
          }
        }
    };
    // the common case without selects and column checks
    if (ncols == 32 * NT && __builtin_amdgcn_ballot_w64(!alive || bad) == 0)
      store(std::true_type{});
    else
      store(std::false_type{});
    if (vpart) continue;
    for (int d = 8 * hi; d < a.Dr; d += 16) {
      const mla_u32x4 v = pkv_ld8(prow + d, a.Dr - d, VEC);
      mla_u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __uint_as_float(v[i] << 16), y = __uint_as_float(v[i] & 0xffff0000u);
        o[i] = alive ? pkv_pack(x * f, y * f) : 0u;
      }
      if (VEC && a.Dn % 8 == 0) {
        *reinterpret_cast<mla_u32x4*>(row + a.Dn + d) = o;
      } else {
        const f16x8_t e8 = __builtin_bit_cast(f16x8_t, o);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (d + e < a.Dr) row[a.Dn + d + e] = e8[e];
      }
    }
    for (int d = a.Dn + a.Dr + hi; d < a.DQp; d += 2) row[d] = (_Float16)0.0f;
  }
}

// ---------------------------------------------------------------- attention
template <int NSTEP, int NV, int NW>
struct PfaCfg {
  static constexpr int DQp = NSTEP * 16;
  static constexpr int DVp = NV * 32;
  static constexpr int KRB = (DQp + 127) / 128 * 256;   // K tile row bytes (mlb_off layout)
  static constexpr int KT = PKV_KB * KRB;               // K tile bytes
  static constexpr int VT = PKV_KB * DVp * 2;           // V tile bytes
  static constexpr int BUF = KT + VT;
  static constexpr int NLK = (KT / 1024 + NW - 1) / NW;  // 1 KB direct loads per wave and tile
  static constexpr int NLV = (VT / 1024 + NW - 1) / NW;
  static constexpr int QB = 32 * NW;
  // two blocks of keys on their way where a third buffer leaves as many waves on a CU (and
  // every wave has as many loads, which the waits count)
  static constexpr bool EVEN = NLK * NW * 1024 == KT && NLV * NW * 1024 == VT;
  static constexpr int NBUF = EVEN && 3 * BUF <= (NW == 8 ? 160 : 80) * 1024 ? 3 : 2;
};

// Query block tnum of the call: block numbers start at floor(offset / QB) + b.
__device__ __forceinline__ bool pfa_block(const PagedAttn& a, int tnum, int QB, PagedSeq& s, int& slot, int& q0) {
  s = paged_at<PAGED_OFFSETS>(a.p, tnum, 1, QB, 1);
  if (s.b < 0) return false;
  slot = __builtin_amdgcn_readfirstlane(a.slot_of[s.b]) - a.slot0;
  q0 = (tnum - s.t0 / QB - s.b) * QB;
  return slot >= 0 && slot < a.pass && q0 >= 0 && q0 < s.n;
}

// What bounds it: of a SIMD's time on two chunks of 2048 and 1332 tokens behind 4096 and 2641 (H 32, D_nope + D_rope 192, D_v
// 128; 343 us, 0.89 PFLOP/s of the products that the masks leave), products take 44 % and the softmax's vector
// instructions as much, and the two waves of a SIMD hardly overlap.  Tried without gain: waves half a
// block apart (388 us), priorities between the waves of a SIMD, blocks of four waves and 32
// keys (366), query blocks sorted by their keys (343), 64 queries a wave with the exponentials of
// one half of the keys beside the products of the other (505: its fragments have no registers to
// arrive in ahead).
template <int NSTEP, int NV, int NW>
__global__ __launch_bounds__(64 * NW) void paged_fa_kernel(const PagedAttn a) {
  using C = PfaCfg<NSTEP, NV, NW>;
  extern __shared__ __attribute__((aligned(16))) char pfa_smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, ql = lane & 31;
  const int tiles = a.p.T / C::QB + a.p.B;
  int h, rank;
  if (!mla_item((int)blockIdx.x, a.H, tiles * a.nsp, h, rank)) return;
  const int split = rank % a.nsp;
  PagedSeq s;
  int slot, q0;
  if (!pfa_block(a, tiles - 1 - rank / a.nsp, C::QB, s, slot, q0)) return;
  const int qw = q0 + 32 * wave;               // the wave's first query
  const int qi = qw + ql, qc = min(qi, s.n - 1);
  const int qpos = s.first + qi;

  // query fragments: step st holds columns 16 st + 8 hi .. +7 of [q_nope | q_pe | 0], in
  // fp16 under the row's own power of two
  f16x8_t qf[NSTEP];
  float cq;
  {
    const bf16_t* qn = a.q_nope + (s.t0 + qc) * a.qn_ts + h * a.qn_hs;
    const bf16_t* qp = a.q_pe + (s.t0 + qc) * a.qp_ts + h * a.qp_hs;
    mla_u32x4 v[NSTEP];
    uint32_t mx = 0;
#pragma unroll
    for (int st = 0; st < NSTEP; ++st) {
      const int d = 16 * st + 8 * hi;
      if (a.qvec) {
        v[st] = *reinterpret_cast<const mla_u32x4*>(d < a.Dn ? qn + d : d < a.Dn + a.Dr ? qp + (d - a.Dn) : qn);
        if (d >= a.Dn + a.Dr) v[st] = mla_u32x4{0u, 0u, 0u, 0u};
      } else {
        bf16_t e8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          e8[e] = d + e < a.Dn ? qn[d + e] : d + e < a.Dn + a.Dr ? qp[d + e - a.Dn] : bf16_t(0);
        v[st] = *reinterpret_cast<const mla_u32x4*>(e8);
      }
      mx = pkv_absmax(v[st], mx);
    }
    const auto sw = __builtin_amdgcn_permlane32_swap(mx, mx, false, false);
    mx = max((uint32_t)sw[0], (uint32_t)sw[1]);
    const int e = (int)(mx >> 23);
    const int n = e == 0 || e == 255 ? 0 : min(127 - e, 126);   // the largest value to [1, 2)
    const float f = a.neg ? -pkv_pow2(n) : pkv_pow2(n);
    cq = a.c * pkv_pow2(-n);
#pragma unroll
    for (int st = 0; st < NSTEP; ++st) {
      mla_u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = pkv_pack(__uint_as_float(v[st][i] << 16) * f, __uint_as_float(v[st][i] & 0xffff0000u) * f);
      qf[st] = __builtin_bit_cast(f16x8_t, o);
    }
  }

  // keys this block needs
  const int kend = max(0, min(s.kv, s.first + min(q0 + C::QB, s.n)));
  const int nkb_all = (kend + PKV_KB - 1) / PKV_KB;
  const int kb0 = (int)((int64_t)nkb_all * split / a.nsp), nkb = (int)((int64_t)nkb_all * (split + 1) / a.nsp);
  const int64_t sh = (int64_t)slot * a.H + h;
  const char* kg = reinterpret_cast<const char*>(a.kbuf + sh * a.cap * C::DQp);
  const char* vg = reinterpret_cast<const char*>(a.vbuf + sh * a.cap * C::DVp);
  const int64_t meta = sh * (a.cap / 32);
  // block j straight into an LDS buffer, 1 KB pieces (lane: the 16 bytes that the
  // tile's swizzle puts at LDS offset 16 lane)
  const auto issue = [&](int j, int buf) {
    const uint32_t lds0 = lds_addr(pfa_smem + buf * C::BUF);
    const int64_t k0 = (int64_t)j * PKV_KB;
#pragma unroll
    for (int u = 0; u < C::NLK; ++u) {
      const int blk = wave * C::NLK + u;
      if (C::NLK * NW * 1024 > C::KT && blk * 1024 >= C::KT) break;
      const int ofs = blk * 1024 + 16 * lane;
      const int row = ofs / C::KRB, pc = (ofs % C::KRB) >> 4;
      const int g = ((row & 3) << 2) | ((row >> 2) & 3);
      const int cl = (pc & ~15) | ((pc & 15) ^ g);
      if (cl < C::DQp / 8)
        dma16s(kg + k0 * C::DQp * 2, (uint32_t)(row * C::DQp * 2 + 16 * cl), lds0 + blk * 1024);
    }
#pragma unroll
    for (int u = 0; u < C::NLV; ++u) {
      const int blk = wave * C::NLV + u;
      if (C::NLV * NW * 1024 > C::VT && blk * 1024 >= C::VT) break;
      const int ofs = blk * 1024 + 16 * lane;
      const int row = ofs / (C::DVp * 2), pc = (ofs % (C::DVp * 2)) >> 4;
      const int cl = pc ^ (mla_vswz<NV>(row) >> 1);
      dma16s(vg + k0 * C::DVp * 2, (uint32_t)(row * C::DVp * 2 + 16 * cl), lds0 + C::KT + blk * 1024);
    }
  };
  const MlbLane<C::KRB> lk(lane);

  mla_f32x16 o[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[v][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  // scale factors and missing keys of a block, asked for one block ahead
  float nkx[2] = {}, nvx[2] = {};
  uint32_t ngone[2] = {};
  const auto ask = [&](int j) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t at = meta + 2 * (int64_t)min(j, nkb - 1) + t;
      nkx[t] = a.kx[at];
      nvx[t] = a.vx[at];
      ngone[t] = a.gone[at];
    }
  };
  constexpr int AHEAD = C::NBUF - 1;
  if (kb0 < nkb) {
    issue(kb0, 0);
    if (AHEAD > 1 && kb0 + 1 < nkb) issue(kb0 + 1, 1);
    ask(kb0);
  }
  int buf = 0;
  for (int kb = kb0; kb < nkb; ++kb) {
    // block kb has landed for every wave, and every wave is done with block kb - 1
    if (AHEAD > 1 && kb + 1 < nkb)
      wait_vm<C::NLK + C::NLV>();
    else
      wait_vm<0>();
    wait_lgkm0();
    lds_barrier();
    if (kb + AHEAD < nkb) issue(kb + AHEAD, buf + AHEAD >= C::NBUF ? buf + AHEAD - C::NBUF : buf + AHEAD);
    const int k0 = kb * PKV_KB;
    const char* kt = pfa_smem + buf * C::BUF;
    const char* vt = kt + C::KT;
    buf = buf + 1 == C::NBUF ? 0 : buf + 1;
    float ct[2], vx[2];
    uint32_t gone[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      ct[t] = fmaxf(cq * nkx[t], 1.17549435e-38f);   // (a masked score stays -infinity)
      vx[t] = nvx[t];
      gone[t] = ngone[t];
    }
    ask(kb + 1);
    if (k0 > s.first + qw + 31) continue;      // behind every query of this wave
    // scores: sub-tile t, register i -> key k0 + 32 t + 8 (i / 4) + 4 hi + i % 4
    mla_f32x16 z[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) z[t][i] = 0.0f;
#pragma unroll
      for (int st = 0; st < NSTEP; ++st)
        z[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, lk.frag(kt, 32 * t, st)), qf[st], z[t], 0,
                                                      0, 0);
    }
    // six fragments on their way (two by the compiler's own order: 357 us for two chunks of 2048
    // and 1332 tokens behind 4096 and 2641, so 343; the widest values have no registers for them)
    if constexpr (NV < 8) {
      constexpr int FRAGS = 2 * NSTEP, EARLY = FRAGS < 6 ? FRAGS : 6;
      __builtin_amdgcn_sched_group_barrier(0x100, EARLY, 0);   // LDS reads
#pragma unroll
      for (int u = 0; u < FRAGS - EARLY; ++u) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);       // a product
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, EARLY, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (k0 + PKV_KB > s.kv || k0 + PKV_KB - 1 > s.first + qw || (gone[0] | gone[1])) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 8 * (i >> 2) + 4 * hi + (i & 3), key = k0 + 32 * t + j;
          if (key >= s.kv || key > qpos || ((gone[t] >> j) & 1)) z[t][i] = -INFINITY;
        }
    }
    float mb = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float mt = z[t][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mt = fmaxf(mt, z[t][i]);
      mb = fmaxf(mb, fmaf(mt, ct[t], vx[t]));
    }
    mb = mla_pair_max(mb);
    // the sums stay under an older maximum until some query's grew by 2^8 (p under it)
    if (__builtin_amdgcn_ballot_w64(mb > m && !(mb - m <= 8.0f))) {
      const float mn = fmaxf(m, mb);
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[v][i] *= alpha;
    }
    // a query whose keys so far are all masked keeps p = 0
    const float mc = m == -INFINITY ? 0.0f : m;
    f16x8_t pf[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float off = vx[t] - mc;
      float ls = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        mla_u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(z[t][8 * half + 2 * e], ct[t], off));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(z[t][8 * half + 2 * e + 1], ct[t], off));
          ls += p0;
          ls += p1;
          w[e] = pkv_pack(p0, p1);
        }
        pf[2 * t + half] = __builtin_bit_cast(f16x8_t, w);
      }
      l = fmaf(ls, __builtin_amdgcn_exp2f(-vx[t]), l);
    }
    // PV: step ps covers keys k0 + 16 ps .. +15 in the order above
    const int gq = lane >> 4, sl = lane & 15;
#pragma unroll
    for (int ps = 0; ps < 4; ++ps) {
      const int kr = 16 * ps + 4 * (gq >> 1) + (sl >> 2);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int u = 8 * v + 4 * (gq & 1) + (sl & 3);
        const mla_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) mla_v4s*)(vt + kr * (C::DVp * 2) + ((u ^ mla_vswz<NV>(kr)) << 3)));
        const mla_v4s hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) mla_v4s*)(vt + (kr + 8) * (C::DVp * 2) +
                                                         ((u ^ mla_vswz<NV>(kr + 8)) << 3)));
        typedef short v8s __attribute__((ext_vector_type(8)));
        const v8s vv = {lo[0], lo[1], lo[2], lo[3], hi4[0], hi4[1], hi4[2], hi4[3]};
        o[v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vv), pf[ps], o[v], 0, 0, 0);
      }
    }
  }

  // lane holds dv = 32 v + 8 (i / 4) + 4 hi + i % 4 of its query
  const float lt = mla_pair_sum(l);
  if (qi >= s.n) return;
  const int64_t grow = (int64_t)(s.t0 + qi) * a.H + h;
  if (a.nsp > 1) {
    const int64_t pr = (int64_t)split * a.p.T * a.H + grow;
    if (hi == 0) a.ml2[pr] = make_float2(m, lt);
    float* pw = a.po2 + pr * C::DVp;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(pw + 32 * v + 8 * g + 4 * hi) =
            make_float4(o[v][4 * g], o[v][4 * g + 1], o[v][4 * g + 2], o[v][4 * g + 3]);
    return;
  }
  const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;   // (a NaN stays one)
  bf16_t* orow = a.out + grow * a.Dv;
  const bool vec = a.Dv % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int dv = 32 * v + 8 * g + 4 * hi;
      if (vec && dv + 3 < a.Dv) {
        *reinterpret_cast<u32x2_t*>(orow + dv) = u32x2_t{pack_bf16x2(o[v][4 * g] * inv, o[v][4 * g + 1] * inv),
                                                         pack_bf16x2(o[v][4 * g + 2] * inv, o[v][4 * g + 3] * inv)};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (dv + e < a.Dv) orow[dv + e] = f2bf(o[v][4 * g + e] * inv);
      }
    }
}

// The key ranges of a query added by their weights 2^(m_i - max m).  A block: 32 tokens
// of a block of queries (as numbered for QB = 32) of one head, DVp / 4 lanes a token.  N: as
// many ranges at least.  7.6 us for 3375 tokens of 12 heads, two ranges of 64 columns (21 MB).
constexpr int PKV_MAX_SPLITS = 8;

template <int N>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedAttn a) {
  PagedSeq s;
  int slot, q0;
  if (!pfa_block(a, blockIdx.x, 32, s, slot, q0)) return;
  const int h = blockIdx.y, lanes = a.DVp / 4, dv = 4 * ((int)threadIdx.x % lanes);
  for (int q = q0 + (int)threadIdx.x / lanes; q < min(q0 + 32, s.n); q += 256 / lanes) {
    const int64_t grow = (int64_t)(s.t0 + q) * a.H + h, step = (int64_t)a.p.T * a.H;
    float2 ml[N];
    float4 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t p = grow + min(i, a.nsp - 1) * step;
      ml[i] = a.ml2[p];
      v[i] = *reinterpret_cast<const float4*>(a.po2 + p * a.DVp + dv);
    }
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, ml[i].x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= a.nsp) continue;
      // (a range whose scores are all NaN has no maximum, and a NaN for its sum)
      const float w = ml[i].x != -INFINITY ? __builtin_amdgcn_exp2f(ml[i].x - m) : 0.0f;
      l = fmaf(w, ml[i].y, l);
      o.x = fmaf(w, v[i].x, o.x);
      o.y = fmaf(w, v[i].y, o.y);
      o.z = fmaf(w, v[i].z, o.z);
      o.w = fmaf(w, v[i].w, o.w);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float f[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    bf16_t* orow = a.out + grow * a.Dv + dv;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (dv + e < a.Dv) orow[e] = f2bf(f[e]);
  }
}

// ------------------------------------------------------------------ host
static int pkv_nstep(int dqk) {
  for (int s : {2, 5, 8, 12, 16})
    if (dqk <= 16 * s) return s;
  return 0;
}
static int pkv_nv(int dv) {
  for (int s : {1, 2, 4, 8})
    if (dv <= 32 * s) return s;
  return 0;
}
// Waves of an attention block: 8 where its two buffers take more than half of the LDS, so
// that a CU has two waves a SIMD either way.
static int pkv_nw(int nstep, int nv) {
  const int buf = PKV_KB * ((16 * nstep + 127) / 128 * 256 + 64 * nv);
  return 2 * buf > 80 * 1024 ? 8 : 4;
}

// K and V of one pass stay within this; a sequence that does not fit is left to the
// latent rows.
constexpr int64_t PKV_BYTES = int64_t(4) << 30;

size_t paged_kv_carve(PagedAttn& a, const dsmoe_mla_paged_dims* d, Carver& c) {
  const int nstep = pkv_nstep(a.Dn + a.Dr), nv = pkv_nv(a.Dv);
  a.DQp = 16 * nstep;
  a.DVp = 32 * nv;
  const int64_t row = (int64_t)a.H * (a.DQp + a.DVp) * 2;
  const int64_t fit = PKV_BYTES / row / PKV_ROWS * PKV_ROWS;
  a.cap = (int)std::min<int64_t>((int64_t)align_up(std::max(d->max_kv, 1), PKV_ROWS), fit);
  a.slots = (int)std::min<int64_t>(a.p.B, a.p.T / (PAGED_FEW + 1));
  // (grids of attention blocks have room for 2^31 of them)
  if (a.cap == 0 || a.slots == 0 || (a.p.T / 32 + (int64_t)a.p.B) * (a.H + 7) * PKV_MAX_SPLITS >= (int64_t(1) << 31)) return 0;
  // about 2048 blocks (K and V) if every slot were full; 1 to 12 tiles a block measure the same
  a.kvt = (int)std::min<int64_t>(8, std::max<int64_t>(1, (int64_t)a.slots * a.H * (a.cap / PKV_ROWS) / 1024));
  a.pass = (int)std::min<int64_t>({a.slots, PKV_BYTES / (row * a.cap), 32767});
  const size_t before = c.off;
  a.slot_of = c.take<int32_t>(a.p.B);
  a.seq_of = c.take<int32_t>(a.slots);
  a.plan_rows = c.take<int32_t>(a.p.B + 1);
  const size_t keys = (size_t)a.pass * a.H * a.cap;
  a.kbuf = c.take<_Float16>(keys * a.DQp);
  a.vbuf = c.take<_Float16>(keys * a.DVp);
  a.kx = c.take<float>(keys / 32);
  a.vx = c.take<float>(keys / 32);
  a.gone = c.take<uint32_t>(keys / 32);
  // ranges of keys where the query blocks leave half of the places on the CUs idle
  const int64_t items = a.H * cdiv(a.p.T, 32 * pkv_nw(nstep, nv));
  const int64_t places = pkv_nw(nstep, nv) == 8 ? 256 : 768;
  a.nsp = (int)std::max<int64_t>(1, std::min<int64_t>({PKV_MAX_SPLITS, places / items, a.cap / 256}));
  if (a.nsp > 1) {
    a.po2 = c.take<float>((size_t)a.nsp * a.p.T * a.H * a.DVp);
    a.ml2 = c.take<float2>((size_t)a.nsp * a.p.T * a.H);
  }
  return c.off - before;
}

int launch_paged_plan(const PagedAttn& a, hipStream_t st) {
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(64), 0, st, a);
  return check_launch("mla_paged_plan");
}

template <int NS, int NT, bool VEC>
static int pkv_launch(const PagedAttn& a, int part, hipStream_t st) {
  constexpr size_t lds = (size_t)NT * 32 * ((NS * 16 + 127) / 128 * 256);
  static_assert(lds <= 160 * 1024, "LDS");
  auto kern = paged_kv_kernel<NS, NT, VEC>;
  if (lds > 64 * 1024) {
    static const hipError_t attr =
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (attr != hipSuccess) return fail(DSMOE_ERR_HIP, "mla_paged: cannot raise LDS limit");
  }
  const unsigned blocks = (unsigned)cdiv(a.cap / PKV_ROWS, a.kvt);
  const dim3 grid(blocks, (unsigned)a.H, (unsigned)a.pass * (part == 2 ? 2 : 1));
  hipLaunchKernelGGL(kern, grid, dim3(256), lds, st, a, part);
  return check_launch("mla_paged_kv");
}

template <int NS>
static int pkv_launch_nt(const PagedAttn& a, int part, hipStream_t st) {
  switch (pkv_nv(part == 1 ? a.Dv : a.Dn)) {
    case 1: return pkv_launch<NS, 1, true>(a, part, st);
    case 2: return pkv_launch<NS, 2, true>(a, part, st);
    case 4: return pkv_launch<NS, 4, true>(a, part, st);
    default: return pkv_launch<NS, 8, true>(a, part, st);
  }
}

template <int NSTEP, int NV>
static int pfa_launch(const PagedAttn& a, hipStream_t st) {
  constexpr int NW = 2 * PfaCfg<NSTEP, NV, 4>::BUF > 80 * 1024 ? 8 : 4;
  using C = PfaCfg<NSTEP, NV, NW>;
  constexpr size_t lds = C::NBUF * (size_t)C::BUF;
  static_assert(lds <= 160 * 1024, "LDS");
  auto kern = paged_fa_kernel<NSTEP, NV, NW>;
  if (lds > 64 * 1024) {
    static const hipError_t attr =
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (attr != hipSuccess) return fail(DSMOE_ERR_HIP, "mla_paged: cannot raise LDS limit");
  }
  const int tiles = a.p.T / C::QB + a.p.B;
  hipLaunchKernelGGL(kern, dim3((unsigned)mla_grid(a.H, tiles * a.nsp)), dim3(64 * NW), lds, st, a);
  int rc = check_launch("mla_paged_fa");
  if (rc || a.nsp == 1) return rc;
  auto merge = a.nsp <= 2 ? paged_merge_kernel<2> : a.nsp <= 4 ? paged_merge_kernel<4> : paged_merge_kernel<PKV_MAX_SPLITS>;
  hipLaunchKernelGGL(merge, dim3((unsigned)(a.p.T / 32 + a.p.B), (unsigned)a.H), dim3(256), 0, st, a);
  return check_launch("mla_paged_merge");
}

template <int NSTEP>
static int pfa_launch_nv(const PagedAttn& a, hipStream_t st) {
  switch (a.DVp / 32) {
    case 1: return pfa_launch<NSTEP, 1>(a, st);
    case 2: return pfa_launch<NSTEP, 2>(a, st);
    case 4: return pfa_launch<NSTEP, 4>(a, st);
    default: return pfa_launch<NSTEP, 8>(a, st);
  }
}

int launch_paged_kv(PagedAttn a, hipStream_t st) {
  const bool vec = a.kvvec && a.wvec;
  for (a.slot0 = 0; a.slot0 < a.slots; a.slot0 += a.pass) {
    a.pass = std::min(a.pass, a.slots - a.slot0);
    int rc = DSMOE_OK;
    // in one launch where both parts have as many column tiles
    const bool one = !vec || pkv_nv(a.Dn) == pkv_nv(a.Dv);
    for (int part = one ? 2 : 0; part <= 2 && (one || part < 2); ++part) {
      if (!vec) {
        rc = pkv_launch<16, 8, false>(a, part, st);
      } else {
        switch (a.Rq / 16) {
          case 2: rc = pkv_launch_nt<2>(a, part, st); break;
          case 4: rc = pkv_launch_nt<4>(a, part, st); break;
          case 8: rc = pkv_launch_nt<8>(a, part, st); break;
          case 12: rc = pkv_launch_nt<12>(a, part, st); break;
          default: rc = pkv_launch_nt<16>(a, part, st); break;
        }
      }
      if (rc) return rc;
    }
    switch (a.DQp / 16) {
      case 2: rc = pfa_launch_nv<2>(a, st); break;
      case 5: rc = pfa_launch_nv<5>(a, st); break;
      case 8: rc = pfa_launch_nv<8>(a, st); break;
      case 12: rc = pfa_launch_nv<12>(a, st); break;
      default: rc = pfa_launch_nv<16>(a, st); break;
    }
    if (rc) return rc;
  }
  return DSMOE_OK;
}

}  // namespace dsmoe
