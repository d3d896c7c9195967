// Attention of few query rows over a paged cache: tiles of 16 rows (single tokens, drafts; every
// float32 call), the keys split over work-groups and over their four waves.
//
// With S^T = K Q^T on 16x16 MFMAs lane (q = l % 16, g = l / 16) holds scores of keys 4 g + 0..3
// of a 16-key segment for row q, and P^T is in its registers as the B operand of O^T += V^T P^T.
//  * f16 / bf16: a wave's step is 32 keys (two segments, 16x16x32).  K rows go straight into the
//    A operand's registers, V rows by LDS DMA into the wave's own two-stage ring, from which
//    transposed reads take V^T (swizzled 16-byte units, as in attn_narrow.hip).
//  * f32: a step is 16 keys (16x16x4).  Contraction index g of the j-th product of a segment is
//    element 4 g + j for the scores and key 4 g + j for the sums, so K is read 16 bytes a lane and
//    V 4, both straight into registers.
// Each wave takes every fourth block of the unit's share, its loads a step ahead of its products,
// with nothing shared between waves until the end.  Segments never straddle pages (a page is a
// multiple of 16 rows), so a segment is one 64-bit offset.
//
// Scores, maxima, sums and O are float32; P is rounded to 16 bits as an MFMA operand only, its
// sum taken before.  Maxima are kept unscaled and p = exp2((x - m) c): a maximum that is rounded
// after its scaling would leave its own p at any power of two where scores are huge.
//
// A lattice leaves few keys of a block live for a few tokens.  Where the tile's tokens are at most three
// quarters of its stride, a wave lists the live keys of 512 at a time and reads their rows alone.
//
// What bounds it: HBM for long lists (64 requests of 300 to 8192 tokens, 32 heads on 8 of 128, bf16:
// 739 MB in 143 us, 5.2 TB/s, where a copy reaches 5.0; two waves a SIMD at 245 registers hold 128 KB a
// CU in flight), and for short ones the chain of trips to memory: requests, pages, rows, states, merge
// (one token over 1001 keys of 4 heads, f32, 8.9 us; drafts under a lattice of 16, 17 MB, 17 us).  In f32
// the 64 requests take 273 to 282 us (4.3 TB/s), and chunks, whose every 16 rows read their keys again,
// 414 to 436 for 512 new tokens of 4096 (76 TFLOP/s of the 152 of a library product).
//
// A dead key contributes nothing whatever its K and V hold: its score is replaced by -inf, and
// where a step is masked for some row and its V rows hold an infinity or NaN, the products are
// taken key by key and added to the rows that the key is live for (a product with a zero would be
// NaN).
#pragma once

#include <math.h>

#include <type_traits>

#include "paged_attn.hpp"

namespace pa {
namespace {

template <typename T>
__device__ __forceinline__ f32x4 mma16x32(typename Mma<T>::frag a, typename Mma<T>::frag b, f32x4 c) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16x4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// max / sum over the four lanes l % 16 + 16 g that hold one query row
__device__ __forceinline__ float quad_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return row_nan_max(nan_max(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
  return row_sum(__builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]));
}

constexpr int kWaves = 4;

// Bits of the words that hold an infinity or NaN in some half (f16 / bf16): the largest magnitude
// of each half against the type's first one that is not finite.
template <typename T>
struct Finite16 {
  uint32_t lo = 0u, hi = 0u;
  __device__ void add(uint32_t w) {
    lo = max(lo, w & 0x7fffu);
    hi = max(hi, w & 0x7fff0000u);
  }
  __device__ bool all() const {
    constexpr uint32_t inf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
    return lo < inf && hi < (inf << 16);
  }
};

template <typename T, int D>
struct RowsShape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int NS = F32 ? 1 : 2;           // 16-key segments of a step
  static constexpr int LG = F32 ? 4 : 5;           // log2 keys of a step
  static constexpr int PER = 64 / NS;              // steps held at a time, a segment per lane
  static constexpr int ROW = D * (int)sizeof(T);   // bytes of a row
  static constexpr int RING = F32 ? 0 : kWaves * 2 * 2 * 16 * ROW;
  static constexpr int OP = D + 4;                 // floats of a row of a wave's O at the end
  static constexpr int ENDS = kWaves * kRows * (OP + 2) * 4;
  static constexpr int LIST = 512;                 // keys of a wave's list of live ones
  static constexpr int LIST_AT = RING > ENDS ? RING : ENDS;
  static constexpr int SMEM = LIST_AT + kWaves * LIST * 4;
};

template <typename T, int D>
__device__ __forceinline__ void rows_body(const PagedK& a, int32_t id, char* smem, int32_t* flag) {
  using S = RowsShape<T, D>;
  constexpr bool F32 = S::F32;
  constexpr int NS = S::NS, PER = S::PER, ROW = S::ROW, ESZ = sizeof(T);
  constexpr int NB = D / 16;                       // blocks of 16 output columns
  constexpr int NK = F32 ? D / 16 : D / 32;        // 16-byte units of a K or Q row that a lane holds
  constexpr int SEG = 16 * ROW, STAGE = 2 * SEG;
  const PagedPart& part = a.rows;

  const int tid = threadIdx.x, lane = tid & 63, q16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  const RawRequest raw = raw_request(a, 0, lane);
  // (what depends on the lane alone, while these are on their way)
  const uint32_t koff = (uint32_t)(q16 * (int32_t)a.c_sn) + 16u * (uint32_t)g;
  uint32_t voff[F32 ? 4 : Rows<D>::NI];
  if constexpr (F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) voff[j] = (uint32_t)((4 * g + j) * (int32_t)a.c_sn) + 4u * (uint32_t)q16;
  } else {
    using R = Rows<D>;
#pragma unroll
    for (int j = 0; j < R::NI; ++j) {
      const int r = R::RPI * j + lane / R::UPR;
      const int sw = D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
      voff[j] = (uint32_t)(r * (int32_t)a.c_sn) + 16u * (uint32_t)((lane % R::UPR) ^ sw);
    }
  }
  const uint32_t ring0 = (uint32_t)(uintptr_t)(lds_char_t*)smem + (uint32_t)(w * 2 * STAGE);
  lds_cptr vptr[F32 ? 1 : NB];
  if constexpr (!F32) {
    // transposed reads of 16 columns (block db) of rows 4 g + q16 / 4 of a segment
#pragma unroll
    for (int db = 0; db < NB; ++db) {
      const int r = 4 * g + (q16 >> 2);
      const int sw = D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
      vptr[db] = (lds_cptr)smem + w * 2 * STAGE + r * ROW + 16 * ((2 * db + ((q16 & 3) >> 1)) ^ sw) + 8 * (q16 & 1);
      asm volatile("" : "+v"(vptr[db]));
    }
  }

  const Unit u = find_unit<kRows, S::LG>(a, part, raw, id, lane);
  if (!u.found) return;

  // ---- the tile's rows -----------------------------------------------------------
  const int rows = u.rq.n * a.G;
  const int i0 = u.tile * kRows;
  const int n_rows = imin(rows - i0, kRows);
  const int i = imin(i0 + q16, rows - 1);          // (a lane past the rows repeats the last)
  const int tok = token_of(a, i), head = u.h * a.G + (i - tok * a.G);
  const int pos0 = u.rq.len - u.rq.n;
  const int q_pos = pos0 + tok;
  const int q_lo = pos0 + token_of(a, i0), q_hi = pos0 + token_of(a, i0 + n_rows - 1);
  const int len = u.rq.len;

  u32x4 qf[NK];
  {
    const char* qrow = a.q + (int64_t)(u.rq.start + tok) * a.q_st + (int64_t)head * a.q_sh + 16 * g;
#pragma unroll
    for (int kc = 0; kc < NK; ++kc) qf[kc] = *reinterpret_cast<const u32x4*>(qrow + 64 * kc);
  }

  // ---- the keys of this share ------------------------------------------------------
  const KernelMask mask = kernel_mask(a);
  const KeyList kl = key_list(mask, q_lo, q_hi, len, S::LG);
  int32_t j0, j1;
  share_of(kl.count(), u.split, u.splits, &j0, &j1);
  const int n_steps = j1 - j0 > w ? (j1 - j0 - w + kWaves - 1) / kWaves : 0;
  const int32_t* table = a.tables + (int64_t)u.r * a.pitch;
  const char* kbase = a.k + u.h * a.c_sh;
  const char* vbase = a.v + u.h * a.c_sh;

  // PER steps at a time: lane l holds segment l, its first key and its offset in the cache; bit l
  // of live / full: some pair of it may be live / all are.  The next ones' pages are loaded
  // halfway through these.
  int32_t c_key = 0, r_page = -1;
  int64_t c_off = 0;
  uint64_t c_live = 0ull, c_full = 0ull;
  // (the lane's segment of step st)
  auto key_at = [&](int st) __attribute__((always_inline)) -> int32_t {
    return st < n_steps ? (kl.block(j0 + w + kWaves * st) << S::LG) + (NS == 2 ? 16 * (lane & 1) : 0) : len;
  };
  auto key_of = [&](int c) __attribute__((always_inline)) -> int32_t { return key_at(c * PER + lane / NS); };
  auto load_raw = [&](int c) __attribute__((always_inline)) {
    const int32_t key = key_of(c);
    r_page = key < len ? table[key >> a.page_lg] : -1;
  };
  auto take_raw = [&](int c) __attribute__((always_inline)) {
    const int32_t key = key_of(c);
    const int32_t page = checked_page(r_page, a.n_pages);
    int v = mask_verdict(mask, q_lo, q_hi, key, key + 15);  // (does not wait for the pages)
    if (v == kFull && key + 15 >= len) v = kPartial;
    if (key >= len || page < 0) v = kDead;
    c_live = __ballot(v != kDead);
    c_full = __ballot(v == kFull);
    c_key = key;
    c_off = (int64_t)imax(page, 0) * a.c_sp + (int64_t)(key & ((1 << a.page_lg) - 1)) * a.c_sn;
    if constexpr (NS == 2) {
      // (a dead segment of a live step holds the other one's rows again)
      const bool dead = !((c_live >> lane) & 1ull);
      const int32_t lo = __shfl_xor((int32_t)c_off, 1), hi = __shfl_xor((int32_t)(c_off >> 32), 1);
      if (dead) c_off = (int64_t)((uint64_t)(uint32_t)lo | ((uint64_t)(uint32_t)hi << 32));
    }
  };

  struct Step {
    int key;
    uint32_t live, full;  // NS bits each
  };
  struct Data {  // what a step needs in registers
    u32x4 k[NS][NK];
    float v[F32 ? 4 : 1][F32 ? NB : 1];
  };
  auto prefetch = [&](int st, int SB, Step& s, Data& d) __attribute__((always_inline)) {
    if (st % PER == 0) take_raw(st / PER);
    if (st % PER == PER / 2) load_raw(st / PER + 1);
    const int l0 = NS * (st % PER);
    s.live = (uint32_t)(c_live >> l0) & ((1u << NS) - 1u);
    s.full = (uint32_t)(c_full >> l0) & ((1u << NS) - 1u);
    s.key = __builtin_amdgcn_readlane(c_key, l0);
    if (s.live == 0u) return;
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)c_off, l0 + t);
      const int32_t hi = __builtin_amdgcn_readlane((int)(c_off >> 32), l0 + t);
      const int64_t off = (int64_t)((uint64_t)lo | ((uint64_t)(uint32_t)hi << 32));
      const char* kp = kbase + off;
      const char* vp = vbase + off;
#pragma unroll
      for (int kc = 0; kc < NK; ++kc) d.k[t][kc] = *reinterpret_cast<const u32x4*>(kp + koff + 64 * kc);
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int db = 0; db < NB; ++db) d.v[j][db] = *reinterpret_cast<const float*>(vp + voff[j] + 64 * db);
      } else {
#pragma unroll
        for (int j = 0; j < Rows<D>::NI; ++j) dma_x4(ring0 + SB * STAGE + t * SEG + j * 1024, vp, voff[j]);
      }
    }
  };

  f32x4 acc[NB];
#pragma unroll
  for (int db = 0; db < NB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_part = 0.f;

  // One step's keys; all: every one is live for every row, else bit i of word: key i is live for this
  // lane's row.
  auto compute = [&](int SB, bool all, uint32_t word, const Data& d) __attribute__((always_inline)) {
    f32x4 x[NS];
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      x[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kc = 0; kc < NK; ++kc) {
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t kx = d.k[t][kc][j], qx = qf[kc][j];
            x[t] = mma16x4(__builtin_bit_cast(float, kx), __builtin_bit_cast(float, qx), x[t]);
          }
        } else {
          using Frag = typename Mma<T>::frag;
          x[t] = mma16x32<T>(__builtin_bit_cast(Frag, d.k[t][kc]), __builtin_bit_cast(Frag, qf[kc]), x[t]);
        }
      }
    }
    if (!all) {
#pragma unroll
      for (int t = 0; t < NS; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((word >> (16 * t + 4 * g + e)) & 1u)) x[t][e] = -INFINITY;
    }
    float mx = nan_max(nan_max(x[0][0], x[0][1]), nan_max(x[0][2], x[0][3]));
    if constexpr (NS == 2) mx = nan_max(mx, nan_max(nan_max(x[1][0], x[1][1]), nan_max(x[1][2], x[1][3])));
    const float m_new = nan_max(m_run, quad_max(mx));
    // (a NaN maximum makes the row NaN by its own probabilities; nothing needs a rescale)
    if (__ballot((m_new - m_run) * a.c > kLazy) != 0ull) {
      const float alpha = __builtin_amdgcn_exp2f((m_run - base_of(m_new)) * a.c);
      m_run = m_new;
      l_part *= alpha;
#pragma unroll
      for (int db = 0; db < NB; ++db) acc[db] *= alpha;
    }
    const float m_base = base_of(m_run);
    float p[4 * NS];
#pragma unroll
    for (int e = 0; e < 4 * NS; ++e) {
      p[e] = __builtin_amdgcn_exp2f((x[e >> 2][e & 3] - m_base) * a.c);
      l_part += p[e];
    }
    if constexpr (F32) {
      bool fin = true;
      if (!all) {
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int db = 0; db < NB; ++db) big = nan_max(big, __builtin_fabsf(d.v[j][db]));
        fin = __ballot(!(big < INFINITY)) == 0ull;
      }
      if (fin) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int db = 0; db < NB; ++db) acc[db] = mma16x4(d.v[j][db], p[j], acc[db]);
      } else {
#pragma unroll 1
        for (int gg = 0; gg < 4; ++gg)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool on = (word >> (4 * gg + j)) & 1u;
#pragma unroll
            for (int db = 0; db < NB; ++db) {
              const f32x4 y = mma16x4(g == gg ? d.v[j][db] : 0.f, g == gg ? p[j] : 0.f, f32x4{0.f, 0.f, 0.f, 0.f});
              if (on) acc[db] += y;
            }
          }
      }
    } else {
      using Frag = typename Mma<T>::frag;
      f32x8 pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = p[e];
      const Frag pf = Mma<T>::cvt(pv);
      auto v_frag = [&](int db) __attribute__((always_inline)) -> u32x4 {
        const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vptr[db] + SB * STAGE));
        const s16x4 x2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vptr[db] + SB * STAGE + SEG));
        return u32x4{__builtin_bit_cast(uint2, x1).x, __builtin_bit_cast(uint2, x1).y, __builtin_bit_cast(uint2, x2).x,
                     __builtin_bit_cast(uint2, x2).y};
      };
      bool fin = true;
      if (!all) {
        Finite16<T> f;
#pragma unroll
        for (int db = 0; db < NB; ++db) {
          const u32x4 vx = v_frag(db);
#pragma unroll
          for (int e = 0; e < 4; ++e) f.add(vx[e]);
        }
        fin = __ballot(!f.all()) == 0ull;
      }
      if (fin) {
#pragma unroll
        for (int db = 0; db < NB; ++db) acc[db] = mma16x32<T>(__builtin_bit_cast(Frag, v_frag(db)), pf, acc[db]);
      } else {
        // key x of segment t is contraction index 4 t + x % 4 of lane group x / 4
        const u32x4 pw = __builtin_bit_cast(u32x4, pf);
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
          const int e = 4 * (key >> 4) + (key & 3), gg = (key >> 2) & 3;
          const uint32_t half = g == gg ? ((e & 1) ? 0xffff0000u : 0x0000ffffu) : 0u;
          u32x4 keep;
#pragma unroll
          for (int z = 0; z < 4; ++z) keep[z] = z == (e >> 1) ? half : 0u;
          const bool on = (word >> key) & 1u;
#pragma unroll
          for (int db = 0; db < NB; ++db) {
            const f32x4 y = mma16x32<T>(__builtin_bit_cast(Frag, v_frag(db) & keep), __builtin_bit_cast(Frag, pw & keep),
                                        f32x4{0.f, 0.f, 0.f, 0.f});
            if (on) acc[db] += y;
          }
        }
      }
    }
  };

  auto compute_block = [&](int SB, const Step& s, const Data& d) __attribute__((always_inline)) {
    if (s.live == 0u) return;
    const bool all = s.full == (1u << NS) - 1u;
    uint32_t word = 0xffffffffu;
    if (!all) {
      word = mask_word(mask, q_pos, s.key, len);
      if (!(s.live & 1u)) word &= 0xffff0000u;
      if (NS == 1 || !(s.live & 2u)) word &= 0x0000ffffu;
    }
    compute(SB, all, word, d);
  };

  Data d0{}, d1{};
  // The step's V rows are in LDS and its K rows in registers once everything issued is done.
  // The memory clobber keeps the ring's reads on their side of the wait (no barrier does),
  // and the last step's are done before the next DMA into their stage; the uses make the
  // compiler's own wait fall here, before the next step's loads.
  auto arrive = [&](const Data& d) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int t = 0; t < NS; ++t)
#pragma unroll
      for (int kc = 0; kc < NK; ++kc) asm volatile("" ::"v"(d.k[t][kc]));
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int db = 0; db < NB; ++db) asm volatile("" ::"v"(d.v[j][db]));
    }
    asm volatile("" ::"v"(r_page));
  };
  const int n_tok = q_hi - q_lo + 1;
  if (n_steps > 0) load_raw(0);
  if (!by_lists(n_tok, a.stride)) {
    // ---- block by block -------------------------------------------------------------
    Step s0{}, s1{};
    if (n_steps > 0) prefetch(0, 0, s0, d0);
    int st = 0;
    for (; st + 1 < n_steps; st += 2) {
      arrive(d0);
      prefetch(st + 1, 1, s1, d1);
      compute_block(0, s0, d0);
      arrive(d1);
      if (st + 2 < n_steps) prefetch(st + 2, 0, s0, d0);
      compute_block(1, s1, d1);
    }
    if (st < n_steps) {
      arrive(d0);
      compute_block(0, s0, d0);
    }
  } else {
    // ---- by lists of live keys -------------------------------------------------------
    // 32 segments at a time: lane l (below 32) finds which of segment l's keys are live for which
    // tokens of the tile, and the wave lists the keys that are for some: segment and key in it, and
    // a bit per token above.  Steps then take 32 (f32: 16) listed keys each, row by row.
    constexpr int PL = S::LIST / 16;            // segments of a list
    uint32_t* list = reinterpret_cast<uint32_t*>(smem + S::LIST_AT) + w * S::LIST;
    const int tq = q_pos - q_lo;                // this lane's token among the tile's
    for (int c = 0; c * (PL / NS) < n_steps; ++c) {
      const int st0 = c * (PL / NS);            // first step (block) of this list
      const int32_t key = lane < PL ? key_at(st0 + lane / NS) : len;
      const int32_t page = checked_page(r_page, a.n_pages);
      const bool some = key < len && page >= 0;
      c_off = (int64_t)imax(page, 0) * a.c_sp + (int64_t)(key & ((1 << a.page_lg) - 1)) * a.c_sn;
      if ((c + 1) * (PL / NS) < n_steps) {
        const int32_t next = lane < PL ? key_at(st0 + PL / NS + lane / NS) : len;
        r_page = next < len ? table[next >> a.page_lg] : -1;
      }
      uint32_t any = 0u, of[8] = {};            // of[p]: tokens of keys 2 p (low half) and 2 p + 1
#pragma unroll 1
      for (int t = 0; t < n_tok; ++t) {
        const uint32_t x = some ? mask_word(mask, q_lo + t, key, len) & 0xffffu : 0u;
        any |= x;
#pragma unroll
        for (int p = 0; p < 8; ++p) of[p] |= ((x >> (2 * p)) & 1u) << t | ((x >> (2 * p + 1)) & 1u) << (16 + t);
      }
      const int n_mine = __builtin_popcount(any), n_in = wave_scan(n_mine);
      const int total = __builtin_amdgcn_readlane(n_in, 63);
      int at = n_in - n_mine;
#pragma unroll
      for (int b = 0; b < 16; ++b)
        if ((any >> b) & 1u)
          list[at++] = (uint32_t)(16 * lane + b) | ((b & 1) ? of[b >> 1] & 0xffff0000u : of[b >> 1] << 16);
      asm volatile("" ::: "memory");  // (a wave's LDS accesses stay in order)
      // offset in the cache of listed key i (past the list: the last one's)
      auto row_off = [&](int i) __attribute__((always_inline)) -> int64_t {
        const uint32_t e = list[imin(i, total - 1)];
        const int l = (e >> 4) & (PL - 1);
        const uint32_t lo = (uint32_t)__shfl((int32_t)(uint32_t)c_off, l);
        const int32_t hi = __shfl((int32_t)(c_off >> 32), l);
        return (int64_t)((uint64_t)lo | ((uint64_t)(uint32_t)hi << 32)) + (int64_t)(e & 15u) * a.c_sn;
      };
      auto fetch = [&](int i0, int SB, Data& d) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NS; ++t) {
          const char* kp = kbase + row_off(i0 + 16 * t + q16) + 16 * g;
#pragma unroll
          for (int kc = 0; kc < NK; ++kc) d.k[t][kc] = *reinterpret_cast<const u32x4*>(kp + 64 * kc);
          if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const char* vp = vbase + row_off(i0 + 4 * g + j) + 4 * q16;
#pragma unroll
              for (int db = 0; db < NB; ++db) d.v[j][db] = *reinterpret_cast<const float*>(vp + 64 * db);
            }
          } else {
            using R = Rows<D>;
#pragma unroll
            for (int j = 0; j < R::NI; ++j) {
              const int r = R::RPI * j + lane / R::UPR;
              const int sw = D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
              dma_x4_va(ring0 + SB * STAGE + t * SEG + j * 1024,
                        vbase + row_off(i0 + 16 * t + r) + 16 * ((lane % R::UPR) ^ sw));
            }
          }
        }
      };
      auto take = [&](int i0, int SB, const Data& d) __attribute__((always_inline)) {
        uint32_t word = 0u;
        const int n = imin(total - i0, 16 * NS);
        if (n_tok == 1) {
          word = n >= 32 ? 0xffffffffu : (1u << n) - 1u;
        } else {
#pragma unroll
          for (int x = 0; x < 4 * NS; ++x) {
            const u32x4 e = *reinterpret_cast<const u32x4*>(list + i0 + 4 * x);
#pragma unroll
            for (int z = 0; z < 4; ++z) word |= ((e[z] >> (16 + tq)) & 1u) << (4 * x + z);
          }
          if (n < 32) word &= (1u << n) - 1u;  // (entries past the list are of an earlier one)
        }
        compute(SB, n_tok == 1 && n == 16 * NS, word, d);
      };
      constexpr int ST = 16 * NS;
      if (total > 0) fetch(0, 0, d0);
      int i = 0;
      for (; i + ST < total; i += 2 * ST) {
        arrive(d0);
        fetch(i + ST, 1, d1);
        take(i, 0, d0);
        arrive(d1);
        if (i + 2 * ST < total) fetch(i + 2 * ST, 0, d0);
        take(i + ST, 1, d1);
      }
      if (i < total) {
        arrive(d0);
        take(i, 0, d0);
      }
      // (the last step's reads of its stage are done before the next list's DMA into it)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }

  // ---- the waves' states become one, and those of the tile's shares ---------------------
  const float l_own = quad_sum(l_part);
  __syncthreads();  // every wave is past its ring
  float* red_o = reinterpret_cast<float*>(smem);                 // [wave][row][OP]
  float* red_ml = red_o + kWaves * kRows * S::OP;                // [wave][row][2]
#pragma unroll
  for (int db = 0; db < NB; ++db)
    *reinterpret_cast<f32x4*>(red_o + (w * kRows + q16) * S::OP + 16 * db + 4 * g) = acc[db];
  if (g == 0) {
    red_ml[2 * (w * kRows + q16)] = m_run;
    red_ml[2 * (w * kRows + q16) + 1] = l_own;
  }
  // thread: a row and D / 16 of its columns
  constexpr int CPT = D / 16;
  const int row = tid >> 4, c0 = (tid & 15) * CPT;
  float M, L, out[CPT];
  auto gather = [&]() __attribute__((always_inline)) {
    __syncthreads();
    float mw[kWaves];
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      mw[x] = red_ml[2 * (x * kRows + row)];
      M = nan_max(M, mw[x]);
    }
#pragma unroll
    for (int e = 0; e < CPT; ++e) out[e] = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const float f = __builtin_amdgcn_exp2f((mw[x] - base_of(M)) * a.c);
      L += f * red_ml[2 * (x * kRows + row) + 1];
#pragma unroll
      for (int e = 0; e < CPT; ++e) out[e] += f * red_o[(x * kRows + row) * S::OP + c0 + e];
    }
  };
  gather();
  if (u.splits > 1) {
    constexpr int SLOT_B = slot_floats(kRows, D) * 4, ML = kRows * D * 4;
    char* first = part.part + (int64_t)u.slot * SLOT_B;  // of the tile's shares
    if (row < n_rows) {
      char* own = first + (int64_t)u.split * SLOT_B;
#pragma unroll
      for (int e = 0; e < CPT; e += 4)
        share_store4(own + (row * D + c0 + e) * 4, f32x4{out[e], out[e + 1], out[e + 2], out[e + 3]});
      if (c0 == 0) {
        share_store(reinterpret_cast<float*>(own + ML) + 2 * row, M);
        share_store(reinterpret_cast<float*>(own + ML) + 2 * row + 1, L);
      }
    }
    if (!last_share(part, u, tid, flag)) return;
    // every fourth share to a wave, two of them at once: lane (row 4 i + l / 16, the columns of l % 16)
    // for all i, every load of a pair on its way before the first is used; then as the waves' states
    // above
    const int r0 = lane >> 4, col = (lane & 15) * CPT;
    const Shares all = shares_at(first, u.splits * SLOT_B);
    float m[4], l[4];
    f32x4 x[4][CPT / 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int e = 0; e < CPT / 4; ++e) x[i][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll 1
    for (int s = w; s < u.splits; s += 2 * kWaves) {
      float ms[2][4], ls[2][4];
      f32x4 os[2][4][CPT / 4];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int32_t at = imin(s + y * kWaves, u.splits - 1) * SLOT_B;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (4 * i >= n_rows) break;
          const f32x2 ml = share_load2(all, 8 * (4 * i + r0), at + ML);
          ms[y][i] = ml[0];
          ls[y][i] = ml[1];
#pragma unroll
          for (int e = 0; e < CPT / 4; ++e) os[y][i][e] = share_load4(all, ((4 * i + r0) * D + col + 4 * e) * 4, at);
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (s + y * kWaves >= u.splits) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (4 * i >= n_rows) break;
          const float mn = nan_max(m[i], ms[y][i]);
          const float f0 = __builtin_amdgcn_exp2f((m[i] - base_of(mn)) * a.c), f1 = __builtin_amdgcn_exp2f((ms[y][i] - base_of(mn)) * a.c);
          m[i] = mn;
          l[i] = f0 * l[i] + f1 * ls[y][i];
#pragma unroll
          for (int e = 0; e < CPT / 4; ++e) x[i][e] = f0 * x[i][e] + f1 * os[y][i][e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + r0;
#pragma unroll
      for (int e = 0; e < CPT / 4; ++e) *reinterpret_cast<f32x4*>(red_o + (w * kRows + r) * S::OP + col + 4 * e) = x[i][e];
      if (col == 0) {
        red_ml[2 * (w * kRows + r)] = m[i];
        red_ml[2 * (w * kRows + r) + 1] = l[i];
      }
    }
    gather();
  }
  if (row >= n_rows) return;
  const int ir = i0 + row, t_r = token_of(a, ir), h_r = u.h * a.G + (ir - t_r * a.G);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  char* orow = a.o + (int64_t)(u.rq.start + t_r) * a.o_st + (int64_t)h_r * a.o_sh;
#pragma unroll
  for (int e = 0; e < CPT; e += 4)
    Mma<T>::store4(orow + (c0 + e) * ESZ, f32x4{out[e], out[e + 1], out[e + 2], out[e + 3]} * inv);
  if (a.lse && c0 == 0)
    a.lse[(int64_t)(u.rq.start + t_r) * a.lse_st + (int64_t)h_r * a.lse_sh] = L == 0.f ? -INFINITY : (M * a.c + log2f(L)) * kLn2;
}

}  // namespace
}  // namespace pa
