// Attention of chunks of new tokens over a paged cache, f16 / bf16: tiles of 128 query rows (new
// tokens times the heads that share a KV head), 64 keys a step.
//
// A work-group is four waves of 32 rows.  Scores are taken transposed (S^T = K Q^T) on 32x32x16
// MFMAs, so a lane owns a query row, a maximum is in its registers but for one exchange, and P^T is
// already the B operand of O^T += V^T P^T.  K and V rows come by LDS DMA into a ring of two slots
// each (layout in lds_rows.hpp), wave w moving segment w (16 rows, inside one page) of a step.  The
// scores of step j + 1 are computed beside the exponentials of step j, whose products follow: one
// straight line of MFMA, LDS and VALU work in an order that is spelled out, behind one wait and one
// barrier per step.
//
// The blocks of keys that may be live for the tile are a list of two ranges (page_math.hpp); its
// entries are held 16 steps at a time, a segment per lane, with each wave's verdicts on its own
// rows; a step that is not all live for a wave is masked by words of 32 keys computed from the mask's
// terms, and its dead pairs have P = 0.
//
// A dead key contributes nothing whatever it holds, but 0 times an infinity or NaN in its V row is
// NaN.  That shows in the sums, so a work-group whose sums are not finite takes its list again, step
// by step, and where a masked chunk of 16 keys has V rows that are not finite it takes the products
// key by key, added only to the rows that the key is live for.  So does one with maxima past 2^24 in
// log2 units: p = exp2(fma(x, c, -m)) has the rounding of m = max(x c) in its exponent, the same for
// all keys of the row, so it falls out of the result while it is small (below 2^24 half a unit at
// most) but empties or overflows the row where m is large; that row's second pass has m in units of
// the scores and p = exp2((x - m) c), and what the rounding of m c leaves out goes with it to the
// merge of its shares.
//
// Scores, maxima, sums and O are float32; P is rounded to 16 bits as an MFMA operand only, its sum
// taken before.
//
// What bounds it: for long lists at D = 128 power (2000 new tokens of 30001, 32 heads on 8, bf16: 873
// to 993 us from card to card, 0.96 to 1.09 PFLOP/s of the 1.07 to 1.12 of a large library product; the
// clock falls to 1.6 to 1.8 GHz with the matrix cores busy 52 to 54% of it), at D = 64 the exponentials'
// issue (4096 of 4096, 32 heads: 104 us, 660 TFLOP/s), and for lists of a few steps what is outside them:
// 5 to 9 us a unit, two units a CU (chunks of 1000 to 4096 under a window of 1024 and 64 sinks, 18 steps a
// unit: 262 to 289 us, 735 to 810 TFLOP/s).
#pragma once

#include <math.h>

#include <type_traits>

#include "page_steps.hpp"
#include "paged_attn.hpp"

namespace pa {
namespace {

template <typename T>
__device__ __forceinline__ bool not_finite16(uint32_t lo, uint32_t hi) {
  constexpr uint32_t inf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  return lo >= inf || hi >= (inf << 16);
}

// Scores of a step's two blocks of 32 keys.
struct StepScores {
  f32x16 x0 = {}, x1 = {};
};

template <typename T, int D>
struct TileShape {
  static constexpr int SLOT = 64 * Rows<D>::ROW;   // a step's K or V
  static constexpr int SMEM = 4 * SLOT;            // aligned to two slots
};

template <typename T, int D, int PART = kWhole>
__device__ __forceinline__ void tile_body(const PagedK& a, int32_t id, char* smem, int32_t* flag) {
  using Frag = typename Mma<T>::frag;
  using R = Rows<D>;
  constexpr int ESZ = 2, NQF = D / 16, NDB = D / 32;
  constexpr int SLOT = TileShape<T, D>::SLOT;
  constexpr int VRING = 0, KRING = 2 * SLOT;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char_t*)smem;
  const PagedPart& part = PART == kPrefix ? a.pre_tiles : a.tiles;

  const int tid = threadIdx.x, lane = tid & 63, G = lane >> 5, m = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  const RawRequest raw = raw_request<PART>(a, 0, lane);
  // (what depends on the lane alone, while these are on their way)
  uint32_t doff[R::NI];
  dma_offsets<D>(doff, a.c_sn, lane);
#pragma unroll
  for (int x = 1; x < R::NI; ++x) doff[x] += (uint32_t)(x * R::RPI * a.c_sn);
  // (K reads are on the slot of the step ahead, V reads on that of the current one; a slot is one bit
  // of an address, as the rings are aligned to two slots)
  TileReads<D> rd = tile_reads<D>((lds_cptr)smem, lane);
  const Unit u = find_unit<kTileRows, kTileLg, PART>(a, part, raw, id, lane);
  if (!u.found) return;
  if (PART == kPrefix && u.slot + u.splits > part.slots) return;  // (a sharing of another step)

  // ---- rows ------------------------------------------------------------------------
  const int rows = u.rq.n * a.G, len = u.rq.len, pos0 = len - u.rq.n;
  const int i0 = u.tile * kTileRows;
  const int n_rows = imin(rows - i0, kTileRows);
  const int w0 = imin(i0 + 32 * w, rows - 1), w1 = imin(i0 + 32 * w + 31, rows - 1);  // this wave's rows
  int q_lo = pos0 + token_of(a, w0), q_hi = pos0 + token_of(a, w1);
  if (PART == kPrefix) {
    const int32_t p = position_of<PART>(a, u, token_of(a, imin(i0 + 32 * w + m, rows - 1)));
    q_lo = lanes_min(p);
    q_hi = lanes_max(p);
  }

  // ---- the keys of this share ---------------------------------------------------------
  const KernelMask mask = kernel_mask(a);
  const KeyList kl = PART == kPrefix ? key_list(mask, u.x0, u.x1, len, kTileLg)
                                     : key_list(mask, pos0 + token_of(a, i0), pos0 + token_of(a, i0 + n_rows - 1), len, kTileLg);
  const int32_t skip = PART == kOwn ? kl.before(u.x0 >> kTileLg) : 0;
  int32_t j0, j1;
  share_of(kl.count() - skip, u.split, u.splits, &j0, &j1);
  if (PART == kOwn) {
    j0 += skip;
    j1 += skip;
  }
  const int n_steps = j1 - j0;
  const int32_t* table = a.tables + (int64_t)u.r * a.pitch;
  const char* kbase = a.k + u.h * a.c_sh;
  const char* vbase = a.v + u.h * a.c_sh;
  // 16 steps: lane 4 s + t holds segment t of step s, its offset in the cache; bit 4 s + t of live /
  // full: some pair of it may be live for this wave / all are.  The next 16 steps' pages are loaded
  // halfway through these.
  int32_t r_page = -1;
  int64_t c_off = 0;
  uint64_t c_live = 0ull, c_full = 0ull;
  auto key_of = [&](int c) __attribute__((always_inline)) -> int32_t {
    const int s = 16 * c + (lane >> 2);
    return s < n_steps ? (kl.block(j0 + s) << kTileLg) + 16 * (lane & 3) : len;
  };
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
    if (PART == kOwn && key < u.x0) v = kDead;
    c_live = __ballot(v != kDead);
    c_full = __ballot(v == kFull);
    // (keys without a page read the cache's first one, and are dead)
    c_off = (int64_t)imax(page, 0) * a.c_sp + (int64_t)(key & ((1 << a.page_lg) - 1)) * a.c_sn;
  };
  load_raw(0);  // (in flight beside the loads of Q)

  // ---- Q ----------------------------------------------------------------------------------
  int q_pos;  // position of this lane's row (a lane past the rows repeats the last)
  Frag qf[NQF];
  {
    const int i = imin(i0 + 32 * w + m, rows - 1), tok = token_of(a, i), head = u.h * a.G + (i - tok * a.G);
    q_pos = PART == kPrefix ? position_of<PART>(a, u, tok) : pos0 + tok;
    const char* qrow = a.q + (int64_t)row_of<PART>(a, u, tok) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
    for (int kc = 0; kc < NQF; ++kc)
      qf[kc] = __builtin_bit_cast(Frag, *reinterpret_cast<const uint4*>(qrow + (16 * kc + 8 * G) * ESZ));
  }

  struct Step {
    int64_t off;          // of the segment that this wave moves
    uint32_t live, full;  // 4 bits: the step's segments
  };
  auto step_of = [&](int j) __attribute__((always_inline)) -> Step {
    if ((j & 15) == 0) take_raw(j >> 4);
    if ((j & 15) == 8) load_raw((j >> 4) + 1);
    const int l0 = 4 * (j & 15);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)c_off, l0 + w);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(c_off >> 32), l0 + w);
    return Step{(int64_t)((uint64_t)lo | ((uint64_t)hi << 32)), (uint32_t)(c_live >> l0) & 15u, (uint32_t)(c_full >> l0) & 15u};
  };
  auto dma = [&](uint32_t ring, const char* base) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < R::NI; ++x) dma_x4(lds0 + ring + (uint32_t)(w * 16 * R::ROW) + x * 1024, base, doff[x]);
  };

  f32x16 acc[NDB];
#pragma unroll
  for (int x = 0; x < NDB; ++x) acc[x] = f32x16{0};
  float m_run = -INFINITY, l_part = 0.f;  // (log2 units)
  StepScores sa, sb;  // of the current step and the next, in turn
  // (held in a register: a scalar load of an argument inside the loop would wait for the LDS reads
  // in flight)
  float c_exp = a.c;
  asm volatile("" : "+s"(c_exp));

  // Scores of both blocks of the step in the K slot that the row reads are on.
  auto qk = [&](f32x16& x0, f32x16& x1) __attribute__((always_inline)) {
    u32x4 ka[NQF], kb[NQF];
#pragma unroll
    for (int kc = 0; kc < NQF; ++kc) ka[kc] = *(lds_u4*)(rd.row(kc) + KRING);
#pragma unroll
    for (int kc = 0; kc < NQF; ++kc) kb[kc] = *(lds_u4*)(rd.row(kc) + KRING + 32 * R::ROW);
    x0 = Mma<T>::mma(__builtin_bit_cast(Frag, ka[0]), qf[0], f32x16{0});
#pragma unroll
    for (int kc = 1; kc < NQF; ++kc) x0 = Mma<T>::mma(__builtin_bit_cast(Frag, ka[kc]), qf[kc], x0);
    x1 = Mma<T>::mma(__builtin_bit_cast(Frag, kb[0]), qf[0], f32x16{0});
#pragma unroll
    for (int kc = 1; kc < NQF; ++kc) x1 = Mma<T>::mma(__builtin_bit_cast(Frag, kb[kc]), qf[kc], x1);
  };
  // -inf for the keys of a block that are dead for this lane's row
  auto mask_block = [&](f32x16& x, uint32_t word) __attribute__((always_inline)) {
    word >>= 4 * G;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float xv = x[e];  // (a scalar copy: bit-casting the vector element reads element 0)
      const int32_t keep = __builtin_amdgcn_sbfe((int32_t)word, 8 * (e >> 2) + (e & 3), 1);
      x[e] = __builtin_bit_cast(float, (__builtin_bit_cast(int32_t, xv) & keep) | (int32_t)(0xff800000u & ~(uint32_t)keep));
    }
  };
  // The word of this lane's row for block b of step j.
  auto word = [&](const Step& s, int j, int b) __attribute__((always_inline)) -> uint32_t {
    const uint32_t live = (s.live >> (2 * b)) & 3u;
    uint32_t x = live ? mask_word(mask, q_pos, (kl.block(j0 + j) << kTileLg) + 32 * b, len) : 0u;
    if (!(live & 1u)) x &= 0xffff0000u;
    if (!(live & 2u)) x &= 0x0000ffffu;
    return x;
  };
  auto shape = [&](const Step& s, int j, f32x16& x0, f32x16& x1) __attribute__((always_inline)) {
    if ((s.full & 3u) != 3u) mask_block(x0, word(s, j, 0));
    if ((s.full & 12u) != 12u) mask_block(x1, word(s, j, 1));
  };
  auto block_max = [&](const f32x16& x, float mx) __attribute__((always_inline)) -> float {
#pragma unroll
    for (int e = 0; e < 16; e += 2) mx = nan_max(mx, nan_max(x[e], x[e + 1]));
    return mx;
  };
  // (huge: this row's m_run is in units of the scores)
  auto raise = [&](float mx, bool huge) __attribute__((always_inline)) {
    const float m_new = nan_max(m_run, huge ? row_nan_max(mx) : row_nan_max(mx) * c_exp);
    if (__ballot(huge ? (m_new - m_run) * c_exp > kLazy : m_new > m_run + kLazy) != 0ull) {
      const float up = m_run - base_of(m_new);
      const float alpha = __builtin_amdgcn_exp2f(huge ? up * c_exp : up);
      m_run = m_new;
      l_part *= alpha;
#pragma unroll
      for (int x = 0; x < NDB; ++x) acc[x] *= alpha;
    }
  };
  // P of chunk c of a block, summed into l_part.  (The empty asm makes the products wait for the sum:
  // left to itself the scheduler sums at the step's end and holds 32 values until then, and the
  // fragments of Q go to scratch memory.)
  auto exps = [&](const f32x16& x, int c, float neg_m, bool huge) __attribute__((always_inline)) -> Frag {
    f32x8 e8;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      e8[e] = __builtin_amdgcn_exp2f(huge ? (x[8 * c + e] + neg_m) * c_exp : __builtin_fmaf(x[8 * c + e], c_exp, neg_m));
    l_part += ((e8[0] + e8[1]) + (e8[2] + e8[3])) + ((e8[4] + e8[5]) + (e8[6] + e8[7]));
    u32x4 pw = __builtin_bit_cast(u32x4, Mma<T>::cvt(e8));
    uint32_t p0 = pw[0];
    asm("" : "+v"(l_part), "+v"(p0));
    pw[0] = p0;
    return __builtin_bit_cast(Frag, pw);
  };
  // Products with chunk x (keys 16 x .. 16 x + 15) of the step in the V slot that the transposed
  // reads are on.
  auto pv = [&](Frag pf, int x) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db] = Mma<T>::mma(tr_frag<T, D>(rd, db, VRING + 16 * x * R::ROW), pf, acc[db]);
  };
  auto sums_step = [&](const f32x16& x0, const f32x16& x1) __attribute__((always_inline)) {
    const float neg_m = -base_of(m_run);
#pragma unroll
    for (int x = 0; x < 4; ++x) pv(exps(x < 2 ? x0 : x1, x & 1, neg_m, false), x);
  };

  Step s_cur{}, s_next{}, s_after{};
  uint32_t p = 0u;  // j & 1, times a slot
  // Iteration j, with a step after it: behind the wait and the barrier, K of step j + 1 and V of step
  // j are in LDS, and the slots that the new DMA writes were last read before the barrier.
  auto next = [&](int j) __attribute__((always_inline)) -> LiveSteps {
    dma_wait_all();
    // (a use that makes the compiler's own wait for the page loads fall here)
    asm volatile("" ::"v"(r_page));
    __syncthreads();
    if (j + 2 < n_steps) {
      s_after = step_of(j + 2);
      dma(KRING + p, kbase + s_after.off);
    }
    dma(VRING + (SLOT - p), vbase + s_next.off);
    return {s_cur.live != 0u, s_next.live != 0u};
  };
  auto body = [&](int j, bool live, const StepScores& x, StepScores& y) __attribute__((always_inline)) {
    // (MFMAs go before the masking, maxima, prologues and epilogues of the other work-group on the
    // CU: sinks in chunks 279 -> 269 us, 16 prompts of 512 92 -> 84, nothing on long lists)
    __builtin_amdgcn_s_setprio(1);
    // (x of a dead step may be an earlier one's scores: every exponential is 0 then, or NaN where that
    // step's sums already were)
    const float neg_m = live ? -base_of(m_run) : -INFINITY;
    const Frag p00 = exps(x.x0, 0, neg_m, false), p01 = exps(x.x0, 1, neg_m, false), p10 = exps(x.x1, 0, neg_m, false),
               p11 = exps(x.x1, 1, neg_m, false);
    qk(y.x0, y.x1);
    pv(p00, 0);
    pv(p01, 1);
    pv(p10, 2);
    pv(p11, 3);
    // 4 K reads ahead; then MFMAs of the scores, each beside a read and exponentials; then those of
    // the products, V reads running 4 MFMAs ahead
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
    for (int z = 0; z < 2 * NQF; ++z) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x002, D == 128 ? 6 : 10, 1);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
    for (int z = 0; z < 4 * NDB; ++z) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
      __builtin_amdgcn_sched_group_barrier(0x002, D == 128 ? 1 : 4, 1);
    }
    __builtin_amdgcn_s_setprio(0);
    shape(s_next, j + 1, y.x0, y.x1);
    raise(block_max(y.x1, block_max(y.x0, -INFINITY)), false);
  };
  auto turn = [&]() __attribute__((always_inline)) {
    s_cur = s_next;
    s_next = s_after;
    rd.template turn_rows<SLOT>();
    rd.template turn_tr<SLOT>();
    p = SLOT - p;
  };
  if (n_steps > 0) {
    s_cur = step_of(0);
    dma(KRING, kbase + s_cur.off);
    dma(VRING, vbase + s_cur.off);
    if (n_steps > 1) s_next = step_of(1);
    dma_wait_all();
#pragma unroll
    for (int kc = 0; kc < NQF; ++kc) asm volatile("" ::"v"(qf[kc]));
    __syncthreads();
    if (n_steps > 1) dma(KRING + SLOT, kbase + s_next.off);
    qk(sa.x0, sa.x1);
    shape(s_cur, 0, sa.x0, sa.x1);
    raise(block_max(sa.x1, block_max(sa.x0, -INFINITY)), false);
    rd.template turn_rows<SLOT>();
    walk_steps(n_steps, sa, sb, next, body, turn);
    dma_wait_all();
    __syncthreads();
    if (s_cur.live != 0u) sums_step(sa.x0, sa.x1);
  }

  // ---- sums that are not finite, scores that are huge: the list again, step by step --------
  float big = 0.f;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; e += 2) big = nan_max(big, nan_max(__builtin_fabsf(acc[db][e]), __builtin_fabsf(acc[db][e + 1])));
  // (a row's maximum may have been huge before it had one near 0: its sum is not finite then; -inf: a
  // row without a live key)
  const bool huge = (__builtin_fabsf(m_run) > 0x1p24f && m_run != -INFINITY) || !(row_sum(l_part) < INFINITY);
  float m_rest = 0.f;  // what the rounding of a huge row's maximum to log2 units left out of m_run
  if (__syncthreads_or(huge || !(big < INFINITY))) {
    rd = tile_reads<D>((lds_cptr)smem, lane);
#pragma unroll
    for (int x = 0; x < NDB; ++x) acc[x] = f32x16{0};
    m_run = -INFINITY;
    l_part = 0.f;
    load_raw(0);
#pragma unroll 1
    for (int j = 0; j < n_steps; ++j) {
      const Step s = step_of(j);
      dma(KRING, kbase + s.off);
      dma(VRING, vbase + s.off);
      dma_wait_all();
      __syncthreads();
      qk(sa.x0, sa.x1);
      uint32_t w0 = ~0u, w1 = ~0u;
      if (s.full != 15u) {
        w0 = word(s, j, 0);
        w1 = word(s, j, 1);
        mask_block(sa.x0, w0);
        mask_block(sa.x1, w1);
      }
      raise(block_max(sa.x1, block_max(sa.x0, -INFINITY)), huge);
      const float neg_m = -base_of(m_run);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const Frag pf = exps(x < 2 ? sa.x0 : sa.x1, x & 1, neg_m, huge);
        if (!((s.live >> x) & 1u)) continue;
        uint32_t lo = 0u, hi = 0u;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const u32x4 v = __builtin_bit_cast(u32x4, tr_frag<T, D>(rd, db, VRING + 16 * x * R::ROW));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t y = v[e];
            lo = max(lo, y & 0x7fffu);
            hi = max(hi, y & 0x7fff0000u);
          }
        }
        if (((s.full >> x) & 1u) || __ballot(not_finite16<T>(lo, hi)) == 0ull) {
          pv(pf, x);
          continue;
        }
        const u32x4 pw = __builtin_bit_cast(u32x4, pf);
        // element e of lane half h is key 8 (e / 4) + 4 h + e % 4 of the chunk
#pragma unroll 1
        for (int y = 0; y < 16; ++y) {
          const int h = y & 1, e = y >> 1;
          const uint32_t half = G == h ? ((e & 1) ? 0xffff0000u : 0x0000ffffu) : 0u;
          u32x4 keep;
#pragma unroll
          for (int z = 0; z < 4; ++z) keep[z] = z == (e >> 1) ? half : 0u;
          const bool on = ((x < 2 ? w0 : w1) >> (16 * (x & 1) + 8 * (e >> 2) + 4 * h + (e & 3))) & 1u;
#pragma unroll
          for (int db = 0; db < NDB; ++db) {
            const u32x4 v = __builtin_bit_cast(u32x4, tr_frag<T, D>(rd, db, VRING + 16 * x * R::ROW)) & keep;
            const f32x16 p = Mma<T>::mma(__builtin_bit_cast(Frag, v), __builtin_bit_cast(Frag, pw & keep), f32x16{0});
#pragma unroll
            for (int z = 0; z < 16; ++z) acc[db][z] = on ? acc[db][z] + p[z] : acc[db][z];
          }
        }
      }
      __syncthreads();  // every wave is past the slots
    }
    if (huge) {
      const float m_x = m_run;
      m_run = m_x * c_exp;
      if (__builtin_fabsf(m_run) < INFINITY) m_rest = __builtin_fmaf(m_x, c_exp, -m_run);
    }
  }

  // ---- the rows leave -------------------------------------------------------------------
  float l_tot = row_sum(l_part);
  int lane_e = lane;  // (opaque: what follows is worked out again instead of held through the loop)
  asm volatile("" : "+v"(lane_e));
  const int m_e = lane_e & 31, G_e = lane_e >> 5;
  const bool mine = 32 * w + m_e < n_rows;
  if (PART != kPrefix && u.splits > 1) {
    // a slot is the waves' registers as they are: 16 bytes of O per lane, then maximum and sum, then
    // what the maximum lacks (which is as large as the difference of two shares' maxima, where these are
    // huge)
    constexpr int SLOT_B = slot_floats(kTileRows, D) * 4, WB = SLOT_B / 4;
    char* first = part.part + (int64_t)u.slot * SLOT_B;
    const bool has = 32 * w < n_rows;  // (a wave without rows stores and merges nothing)
    if (has) {
      char* own = first + (int64_t)u.split * SLOT_B + w * WB + 16 * lane_e;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          share_store4(own + (4 * db + e) * 1024, f32x4{acc[db][4 * e], acc[db][4 * e + 1], acc[db][4 * e + 2], acc[db][4 * e + 3]});
      if (G_e == 0) {
        float* ml = reinterpret_cast<float*>(own + NDB * 4096 - 8 * lane_e);
        share_store(ml, m_run);
        share_store(ml + 1, l_tot);
        share_store(reinterpret_cast<float*>(own + NDB * 4096 + 256 - 12 * lane_e), m_rest);
      }
    }
    if (!last_share(part, u, tid, flag) || !has) return;
    const Shares all = shares_at(first, u.splits * SLOT_B);
    m_run = -INFINITY;
    m_rest = 0.f;
#pragma unroll 8
    for (int s = 0; s < u.splits; ++s) {
      const int32_t at = s * SLOT_B + w * WB + NDB * 4096;
      const float ms = share_load2(all, 8 * m_e, at)[0], rs = share_load1(all, 4 * m_e, at + 256);
      m_rest = ms > m_run ? rs : ms == m_run ? nan_max(m_rest, rs) : m_rest;
      m_run = nan_max(m_run, ms);
    }
    l_tot = 0.f;
#pragma unroll
    for (int x = 0; x < NDB; ++x) acc[x] = f32x16{0};
#pragma unroll 2
    for (int s = 0; s < u.splits; ++s) {
      const int32_t at = s * SLOT_B + w * WB;
      f32x4 x[NDB][4];
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[db][e] = share_load4(all, 16 * lane_e, at + (4 * db + e) * 1024);
      const f32x2 ml = share_load2(all, 8 * m_e, at + NDB * 4096);
      const float rest = share_load1(all, 4 * m_e, at + NDB * 4096 + 256);
      const float f = __builtin_amdgcn_exp2f((ml[0] - base_of(m_run)) + (rest - m_rest));
      l_tot += f * ml[1];
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int z = 0; z < 4; ++z) acc[db][4 * e + z] += f * x[db][e][z];
    }
  }
  if (PART == kPrefix || (PART == kOwn && u.x0 > 0)) {
    // (a lane has columns 32 db + 8 e + 4 G .. + 3 of its row)
    if (!mine) return;
    const int ir = i0 + 32 * w + m_e, tok = token_of(a, ir), head = u.h * a.G + (ir - tok * a.G);
    float* to = PART == kPrefix ? prefix_state<kTileRows, D>(a, part, u, 32 * w + m_e, tok, head, G_e == 0)
                                : a.own + ((int64_t)(u.rq.start + tok) * (a.Hkv * a.G) + head) * state_floats(D);
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(to + 32 * db + 8 * e + 4 * G_e) =
            f32x4{acc[db][4 * e], acc[db][4 * e + 1], acc[db][4 * e + 2], acc[db][4 * e + 3]};
    if (G_e == 0) *reinterpret_cast<f32x4*>(to + D) = f32x4{m_run, m_rest, l_tot, 0.f};
    return;
  }
  const float inv = l_tot == 0.f ? 0.f : 1.f / l_tot;
  if (a.lse && G_e == 0 && mine) {
    const int ir = i0 + 32 * w + m_e, tok = token_of(a, ir), head = u.h * a.G + (ir - tok * a.G);
    a.lse[(int64_t)(u.rq.start + tok) * a.lse_st + (int64_t)head * a.lse_sh] =
        l_tot == 0.f ? -INFINITY : (m_run + log2f(l_tot)) * kLn2;
  }
  // Through LDS (32 rows a wave, 16-byte units swizzled), so that they are stored as whole rows.
  // (every wave is past its last read of the rings: the sums' check was a barrier)
  lds_char_t* stage = (lds_char_t*)smem + w * 32 * R::ROW;
  typedef __attribute__((address_space(3))) u32x2 lds_w2;
  constexpr int UM = R::UPR - 1;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x4 x = f32x4{acc[db][4 * e], acc[db][4 * e + 1], acc[db][4 * e + 2], acc[db][4 * e + 3]} * inv;
      *(lds_w2*)(stage + m_e * R::ROW + 16 * ((4 * db + e) ^ (m_e & UM)) + 8 * G_e) = __builtin_bit_cast(u32x2, Mma<T>::cvt4(x));
    }
  // (each wave reads back only the rows it wrote: LDS keeps a wave's accesses in order; a row's
  // place in the output is worked out by its own lane)
  int64_t o_off;
  {
    const int ir = i0 + 32 * w + m_e, t = token_of(a, ir), h = u.h * a.G + (ir - t * a.G);
    o_off = (int64_t)(u.rq.start + t) * a.o_st + (int64_t)h * a.o_sh;
  }
#pragma unroll
  for (int x = 0; x < 32 / R::RPI; ++x) {
    const int rr = R::RPI * x + lane_e / R::UPR, un = lane_e % R::UPR;
    const u32x4 v = *(lds_u4*)(stage + rr * R::ROW + 16 * (un ^ (rr & UM)));
    const uint32_t lo = (uint32_t)__shfl((int32_t)(uint32_t)o_off, rr);
    const int32_t hi = __shfl((int32_t)(o_off >> 32), rr);
    if (32 * w + rr < n_rows)
      *reinterpret_cast<u32x4*>(a.o + (int64_t)((uint64_t)lo | ((uint64_t)(uint32_t)hi << 32)) + 16 * un) = v;
  }
}

}  // namespace
}  // namespace pa
