// Attention over a paged cache: the arguments its kernels share, how their work-groups find their
// work, and how the shares of a split tile become one.
//
// Query rows of a request are its new tokens times the G = Hq / Hkv heads that share a KV head
// (row i: token i / G, head i % G), cut into tiles of BM rows.  A unit of work is one tile, one
// KV head and one of the tile's `splits` equal shares of the blocks of keys that may be live for
// it.  Lengths are on the device, so every wave works out the split itself: a first pass over
// the requests sums tiles x blocks, which gives the blocks of a share, and a second one finds
// the unit's request (both are one load and a few scans for up to 64 requests).
//
// The units of a split tile write their states to slots of the workspace, count themselves, and the
// last one merges them all, in the order of the shares whichever it is.  (A second launch that
// merges took 5 us where nothing was split, and 30 to 70 behind large grids of chunks.)
#pragma once

#include <stddef.h>

#include "lds_rows.hpp"
#include "page_math.hpp"

namespace pa {

constexpr int kRows = 16;       // query rows of a tile of few rows
constexpr int kTileRows = 128;  // and of a chunk's tile
constexpr int kTileLg = 6;      // log2 keys of a step of a chunk's tile

// Which rows and keys a body takes.  Requests that share a prefix are attended in two parts: the rows of
// all of a group's requests against the prefix (kPrefix: "request" g is the group of holder g, its rows
// found through a list, at positions of their own), and each request's rows against its own keys (kOwn).
// Both leave the rows' states in memory, a prefix one for each share of it, and a second launch merges them.
enum Part { kWhole = 0, kPrefix = 1, kOwn = 2 };

// What one of the two kernels' bodies does in a call.
struct PagedPart {
  char* part;           // [slots] states of split tiles' units
  int32_t* count;       // [slots] units done, at a tile's first slot; zero between calls
  int32_t slots;
  // A share is at least `least` blocks, and the root of its tile's blocks times root_over (the time of
  // a share against that of merging them all).
  int32_t least;
  float root_over;
  float by_shares;      // 1.0001 / the most shares that all the work is cut into, beyond one a tile
  int32_t span;         // new tokens that a tile can hold rows of
  int32_t row_min, row_max;  // requests with row_min < rows <= row_max
  int32_t grid;
};

struct PagedK {
  const char* q;
  int64_t q_st, q_sh;  // bytes, as every stride here
  const char* k;
  const char* v;
  int64_t c_sp, c_sh, c_sn;
  int64_t n_pages;
  int32_t page_lg, cols;
  const int32_t* tables;
  int64_t pitch;
  const int32_t* lengths;
  const int32_t* q_start;
  int32_t R, T, Hkv, G;
  Divisor by_G, by_Hkv;
  float c;  // scale * log2(e)
  int32_t n_include, n_exclude;
  pa_term terms[PA_MAX_TERMS];
  float few_weight;  // time of a block of few rows' keys, of that of a chunk's step (see find_unit)
  int32_t stride;  // of a mask that is a lattice beyond a band: 1 in `stride` keys is live for a token; else 0
  char* o;
  int64_t o_st, o_sh;
  float* lse;
  int64_t lse_st, lse_sh;  // elements
  PagedPart tiles, rows;
  // ---- requests that share prefixes (kPrefix, kOwn) ----
  pa_sharing share;
  PagedPart pre_tiles, pre_rows;
  // States: D floats of O, then maximum (log2 units), what its rounding left out, sum, and one unused.
  float* states;       // of the prefixes' shares, a slot of pre_tiles or pre_rows each, at their `part`
  float* own;          // [T, Hq] states over the requests' own keys
  struct StatesAt* at; // [T, Hq] by place among the groups' rows
  int64_t n_states;    // floats of `states`, a multiple of 4
  int32_t* end;        // rows of requests end here, for the merge (q_start's last entry may have fallen back)
};

// Where a row's states over its prefix are: units of 4 floats.
struct StatesAt {
  uint32_t first, step;
  int32_t n;
  int32_t unused;
};

// The mask of a kernel whose first argument is a PagedK.
typedef const __attribute__((address_space(4))) pa_term cterm;
typedef PageMask<cterm*> KernelMask;
__device__ __forceinline__ KernelMask kernel_mask(const PagedK& a) {
  typedef const __attribute__((address_space(4))) char cchar;
  cchar* args = (cchar*)__builtin_amdgcn_kernarg_segment_ptr();
  return {a.n_include, a.n_exclude, a.terms[0], (cterm*)(args + offsetof(PagedK, terms))};
}

// Whether a tile of few rows with that many tokens is taken by lists of live keys (paged_rows.hpp; one
// in `stride` keys of a lattice is live for each: beyond, most of a block is listed.  16 requests of
// 4000, stride 16, 8 heads: 8 tokens 48 us block by block, 37 by lists; 10 50 and 43; 14 51 and 55).
__device__ __forceinline__ bool by_lists(int32_t tokens, int32_t stride) { return tokens <= stride - stride / 4; }

struct Work {
  int32_t tiles, blocks, least;  // least: blocks of a share
  int32_t few;                   // blocks of a request with fewer rows than the part takes
};

struct Unit {
  bool found;
  Request rq;
  int32_t r, tile, h, split, splits;
  int32_t slot;  // of the tile's first share
  int32_t x0, x1;  // kPrefix: the group's positions; kOwn: the request's first own key
};

// Tiles of a request and blocks of 1 << LG keys of its last whole one (a causal mask's longest).
template <int BM, int LG, int PART>
__device__ __forceinline__ Work work_of(const PagedK& a, const PagedPart& p, const Request& q, int32_t x0, int32_t x1) {
  const int32_t rows = q.n * a.G;
  if (rows == 0 || rows > p.row_max || (BM == kRows && rows <= p.row_min)) return {0, 0, 1, 0};
  const int32_t span = imin(q.n, p.span);
  // (a share that is taken by lists: for one token a list of 512 keys for each wave, for more fewer)
  const int32_t least = PART != kPrefix && BM == kRows && by_lists(span, a.stride) ? imax((2048 >> LG) >> (31 - __builtin_clz((uint32_t)imax(span, 1))), p.least) : p.least;
  const KeyList kl = PART == kPrefix ? key_list(kernel_mask(a), x0, x1, q.len, LG) : key_list(kernel_mask(a), q.len - span, q.len - 1, q.len, LG);
  const int32_t blocks = kl.count() - (PART == kOwn ? kl.before(x0 >> LG) : 0);
  if (BM == kTileRows && rows <= p.row_min) return {0, 0, 1, blocks};
  return {(rows + BM - 1) / BM, blocks, least, 0};
}

// Sum over lanes 0 .. l, by DPP moves inside rows of 16 lanes and broadcasts of their last ones.
template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t dpp_move(int32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int32_t wave_scan(int32_t x) {
  x += dpp_move<0x111, 0xf>(x);
  x += dpp_move<0x112, 0xf>(x);
  x += dpp_move<0x114, 0xf>(x);
  x += dpp_move<0x118, 0xf>(x);
  x += dpp_move<0x142, 0xa>(x);
  x += dpp_move<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ float wave_total(float x) {
  auto add = [&](int32_t y) __attribute__((always_inline)) { x += __builtin_bit_cast(float, y); };
  add(dpp_move<0x111, 0xf>(__builtin_bit_cast(int32_t, x)));
  add(dpp_move<0x112, 0xf>(__builtin_bit_cast(int32_t, x)));
  add(dpp_move<0x114, 0xf>(__builtin_bit_cast(int32_t, x)));
  add(dpp_move<0x118, 0xf>(__builtin_bit_cast(int32_t, x)));
  add(dpp_move<0x142, 0xa>(__builtin_bit_cast(int32_t, x)));
  add(dpp_move<0x143, 0xc>(__builtin_bit_cast(int32_t, x)));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, x), 63));
}

// What q_start and lengths hold for request r0 + lane (past R: zeros).
struct RawRequest {
  int32_t s0, s1, len, x0, x1;
};
template <int PART = kWhole>
__device__ __forceinline__ RawRequest raw_request(const PagedK& a, int r0, int lane) {
  RawRequest x{0, 0, 0, 0, 0};
  const int r = r0 + lane;
  if (r < a.R) {
    const int32_t* start = PART == kPrefix ? a.share.start : a.q_start;
    x.s0 = start[r];
    x.s1 = start[r + 1];
    x.len = PART == kPrefix ? a.share.prefix[r] : a.lengths[r];
    if (PART == kPrefix) {
      x.x0 = imin(imax(a.share.low[r], 0), kMaxPosition);
      x.x1 = imin(imax(a.share.high[r], 0), kMaxPosition);
    }
    // (whole segments of 16 keys, as pages are)
    if (PART == kOwn) x.x0 = imin(imax(a.share.first[r], 0), a.cols << a.page_lg) & ~15;
  }
  return x;
}

// Request r0 + lane (past R: none).  `end`: the largest start so far.  Starts that fall back are
// taken as that, so whatever q_start holds the requests' rows are disjoint, and the units and slots
// stay within what the host sized for T rows.
__device__ __forceinline__ Request load_request(const PagedK& a, const RawRequest& x, int r0, int lane, int32_t& end) {
  const int r = r0 + lane;
  int32_t s0 = imin(imax(x.s0, 0), a.T), s1 = imin(imax(x.s1, 0), a.T);
  if (__ballot(r < a.R && (s1 < s0 || s0 < end)) != 0ull) {
    s0 = imax(s0, end);
#pragma unroll 1
    for (int o = 1; o < 64; o <<= 1) {
      const int32_t y = __shfl_up(s0, o);
      if (lane >= o) s0 = imax(s0, y);
    }
    s1 = imax(s1, s0);
  }
  end = __builtin_amdgcn_readlane(s1, imin(a.R - 1 - r0, 63));
  return request_of(s0, s1, x.len, a.T, a.cols << a.page_lg);
}

// A prefix's tiles are few, and the root of their blocks may leave places without work: then a third of the most
// shares at least, as a row's states are merged by a work-group of their own.  (24 requests of a token, 4 heads over
// one of 128, behind 6700 to 26800: 32.6 -> 28.5 us; 9 of up to 29 tokens behind three of up to 62000: 49 -> 44, with
// half of the shares 37, but 64 behind 8192 then 56 -> 61.)
constexpr float kFewShares = 3.f;

template <int BM, int LG, int PART = kWhole>
__device__ __forceinline__ Unit find_unit(const PagedK& a, const PagedPart& p, const RawRequest& raw, int32_t id, int lane) {
  Unit u;
  u.found = false;
  u.x0 = u.x1 = 0;
  Request q{0, 0, 0};
  RawRequest x = raw;
  Work w{0, 0, 1, 0};
  float total = 0.f, few = 0.f;  // (a share needs no exact total)
  int32_t end = 0;
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    if (r0) x = raw_request<PART>(a, r0, lane);
    q = load_request(a, x, r0, lane, end);
    w = work_of<BM, LG, PART>(a, p, q, x.x0, x.x1);
    total += wave_total((float)w.tiles * (float)w.blocks);
    if (BM == kTileRows) few += wave_total((float)w.few);
  }
  if (PART == kOwn && BM == kRows && id == 0 && lane == 0) *a.end = end;
  // Blocks of a share: all of the part's work over `shares` (rounded up, so the units stay within shares
  // + tiles Hkv, which the grid is sized for).  Two work-groups run per CU, so 1024 shares of few rows are
  // two rounds, which suits long lists of uneven lengths (64 requests of 300 to 8192 in one round of
  // 512: 160 us, in two 148); short ones are cut for one round.  A little fewer than the round holds, as
  // shares are rounded to whole blocks and tiles, and a few units more cost a round of their own: 8
  // requests of 300 to 8192 30 -> 24 us, 16 49 -> 44, 5 of 6000 32 -> 27, the 64 148 -> 144.
  float share = total * (float)a.Hkv * p.by_shares;
  if (BM == kRows) share *= share < 24.f ? 2.4f : 1.08f;
  // Where the requests with few rows take longer than the chunks, those get one place of a CU's two, and
  // their MFMAs run beside the loads of the others instead of before them: 61 requests of a token and 3
  // chunks 166 -> 150 us, 29 and 3 307 -> 284.  (36 requests of which the chunks take longer: 52 -> 70,
  // units as long as the whole launch.)
  if (BM == kTileRows && few * a.few_weight >= total) share *= 2.f;

  int32_t before = 0, slot = 0;  // units and slots of earlier requests
  end = 0;
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    if (a.R > 64) {
      x = r0 ? raw_request<PART>(a, r0, lane) : raw;
      q = load_request(a, x, r0, lane, end);
      w = work_of<BM, LG, PART>(a, p, q, x.x0, x.x1);
    }
    // (to the nearest: a tile little longer than a share stays whole)
    const float b = (float)w.blocks, root = __builtin_amdgcn_sqrtf(b) * p.root_over;
    const float mine = fmaxf(fmaxf(share, (float)w.least), PART == kPrefix ? fminf(root, kFewShares * share) : root);
    const int32_t splits = imax((int32_t)(b * __builtin_amdgcn_rcpf(mine) + 0.5f), 1);
    const int32_t units = w.tiles * a.Hkv * splits, slotted = PART == kPrefix || splits > 1 ? units : 0;
    const int32_t n_in = wave_scan(units), s_in = wave_scan(slotted);
    const int32_t at = before + n_in - units;
    const uint64_t hit = __ballot(at <= id && id < at + units);
    if (hit) {
      const int l = (int)__builtin_ctzll(hit);
      auto get = [&](int32_t x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, l); };
      u.found = true;
      u.r = r0 + l;
      u.rq = {get(q.start), get(q.n), get(q.len)};
      u.splits = get(splits);
      if (PART != kWhole) u.x0 = get(x.x0);
      if (PART == kPrefix) u.x1 = get(x.x1);
      // KV heads side by side, so that those of one head are Hkv units apart: with 8 of them a head's
      // work falls on one XCD (work-groups are dealt to the XCDs in turn) and shares its L2
      const int32_t i = id - get(at), y = divide(i, a.by_Hkv);
      u.h = i - y * a.Hkv;
      const int32_t tile = u.splits == 1 ? y : (int32_t)((uint32_t)y / (uint32_t)u.splits);
      u.split = y - tile * u.splits;
      u.slot = slot + get(s_in - slotted) + (tile * a.Hkv + u.h) * u.splits;
      // (a causal mask's longest tile first)
      u.tile = get(w.tiles) - 1 - tile;
      return u;
    }
    before += __builtin_amdgcn_readlane(n_in, 63);
    slot += __builtin_amdgcn_readlane(s_in, 63);
  }
  return u;
}

// Token of a request's row i (its head of the group: i - token G).
__device__ __forceinline__ int32_t token_of(const PagedK& a, int32_t i) { return divide(i, a.by_G); }

// Blocks j0 .. j1 - 1 of a list of n are share `split` of `splits`.
__device__ __forceinline__ void share_of(int32_t n, int32_t split, int32_t splits, int32_t* j0, int32_t* j1) {
  const int32_t per = (int32_t)((uint32_t)n / (uint32_t)splits), more = n - per * splits;
  *j0 = split * per + imin(split, more);
  *j1 = *j0 + per + (split < more ? 1 : 0);
}

// The states of a tile's shares pass from one work-group to another, maybe on another XCD, whose L2
// does not see this one's: agent-scope stores and loads go past it, and a store is complete (the
// wait below) before the tile's count says so.
__device__ __forceinline__ void share_store(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The states of a tile's shares as a buffer: loads of 16 bytes at agent scope, which no atomic load has.
// (As pairs of 8-byte ones every line is asked for twice.)
typedef __amdgpu_buffer_rsrc_t Shares;
__device__ __forceinline__ Shares shares_at(char* first, int32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(first, 0, bytes, 0x00027000);  // (raw 32-bit data)
}
constexpr int kSc1 = 16;  // agent scope
__device__ __forceinline__ f32x4 share_load4(Shares s, int32_t lane_off, int32_t off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(s, lane_off, off, kSc1));
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x2 share_load2(Shares s, int32_t lane_off, int32_t off) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(s, lane_off, off, kSc1));
}
__device__ __forceinline__ float share_load1(Shares s, int32_t lane_off, int32_t off) {
  return __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(s, lane_off, off, kSc1));
}
__device__ __forceinline__ void share_store4(char* p, f32x4 x) {
  const u32x4 y = __builtin_bit_cast(u32x4, x);
  store_x4_sc1(p, y.x, y.y, y.z, y.w);
}
// After its stores by the whole work-group: whether this is the tile's last share (told through
// `flag` in LDS).  The last one clears the count for the next call.
__device__ __forceinline__ bool last_share(const PagedPart& p, const Unit& u, int tid, int32_t* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const int32_t n = __hip_atomic_fetch_add(p.count + u.slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = n == u.splits - 1;
    if (n == u.splits - 1) __hip_atomic_store(p.count + u.slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *flag != 0;
}

// The maximum m of a row's scores so far as the base of its exponentials: 0 for -inf (no live key
// so far; every score is -inf then).
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// The packed row of token `tok` of a unit's rows, and (kPrefix) its position.
template <int PART>
__device__ __forceinline__ int32_t row_of(const PagedK& a, const Unit& u, int32_t tok) {
  return PART == kPrefix ? imin(imax(a.share.rows[u.rq.start + tok], 0), a.T - 1) : u.rq.start + tok;
}
template <int PART>
__device__ __forceinline__ int32_t position_of(const PagedK& a, const Unit& u, int32_t tok) {
  return PART == kPrefix ? imin(imax(a.share.positions[u.rq.start + tok], 0), kMaxPosition) : u.rq.len - u.rq.n + tok;
}
__device__ __forceinline__ int32_t lanes_min(int32_t x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x = imin(x, __shfl_xor(x, o));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int32_t lanes_max(int32_t x) { return ~lanes_min(~x); }

// What the rounding of m = x c left out (0 where m is not finite: nothing needs it there).
__device__ __forceinline__ float rest_of(float x, float c, float m) {
  return __builtin_fabsf(m) < INFINITY ? __builtin_fmaf(x, c, -m) : 0.f;
}
// floats of a slot: O of every row, then maximum and sum (and of a chunk's tile what the maximum lacks)
constexpr int slot_floats(int BM, int D) { return BM * (D + (BM == kTileRows ? 3 : 2)); }

// and of a slot of a prefix's share
constexpr int state_floats(int D) { return D + 4; }

// Where a row over a prefix leaves its state, row `row` of the unit's slot; the first share says where all are.
template <int BM, int D>
__device__ __forceinline__ float* prefix_state(const PagedK& a, const PagedPart& p, const Unit& u, int32_t row, int32_t tok, int32_t head, bool tell) {
  constexpr int SLOT = BM * state_floats(D);
  float* first = reinterpret_cast<float*>(p.part) + (int64_t)u.slot * SLOT + row * state_floats(D);
  if (tell && u.split == 0)
    a.at[(int64_t)(u.rq.start + tok) * (a.Hkv * a.G) + head] = StatesAt{(uint32_t)((first - a.states) / 4), SLOT / 4, u.splits, 0};
  return first + (int64_t)u.split * SLOT;
}

int check_pages(const char* who, int64_t n_pages, int32_t page_size, int* page_lg);

// Launches the parts whose grid is not 0.
int launch_paged_bf16(const PagedK& a, int D, hipStream_t s);
int launch_paged_f16(const PagedK& a, int D, hipStream_t s);
int launch_paged_f32(const PagedK& a, int D, hipStream_t s);

// The same for requests that share prefixes.
int launch_shared_bf16(const PagedK& a, int D, hipStream_t s);
int launch_shared_f16(const PagedK& a, int D, hipStream_t s);
int launch_shared_f32(const PagedK& a, int D, hipStream_t s);

}  // namespace pa
