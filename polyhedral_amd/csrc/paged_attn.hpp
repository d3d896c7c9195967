// Attention over a paged cache: the arguments its kernels share, and how their work-groups find
// their work.
//
// Query rows of a request are its new tokens times the G = Hq / Hkv heads that share a KV head
// (row i: token i / G, head i % G), cut into tiles of BM rows.  A unit of work is one tile, one
// KV head and one of the tile's `splits` equal shares of the blocks of keys that may be live for
// it.  Lengths are on the device, so every wave works out the split itself: a first pass over
// the requests sums tiles x blocks, which gives the blocks of a share, and a second one finds
// the unit's request (both are one load and a few scans for up to 64 requests).
// A request whose tiles are split has a slot of the workspace per unit, numbered in unit order.
#pragma once

#include <stddef.h>

#include "lds_rows.hpp"
#include "page_math.hpp"

namespace pa {

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
  float c;  // scale * log2(e)
  int32_t n_include, n_exclude;
  pa_term terms[PA_MAX_TERMS];
  char* o;
  int64_t o_st, o_sh;
  float* lse;
  int64_t lse_st, lse_sh;  // elements
  float* part_o;   // [slots][BM][D]: unnormalised
  float* part_ml;  // [slots][BM][2]: maximum (tiles of 128 rows: times c) and sum
  int32_t slots;
  int32_t target;     // units a split aims for
  int32_t least;      // least blocks of a share
  int32_t row_min, row_max;  // requests with row_min < rows <= row_max are this kernel's
};

// The mask of a kernel whose first argument is a PagedK.
typedef const __attribute__((address_space(4))) pa_term cterm;
typedef PageMask<cterm*> KernelMask;
__device__ __forceinline__ KernelMask kernel_mask(const PagedK& a) {
  typedef const __attribute__((address_space(4))) char cchar;
  cchar* args = (cchar*)__builtin_amdgcn_kernarg_segment_ptr();
  return {a.n_include, a.n_exclude, (cterm*)(args + offsetof(PagedK, terms))};
}

struct Work {
  int32_t tiles, blocks;
};

struct Unit {
  bool found;
  Request rq;
  int32_t r, tile, tiles, h, split, splits;
  int32_t slot;   // of this unit (merge: of the group's first unit)
};

__device__ __forceinline__ Request load_request(const PagedK& a, int r) {
  return request_of(a.q_start[r], a.q_start[r + 1], a.lengths[r], a.T, a.cols << a.page_lg);
}

// Tiles of a request and blocks of 1 << LG keys of its last whole one (a causal mask's longest).
template <int BM, int LG>
__device__ __forceinline__ Work work_of(const PagedK& a, const Request& q) {
  const int32_t rows = q.n * a.G;
  if (rows <= a.row_min || rows > a.row_max) return {0, 0};
  const int32_t span = imin(q.n, (BM + a.G - 1) / a.G + 1);
  return {(rows + BM - 1) / BM, key_list(kernel_mask(a), q.len - span, q.len - 1, q.len, LG).count()};
}

__device__ __forceinline__ int32_t wave_scan(int32_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Unit (GROUP: the group of all splits of a tile and head, of tiles with more than one) `id`.
template <int BM, int LG, bool GROUP>
__device__ __forceinline__ Unit find_unit(const PagedK& a, int32_t id, int lane) {
  Unit u;
  u.found = false;
  Request q{0, 0, 0};
  Work w{0, 0};
  float total = 0.f;  // (a share needs no exact total)
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    const int r = r0 + lane;
    w = {0, 0};
    if (r < a.R) {
      q = load_request(a, r);
      w = work_of<BM, LG>(a, q);
    }
    total += (float)w.tiles * (float)w.blocks;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o);
  // (rounded up, so the units stay within target + tiles Hkv, which the grid is sized for)
  const float share = total * (float)a.Hkv / (float)a.target * 1.0001f;
  const int32_t chunk = imax(a.least, share < 1e9f ? (int32_t)share + 1 : (1 << 30));

  int32_t before = 0, slot = 0;  // units (groups) and slots of earlier requests
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    const int r = r0 + lane;
    if (a.R > 64) {
      w = {0, 0};
      if (r < a.R) {
        q = load_request(a, r);
        w = work_of<BM, LG>(a, q);
      }
    }
    const int32_t splits = imax((w.blocks + chunk - 1) / chunk, 1);
    const int32_t units = w.tiles * a.Hkv * splits, mine = splits > 1 ? units : 0;
    const int32_t n = GROUP ? (splits > 1 ? w.tiles * a.Hkv : 0) : units;
    const int32_t n_in = wave_scan(n, lane), s_in = wave_scan(mine, lane);
    const int32_t at = before + n_in - n;
    const uint64_t hit = __ballot(at <= id && id < at + n);
    if (hit) {
      const int l = (int)__builtin_ctzll(hit);
      auto get = [&](int32_t x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, l); };
      u.found = true;
      u.r = r0 + l;
      u.rq = {get(q.start), get(q.n), get(q.len)};
      u.tiles = get(w.tiles);
      u.splits = get(splits);
      int32_t x = id - get(at);
      const int32_t s0 = slot + get(s_in - mine);
      if (GROUP) {
        u.tile = x / a.Hkv;
        u.h = x - u.tile * a.Hkv;
        u.split = 0;
        u.slot = s0 + x * u.splits;
      } else {
        // a KV head's shares side by side, its tiles a multiple of Hkv units apart: with 8 KV heads
        // the tiles of one fall on one XCD (work-groups are dealt to the XCDs in turn) and share
        // its L2
        const int32_t per = a.Hkv * u.splits;
        u.tile = x / per;
        u.slot = s0 + x;
        x -= u.tile * per;
        u.h = x / u.splits;
        u.split = x - u.h * u.splits;
      }
      // (a causal mask's longest tile first)
      u.tile = u.tiles - 1 - u.tile;
      return u;
    }
    before += __builtin_amdgcn_readlane(n_in, 63);
    slot += __builtin_amdgcn_readlane(s_in, 63);
  }
  return u;
}

// Blocks j0 .. j1 - 1 of a list of n are share `split` of `splits`.
__device__ __forceinline__ void share_of(int32_t n, int32_t split, int32_t splits, int32_t* j0, int32_t* j1) {
  const int32_t per = n / splits, more = n - per * splits;
  *j0 = split * per + imin(split, more);
  *j1 = *j0 + per + (split < more ? 1 : 0);
}

int check_pages(const char* who, int64_t n_pages, int32_t page_size, int* page_lg);

// The maximum m of a row's scores so far as the base of its exponentials: 0 for -inf (no live key
// so far; every score is -inf then).
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

constexpr int kRows = 16;       // query rows of a tile of paged_rows_kernel
constexpr int kTileRows = 128;  // and of paged_tile_kernel
constexpr int kTileLg = 6;      // log2 keys of a step of paged_tile_kernel

int launch_paged_rows(const PagedK& a, int dtype, int D, int64_t max_tiles, hipStream_t s);
int launch_paged_tile(const PagedK& a, int dtype, int D, int64_t max_tiles, hipStream_t s);
int launch_paged_tile_merge(const PagedK& a, int dtype, int D, int64_t max_tiles, hipStream_t s);

}  // namespace pa
