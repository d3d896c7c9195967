// The attention weight that cached keys receive, over a paged cache (gfx950): for every key and KV head
// the sum over its request's new tokens and the heads of the group of exp(scale q . k - lse).
//
// Sums of different keys are independent, so the keys are what is cut.  Requests of few rows (new tokens times
// heads of a group) are bound by the bytes of K: weigh_blocks, a wave for some blocks of 64 keys (f32: 32), K straight
// into registers.  64 requests of 300..8192 tokens, a new one each (8 KV heads of 128, bf16, 317 MB of K): 75 us, 4.2
// TB/s of the 5.0 that a copy reaches; one request of 1001 tokens, 4 heads of 64 in f32: 6.0 us, latency.  Requests of
// many rows are bound by products and exponentials: weigh_keys, a work-group for 256 keys, which stay in registers
// while rows of Q pass by.  8 chunks of 256..1500 tokens behind 1000..8000 (32 heads over 8 of 128, f16, 127
// GFLOP of products and 0.5 G exponentials): 172 to 178 us from card to card, 0.72 PFLOP/s; matrix instructions run in a third of the
// cycles and vector instructions, mostly the exponentials' chains, in near half, beside each other; about 40 us go to the units'
// beginnings and ends (keys' loads, reduction over lanes).  By blocks alone it takes 610 us.
//
// Scores, exponentials and sums are float32.  A dead pair adds 0 whatever its key or its row's lse holds: by selection
// (of its exponential, or of its score, as -inf beside a base of the row that is neither NaN nor infinite above).
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "page_checks.hpp"
#include "paged_rows.hpp"

namespace pa {
namespace {

struct WeightsK {
  const char* q;
  int64_t q_st, q_sh;  // bytes, as every stride of q and k
  const char* k;
  int64_t c_sp, c_sh, c_sn;
  int64_t n_pages;
  int32_t page_lg, cols;
  const int32_t* tables;
  int64_t pitch;
  const int32_t* lengths;
  const int32_t* q_start;
  const int32_t* first;
  int32_t R, T, Hkv, G;
  Divisor by_G;
  float c;  // scale * log2(e)
  int32_t n_include, n_exclude;
  pa_term terms[PA_MAX_TERMS];
  const float* lse;
  int64_t lse_st, lse_sh;  // elements
  float* scores;
  int64_t s_sp, s_sh;  // elements
  // requests with more rows (new tokens times heads of a group) than row_max are taken by units of 256 keys, where
  // the grid has tile_grid work-groups, the others by blocks
  int32_t row_max, tile_grid;
  int32_t near;        // no token sees all before it
  int32_t even;        // a step's rows are whole tokens, whose offsets in q and lse fit 31 bits
  float by_shares;     // 1 / the shares that the former's work is cut into
  float* part;         // [slots][256] sums of split groups' shares
  int32_t* count;      // [slots] shares done, at a group's first slot; zero between calls
  int32_t* queue;      // units drawn, 16 ints apart; zero between calls
};

__device__ __forceinline__ KernelMask weights_mask(const WeightsK& a) {
  typedef const __attribute__((address_space(4))) char cchar;
  cchar* args = (cchar*)__builtin_amdgcn_kernarg_segment_ptr();
  return {a.n_include, a.n_exclude, a.terms[0], (cterm*)(args + offsetof(WeightsK, terms))};
}

template <typename T, int D>
struct WeightsShape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int NS = F32 ? 2 : 4;           // 16-key segments of a block
  static constexpr int LG = F32 ? 5 : 6;           // log2 keys of a block
  static constexpr int NK = F32 ? D / 16 : D / 32; // 16-byte units of a row that a lane holds
  static constexpr int PER = 64 / NS;              // blocks whose pages are held at a time
};

// One request's share of the work: blocks of each head, `cost` each: those from the `first` key's on and, where a
// window leaves some dead, which hold a key that may be live or a new token's (whose score begins), a list of two runs.
// (32 requests of 16000 to 32000 under a window of 1024 and 64 sinks: 25 us, 311 of all blocks.)
struct BlockList {
  int32_t low, base0, base1;
  __device__ __forceinline__ int32_t block(int32_t j) const { return j + (j < low ? base0 : base1); }
};
struct WeighedRequest {
  Request rq;
  int32_t first;
  BlockList list;
  int32_t blocks, cost;
};
template <int LG, bool LIST>
__device__ __forceinline__ WeighedRequest weighed(const WeightsK& a, int r0, int lane, int32_t& end) {
  WeighedRequest x{{0, 0, 0}, 0, {0, 0, 0}, 0, 0};
  const int r = r0 + lane;
  int32_t s0 = 0, s1 = 0, len = 0, first = 0;
  if (r < a.R) {
    s0 = a.q_start[r];
    s1 = a.q_start[r + 1];
    len = a.lengths[r];
    first = a.first ? a.first[r] : 0;
  }
  s0 = imin(imax(s0, 0), a.T);
  s1 = imin(imax(s1, 0), a.T);
  // (starts that fall back are taken as the largest so far, as in load_request)
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
  x.rq = request_of(s0, s1, len, a.T, a.cols << a.page_lg);
  x.first = imin(imax(first, 0), x.rq.len);
  const int32_t block0 = x.first >> LG, end_block = (x.rq.len + (1 << LG) - 1) >> LG;
  x.list = {0, block0, block0};
  // (without new tokens nothing changes)
  x.blocks = r < a.R && x.rq.n > 0 ? end_block - block0 : 0;
  if (LIST && a.near && x.blocks) {
    const int32_t pos0 = x.rq.len - x.rq.n;
    KeyList kl = key_list(weights_mask(a), pos0, x.rq.len - 1, x.rq.len, LG);
    const int32_t fresh = imax(imax(pos0, 0) >> LG, kl.low);
    kl.first = kl.high ? imin(kl.first, fresh) : fresh;
    kl.high = imax(end_block - kl.first, 0);
    const int32_t skip = kl.before(block0);
    x.list = {kl.low - skip, skip, kl.first - kl.low + skip};
    x.blocks = kl.count() - skip;
  }
  x.cost = 2 + (x.rq.n * a.G + kRows - 1) / kRows;
  return x;
}

// Those of few rows.
template <int LG>
__device__ __forceinline__ WeighedRequest few(const WeightsK& a, int r0, int lane, int32_t& end) {
  WeighedRequest x = weighed<LG, true>(a, r0, lane, end);
  if (x.rq.n * a.G > a.row_max) x.blocks = 0;
  return x;
}

__device__ __forceinline__ int64_t wave_scan64(int64_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)x, o);
    const int32_t hi = __shfl_up((int)(x >> 32), o);
    if (lane >= o) x += (int64_t)((uint64_t)lo | (uint64_t)(uint32_t)hi << 32);
  }
  return x;
}
__device__ __forceinline__ int64_t readlane64(int64_t x, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l);
  const int32_t hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
  return (int64_t)((uint64_t)lo | (uint64_t)(uint32_t)hi << 32);
}

// A row's -lse in log2 units, NaN where that is, and at most the largest number, so that beside it a dead score's -inf
// stays what it is.
__device__ __forceinline__ float neg_of(float lse) {
  return __builtin_elementwise_minimum(-lse * 1.4426950408889634f, FLT_MAX);
}

// ---- few rows a request -------------------------------------------------------------------------
// A wave takes a run of consecutive blocks, an equal share of all blocks times the row tiles each meets: K rows go
// straight into the A operand's registers of 16x16 MFMAs (S^T = K Q^T, as in paged_rows.hpp), once for all
// rows of the request, the next block's loads ahead of this one's products.  Lane (q = l % 16, g = l / 16) holds
// scores of keys 4 g + 0..3 of each 16 keys for row q; their exponentials are added up over the row tiles, and
// over the 16 rows at the end, in a fixed order.
template <typename T, int D>
__device__ __forceinline__ void weigh_blocks(const WeightsK& a, int32_t id, int32_t grid) {
  using S = WeightsShape<T, D>;
  constexpr int NS = S::NS, NK = S::NK, LG = S::LG, PER = S::PER;
  const int tid = threadIdx.x, lane = tid & 63, q16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const KernelMask mask = weights_mask(a);
  const uint32_t koff = (uint32_t)(q16 * (int32_t)a.c_sn) + 16u * (uint32_t)g;

  // ---- this wave's share of all blocks, by their cost --------------------------------------
  int64_t total = 0;
  int32_t end = 0;
  WeighedRequest x{};
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    x = few<LG>(a, r0, lane, end);
    total += readlane64(wave_scan64((int64_t)x.blocks * a.Hkv * x.cost, lane), 63);
  }
  const int64_t waves = (int64_t)grid * 4, me = (int64_t)id * 4 + w;
  const int64_t per = total / waves, more = total - per * waves;
  const int64_t lo = per * me + (me < more ? me : more), hi = lo + per + (me < more ? 1 : 0);
  if (lo >= hi) return;

  int64_t before = 0;
  end = 0;
  for (int r0 = 0; r0 < a.R && before < hi; r0 += 64) {
    if (a.R > 64) x = few<LG>(a, r0, lane, end);
    const int64_t mine = (int64_t)x.blocks * a.Hkv * x.cost, in = wave_scan64(mine, lane), at = before + in - mine;
    uint64_t hit = __ballot(at < hi && at + mine > lo);
    before += readlane64(in, 63);
    while (hit) {
      const int l = (int)__builtin_ctzll(hit);
      hit &= hit - 1;
      auto get = [&](int32_t y) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(y, l); };
      const int r = r0 + l;
      const Request rq{get(x.rq.start), get(x.rq.n), get(x.rq.len)};
      const int32_t first = get(x.first), blocks = get(x.blocks), cost = get(x.cost);
      const BlockList list{get(x.list.low), get(x.list.base0), get(x.list.base1)};
      const int64_t from = readlane64(at, l);
      // the blocks that begin within the share (all heads of the request one after the other)
      const int64_t all = (int64_t)blocks * a.Hkv;
      int64_t b0 = lo <= from ? 0 : (lo - from + cost - 1) / cost, b1 = (hi - from + cost - 1) / cost;
      if (b1 > all) b1 = all;
      const int32_t* table = a.tables + (int64_t)r * a.pitch;
      const int rows = rq.n * a.G, pos0 = rq.len - rq.n, tiles = (rows + kRows - 1) / kRows;
      while (b0 < b1) {
        const int h = (int)((uint64_t)b0 / (uint32_t)blocks);
        const int32_t i0 = (int32_t)(b0 - (int64_t)h * blocks);
        const int n_blocks = (int)(b1 - b0 < blocks - i0 ? b1 - b0 : blocks - i0);
        b0 += n_blocks;
        const char* kbase = a.k + h * a.c_sh;
        float* sbase = a.scores + h * a.s_sh;

        // rows of a tile: this lane's, its -lse in log2 units, its position (a lane past the rows: none)
        u32x4 qf[NK];
        float neg = 0.f;
        int32_t q_pos = 0, q_lo = 0, q_hi = 0;
        bool row_ok = false;
        auto take_rows = [&](int tile) __attribute__((always_inline)) {
          const int i = imin(tile * kRows + q16, rows - 1), tok = divide(i, a.by_G), head = h * a.G + (i - tok * a.G);
          const char* qrow = a.q + (int64_t)(rq.start + tok) * a.q_st + (int64_t)head * a.q_sh + 16 * g;
#pragma unroll
          for (int kc = 0; kc < NK; ++kc) qf[kc] = *reinterpret_cast<const u32x4*>(qrow + 64 * kc);
          const float z = a.lse[(int64_t)(rq.start + tok) * a.lse_st + (int64_t)head * a.lse_sh];
          neg = neg_of(z);
          row_ok = tile * kRows + q16 < rows && z != -INFINITY;
          q_pos = pos0 + tok;
          q_lo = pos0 + divide(tile * kRows, a.by_G);
          q_hi = pos0 + divide(imin(tile * kRows + kRows, rows) - 1, a.by_G);
        };
        if (tiles == 1) take_rows(0);

        // ---- PER blocks at a time: lane l holds segment l's page --------------------------------
        int32_t c_page = -1;
        auto key_of = [&](int c) __attribute__((always_inline)) -> int32_t {
          const int b = c * PER + lane / NS;
          return b < n_blocks ? (list.block(i0 + b) << LG) + 16 * (lane % NS) : rq.len;
        };
        auto take_pages = [&](int c) __attribute__((always_inline)) {
          const int32_t key = key_of(c);
          c_page = key < rq.len ? checked_page(table[key >> a.page_lg], a.n_pages) : -1;
        };
        struct Data {
          u32x4 k[NS][NK];
          float old;       // score of key 16 (q16 / 4) + 4 g + q16 % 4 of the block (NS = 2: of q16 < 8)
          float* to;       // its place, null where it is none of ours
          int32_t key;     // the block's first
        };
        auto fetch = [&](int b, Data& d) __attribute__((always_inline)) {
          if (b % PER == 0) take_pages(b / PER);
          const int l0 = NS * (b % PER);
          d.key = list.block(i0 + b) << LG;
#pragma unroll
          for (int t = 0; t < NS; ++t) {
            const int32_t page = __builtin_amdgcn_readlane(c_page, l0 + t);
            const int64_t off = (int64_t)imax(page, 0) * a.c_sp + (int64_t)((d.key + 16 * t) & ((1 << a.page_lg) - 1)) * a.c_sn;
#pragma unroll
            for (int kc = 0; kc < NK; ++kc) d.k[t][kc] = *reinterpret_cast<const u32x4*>(kbase + off + koff + 64 * kc);
          }
          const int seg = (q16 >> 2) % NS;
          const int32_t page = __shfl(c_page, l0 + seg), key = d.key + 16 * seg + 4 * g + (q16 & 3);
          d.to = nullptr;
          d.old = 0.f;
          if (q16 < 4 * NS && page >= 0 && key >= first && key < rq.len) {
            d.to = sbase + (int64_t)page * a.s_sp + (key & ((1 << a.page_lg) - 1));
            if (key < pos0) d.old = *d.to;
          }
        };
        auto compute = [&](const Data& d) __attribute__((always_inline)) {
          float sum[4 * NS];
#pragma unroll
          for (int e = 0; e < 4 * NS; ++e) sum[e] = 0.f;
          for (int tile = 0; tile < tiles; ++tile) {
            if (tiles > 1) take_rows(tile);
            int v = mask_verdict(mask, q_lo, q_hi, d.key, d.key + 16 * NS - 1);
            if (v == kDead) continue;
            if (v == kFull && d.key + 16 * NS > rq.len) v = kPartial;
            uint64_t word = ~0ull;
            if (v != kFull) {
              word = mask_word(mask, q_pos, d.key, rq.len);
              if (NS == 4) word |= (uint64_t)mask_word(mask, q_pos, d.key + 32, rq.len) << 32;
            }
            if (!row_ok) word = 0ull;
#pragma unroll
            for (int t = 0; t < NS; ++t) {
              f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int kc = 0; kc < NK; ++kc) {
                if constexpr (S::F32) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    const uint32_t kx = d.k[t][kc][j], qx = qf[kc][j];
                    s = mma16x4(__builtin_bit_cast(float, kx), __builtin_bit_cast(float, qx), s);
                  }
                } else {
                  using Frag = typename Mma<T>::frag;
                  s = mma16x32<T>(__builtin_bit_cast(Frag, d.k[t][kc]), __builtin_bit_cast(Frag, qf[kc]), s);
                }
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.c, neg));
                sum[4 * t + e] += (word >> (16 * t + 4 * g + e)) & 1ull ? p : 0.f;
              }
            }
          }
          // over the 16 rows, halving: lane q16 ends with the sum of key 16 (q16 / 4) + 4 g + q16 % 4
          float total = 0.f;
#pragma unroll
          for (int e = 0; e < 4 * NS; ++e) {
            float y = sum[e];
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) y += __shfl_xor(y, o);
            if (q16 == e) total = y;
          }
          if (d.to) *d.to = d.old + total;
        };
        Data d0{}, d1{};
        fetch(0, d0);
        int b = 0;
        for (; b + 1 < n_blocks; b += 2) {
          fetch(b + 1, d1);
          compute(d0);
          if (b + 2 < n_blocks) fetch(b + 2, d0);
          compute(d1);
        }
        if (b < n_blocks) compute(d0);
      }
    }
  }
}

// ---- many rows a request ------------------------------------------------------------------------
// A unit is 256 keys of one KV head and one of `splits` equal shares of the 64-row steps that may see them.  A
// wave holds 64 keys in registers, as the A operand of 32x32 MFMAs; the rows of Q come by LDS DMA, 64 a step in
// two slots, and are read as the B operand by all four waves.  Lane l then has row l % 32 and 16 of 32 keys,
// whose exponentials it adds up over all steps, those of one 32 rows beside the MFMAs of the next; at the end
// the 32 lanes' sums are added by halves.  Shares of a group leave their sums in the workspace, and the last
// one adds them in order.
constexpr int kQueues = 8;
constexpr int kKeysLg = 8, kKeys = 1 << kKeysLg, kStepRows = 64;

template <typename T, int D>
struct WeighTile {
  static constexpr int ROW = 2 * D, SLOT = kStepRows * ROW;
};

struct KeyUnit {
  Request rq;
  int32_t r, first, h, group, share, splits, slot;
};
struct KeyWork {
  Request rq;
  int32_t first, group0, groups, steps;
};
__device__ __forceinline__ KeyWork key_work(const WeightsK& a, int r0, int lane, int32_t& end) {
  const WeighedRequest x = weighed<kKeysLg, false>(a, r0, lane, end);
  KeyWork k{x.rq, x.first, x.list.base1, 0, 0};
  const int32_t rows = x.rq.n * a.G;
  if (r0 + lane < a.R && rows > a.row_max) {
    k.groups = x.blocks;
    k.steps = (rows + kStepRows - 1) / kStepRows;
  }
  return k;
}
// Unit `id`; past the last: false, and units is how many there are.  share: steps of a share (0 at first).
__device__ __forceinline__ bool find_keys(const WeightsK& a, int32_t id, int lane, float& share, KeyUnit& u, int64_t& units_all) {
  KeyWork k{};
  int32_t end = 0;
  if (share == 0.f || a.R <= 64) {
    float total = 0.f;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
      k = key_work(a, r0, lane, end);
      total += wave_total((float)k.groups * (float)k.steps);
    }
    share = fmaxf(total * (float)a.Hkv * a.by_shares, 8.f);
  }
  int64_t before = 0;
  int32_t slot = 0;
  end = 0;
  for (int r0 = 0; r0 < a.R; r0 += 64) {
    if (a.R > 64) k = key_work(a, r0, lane, end);
    const int32_t splits = imax((int32_t)((float)k.steps / share + 0.5f), 1);
    const int64_t units = (int64_t)k.groups * a.Hkv * splits;
    const int32_t slotted = splits > 1 ? (int32_t)units : 0;
    const int64_t n_in = wave_scan64(units, lane), at = before + n_in - units;
    const int32_t s_in = wave_scan(slotted);
    const uint64_t hit = __ballot(at <= id && id < at + units);
    if (hit) {
      const int l = (int)__builtin_ctzll(hit);
      auto get = [&](int32_t y) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(y, l); };
      u.rq = {get(k.rq.start), get(k.rq.n), get(k.rq.len)};
      u.r = r0 + l;
      u.first = get(k.first);
      u.splits = get(splits);
      // heads side by side, as in find_unit
      const uint32_t i = (uint32_t)(id - readlane64(at, l)), y = i / (uint32_t)a.Hkv;
      u.h = (int32_t)(i - y * (uint32_t)a.Hkv);
      const int32_t group = (int32_t)(y / (uint32_t)u.splits);
      u.share = (int32_t)y - group * u.splits;
      u.group = get(k.group0) + group;
      u.slot = slot + get(s_in - slotted) + (group * a.Hkv + u.h) * u.splits;
      return true;
    }
    before += readlane64(n_in, 63);
    slot += __builtin_amdgcn_readlane(s_in, 63);
  }
  units_all = before;
  return false;
}

template <typename T, int D>
__device__ __forceinline__ void weigh_keys(const WeightsK& a, const KeyUnit& u, char* smem, int32_t* flag) {
  using Frag = typename Mma<T>::frag;
  using R = Rows<D>;
  constexpr int NQF = D / 16, SLOT = WeighTile<T, D>::SLOT;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, m = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char_t*)smem;
  const KernelMask mask = weights_mask(a);
  const int32_t len = u.rq.len, pos0 = len - u.rq.n, rows = u.rq.n * a.G;
  const int32_t key0 = (u.group << kKeysLg) + 64 * w;  // this wave's first key
  const int32_t* table = a.tables + (int64_t)u.r * a.pitch;
  const int one = (1 << a.page_lg) - 1;

  // (a group that a window leaves dead, with no score that begins)
  if (a.near && (u.group + 1) << kKeysLg <= pos0) {
    const QueryRange q = query_range(mask, u.group << kKeysLg, (u.group << kKeysLg) + kKeys - 1);
    if (q.hi < pos0 || q.lo >= len) return;
  }

  // ---- the keys (one past the length or without a page: some row of page 0, whose sum goes nowhere) ----
  Frag kf[2][NQF];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int32_t key = key0 + 32 * b + m;
    const int32_t page = key < len ? checked_page(table[key >> a.page_lg], a.n_pages) : -1;
    const char* row = a.k + (int64_t)imax(page, 0) * a.c_sp + u.h * a.c_sh + (int64_t)(key & one) * a.c_sn + 16 * half;
#pragma unroll
    for (int kc = 0; kc < NQF; ++kc) kf[b][kc] = __builtin_bit_cast(Frag, *reinterpret_cast<const u32x4*>(row + 32 * kc));
  }

  // ---- the steps: rows of tokens that may see one of the group's keys ----
  const QueryRange q = query_range(mask, u.group << kKeysLg, imin((u.group << kKeysLg) + kKeys, len) - 1);
  const int32_t t0 = imin(imax(q.lo - pos0, 0), u.rq.n), t1 = imin(imax(imin(q.hi, len) - pos0 + 1, t0), u.rq.n);
  const int32_t first_step = t0 * a.G / kStepRows, n_steps = t1 > t0 ? (t1 * a.G + kStepRows - 1) / kStepRows - first_step : 0;
  int32_t j0, j1;
  share_of(n_steps, u.share, u.splits, &j0, &j1);
  j0 += first_step;
  j1 += first_step;

  lds_cptr rd[NQF];  // row m of 32 staged ones, units 2 kc + half
#pragma unroll
  for (int kc = 0; kc < NQF; ++kc) rd[kc] = (lds_cptr)smem + m * R::ROW + 16 * ((2 * kc + half) ^ R::swz(m));
  // Step j's rows, 16 a wave, and -lse of row l for lane l (a row past the last: -inf).  Where a step is whole
  // tokens it is one uniform pointer and the lanes' offsets, which stay.
  uint32_t off[R::NI];
#pragma unroll
  for (int x = 0; x < R::NI; ++x) {
    const int i = 16 * w + R::RPI * x + lane / R::UPR, tok = divide(i, a.by_G);
    off[x] = (uint32_t)tok * (uint32_t)a.q_st + (uint32_t)(i - tok * a.G) * (uint32_t)a.q_sh +
             16u * (uint32_t)((lane % R::UPR) ^ R::swz(R::RPI * x + lane / R::UPR));
  }
  const int lse_tok = divide(lane, a.by_G);
  const int32_t lse_off = (int32_t)(lse_tok * (int32_t)a.lse_st + (lane - lse_tok * a.G) * (int32_t)a.lse_sh);
  const int32_t whole = a.even ? rows / kStepRows : 0;  // steps that are
  const char* q0 = a.q + (int64_t)u.rq.start * a.q_st + (int64_t)u.h * a.G * a.q_sh;
  const float* lse0 = a.lse + (int64_t)u.rq.start * a.lse_st + (int64_t)u.h * a.G * a.lse_sh;
  auto stage = [&](int32_t j, int slot) __attribute__((always_inline)) -> float {
    const uint32_t to = lds0 + slot * SLOT + 16 * w * R::ROW;
    if (j < whole) {
      const int32_t tok = divide(j * kStepRows, a.by_G);
      const char* base = q0 + (int64_t)tok * a.q_st;
#pragma unroll
      for (int x = 0; x < R::NI; ++x) dma_x4(to + x * 1024, base, off[x]);
      return (lse0 + (int64_t)tok * a.lse_st)[lse_off];
    }
#pragma unroll
    for (int x = 0; x < R::NI; ++x) {
      const int i = imin(j * kStepRows + 16 * w + R::RPI * x + lane / R::UPR, rows - 1), tok = divide(i, a.by_G);
      dma_x4_va(to + x * 1024, q0 + (int64_t)tok * a.q_st + (int64_t)(i - tok * a.G) * a.q_sh +
                                   16 * ((lane % R::UPR) ^ R::swz(R::RPI * x + lane / R::UPR)));
    }
    const int32_t i = imin(j * kStepRows + lane, rows - 1), tok = divide(i, a.by_G);
    const float z = lse0[(int64_t)tok * a.lse_st + (int64_t)(i - tok * a.G) * a.lse_sh];
    return j * kStepRows + lane < rows ? z : -INFINITY;
  };
  // 64 steps at a time: bit l of live / full: some pair of this wave's keys and step l's rows may be live / all are
  uint64_t live = 0ull, full = 0ull;
  auto verdicts = [&](int32_t j) __attribute__((always_inline)) {
    const int32_t i0 = imin((j + lane) * kStepRows, rows - 1), i1 = imin(i0 + kStepRows, rows) - 1;
    const int v = mask_verdict(mask, pos0 + divide(i0, a.by_G), pos0 + divide(i1, a.by_G), key0, key0 + 63);
    live = __ballot(v != kDead);
    full = key0 + 63 < len ? __ballot(v == kFull) : 0ull;
  };

  float sum[32] = {};
  float c_exp = a.c;
  asm volatile("" : "+s"(c_exp));
  auto add = [&](const f32x16& x, float neg, float* to) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) to[e] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], c_exp, neg));
    // (or they are moved behind the branches that follow, away from the MFMAs)
#pragma unroll
    for (int e = 0; e < 16; e += 8)
      asm volatile("" : "+v"(to[e]), "+v"(to[e + 1]), "+v"(to[e + 2]), "+v"(to[e + 3]), "+v"(to[e + 4]), "+v"(to[e + 5]), "+v"(to[e + 6]),
                   "+v"(to[e + 7]));
  };
  auto mask_block = [&](f32x16& x, uint32_t word) __attribute__((always_inline)) {
    word >>= 4 * half;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float xv = x[e];
      const int32_t keep = __builtin_amdgcn_sbfe((int32_t)word, 8 * (e >> 2) + (e & 3), 1);
      x[e] = __builtin_bit_cast(float, (__builtin_bit_cast(int32_t, xv) & keep) | (int32_t)(0xff800000u & ~(uint32_t)keep));
    }
  };
  // Scores of the wave's keys and 32 rows, in two places in turn: the exponentials of one are added beside the MFMAs
  // of the other, which are two chains (one, of 32 keys at a time, waits for itself).
  f32x16 xa[2], xb[2];
#pragma unroll
  for (int e = 0; e < 16; ++e) xb[0][e] = xb[1][e] = -INFINITY;  // (dead)
  float neg = 0.f;  // of the rows of the scores that are still to be added
  auto block = [&](const u32x4* qf, f32x16* y, const f32x16* x) __attribute__((always_inline)) {
    y[0] = Mma<T>::mma(kf[0][0], __builtin_bit_cast(Frag, qf[0]), f32x16{0});
    y[1] = Mma<T>::mma(kf[1][0], __builtin_bit_cast(Frag, qf[0]), f32x16{0});
#pragma unroll
    for (int kc = 1; kc < NQF; ++kc) {
      y[0] = Mma<T>::mma(kf[0][kc], __builtin_bit_cast(Frag, qf[kc]), y[0]);
      y[1] = Mma<T>::mma(kf[1][kc], __builtin_bit_cast(Frag, qf[kc]), y[1]);
    }
    add(x[0], neg, sum);
    add(x[1], neg, sum + 16);
#pragma unroll
    for (int z = 0; z < 2 * NQF; ++z) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 2);
      __builtin_amdgcn_sched_group_barrier(0x002, D == 128 ? 4 : 8, 2);
      __builtin_amdgcn_sched_group_barrier(0x400, D == 128 ? 2 : 4, 2);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (j0 < j1) {
    float z = stage(j0, 0);
#pragma unroll 1
    for (int32_t j = j0; j < j1; ++j) {
      const int slot = (j - j0) & 1;
      dma_wait_all();
      asm volatile("" ::"v"(z));
      __syncthreads();
      const float z_now = z;
      if (j + 1 < j1) z = stage(j + 1, 1 - slot);
      if (((j - j0) & 63) == 0) verdicts(j);
      if (!((live >> ((j - j0) & 63)) & 1ull)) continue;
      const int32_t i0 = j * kStepRows;
      const uint64_t ok = __ballot(z_now != -INFINITY);  // (rows past the last have no weight)
      const float neg_now = z_now == -INFINITY ? 0.f : neg_of(z_now);
      const bool is_full = (full >> ((j - j0) & 63)) & 1ull, all = is_full && ok == ~0ull;
      // words of this lane's rows and the wave's keys (rolled, for one copy of the mask's code)
      uint32_t word[2][2] = {};
      if (!all) {
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          const int i = 32 * (x >> 1) + m;
          uint32_t y = ~0u;  // (full: rows without weight alone are dead)
          if (!is_full) y = mask_word(mask, pos0 + divide(imin(i0 + i, rows - 1), a.by_G), key0 + 32 * (x & 1), len);
          y = (uint32_t)(ok >> i) & 1u ? y : 0u;
#pragma unroll
          for (int z = 0; z < 4; ++z) word[z >> 1][z & 1] = z == x ? y : word[z >> 1][z & 1];
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float neg_b = __shfl(neg_now, 32 * b + m);
        u32x4 qf[NQF];
#pragma unroll
        for (int kc = 0; kc < NQF; ++kc) qf[kc] = *(lds_u4*)(rd[kc] + slot * SLOT + 32 * b * R::ROW);
        // (a row whose lse is NaN: in its scores, of which the live ones keep it, and not in their base)
        if (__ballot(neg_now != neg_now) && neg_b != neg_b) {
          qf[0][0] = ~0u;
          neg_b = 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x16* y = b ? xb : xa;
        block(qf, y, b ? xa : xb);
        neg = neg_b;
        if (!all) {
          mask_block(y[0], word[b][0]);
          mask_block(y[1], word[b][1]);
        }
      }
    }
    add(xb[0], neg, sum);
    add(xb[1], neg, sum + 16);
  }

  // ---- over the 32 rows: lane l ends with the sum of key 32 (l / 16 % 2) + 8 (l / 4 % 4) + 4 half + l % 4 ----
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int e = 0; e < o; ++e) {
      float x = sum[e], y = sum[e + o];
      asm("" : "+v"(x), "+v"(y));  // (or the index is selected, and the value by as many comparisons)
      sum[e] = (up ? y : x) + __shfl_xor(up ? x : y, o);
    }
  }
  float total = sum[0];
  const int in_wave = 32 * ((lane >> 4) & 1) + 8 * ((lane >> 2) & 3) + 4 * half + (lane & 3);
  if (u.splits > 1) {
    float* first = a.part + (int64_t)u.slot * kKeys + 64 * w + lane;
    share_store(first + u.share * kKeys, total);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      const int32_t n = __hip_atomic_fetch_add(a.count + u.slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *flag = n == u.splits - 1;
      if (n == u.splits - 1) __hip_atomic_store(a.count + u.slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (*flag == 0) return;
    total = 0.f;
#pragma unroll 4
    for (int s = 0; s < u.splits; ++s) total += __hip_atomic_load(first + s * kKeys, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const int32_t key = key0 + in_wave;
  if (key < u.first || key >= len) return;
  const int32_t page = checked_page(table[key >> a.page_lg], a.n_pages);
  if (page < 0) return;
  float* to = a.scores + page * a.s_sp + u.h * a.s_sh + (key & one);
  *to = (key < pos0 ? *to : 0.f) + total;
}

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void weights_kernel(const WeightsK a) {
  // Equal shares of the blocks first, then units as there is time (work-groups of their own for the blocks, 1024
  // behind these, mostly had none: 183 us of chunks that take 178).
  weigh_blocks<T, D>(a, (int32_t)blockIdx.x, (int32_t)gridDim.x);
  if constexpr (sizeof(T) == 2) {
    __shared__ __attribute__((aligned(256))) char smem[2 * WeighTile<T, D>::SLOT];
    __shared__ int32_t flag;
    if (a.tile_grid) {
      // Units are of different lengths and go to whom has time: the first by the work-group's number, the
      // others from a queue for each XCD (work-groups are dealt to those in turn), so that a head's rows stay in
      // one L2.  Who draws its last number clears the queue.
      const int32_t x = (int32_t)blockIdx.x % kQueues, of_x = a.tile_grid / kQueues;
      float share = 0.f;
      KeyUnit u;
      int32_t n = (int32_t)blockIdx.x / kQueues;
      int64_t units = 0;
      while (find_keys(a, n * kQueues + x, (int)threadIdx.x & 63, share, u, units)) {
        weigh_keys<T, D>(a, u, smem, &flag);
        __syncthreads();  // (the slots and the flag have been read)
        if (threadIdx.x == 0)
          flag = of_x + __hip_atomic_fetch_add(a.queue + 16 * x, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        n = flag;
        __syncthreads();
      }
      // (a number is drawn after every unit)
      if (threadIdx.x == 0 && n >= of_x && n - of_x == (int32_t)((units - x + kQueues - 1) / kQueues) - 1)
        __hip_atomic_store(a.queue + 16 * x, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// The most rows of a request that is taken by blocks.  32 requests of 300..8192 tokens (bf16, 8 KV heads of 128): by
// blocks / by 256 keys 47 / 54 us at 24 rows, 48 / 54 at 32, 53 / 54 at 48, 59 / 52 at 64, 70 / 63 at 96; 4 requests of
// 2000..16000: 16 / 16 at 12, 19 / 16 at 32, 25 / 15 at 64.
constexpr int kFewRows = 32;
// Work-groups of the others, two a CU, whose registers are full (one: 228 us of the chunks' 177), and the shares that
// the work is cut into at least (512: 176, 768: 176, 1024: 178, 1536: 191, for each reads its keys anew).
constexpr int kTileGroups = 512, kTileShares = 768;

struct WeightsPlan {
  bool tile;
  int64_t slots, zero, bytes;
};
WeightsPlan weights_plan(const pa_weights_args* x) {
  const int64_t most = x->max_fresh < x->T ? x->max_fresh : x->T;
  WeightsPlan p;
  p.tile = x->dtype != PA_F32 && most * (x->Hq / x->Hkv) > kFewRows;
  p.slots = p.tile ? 2 * kTileShares : 0;  // (a group that is split has at most 4/3 of the shares that its work fills)
  p.zero = p.tile ? (4 * (p.slots + 16 * kQueues) + 255) / 256 * 256 : 0;
  p.bytes = p.zero + 4 * p.slots * kKeys;
  return p;
}

template <typename T, int D>
int launch_weights(const WeightsK& a, hipStream_t s) {
  hipLaunchKernelGGL((weights_kernel<T, D>), dim3((unsigned)(a.tile_grid ? a.tile_grid : 1024)), dim3(256), 0, s, a);
  PA_LAUNCH_CHECK("weights_kernel");
  return PA_OK;
}

int check_weights(const char* who, const pa_weights_args* x, int* page_lg) {
  PA_CHECK_ARG(x, "%s: null arguments", who);
  if (int rc = check_pages(who, x->n_pages, x->page_size, page_lg)) return rc;
  PA_CHECK_ARG(x->dtype == PA_BF16 || x->dtype == PA_F16 || x->dtype == PA_F32, "%s: dtype %d", who, x->dtype);
  PA_CHECK_ARG(x->D == 64 || x->D == 128, "%s: D=%d (64 or 128)", who, x->D);
  PA_CHECK_ARG(x->Hkv >= 1 && x->Hq >= x->Hkv && x->Hq % x->Hkv == 0 && x->Hq <= 65535,
               "%s: %d query heads and %d KV heads (a multiple, at most 65535)", who, x->Hq, x->Hkv);
  PA_CHECK_ARG(x->R >= 0 && x->T >= 0 && x->T <= kMaxPosition && x->T * x->Hq <= kMaxPosition, "%s: R=%d T=%lld Hq=%d (T Hq < 2^30)", who,
               x->R, (long long)x->T, x->Hq);
  PA_CHECK_ARG(x->max_fresh >= 0, "%s: max_fresh=%lld", who, (long long)x->max_fresh);
  PA_CHECK_ARG(x->cols >= 0 && ((int64_t)x->cols << *page_lg) <= kMaxPosition && x->pitch >= x->cols, "%s: %d columns of %d, pitch %lld", who,
               x->cols, x->page_size, (long long)x->pitch);
  PA_CHECK_ARG(!x->mask.perm_q && !x->mask.perm_kv, "%s: the mask takes no permutation tables", who);
  for (int i = 0; i < x->mask.n_include + x->mask.n_exclude && i < PA_MAX_TERMS; ++i)
    PA_CHECK_ARG(x->mask.terms[i].kind != PA_DENSE, "%s: PA_DENSE has no meaning here", who);
  if (int rc = check_mask(&x->mask, 0)) return rc;
  PA_CHECK_ARG(x->scale > 0.f && x->scale < INFINITY, "%s: scale=%g must be positive", who, (double)x->scale);
  return PA_OK;
}

}  // namespace
}  // namespace pa

extern "C" int pa_weights_workspace(const pa_weights_args* x, int64_t* bytes, int64_t* zero) {
  using namespace pa;
  int lg;
  if (int rc = check_weights("pa_paged_weights", x, &lg)) return rc;
  PA_CHECK_ARG(bytes && zero, "pa_paged_weights: null output");
  const WeightsPlan p = weights_plan(x);
  *bytes = p.bytes;
  *zero = p.zero;
  return PA_OK;
}

extern "C" int pa_paged_weights(const pa_weights_args* x, void* stream) {
  using namespace pa;
  const char* who = "pa_paged_weights";
  int lg;
  if (int rc = check_weights(who, x, &lg)) return rc;
  if (x->R == 0 || x->T == 0 || x->n_pages == 0 || x->cols == 0) return PA_OK;
  const WeightsPlan p = weights_plan(x);
  // (units are counted in 32 bits: those of whole groups of keys, at most one to each of a table, and the shares)
  const int64_t many = std::min<int64_t>(x->R, x->T * (x->Hq / x->Hkv) / (kFewRows + 1)), groups = ((int64_t)x->cols << lg >> kKeysLg) + 1;
  PA_CHECK_ARG(!p.tile || (wide)many * groups * x->Hkv < INT_MAX - 4 * kTileShares,
               "%s: %lld requests of %d heads and tables of %d pages of %d exceed the units that can be counted", who, (long long)many,
               x->Hkv, x->cols, x->page_size);
  PA_CHECK_ARG(x->q && x->k && x->lse && x->scores && x->tables && x->lengths && x->q_start, "%s: null pointer", who);
  const int64_t esz = x->dtype == PA_F32 ? 4 : 2, row = x->D * esz, R = x->R;
  auto al = [&](const void* p, int64_t s0, int64_t s1, int64_t s2) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (s0 * esz) % 16 == 0 && (s1 * esz) % 16 == 0 && (s2 * esz) % 16 == 0;
  };
  PA_CHECK_ARG(al(x->q, x->q_st, x->q_sh, 0) && al(x->k, x->c_sp, x->c_sh, x->c_sn), "%s: rows must be 16-byte aligned", who);
  PA_CHECK_ARG(x->q_st >= 0 && x->q_sh >= 0 && x->c_sp >= 0 && x->c_sh >= 0 && x->c_sn >= x->D && x->c_sn <= (1 << 21),
               "%s: negative strides, or cache rows closer than D or further than 2^21", who);
  PA_CHECK_ARG(x->s_sp >= 0 && x->s_sh >= 0, "%s: negative strides of scores", who);
  // scores are written while the inputs are read, a page's by different waves
  const Strided<2> scores = strided<2>(x->scores, 4ll * x->page_size, {x->n_pages, x->Hkv}, {x->s_sp, x->s_sh}, 4);
  PA_CHECK_ARG(nested(scores), "%s: rows of scores overlap", who);
  auto in_of = [&](const auto& out) -> const char* {
    return overlap(out, strided<2>(x->q, row, {x->T, x->Hq}, {x->q_st, x->q_sh}, (int)esz)) ? "q"
           : overlap(out, strided<3>(x->k, row, {x->n_pages, x->Hkv, x->page_size}, {x->c_sp, x->c_sh, x->c_sn}, (int)esz)) ? "k"
           : overlap(out, strided<2>(x->lse, 4, {x->T, x->Hq}, {x->lse_st, x->lse_sh}, 4)) ? "lse"
           : overlap(out, tables_span(x->tables, x->R, x->pitch, x->cols)) ? "tables"
           : overlap(out, flat(x->lengths, 4 * R)) ? "lengths"
           : overlap(out, flat(x->q_start, 4 * (R + 1))) ? "q_start"
           : overlap(out, flat(x->first, x->first ? 4 * R : 0)) ? "first" : nullptr;
  };
  const char* other = in_of(scores);
  PA_CHECK_ARG(!other, "%s: scores and %s overlap", who, other);
  PA_CHECK_ARG(p.bytes == 0 || (x->workspace && reinterpret_cast<uintptr_t>(x->workspace) % 256 == 0 && x->workspace_bytes >= p.bytes),
               "%s: needs a 256-byte aligned workspace of %lld bytes", who, (long long)p.bytes);
  const Strided<1> ws = flat(x->workspace, p.bytes);
  other = in_of(ws);
  PA_CHECK_ARG(!other, "%s: workspace and %s overlap", who, other);
  PA_CHECK_ARG(!overlap(ws, scores), "%s: workspace and scores overlap", who);
  WeightsK a;
  a.q = static_cast<const char*>(x->q);
  a.q_st = x->q_st * esz;
  a.q_sh = x->q_sh * esz;
  a.k = static_cast<const char*>(x->k);
  a.c_sp = x->c_sp * esz;
  a.c_sh = x->c_sh * esz;
  a.c_sn = x->c_sn * esz;
  a.n_pages = x->n_pages;
  a.page_lg = lg;
  a.cols = x->cols;
  a.tables = x->tables;
  a.pitch = x->pitch;
  a.lengths = x->lengths;
  a.q_start = x->q_start;
  a.first = x->first;
  a.R = x->R;
  a.T = (int32_t)x->T;
  a.Hkv = x->Hkv;
  a.G = x->Hq / x->Hkv;
  a.by_G = divisor_of((uint32_t)a.G);
  a.c = x->scale * 1.4426950408889634f;
  a.n_include = x->mask.n_include;
  a.n_exclude = x->mask.n_exclude;
  for (int i = 0; i < PA_MAX_TERMS; ++i) {
    pa_term t = x->mask.terms[i];
    // (no distance reaches the clamp)
    t.p0 = imin(t.p0, kMaxPosition);
    t.p1 = imin(t.p1, kMaxPosition);
    t.p2 = imin(t.p2, kMaxPosition);
    a.terms[i] = t;
  }
  a.lse = x->lse;
  a.lse_st = x->lse_st;
  a.lse_sh = x->lse_sh;
  a.scores = x->scores;
  a.s_sp = x->s_sp;
  a.s_sh = x->s_sh;
  a.near = a.n_include > 0;
  for (int i = 0; i < a.n_include; ++i) {
    const int32_t kind = a.terms[i].kind;
    a.near = a.near && (kind == PA_WINDOW || kind == PA_SINKS || kind == PA_TWOBAND);
  }
  a.row_max = p.tile ? kFewRows : INT_MAX;
  a.tile_grid = p.tile ? kTileGroups : 0;
  auto near = [&](int64_t st, int64_t sh) { return st <= (1 << 24) && sh <= (1 << 24) && st >= -(1 << 24) && sh >= -(1 << 24); };
  a.even = kStepRows % a.G == 0 && near(a.q_st, a.q_sh) && near(a.lse_st, a.lse_sh);
  a.by_shares = 1.f / (float)kTileShares;
  a.queue = reinterpret_cast<int32_t*>(x->workspace);
  a.count = a.queue + 16 * kQueues;
  a.part = reinterpret_cast<float*>(static_cast<char*>(x->workspace) + p.zero);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (x->D == 64)
    return x->dtype == PA_F32 ? launch_weights<float, 64>(a, s) : x->dtype == PA_BF16 ? launch_weights<__bf16, 64>(a, s) : launch_weights<_Float16, 64>(a, s);
  return x->dtype == PA_F32 ? launch_weights<float, 128>(a, s) : x->dtype == PA_BF16 ? launch_weights<__bf16, 128>(a, s) : launch_weights<_Float16, 128>(a, s);
}
