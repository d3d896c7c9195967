// Which cached keys stay, and their move to the front of their request's pages (gfx950).
//
// pa_choose_keys: a work-group for the keys of one layer, request and KV head.  Their scores become
// unsigned numbers of the same order and stay in registers, four keys side by side a load (beyond 16384
// they are read again for every pass).  The keep - recent-th largest is found 11, 11 and 10 bits at a
// time, each from counts in LDS of the keys that agree so far; where a bin's keys just make up the number the
// search ends, else the keys equal to the bound go by place.  Ranks among the kept are sums over the waves.
// What bounds it: for one layer of a few requests the launch and its trips to memory (4 requests of 1000, 4
// heads: 5.5 us), for many the counts' and ranks' instructions beside the barriers of three work-groups a CU
// (8 layers of 32 requests of 1500 to 16384, 8 heads, 51 MB: 43 us, of which the loads 16).
//
// pa_evict_rows: kept[j] >= first + j, so the row that place first + j gives up was read for some j' <= j: a
// work-group that takes the rows of one layer, request, KV head and tensor in order, a batch into
// registers before any of it is stored and the next one's on their way meanwhile, moves them in place with
// no scratch memory.  What bounds it: HBM (1.8 GB in 375 us, 4.9 TB/s, where a copy reaches 5.0), and for
// a few heads four trips to memory (2 requests of about 1000, 4 heads of 64 in f32: 4.8 us).
#include <limits.h>

#include "page_checks.hpp"
#include "paged_attn.hpp"

namespace pa {
namespace {

struct Pages {
  const int32_t* tables;
  int64_t pitch, n_pages;
  int32_t cols, page_lg;
  const int32_t* lengths;
  const int32_t* first;
};
struct Held {
  int32_t len, first;
};
__device__ __forceinline__ Held held_of(const Pages& p, int r) {
  const int32_t len = imin(imax(p.lengths[r], 0), p.cols << p.page_lg);
  return {len, p.first ? imin(imax(p.first[r], 0), len) : 0};
}

// ---- which stay ---------------------------------------------------------------------------------
constexpr int kChooseThreads = 512, kChooseWaves = kChooseThreads / 64, kMostQuads = 8;

struct ChooseK {
  const float* scores;
  int64_t s_sl, s_sp, s_sh;
  uint32_t s_bytes;  // of a head's scores from its first to its last (0: not by 32-bit offsets of 16 bytes)
  Pages pages;
  int32_t R, Hkv, keep, recent, limit;
  int32_t* kept;
  int32_t* after;
  int32_t* missing;      // null, or where a request that cannot be evicted for want of pages shows
  int32_t missing_bits;
};

// A number of the order of the scores: NaN above all, -0 as 0, never 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The counts of the upper 11 bits are kept kCopies times, lane l adding to the l % kCopies-th: scores that are
// equal (keys that nothing has looked at) or near queue for a word otherwise, some 6 cycles a lane (2048 lists
// of 1500 to 16384, a fifth of them 0: the counts alone 33 us with one copy).  A copy's pitch puts a bin's
// words on different banks.
constexpr int kBins = 2048, kCopies = 4, kPitch = kBins + 64 / kCopies;
struct ChooseShared {
  __attribute__((aligned(16))) int32_t bins[kCopies * kPitch + kBins + kBins / 2];  // .. then those of the next bits
  int32_t pre[2][kMostQuads * kChooseWaves];
  int32_t wave[3][kChooseWaves];
  int32_t bin[3], above[3], held[3];
};

// The keys first .. first + n - 1 of a list, `want` of which stay.  Thread t holds QUADS times 4 of them side by
// side (a page is a multiple of 16 rows, so they are in one), from the multiple of 4 at or below first.
template <int QUADS, bool ANY>
__device__ __forceinline__ void choose_body(const ChooseK& a, const float* scores, const int32_t* table, int32_t first,
                                            int32_t n, int32_t want, int32_t* kept, ChooseShared& s) {
  constexpr int SPAN = 4 * QUADS * kChooseThreads;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t base = first & ~3, end = first + n;
  const int chunks = QUADS == kMostQuads ? (end - base + SPAN - 1) / SPAN : 1;
  const int one = (1 << a.pages.page_lg) - 1;
  uint32_t u[QUADS][4];
  auto at = [&](int c, int i) __attribute__((always_inline)) { return base + c * SPAN + 4 * (i * kChooseThreads + tid); };
  auto load = [&](int c) __attribute__((always_inline)) {
    // All pages on their way at once, then all scores.  (A place past the table reads page 0, and what has no
    // page the first scores; neither is used.)
    const __amdgpu_buffer_rsrc_t pages = __builtin_amdgcn_make_buffer_rsrc((void*)table, 0, 4 * a.pages.cols, 0x00027000);
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc((void*)scores, 0, (int)a.s_bytes, 0x00027000);
    int32_t page[QUADS];
#pragma unroll
    for (int i = 0; i < QUADS; ++i) page[i] = (int32_t)__builtin_amdgcn_raw_buffer_load_b32(pages, (at(c, i) >> a.pages.page_lg) << 2, 0, 0);
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      page[i] = checked_page(page[i], a.pages.n_pages);
      u32x4 x;
      if constexpr (ANY) {
        x = u32x4{0u, 0u, 0u, 0u};
        if (page[i] >= 0) {
          const float* y = scores + (int64_t)page[i] * a.s_sp + (at(c, i) & one);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(uint32_t, y[e]);
        }
      } else {
        const uint32_t off = (uint32_t)page[i] * (uint32_t)a.s_sp + (uint32_t)(at(c, i) & one);
        x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, page[i] < 0 ? 0u : off << 2, 0, 0));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) u[i][e] = x[e];
    }
#pragma unroll
    for (int i = 0; i < QUADS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = at(c, i) + e;
        u[i][e] = t < first || t >= end ? 0u : page[i] < 0 ? 1u : rank_of(__builtin_bit_cast(float, u[i][e]));
      }
  };
#pragma unroll
  for (int i = tid; i < (int)(sizeof(s.bins) / 16); i += kChooseThreads) reinterpret_cast<u32x4*>(s.bins)[i] = u32x4{0u, 0u, 0u, 0u};
  load(0);
  __syncthreads();
  // ---- the bound: its upper 11 bits, the next 11, the last 10, each by the counts of the keys that have
  // the bits so far (what is no key is 0, below all) ----
  uint32_t bound = 0u;
  int32_t rest = want;  // of the keys at the bound's bits so far that many stay
  bool just = false;    // all of them do
#pragma unroll 1
  for (int round = 0; round < 3 && !just; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
    const uint32_t mask = (1u << bits) - 1u;
    int32_t* bins = s.bins + (round == 0 ? 0 : round == 1 ? kCopies * kPitch : kCopies * kPitch + kBins);
    int32_t* mine_of = round == 0 ? bins + lane % kCopies * kPitch : bins;
    for (int c = 0; c < chunks; ++c) {
      if (chunks > 1) load(c);
#pragma unroll
      for (int i = 0; i < QUADS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          // (largest first)
          if (round == 0 || (u[i][e] ^ bound) >> (shift + bits) == 0u) atomicAdd(&mine_of[mask - ((u[i][e] >> shift) & mask)], 1);
    }
    __syncthreads();
    constexpr int PER = kBins / kChooseThreads;
    static_assert(PER == 4, "16 bytes a thread");
    u32x4 mine = u32x4{0u, 0u, 0u, 0u};
    if (round < 2 || tid < kChooseThreads / 2)
      for (int z = 0; z < (round == 0 ? kCopies : 1); ++z) mine += *reinterpret_cast<const u32x4*>(bins + z * kPitch + PER * tid);
    const int32_t sum = (int32_t)((mine[0] + mine[1]) + (mine[2] + mine[3])), in = wave_scan(sum);
    if (lane == 63) s.wave[round][w] = in;
    __syncthreads();
    int32_t above = in - sum;
#pragma unroll
    for (int y = 0; y < kChooseWaves; ++y) above += y < w ? s.wave[round][y] : 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < rest && rest <= above + (int32_t)mine[i]) {
        s.bin[round] = PER * tid + i;
        s.above[round] = above;
        s.held[round] = (int32_t)mine[i];
      }
      above += (int32_t)mine[i];
    }
    __syncthreads();
    bound |= (mask - (uint32_t)s.bin[round]) << shift;
    rest -= s.above[round];
    just = rest == s.held[round];
  }
  // Those above the bound stay (just: those not below it), and of those at it the first `rest`.
  const uint32_t least = just ? bound : bound + 1u;
  const bool top = !just && bound == 0xffffffffu;  // (NaNs beyond the number wanted: nothing is above)
  int32_t ties = 0, done = 0;
  // Ranks of the keys for which `is` holds, in order of place: quad, thread, key.  rank(i): of the first key of
  // this thread's quad i; from: those of earlier chunks, and of this one after it.
  int32_t in[QUADS];
  auto ranks = [&](auto is, int32_t* from, int32_t* counts) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const int32_t x = (is(u[i][0]) + is(u[i][1])) + (is(u[i][2]) + is(u[i][3]));
      in[i] = wave_scan(x);
      if (lane == 63) counts[i * kChooseWaves + w] = in[i];
      in[i] -= x;
    }
    __syncthreads();
    static_assert(kMostQuads * kChooseWaves <= 64, "one entry a lane");
    const int32_t one_of = lane < QUADS * kChooseWaves ? counts[lane] : 0, upto = wave_scan(one_of);
#pragma unroll
    for (int i = 0; i < QUADS; ++i) in[i] += *from + __builtin_amdgcn_readlane(upto - one_of, i * kChooseWaves + w);
    *from += __builtin_amdgcn_readlane(upto, 63);
  };
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) {
      __syncthreads();  // (the last one's counts have been read)
      load(c);
    }
    if (!just) {
      ranks([&](uint32_t x) __attribute__((always_inline)) { return x == bound ? 1 : 0; }, &ties, s.pre[0]);
#pragma unroll
      for (int i = 0; i < QUADS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool tie = u[i][e] == bound;
          u[i][e] = (!top && u[i][e] >= least) || (tie && in[i] < rest) ? 1u : 0u;
          in[i] += tie ? 1 : 0;
        }
    } else {
#pragma unroll
      for (int i = 0; i < QUADS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) u[i][e] = u[i][e] >= least ? 1u : 0u;
    }
    ranks([&](uint32_t x) __attribute__((always_inline)) { return (int32_t)x; }, &done, s.pre[1]);
#pragma unroll
    for (int i = 0; i < QUADS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (u[i][e]) kept[in[i]++] = at(c, i) + e;
  }
}

// ANY: scores that are not aligned to 16 bytes, or span more than 32 bits of bytes.
template <bool ANY>
__global__ __launch_bounds__(kChooseThreads) __attribute__((amdgpu_waves_per_eu(6))) void choose_kernel(const ChooseK a) {
  __shared__ ChooseShared s;
  const int tid = threadIdx.x;
  const int h = (int)(blockIdx.x % (unsigned)a.Hkv), lr = (int)(blockIdx.x / (unsigned)a.Hkv);
  const int r = lr % a.R, layer = lr / a.R;
  const Held q = held_of(a.pages, r);
  const int32_t m = q.len - q.first;
  int32_t* kept = a.kept + (((int64_t)layer * a.R + r) * a.Hkv + h) * a.keep;
  const int32_t* table = a.pages.tables + r * a.pages.pitch;
  // (all layers and heads of a request see the same table; a trip to memory more, where it is asked for)
  bool whole = m <= a.limit;
  if (a.missing && !whole) {
    bool none = false;
    for (int32_t c = (q.first >> a.pages.page_lg) + tid; c <= (q.len - 1) >> a.pages.page_lg; c += kChooseThreads)
      none |= checked_page(table[c], a.pages.n_pages) < 0;
    whole = __syncthreads_or(none);
    if (whole && layer == 0 && h == 0 && tid == 0) atomicOr(a.missing, a.missing_bits);
  }
  if (layer == 0 && h == 0 && tid == 0) a.after[r] = whole ? a.pages.lengths[r] : q.first + a.keep;
  if (whole) {
    for (int j = tid; j < a.keep; j += kChooseThreads) kept[j] = -1;
    return;
  }
  const int32_t want = a.keep - a.recent, n = m - a.recent;
  for (int j = tid; j < a.recent; j += kChooseThreads) kept[want + j] = q.len - a.recent + j;
  if (want == 0) return;
  const float* scores = a.scores + layer * a.s_sl + h * a.s_sh;
  const int32_t held = n + (q.first & 3);
  if (held <= 4 * kChooseThreads)
    choose_body<1, ANY>(a, scores, table, q.first, n, want, kept, s);
  else if (held <= 8 * kChooseThreads)
    choose_body<2, ANY>(a, scores, table, q.first, n, want, kept, s);
  else if (held <= 16 * kChooseThreads)
    choose_body<4, ANY>(a, scores, table, q.first, n, want, kept, s);
  else
    choose_body<kMostQuads, ANY>(a, scores, table, q.first, n, want, kept, s);
}

// ---- their move -----------------------------------------------------------------------------------
// Heads from which there are work-groups enough with 512 threads (1024: 4 layers of 32 requests, 8 heads, 1.8 GB
// 389 us and 375; a layer of 2 requests, 4 heads, 4 MB 7.1 us and 7.6).
constexpr int64_t kManyHeads = 512;

// Where heads times K and V are fewer than the CUs, a row is cut into slices of 64 bytes or more (each takes more rows
// at a time then, and a head's columns move independently): one request of 7000, 4 heads of 128 in f16, to 2500:
// 24.8 us whole, 14.6 in slices of 128 bytes, 9.6 of 64; 4 requests of 9000, 8 heads in f32, to 2048: 47 and
// 26; two requests of about 1000, 4 heads of 64 in f32: 7.1 and 4.8; 16 requests of 8 heads are as fast whole.
constexpr int kSliceLg = 2;
constexpr int64_t kSliceGroups = 256;

struct EvictK {
  const int32_t* kept;
  char* k;
  char* v;
  float* scores;
  int64_t c_sl, c_sp, c_sh, c_sn;  // bytes
  int64_t s_sl, s_sp, s_sh;        // floats
  Pages pages;
  int32_t R, Hkv, keep, row_lg;    // row_lg: log2 of the 16-byte units of a row
  int32_t cut_lg;                  // and of the slices of a row that go to work-groups of their own
};

// Units of type U (1 << lg of them a row) of the kept rows of one head, in order, by THREADS threads.  A batch's
// rows are loaded before the last one's are stored: they come from places past those.
template <typename U, int UNROLL, int THREADS, typename At>
__device__ __forceinline__ void move_rows(const EvictK& a, const int32_t* kept, const int32_t* table, const Held& q, int lg, At at) {
  const int tid = threadIdx.x, unit = tid & ((1 << lg) - 1);
  const int per = THREADS >> lg;  // rows that one load of the work-group takes
  const int one = (1 << a.pages.page_lg) - 1;
  const int32_t reach = a.pages.cols << a.pages.page_lg;
  // (a place past the table takes nothing; and sums of places stay below 2^31, however long the list)
  const int32_t most = imin(a.keep, reach - q.first);
  if (most <= 0) return;
  struct Batch {
    U x[UNROLL];
    U* from[UNROLL];
    U* to[UNROLL];  // null where nothing moves
  };
  auto places = [&](int j0, Batch& b) __attribute__((always_inline)) {
    int32_t of[UNROLL], p[UNROLL], d[UNROLL];
    if (j0 >= most) {
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) b.to[i] = nullptr;
      return;
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) of[i] = kept[imin(j0 + i * per + (tid >> lg), most - 1)];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int32_t dst = imin(q.first + j0 + i * per + (tid >> lg), reach - 1);
      p[i] = table[imin(imax(of[i], 0), reach - 1) >> a.pages.page_lg];
      d[i] = table[dst >> a.pages.page_lg];
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int j = j0 + i * per + (tid >> lg), dst = q.first + j;
      p[i] = checked_page(p[i], a.pages.n_pages);
      d[i] = checked_page(d[i], a.pages.n_pages);
      b.from[i] = at(imax(p[i], 0), of[i] & one) + unit;
      b.to[i] = j < most && of[i] > dst && of[i] < reach && p[i] >= 0 && d[i] >= 0 ? at(d[i], dst & one) + unit : nullptr;
    }
  };
  auto fetch = [&](Batch& b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      b.x[i] = U{};
      if (b.to[i]) b.x[i] = *b.from[i];
    }
  };
  auto step = [&](int j0, Batch& b, Batch& next) __attribute__((always_inline)) {
    // (all of the batch has been read, by every wave, before any of it is written)
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) asm volatile("" ::"v"(b.x[i]));
    __syncthreads();
    fetch(next);
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
      if (b.to[i]) *b.to[i] = b.x[i];
    places(j0 + 2 * per * UNROLL, b);
  };
  Batch b0, b1;
  places(0, b0);
  fetch(b0);
  places(per * UNROLL, b1);
  for (int j0 = 0; j0 < most; j0 += 2 * per * UNROLL) {
    step(j0, b0, b1);
    step(j0 + per * UNROLL, b1, b0);
  }
}

typedef uint32_t unit16 __attribute__((ext_vector_type(4)));

template <int THREADS>
__global__ __launch_bounds__(THREADS) void evict_kernel(const EvictK a) {
  const int h = (int)(blockIdx.x % (unsigned)a.Hkv), lr = (int)(blockIdx.x / (unsigned)a.Hkv);
  const int r = lr % a.R, layer = lr / a.R;
  const Held q = held_of(a.pages, r);
  const int32_t* kept = a.kept + (((int64_t)layer * a.R + r) * a.Hkv + h) * a.keep;
  const int32_t* table = a.pages.tables + r * a.pages.pitch;
  if (blockIdx.y < 2u << a.cut_lg) {
    const int lg = a.row_lg - a.cut_lg;
    char* base = (blockIdx.y & 1 ? a.v : a.k) + layer * a.c_sl + h * a.c_sh + ((int)(blockIdx.y >> 1) << lg << 4);
    move_rows<unit16, 4, THREADS>(a, kept, table, q, lg, [&](int32_t page, int32_t row) __attribute__((always_inline)) {
      return reinterpret_cast<unit16*>(base + page * a.c_sp + row * a.c_sn);
    });
  } else {
    float* base = a.scores + layer * a.s_sl + h * a.s_sh;
    move_rows<float, 4, THREADS>(a, kept, table, q, 0, [&](int32_t page, int32_t row) __attribute__((always_inline)) {
      return base + page * a.s_sp + row;
    });
  }
}

// The checks that both calls share; p is filled in.
int check_keys(const char* who, int64_t n_pages, int32_t page_size, const int32_t* tables, int64_t pitch, int32_t cols,
               const int32_t* lengths, const int32_t* first, int32_t layers, int32_t R, int32_t Hkv, int32_t keep, Pages* p) {
  int lg;
  if (int rc = check_pages(who, n_pages, page_size, &lg)) return rc;
  PA_CHECK_ARG(cols >= 0 && ((int64_t)cols << lg) <= kMaxPosition && pitch >= cols, "%s: %d columns of %d, pitch %lld", who, cols,
               page_size, (long long)pitch);
  PA_CHECK_ARG(layers >= 0 && R >= 0 && Hkv >= 1 && Hkv <= 65535, "%s: layers=%d R=%d Hkv=%d", who, layers, R, Hkv);
  PA_CHECK_ARG(keep >= 1 && keep <= kMaxPosition, "%s: keep=%d", who, keep);
  // (a grid of up to 1024 threads a work-group has less than 2^32 of them)
  PA_CHECK_ARG((wide)layers * R * Hkv < (1 << 22), "%s: %d layers of %d requests of %d heads exceed the grid limit", who, layers, R, Hkv);
  PA_CHECK_ARG(R == 0 || (lengths && (cols == 0 || tables)), "%s: null lengths / tables", who);
  *p = Pages{tables, pitch, n_pages, cols, lg, lengths, first};
  return PA_OK;
}

}  // namespace
}  // namespace pa

extern "C" int pa_choose_keys(const pa_choose_args* x, void* stream) {
  using namespace pa;
  PA_CHECK_ARG(x, "pa_choose_keys: null arguments");
  ChooseK a;
  if (int rc = check_keys("pa_choose_keys", x->n_pages, x->page_size, x->tables, x->pitch, x->cols, x->lengths, x->first, x->layers,
                          x->R, x->Hkv, x->keep, &a.pages))
    return rc;
  PA_CHECK_ARG(x->recent >= 0 && x->recent <= x->keep && x->limit >= x->keep, "pa_choose_keys: recent=%d keep=%d limit=%d (ascending)",
               x->recent, x->keep, x->limit);
  if (x->R == 0 || x->layers == 0) return PA_OK;
  PA_CHECK_ARG(x->kept && x->after && (x->n_pages == 0 || x->scores), "pa_choose_keys: null kept / after / scores");
  PA_CHECK_ARG(x->s_sl >= 0 && x->s_sp >= 0 && x->s_sh >= 0, "pa_choose_keys: negative strides");
  const int64_t R = x->R;
  const Strided<3> scores = strided<3>(x->scores, 4ll * x->page_size, {x->layers, x->n_pages, x->Hkv}, {x->s_sl, x->s_sp, x->s_sh}, 4);
  const Strided<1> kept = strided<1>(x->kept, 4ll * x->keep, {(int64_t)x->layers * R * x->Hkv}, {x->keep}, 4);
  if (int rc = check_apart("pa_choose_keys",
                           {{"lengths", flat(x->lengths, 4 * R)}, {"first", flat(x->first, x->first ? 4 * R : 0)},
                            {"tables", tables_span(x->tables, x->R, x->pitch, x->cols)}},
                           {{"kept", kept}, {"after", flat(x->after, 4 * R)}, {"missing", flat(x->missing, x->missing ? 4 : 0)}}))
    return rc;
  PA_CHECK_ARG(!overlap(kept, scores) && !overlap(flat(x->after, 4 * R), scores) && !overlap(flat(x->missing, x->missing ? 4 : 0), scores),
               "pa_choose_keys: kept, after or missing and scores overlap");
  a.scores = x->scores;
  a.s_sl = x->s_sl;
  a.s_sp = x->s_sp;
  a.s_sh = x->s_sh;
  const wide bytes = x->n_pages ? span(strided<1>(x->scores, 4ll * x->page_size, {x->n_pages}, {x->s_sp}, 4)) : 4;
  const bool aligned = reinterpret_cast<uintptr_t>(x->scores) % 16 == 0 && x->s_sl % 4 == 0 && x->s_sp % 4 == 0 && x->s_sh % 4 == 0;
  a.s_bytes = x->n_pages && aligned && bytes < (1ll << 32) ? (uint32_t)bytes : 0u;
  a.R = x->R;
  a.Hkv = x->Hkv;
  a.keep = x->keep;
  a.recent = x->recent;
  a.limit = x->limit;
  a.kept = x->kept;
  a.after = x->after;
  a.missing = x->missing;
  a.missing_bits = x->missing_bits;
  const dim3 grid((unsigned)(x->layers * R * x->Hkv));
  if (a.s_bytes)
    hipLaunchKernelGGL(choose_kernel<false>, grid, dim3(kChooseThreads), 0, static_cast<hipStream_t>(stream), a);
  else
    hipLaunchKernelGGL(choose_kernel<true>, grid, dim3(kChooseThreads), 0, static_cast<hipStream_t>(stream), a);
  PA_LAUNCH_CHECK("choose_kernel");
  return PA_OK;
}

extern "C" int pa_evict_rows(const pa_evict_args* x, void* stream) {
  using namespace pa;
  PA_CHECK_ARG(x, "pa_evict_rows: null arguments");
  EvictK a;
  if (int rc = check_keys("pa_evict_rows", x->n_pages, x->page_size, x->tables, x->pitch, x->cols, x->lengths, x->first, x->layers, x->R,
                          x->Hkv, x->keep, &a.pages))
    return rc;
  PA_CHECK_ARG(x->dtype == PA_BF16 || x->dtype == PA_F16 || x->dtype == PA_F32, "pa_evict_rows: dtype %d", x->dtype);
  PA_CHECK_ARG(x->D == 64 || x->D == 128, "pa_evict_rows: D=%d (64 or 128)", x->D);
  if (x->R == 0 || x->layers == 0 || x->n_pages == 0) return PA_OK;
  PA_CHECK_ARG(x->kept && x->k && x->v, "pa_evict_rows: null kept / k / v");
  const int64_t esz = x->dtype == PA_F32 ? 4 : 2, row = x->D * esz, R = x->R;
  auto al = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  PA_CHECK_ARG(al(x->k) && al(x->v) && (x->c_sl * esz) % 16 == 0 && (x->c_sp * esz) % 16 == 0 && (x->c_sh * esz) % 16 == 0 &&
                   (x->c_sn * esz) % 16 == 0,
               "pa_evict_rows: rows must be 16-byte aligned");
  PA_CHECK_ARG(x->c_sl >= 0 && x->c_sp >= 0 && x->c_sh >= 0 && x->c_sn >= x->D && x->s_sl >= 0 && x->s_sp >= 0 && x->s_sh >= 0,
               "pa_evict_rows: negative strides, or rows closer than D");
  // Rows of k, v and scores are written while others are read: none shares a byte with another, or with an
  // input.
  const int64_t n[] = {x->layers, x->n_pages, x->Hkv, x->page_size}, c[] = {x->c_sl, x->c_sp, x->c_sh, x->c_sn};
  const Strided<4> k = strided<4>(x->k, row, n, c, (int)esz), v = strided<4>(x->v, row, n, c, (int)esz);
  const Strided<3> scores = strided<3>(x->scores, 4ll * x->page_size, {x->scores ? x->layers : 0, x->n_pages, x->Hkv},
                                       {x->s_sl, x->s_sp, x->s_sh}, 4);
  PA_CHECK_ARG(nested(k) && (!x->scores || nested(scores)), "pa_evict_rows: rows of k, v or scores overlap");
  Strided<5> kv;
  kv.at = k.at < v.at ? k.at : v.at;
  kv.w = row;
  for (int i = 0; i < 4; ++i) {
    kv.n[i] = k.n[i];
    kv.s[i] = k.s[i];
  }
  kv.n[4] = 2;
  kv.s[4] = k.at < v.at ? v.at - k.at : k.at - v.at;
  PA_CHECK_ARG(!overlap(k, v) || nested(kv), "pa_evict_rows: k and v overlap");
  auto apart = [&](const char* name, const auto& out) {
    const char* other = overlap(out, strided<1>(x->kept, 4ll * x->keep, {(int64_t)x->layers * R * x->Hkv}, {x->keep}, 4)) ? "kept"
                        : overlap(out, tables_span(x->tables, x->R, x->pitch, x->cols))                                   ? "tables"
                        : overlap(out, flat(x->lengths, 4 * R))                                                           ? "lengths"
                        : overlap(out, flat(x->first, x->first ? 4 * R : 0))                                              ? "first"
                                                                                                                          : nullptr;
    PA_CHECK_ARG(!other, "pa_evict_rows: %s and %s overlap", name, other);
    return (int)PA_OK;
  };
  if (int rc = apart("k", k)) return rc;
  if (int rc = apart("v", v)) return rc;
  if (int rc = apart("scores", scores)) return rc;
  PA_CHECK_ARG(!overlap(scores, k) && !overlap(scores, v), "pa_evict_rows: scores and k or v overlap");
  a.kept = x->kept;
  a.k = static_cast<char*>(x->k);
  a.v = static_cast<char*>(x->v);
  a.scores = x->scores;
  a.c_sl = x->c_sl * esz;
  a.c_sp = x->c_sp * esz;
  a.c_sh = x->c_sh * esz;
  a.c_sn = x->c_sn * esz;
  a.s_sl = x->s_sl;
  a.s_sp = x->s_sp;
  a.s_sh = x->s_sh;
  a.R = x->R;
  a.Hkv = x->Hkv;
  a.keep = x->keep;
  a.row_lg = row == 128 ? 3 : row == 256 ? 4 : 5;
  const int64_t heads = x->layers * R * x->Hkv;
  a.cut_lg = 0;
  while (a.row_lg - a.cut_lg > kSliceLg && heads << (a.cut_lg + 1) < kSliceGroups) ++a.cut_lg;
  const dim3 grid((unsigned)heads, (2u << a.cut_lg) + (x->scores ? 1 : 0));
  if (heads < kManyHeads)
    hipLaunchKernelGGL(evict_kernel<1024>, grid, dim3(1024), 0, static_cast<hipStream_t>(stream), a);
  else
    hipLaunchKernelGGL(evict_kernel<512>, grid, dim3(512), 0, static_cast<hipStream_t>(stream), a);
  PA_LAUNCH_CHECK("evict_kernel");
  return PA_OK;
}
