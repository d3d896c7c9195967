// Which cached keys stay, and their move to the front of their request's pages (gfx950).
//
// pa_choose_keys: a work-group for the keys of one layer, request and KV head.  Their scores become
// unsigned numbers of the same order and stay in registers (beyond 32768 of them they are read again for
// every pass); the keep - recent-th largest is found bit by bit from the top, each pass counting by
// ballots how many are not below the bound tried (no histogram: scores that are equal, as those of
// keys that were never looked at, would queue for one LDS word).  Where a bound passes just the
// number wanted the search ends, else the keys equal to it go by place; ranks among the kept are the
// same ballots' counts, summed over waves.
//
// pa_evict_rows: kept[j] >= first + j, so the row that place first + j gives up was read for some j' <= j: a
// work-group that takes the rows of one layer, request, KV head and tensor in order, a batch into
// registers before any of it is stored, moves them in place with no scratch memory.
#include <limits.h>

#include "page_checks.hpp"

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
constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;

struct ChooseK {
  const float* scores;
  int64_t s_sl, s_sp, s_sh;
  Pages pages;
  int32_t R, Hkv, keep, recent, limit;
  int32_t* kept;
  int32_t* after;
};

// A number of the order of the scores: NaN above all, -0 as 0, never 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct ChooseShared {
  int32_t n[2][kChooseWaves];
  uint64_t pre[32 * kChooseWaves];
  uint64_t wave[kChooseWaves];
};

template <int ITEMS>
__device__ __forceinline__ void choose_body(const ChooseK& a, const float* scores, const int32_t* table, int32_t first,
                                            int32_t n, int32_t want, int32_t* kept, ChooseShared& s) {
  constexpr int SPAN = ITEMS * kChooseThreads;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunks = (n + SPAN - 1) / SPAN;
  uint32_t u[ITEMS];
  auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int x = c * SPAN + i * kChooseThreads + tid;
      u[i] = 0u;
      if (x < n) {
        const int32_t t = first + x, page = checked_page(table[t >> a.pages.page_lg], a.pages.n_pages);
        u[i] = page < 0 ? 1u : rank_of(scores[(int64_t)page * a.s_sp + (t & ((1 << a.pages.page_lg) - 1))]);
      }
    }
  };
  load(0);
  // ---- the largest bound that `want` of them are not below ----
  uint32_t bound = 0u;
  int buf = 0;
  bool just = false;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit && !just; bit >>= 1) {
    const uint32_t x = bound | bit;
    int32_t mine = 0;
    for (int c = 0; c < chunks; ++c) {
      if (chunks > 1) load(c);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) mine += __builtin_popcountll(__ballot(u[i] >= x));
    }
    if (lane == 0) s.n[buf][w] = mine;
    __syncthreads();
    int32_t all = 0;
#pragma unroll
    for (int y = 0; y < kChooseWaves; ++y) all += s.n[buf][y];
    buf ^= 1;
    if (all >= want) bound = x;
    just = all == want;
  }
  // `above` of them are past the bound (just: not below it), and the first of those at it make up the rest
  const uint32_t past = just ? bound : bound + 1u;  // (bound is no 0xffffffff unless just: it is below)
  const bool top = !just && bound == 0xffffffffu;   // (NaNs beyond the number wanted)
  int32_t above = want;
  if (!just) {
    int32_t mine = 0;
    for (int c = 0; c < chunks; ++c) {
      if (chunks > 1) load(c);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) mine += __builtin_popcountll(__ballot(!top && u[i] >= past));
    }
    if (lane == 0) s.n[buf][w] = mine;
    __syncthreads();
    above = 0;
#pragma unroll
    for (int y = 0; y < kChooseWaves; ++y) above += s.n[buf][y];
  }
  const int32_t at_bound = want - above;
  // ---- their ranks, in order of place: item, wave, lane ----
  uint64_t done = 0ull;  // of earlier chunks: past the bound, at it (high half)
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint64_t g = __ballot(!top && u[i] >= past), e = __ballot(!just && u[i] == bound);
      if (lane == 0)
        s.pre[i * kChooseWaves + w] = (uint64_t)__builtin_popcountll(g) | (uint64_t)__builtin_popcountll(e) << 32;
    }
    __syncthreads();
    // exclusive sums of ITEMS x waves entries, one a thread
    const uint64_t own = tid < ITEMS * kChooseWaves ? s.pre[tid] : 0ull;
    uint64_t in = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)in, o), hi = (uint32_t)__shfl_up((int)(in >> 32), o);
      if (lane >= o) in += (uint64_t)lo | (uint64_t)hi << 32;
    }
    if (lane == 63) s.wave[w] = in;
    __syncthreads();
    uint64_t base = done;
#pragma unroll
    for (int y = 0; y < kChooseWaves; ++y) {
      if (y < w) base += s.wave[y];
      done += s.wave[y];
    }
    if (tid < ITEMS * kChooseWaves) s.pre[tid] = base + in - own;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool gt = !top && u[i] >= past, eq = !just && u[i] == bound;
      const uint64_t g = __ballot(gt), e = __ballot(eq), below = (1ull << lane) - 1ull;
      const uint64_t p = s.pre[i * kChooseWaves + w];
      const int32_t gr = (int32_t)(uint32_t)p + (int32_t)__builtin_popcountll(g & below);
      const int32_t er = (int32_t)(p >> 32) + (int32_t)__builtin_popcountll(e & below);
      if (gt || (eq && er < at_bound)) kept[gr + imin(er, at_bound)] = first + c * SPAN + i * kChooseThreads + tid;
    }
  }
}

__global__ __launch_bounds__(kChooseThreads) void choose_kernel(const ChooseK a) {
  __shared__ ChooseShared s;
  const int tid = threadIdx.x;
  const int h = (int)(blockIdx.x % (unsigned)a.Hkv), lr = (int)(blockIdx.x / (unsigned)a.Hkv);
  const int r = lr % a.R, layer = lr / a.R;
  const Held q = held_of(a.pages, r);
  const int32_t m = q.len - q.first;
  int32_t* kept = a.kept + (((int64_t)layer * a.R + r) * a.Hkv + h) * a.keep;
  if (layer == 0 && h == 0 && tid == 0) a.after[r] = m > a.limit ? q.first + a.keep : a.pages.lengths[r];
  if (m <= a.limit) {
    for (int j = tid; j < a.keep; j += kChooseThreads) kept[j] = -1;
    return;
  }
  const int32_t want = a.keep - a.recent, n = m - a.recent;
  for (int j = tid; j < a.recent; j += kChooseThreads) kept[want + j] = q.len - a.recent + j;
  if (want == 0) return;
  const float* scores = a.scores + layer * a.s_sl + h * a.s_sh;
  const int32_t* table = a.pages.tables + r * a.pages.pitch;
  if (n <= 4 * kChooseThreads)
    choose_body<4>(a, scores, table, q.first, n, want, kept, s);
  else if (n <= 16 * kChooseThreads)
    choose_body<16>(a, scores, table, q.first, n, want, kept, s);
  else
    choose_body<32>(a, scores, table, q.first, n, want, kept, s);
}

// ---- their move -----------------------------------------------------------------------------------
constexpr int kEvictThreads = 256;

struct EvictK {
  const int32_t* kept;
  char* k;
  char* v;
  float* scores;
  int64_t c_sl, c_sp, c_sh, c_sn;  // bytes
  int64_t s_sl, s_sp, s_sh;        // floats
  Pages pages;
  int32_t R, Hkv, keep, row_lg;    // row_lg: log2 of the 16-byte units of a row
};

// Units of type U (1 << lg of them a row) of the kept rows of one head, in order.
template <typename U, int UNROLL, typename At>
__device__ __forceinline__ void move_rows(const EvictK& a, const int32_t* kept, const int32_t* table, const Held& q, int lg, At at) {
  const int tid = threadIdx.x;
  const int per = kEvictThreads >> lg;  // rows that one load of the work-group takes
  const int one = (1 << a.pages.page_lg) - 1;
  const int32_t reach = a.pages.cols << a.pages.page_lg;
  for (int j0 = 0; j0 < a.keep; j0 += per * UNROLL) {
    U x[UNROLL];
    U* to[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int j = j0 + i * per + (tid >> lg);
      to[i] = nullptr;
      x[i] = U{};
      if (j >= a.keep) continue;
      const int32_t of = kept[j], dst = q.first + j;
      if (of <= dst || of >= reach) continue;
      const int32_t p = checked_page(table[of >> a.pages.page_lg], a.pages.n_pages);
      const int32_t d = checked_page(table[dst >> a.pages.page_lg], a.pages.n_pages);
      if (p < 0 || d < 0) continue;
      to[i] = at(d, dst & one) + (tid & ((1 << lg) - 1));
      x[i] = *(at(p, of & one) + (tid & ((1 << lg) - 1)));
    }
    // (all of the batch has been read, by every wave, before any of it is written)
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) asm volatile("" ::"v"(x[i]));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
      if (to[i]) *to[i] = x[i];
  }
}

typedef uint32_t unit16 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kEvictThreads) void evict_kernel(const EvictK a) {
  const int h = (int)(blockIdx.x % (unsigned)a.Hkv), lr = (int)(blockIdx.x / (unsigned)a.Hkv);
  const int r = lr % a.R, layer = lr / a.R;
  const Held q = held_of(a.pages, r);
  const int32_t* kept = a.kept + (((int64_t)layer * a.R + r) * a.Hkv + h) * a.keep;
  const int32_t* table = a.pages.tables + r * a.pages.pitch;
  if (blockIdx.y < 2) {
    char* base = (blockIdx.y ? a.v : a.k) + layer * a.c_sl + h * a.c_sh;
    move_rows<unit16, 8>(a, kept, table, q, a.row_lg, [&](int32_t page, int32_t row) __attribute__((always_inline)) {
      return reinterpret_cast<unit16*>(base + page * a.c_sp + row * a.c_sn);
    });
  } else {
    float* base = a.scores + layer * a.s_sl + h * a.s_sh;
    move_rows<float, 8>(a, kept, table, q, 0, [&](int32_t page, int32_t row) __attribute__((always_inline)) {
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
                           {{"kept", kept}, {"after", flat(x->after, 4 * R)}}))
    return rc;
  PA_CHECK_ARG(!overlap(kept, scores) && !overlap(flat(x->after, 4 * R), scores), "pa_choose_keys: kept or after and scores overlap");
  a.scores = x->scores;
  a.s_sl = x->s_sl;
  a.s_sp = x->s_sp;
  a.s_sh = x->s_sh;
  a.R = x->R;
  a.Hkv = x->Hkv;
  a.keep = x->keep;
  a.recent = x->recent;
  a.limit = x->limit;
  a.kept = x->kept;
  a.after = x->after;
  hipLaunchKernelGGL(choose_kernel, dim3((unsigned)(x->layers * R * x->Hkv)), dim3(kChooseThreads), 0,
                     static_cast<hipStream_t>(stream), a);
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
  hipLaunchKernelGGL(evict_kernel, dim3((unsigned)(x->layers * R * x->Hkv), x->scores ? 3 : 2), dim3(kEvictThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  PA_LAUNCH_CHECK("evict_kernel");
  return PA_OK;
}
