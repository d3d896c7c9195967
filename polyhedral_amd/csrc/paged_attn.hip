// Attention over a paged cache: the entry points' checks, the workspace and the choice of kernels.
#include <limits.h>
#include <math.h>

#include "page_checks.hpp"
#include "paged_attn.hpp"

namespace pa {
namespace {

// Rows of a request (new tokens times heads of a group) up to which it is a tile of few rows.  Over
// 4000 keys of 8 heads of 128, as tiles of 16 and as one of 128: 24 rows 23 and 28 us of 4 requests (204
// and 200 of 64), 48 rows 28 and 31 (273 and 203), 64 rows 32 and 31 (330 and 210).
constexpr int kFewRows = 32;

// Work-groups of a launch: a grid of 256 threads each has less than 2^32 of them.
constexpr int64_t kMaxGroups = 0xffffffffll / 256;

// One in how many keys a mask leaves live for a token far from it: the stride of a mask's one lattice
// when its other terms are bands (windows, sinks); 0 for any other mask.
int stride_of(const pa_mask& m) {
  int stride = 0;
  for (int i = 0; i < m.n_include; ++i) {
    const pa_term& t = m.terms[i];
    if (t.kind == PA_WINDOW || t.kind == PA_SINKS || t.kind == PA_TWOBAND) continue;
    if ((t.kind != PA_DILATED && t.kind != PA_LOCAL_STRIDED) || stride) return 0;
    stride = t.kind == PA_DILATED ? t.p0 : t.p1;
  }
  return stride;
}

// Workspace: the counts of both parts, then their slots.
struct PagedPlan {
  int page_lg;
  bool tile;            // some request may have more rows than a tile of few rows takes
  int stride;
  PagedPart rows, tiles;
  PagedPart pre_rows, pre_tiles;  // of the prefixes that requests share
  int64_t zero, bytes;
  int64_t states, own, at, end;   // where the states of their shares begin, those of own keys, their places, and the last row's
};

// A part whose requests have at most max_tiles tiles: its grid and slots.  (The shares of all tiles are
// at most `shares` and one more for each tile and KV head; a tile that is split has two shares at
// least, and then less than twice those that its blocks fill.  The work-groups without a unit each
// hold a place on a CU for 1.5 us; a grid without them, whose groups loop over units, costs more: 276
// -> 296 us of sinks in chunks, 15 -> 17 us of one token over 8000, by registers that the loop holds.)
// blocks: the most that all its requests have, where the grid goes by that too (-1: not).
int part_of(const char* who, const pa_paged_args* x, int BM, int shares, int32_t least, int64_t max_tiles, int64_t blocks, PagedPart* p) {
  p->by_shares = 1.0001f / (float)shares;
  if (blocks >= 0 && blocks / least < shares) shares = (int)(blocks / least);
  const int64_t most = shares + max_tiles * x->Hkv;
  PA_CHECK_ARG(most <= kMaxGroups, "%s: %lld work-groups exceed the grid limit", who, (long long)most);
  p->grid = (int32_t)most;
  p->slots = (int32_t)(2 * shares < most ? 2 * shares : most);
  p->least = least;
  const int G = x->Hq / x->Hkv;
  p->span = (BM + G - 1) / G + 1;
  return PA_OK;
}

int plan_of(const char* who, const pa_paged_args* x, bool sharing, PagedPlan* p) {
  PA_CHECK_ARG(x, "%s: null arguments", who);
  if (int rc = check_pages(who, x->n_pages, x->page_size, &p->page_lg)) return rc;
  PA_CHECK_ARG(x->dtype == PA_BF16 || x->dtype == PA_F16 || x->dtype == PA_F32, "%s: dtype %d", who, x->dtype);
  PA_CHECK_ARG(x->D == 64 || x->D == 128, "%s: D=%d (64 or 128)", who, x->D);
  PA_CHECK_ARG(x->Hkv >= 1 && x->Hq >= x->Hkv && x->Hq % x->Hkv == 0 && x->Hq <= 65535,
               "%s: %d query heads and %d KV heads (a multiple, at most 65535)", who, x->Hq, x->Hkv);
  PA_CHECK_ARG(x->R >= 0 && x->T >= 0 && x->T <= kMaxPosition && x->T * x->Hq <= kMaxPosition, "%s: R=%d T=%lld Hq=%d (T Hq < 2^30)", who,
               x->R, (long long)x->T, x->Hq);
  PA_CHECK_ARG(x->max_fresh >= 0, "%s: max_fresh=%lld", who, (long long)x->max_fresh);
  PA_CHECK_ARG(x->cols >= 0 && ((int64_t)x->cols << p->page_lg) <= kMaxPosition && x->pitch >= x->cols,
               "%s: %d columns of %d, pitch %lld", who, x->cols, x->page_size, (long long)x->pitch);
  PA_CHECK_ARG(!x->mask.perm_q && !x->mask.perm_kv, "%s: the mask takes no permutation tables", who);
  for (int i = 0; i < x->mask.n_include + x->mask.n_exclude && i < PA_MAX_TERMS; ++i)
    PA_CHECK_ARG(x->mask.terms[i].kind != PA_DENSE, "%s: PA_DENSE has no meaning here", who);
  if (int rc = check_mask(&x->mask, 0)) return rc;
  PA_CHECK_ARG(x->scale > 0.f && x->scale < INFINITY, "%s: scale=%g must be positive", who, (double)x->scale);
  p->stride = stride_of(x->mask);
  const int64_t G = x->Hq / x->Hkv, some = x->T < x->R ? x->T : x->R;  // some: requests with rows, at most
  // (Tiles of few rows that take lists read 1 / stride of the keys for each token, a chunk's tile all: 64
  // rows of 16 requests, stride 16, over 8000 keys 74 us and 141, 96 rows 146 both.)
  const int span = (int)((kRows + G - 1) / G) + 1;
  const int64_t few_rows = 2 * span <= p->stride && G * p->stride / 2 > kFewRows ? (G * p->stride / 2 < kTileRows ? G * p->stride / 2 : kTileRows) : kFewRows;
  const int64_t most = x->max_fresh < x->T ? x->max_fresh : x->T;  // new tokens of a request
  p->tile = x->dtype != PA_F32 && x->n_pages > 0 && most * G > few_rows;
  int64_t few = x->T * G / kRows + some;
  if (p->tile && few > some * ((few_rows + kRows - 1) / kRows)) few = some * ((few_rows + kRows - 1) / kRows);
  // (a call that shares: the tables' reach in blocks of 16 or 32 keys, for each tile of few rows)
  const int64_t row_blocks = sharing ? few * x->Hkv * (((int64_t)x->cols << p->page_lg) / (x->dtype == PA_F32 ? 16 : 32) + 1) : -1;
  // (beside chunks too: 61 requests of a token and 3 chunks with 256 shares 232 us, with 512 177, with 1024
  // 166; 36 requests of which most are chunks 53 with any)
  if (int rc = part_of(who, x, kRows, 1024, 4, few, row_blocks, &p->rows)) return rc;
  p->rows.root_over = 0.7f;
  p->rows.row_min = 0;
  p->rows.row_max = p->tile ? (int32_t)few_rows : INT_MAX;
  p->tiles = PagedPart{};
  if (p->tile) {
    if (int rc = part_of(who, x, kTileRows, 512, 8, x->T * G / kTileRows + some, -1, &p->tiles)) return rc;
    p->tiles.root_over = 1.f;
    p->tiles.row_min = (int32_t)few_rows;
    p->tiles.row_max = INT_MAX;
  }
  PA_CHECK_ARG((int64_t)p->rows.grid + p->tiles.grid <= kMaxGroups, "%s: %lld work-groups exceed the grid limit", who,
               (long long)p->rows.grid + p->tiles.grid);
  p->pre_rows = p->pre_tiles = PagedPart{};
  if (sharing && some > 1) {
    // (a group is two requests or more, so its rows may be many where each request's are few)
    const bool tile = x->dtype != PA_F32 && x->n_pages > 0 && x->T * G > kFewRows;
    const int64_t groups = some / 2;
    few = x->T * G / kRows + groups;
    if (tile && few > groups * (kFewRows / kRows)) few = groups * (kFewRows / kRows);
    // (beside tiles fewer shares, as its work-groups are mostly without work: 64 requests behind 8192 tokens 64 us
    // with 1024, 61 with 256)
    if (int rc = part_of(who, x, kRows, tile ? 256 : 1024, 4, few, row_blocks, &p->pre_rows)) return rc;
    p->pre_rows.root_over = 0.7f;
    p->pre_rows.row_max = tile ? kFewRows : INT_MAX;
    if (tile) {
      if (int rc = part_of(who, x, kTileRows, 512, 8, x->T * G / kTileRows + groups, -1, &p->pre_tiles)) return rc;
      p->pre_tiles.root_over = 1.f;
      p->pre_tiles.row_min = kFewRows;
      p->pre_tiles.row_max = INT_MAX;
    }
    PA_CHECK_ARG((int64_t)p->pre_rows.grid + p->pre_tiles.grid + p->rows.grid + p->tiles.grid <= kMaxGroups,
                 "%s: %lld work-groups exceed the grid limit", who,
                 (long long)p->pre_rows.grid + p->pre_tiles.grid + p->rows.grid + p->tiles.grid);
    // every unit over a prefix has a slot
    p->pre_rows.slots = p->pre_rows.grid;
    p->pre_tiles.slots = p->pre_tiles.grid;
  }
  p->zero = (4 * ((int64_t)p->rows.slots + p->tiles.slots) + 255) / 256 * 256;
  p->states = p->zero + 4ll * p->rows.slots * slot_floats(kRows, x->D) + 4ll * p->tiles.slots * slot_floats(kTileRows, x->D);
  const int64_t state = 4 * state_floats(x->D), rows = sharing ? x->T * x->Hq : 0;
  p->own = p->states + state * ((int64_t)p->pre_rows.slots * kRows + (int64_t)p->pre_tiles.slots * kTileRows);
  p->at = p->own + state * rows;
  p->end = p->at + (int64_t)sizeof(StatesAt) * rows;
  p->bytes = p->end + (sharing ? 16 : 0);
  PA_CHECK_ARG(p->own - p->states < (1ll << 36) && rows * (x->D / 4) <= kMaxGroups * 256,
               "%s: %lld rows leave too many states (%lld bytes)", who, (long long)rows, (long long)(p->own - p->states));
  return PA_OK;
}

// Work-groups write o, lse and the workspace while others read the inputs: no two of them, and no two
// rows of o or lse, share a byte.  (Heads of one buffer may be q and o in turn.)
int check_overlaps(const char* who, const pa_paged_args* x, const pa_sharing* share, int esz, int64_t workspace) {
  const int64_t row = x->D * esz;
  const Strided<2> o = strided<2>(x->o, row, {x->T, x->Hq}, {x->o_st, x->o_sh}, esz);
  const Strided<2> q = strided<2>(x->q, row, {x->T, x->Hq}, {x->q_st, x->q_sh}, esz);
  const Strided<2> lse = strided<2>(x->lse, 4, {x->lse ? x->T : 0, x->Hq}, {x->lse_st, x->lse_sh}, 4);
  PA_CHECK_ARG(!overlaps_itself(o), "%s: rows of o overlap", who);
  PA_CHECK_ARG(!overlaps_itself(lse), "%s: rows of lse overlap", who);
  const int64_t pages[] = {x->n_pages, x->Hkv, x->page_size}, steps[] = {x->c_sp, x->c_sh, x->c_sn};
  const Strided<3> k = strided<3>(x->k, row, pages, steps, esz), v = strided<3>(x->v, row, pages, steps, esz);
  const Strided<1> tables = strided<1>(x->tables, 4ll * x->cols, {x->cols ? x->R : 0}, {x->pitch}, 4);
  const Strided<1> lengths = flat(x->lengths, 4ll * x->R), starts = flat(x->q_start, 4ll * (x->R + 1ll));
  const Strided<1> ws = flat(x->workspace, workspace);
  auto apart = [&](const char* name, const auto& out) {
    const char* other = overlap(out, q) ? "q" : overlap(out, k) ? "k" : overlap(out, v) ? "v" : overlap(out, tables) ? "tables"
                        : overlap(out, lengths) ? "lengths" : overlap(out, starts) ? "q_start" : nullptr;
    if (share && !other) {
      const int64_t R = x->R, n[] = {R + 1, x->T, x->T, R, R, R, R};
      const int32_t* at[] = {share->start, share->rows, share->positions, share->prefix, share->low, share->high, share->first};
      for (int i = 0; i < 7; ++i)
        if (overlap(out, flat(at[i], 4 * n[i]))) other = "sharing";
    }
    PA_CHECK_ARG(!other, "%s: %s and %s overlap", who, name, other);
    return (int)PA_OK;
  };
  if (int rc = apart("o", o)) return rc;
  if (int rc = apart("lse", lse)) return rc;
  if (int rc = apart("workspace", ws)) return rc;
  PA_CHECK_ARG(!overlap(o, lse), "%s: o and lse overlap", who);
  PA_CHECK_ARG(!overlap(ws, o), "%s: workspace and o overlap", who);
  PA_CHECK_ARG(!overlap(ws, lse), "%s: workspace and lse overlap", who);
  return PA_OK;
}

int workspace_of(const char* who, const pa_paged_args* x, bool sharing, int64_t* bytes, int64_t* zero) {
  PagedPlan p;
  if (int rc = plan_of(who, x, sharing, &p)) return rc;
  PA_CHECK_ARG(bytes && zero, "%s: null output", who);
  *bytes = p.bytes;
  *zero = p.zero;
  return PA_OK;
}

int run_paged(const char* who, const pa_paged_args* x, const pa_sharing* share, void* stream) {
  PagedPlan p;
  if (int rc = plan_of(who, x, share != nullptr, &p)) return rc;
  if (x->R == 0 || x->T == 0) return PA_OK;
  PA_CHECK_ARG(x->q && x->o && x->lengths && x->q_start, "%s: null q / o / lengths / q_start", who);
  PA_CHECK_ARG(!share || (share->start && share->rows && share->positions && share->prefix && share->low && share->high && share->first),
               "%s: null sharing", who);
  PA_CHECK_ARG(x->cols == 0 || x->tables, "%s: null tables", who);
  PA_CHECK_ARG(x->n_pages == 0 || (x->k && x->v), "%s: null k / v", who);
  const int64_t esz = x->dtype == PA_F32 ? 4 : 2;
  auto al = [&](const void* q, int64_t s0, int64_t s1, int64_t s2) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (s0 * esz) % 16 == 0 && (s1 * esz) % 16 == 0 && (s2 * esz) % 16 == 0;
  };
  PA_CHECK_ARG(al(x->q, x->q_st, x->q_sh, 0) && al(x->o, x->o_st, x->o_sh, 0) && al(x->k, x->c_sp, x->c_sh, x->c_sn) &&
                   al(x->v, x->c_sp, x->c_sh, x->c_sn),
               "%s: rows must be 16-byte aligned", who);
  PA_CHECK_ARG(x->q_st >= 0 && x->q_sh >= 0 && x->o_st >= 0 && x->o_sh >= 0 && x->c_sp >= 0 && x->c_sh >= 0 &&
                   x->c_sn >= x->D && x->c_sn <= (1 << 21),
               "%s: negative strides, or cache rows closer than D or further than 2^21", who);
  PA_CHECK_ARG(x->workspace && reinterpret_cast<uintptr_t>(x->workspace) % 256 == 0 && x->workspace_bytes >= p.bytes,
               "%s: needs a 256-byte aligned workspace of %lld bytes", who, (long long)p.bytes);
  if (int rc = check_overlaps(who, x, share, (int)esz, p.bytes)) return rc;
  PagedK a{};
  a.q = static_cast<const char*>(x->q);
  a.q_st = x->q_st * esz;
  a.q_sh = x->q_sh * esz;
  a.k = static_cast<const char*>(x->k);
  a.v = static_cast<const char*>(x->v);
  a.c_sp = x->c_sp * esz;
  a.c_sh = x->c_sh * esz;
  a.c_sn = x->c_sn * esz;
  a.n_pages = x->n_pages;
  a.page_lg = p.page_lg;
  a.cols = x->cols;
  a.tables = x->tables;
  a.pitch = x->pitch;
  a.lengths = x->lengths;
  a.q_start = x->q_start;
  a.R = x->R;
  a.T = (int32_t)x->T;
  a.Hkv = x->Hkv;
  a.G = x->Hq / x->Hkv;
  a.by_G = divisor_of((uint32_t)a.G);
  a.by_Hkv = divisor_of((uint32_t)a.Hkv);
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
  // (rows of 64 keys at 5 TB/s against a step's 1.9 us on 512 places, less a tenth)
  a.few_weight = x->D == 128 ? 1.6f : 0.8f;
  a.stride = p.stride;
  a.o = static_cast<char*>(x->o);
  a.o_st = x->o_st * esz;
  a.o_sh = x->o_sh * esz;
  a.lse = x->lse;
  a.lse_st = x->lse_st;
  a.lse_sh = x->lse_sh;
  a.tiles = p.tiles;
  a.rows = p.rows;
  char* ws = static_cast<char*>(x->workspace);
  a.rows.count = reinterpret_cast<int32_t*>(ws);
  a.tiles.count = a.rows.count + p.rows.slots;
  a.rows.part = ws + p.zero;
  a.tiles.part = a.rows.part + 4ll * p.rows.slots * slot_floats(kRows, x->D);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (share && p.pre_rows.grid) {
    a.share = *share;
    a.pre_rows = p.pre_rows;
    a.pre_tiles = p.pre_tiles;
    a.states = reinterpret_cast<float*>(ws + p.states);
    a.n_states = (p.own - p.states) / 4;
    a.pre_rows.part = ws + p.states;
    a.pre_tiles.part = a.pre_rows.part + 4ll * p.pre_rows.slots * kRows * state_floats(x->D);
    a.own = reinterpret_cast<float*>(ws + p.own);
    a.at = reinterpret_cast<StatesAt*>(ws + p.at);
    a.end = reinterpret_cast<int32_t*>(ws + p.end);
    if (x->dtype == PA_F32) return launch_shared_f32(a, x->D, s);
    return x->dtype == PA_BF16 ? launch_shared_bf16(a, x->D, s) : launch_shared_f16(a, x->D, s);
  }
  if (x->dtype == PA_F32) return launch_paged_f32(a, x->D, s);
  return x->dtype == PA_BF16 ? launch_paged_bf16(a, x->D, s) : launch_paged_f16(a, x->D, s);
}

}  // namespace
}  // namespace pa

extern "C" int pa_paged_workspace(const pa_paged_args* x, int64_t* bytes, int64_t* zero) {
  return pa::workspace_of("pa_paged_attn", x, false, bytes, zero);
}

extern "C" int pa_paged_attn(const pa_paged_args* x, void* stream) { return pa::run_paged("pa_paged_attn", x, nullptr, stream); }

extern "C" int pa_shared_workspace(const pa_paged_args* x, int64_t* bytes, int64_t* zero) {
  return pa::workspace_of("pa_shared_attn", x, true, bytes, zero);
}

extern "C" int pa_shared_attn(const pa_paged_args* x, const pa_sharing* sharing, void* stream) {
  PA_CHECK_ARG(sharing, "pa_shared_attn: null sharing");
  return pa::run_paged("pa_shared_attn", x, sharing, stream);
}
