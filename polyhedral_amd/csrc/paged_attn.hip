// Attention over a paged cache: the entry points' checks, the workspace and the choice of kernels.
#include <limits.h>
#include <math.h>

#include "page_spans.hpp"
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
  int64_t zero, bytes;
};

// A part whose requests have at most max_tiles tiles: its grid and slots.  (The shares of all tiles are
// at most `shares` and one more for each tile and KV head; a tile that is split has two shares at
// least, and then less than twice those that its blocks fill.  The work-groups without a unit each
// hold a place on a CU for 1.5 us; a grid without them, whose groups loop over units, costs more: 276
// -> 296 us of sinks in chunks, 15 -> 17 us of one token over 8000, by registers that the loop holds.)
int part_of(const pa_paged_args* x, int BM, int shares, int64_t max_tiles, PagedPart* p) {
  const int64_t most = shares + max_tiles * x->Hkv;
  PA_CHECK_ARG(most <= kMaxGroups, "pa_paged_attn: %lld work-groups exceed the grid limit", (long long)most);
  p->grid = (int32_t)most;
  p->slots = (int32_t)(2 * shares < most ? 2 * shares : most);
  p->by_shares = 1.0001f / (float)shares;
  const int G = x->Hq / x->Hkv;
  p->span = (BM + G - 1) / G + 1;
  return PA_OK;
}

int plan_of(const pa_paged_args* x, PagedPlan* p) {
  PA_CHECK_ARG(x, "pa_paged_attn: null arguments");
  if (int rc = check_pages("pa_paged_attn", x->n_pages, x->page_size, &p->page_lg)) return rc;
  PA_CHECK_ARG(x->dtype == PA_BF16 || x->dtype == PA_F16 || x->dtype == PA_F32, "pa_paged_attn: dtype %d", x->dtype);
  PA_CHECK_ARG(x->D == 64 || x->D == 128, "pa_paged_attn: D=%d (64 or 128)", x->D);
  PA_CHECK_ARG(x->Hkv >= 1 && x->Hq >= x->Hkv && x->Hq % x->Hkv == 0 && x->Hq <= 65535,
               "pa_paged_attn: %d query heads and %d KV heads (a multiple, at most 65535)", x->Hq, x->Hkv);
  PA_CHECK_ARG(x->R >= 0 && x->T >= 0 && x->T <= kMaxPosition && x->T * x->Hq <= kMaxPosition, "pa_paged_attn: R=%d T=%lld Hq=%d (T Hq < 2^30)",
               x->R, (long long)x->T, x->Hq);
  PA_CHECK_ARG(x->max_fresh >= 0, "pa_paged_attn: max_fresh=%lld", (long long)x->max_fresh);
  PA_CHECK_ARG(x->cols >= 0 && ((int64_t)x->cols << p->page_lg) <= kMaxPosition && x->pitch >= x->cols,
               "pa_paged_attn: %d columns of %d, pitch %lld", x->cols, x->page_size, (long long)x->pitch);
  PA_CHECK_ARG(!x->mask.perm_q && !x->mask.perm_kv, "pa_paged_attn: the mask takes no permutation tables");
  for (int i = 0; i < x->mask.n_include + x->mask.n_exclude && i < PA_MAX_TERMS; ++i)
    PA_CHECK_ARG(x->mask.terms[i].kind != PA_DENSE, "pa_paged_attn: PA_DENSE has no meaning here");
  if (int rc = check_mask(&x->mask, 0)) return rc;
  PA_CHECK_ARG(x->scale > 0.f && x->scale < INFINITY, "pa_paged_attn: scale=%g must be positive", (double)x->scale);
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
  // (beside chunks too: 61 requests of a token and 3 chunks with 256 shares 232 us, with 512 177, with 1024
  // 166; 36 requests of which most are chunks 53 with any)
  if (int rc = part_of(x, kRows, 1024, few, &p->rows)) return rc;
  p->rows.least = 4;
  p->rows.root_over = 0.7f;
  p->rows.row_min = 0;
  p->rows.row_max = p->tile ? (int32_t)few_rows : INT_MAX;
  p->tiles = PagedPart{};
  if (p->tile) {
    if (int rc = part_of(x, kTileRows, 512, x->T * G / kTileRows + some, &p->tiles)) return rc;
    p->tiles.least = 8;
    p->tiles.root_over = 1.f;
    p->tiles.row_min = (int32_t)few_rows;
    p->tiles.row_max = INT_MAX;
  }
  PA_CHECK_ARG((int64_t)p->rows.grid + p->tiles.grid <= kMaxGroups, "pa_paged_attn: %lld work-groups exceed the grid limit",
               (long long)p->rows.grid + p->tiles.grid);
  p->zero = (4 * ((int64_t)p->rows.slots + p->tiles.slots) + 255) / 256 * 256;
  p->bytes = p->zero + 4ll * p->rows.slots * slot_floats(kRows, x->D) + 4ll * p->tiles.slots * slot_floats(kTileRows, x->D);
  return PA_OK;
}

// Work-groups write o, lse and the workspace while others read the inputs: no two of them, and no two
// rows of o or lse, share a byte.  (Heads of one buffer may be q and o in turn.)
int check_overlaps(const pa_paged_args* x, int esz, int64_t workspace) {
  const int64_t row = x->D * esz;
  const Strided<2> o = strided<2>(x->o, row, {x->T, x->Hq}, {x->o_st, x->o_sh}, esz);
  const Strided<2> q = strided<2>(x->q, row, {x->T, x->Hq}, {x->q_st, x->q_sh}, esz);
  const Strided<2> lse = strided<2>(x->lse, 4, {x->lse ? x->T : 0, x->Hq}, {x->lse_st, x->lse_sh}, 4);
  PA_CHECK_ARG(!overlaps_itself(o), "pa_paged_attn: rows of o overlap");
  PA_CHECK_ARG(!overlaps_itself(lse), "pa_paged_attn: rows of lse overlap");
  const int64_t pages[] = {x->n_pages, x->Hkv, x->page_size}, steps[] = {x->c_sp, x->c_sh, x->c_sn};
  const Strided<3> k = strided<3>(x->k, row, pages, steps, esz), v = strided<3>(x->v, row, pages, steps, esz);
  const Strided<1> tables = strided<1>(x->tables, 4ll * x->cols, {x->cols ? x->R : 0}, {x->pitch}, 4);
  const Strided<1> lengths = flat(x->lengths, 4ll * x->R), starts = flat(x->q_start, 4ll * (x->R + 1ll));
  const Strided<1> ws = flat(x->workspace, workspace);
  auto apart = [&](const char* name, const auto& out) {
    const char* other = overlap(out, q) ? "q" : overlap(out, k) ? "k" : overlap(out, v) ? "v" : overlap(out, tables) ? "tables"
                        : overlap(out, lengths) ? "lengths" : overlap(out, starts) ? "q_start" : nullptr;
    PA_CHECK_ARG(!other, "pa_paged_attn: %s and %s overlap", name, other);
    return (int)PA_OK;
  };
  if (int rc = apart("o", o)) return rc;
  if (int rc = apart("lse", lse)) return rc;
  if (int rc = apart("workspace", ws)) return rc;
  PA_CHECK_ARG(!overlap(o, lse), "pa_paged_attn: o and lse overlap");
  PA_CHECK_ARG(!overlap(ws, o), "pa_paged_attn: workspace and o overlap");
  PA_CHECK_ARG(!overlap(ws, lse), "pa_paged_attn: workspace and lse overlap");
  return PA_OK;
}

}  // namespace
}  // namespace pa

extern "C" int pa_paged_workspace(const pa_paged_args* x, int64_t* bytes, int64_t* zero) {
  pa::PagedPlan p;
  if (int rc = pa::plan_of(x, &p)) return rc;
  PA_CHECK_ARG(bytes && zero, "pa_paged_workspace: null output");
  *bytes = p.bytes;
  *zero = p.zero;
  return PA_OK;
}

extern "C" int pa_paged_attn(const pa_paged_args* x, void* stream) {
  using namespace pa;
  PagedPlan p;
  if (int rc = plan_of(x, &p)) return rc;
  if (x->R == 0 || x->T == 0) return PA_OK;
  PA_CHECK_ARG(x->q && x->o && x->lengths && x->q_start, "pa_paged_attn: null q / o / lengths / q_start");
  PA_CHECK_ARG(x->cols == 0 || x->tables, "pa_paged_attn: null tables");
  PA_CHECK_ARG(x->n_pages == 0 || (x->k && x->v), "pa_paged_attn: null k / v");
  const int64_t esz = x->dtype == PA_F32 ? 4 : 2;
  auto al = [&](const void* q, int64_t s0, int64_t s1, int64_t s2) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (s0 * esz) % 16 == 0 && (s1 * esz) % 16 == 0 && (s2 * esz) % 16 == 0;
  };
  PA_CHECK_ARG(al(x->q, x->q_st, x->q_sh, 0) && al(x->o, x->o_st, x->o_sh, 0) && al(x->k, x->c_sp, x->c_sh, x->c_sn) &&
                   al(x->v, x->c_sp, x->c_sh, x->c_sn),
               "pa_paged_attn: rows must be 16-byte aligned");
  PA_CHECK_ARG(x->q_st >= 0 && x->q_sh >= 0 && x->o_st >= 0 && x->o_sh >= 0 && x->c_sp >= 0 && x->c_sh >= 0 &&
                   x->c_sn >= x->D && x->c_sn <= (1 << 21),
               "pa_paged_attn: negative strides, or cache rows closer than D or further than 2^21");
  PA_CHECK_ARG(x->workspace && reinterpret_cast<uintptr_t>(x->workspace) % 256 == 0 && x->workspace_bytes >= p.bytes,
               "pa_paged_attn: needs a 256-byte aligned workspace of %lld bytes", (long long)p.bytes);
  if (int rc = check_overlaps(x, (int)esz, p.bytes)) return rc;
  PagedK a;
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
  if (x->dtype == PA_F32) return launch_paged_f32(a, x->D, s);
  return x->dtype == PA_BF16 ? launch_paged_bf16(a, x->D, s) : launch_paged_f16(a, x->D, s);
}
