// The paged cache's tables, its free list and the write of new keys and values (gfx950).
//
// pa_page_tables: with first[r] = ceil(before[r] / ps) and need[r] = ceil((before[r] +
// fresh[r]) / ps) - first[r], the exclusive sums of fresh give the rows of each request, those
// of need its place in the run of free pages that is taken, and then every token's slot and every
// new table entry follow from one binary search each.  A work-group takes all the sums and holds
// them in LDS; where there are many tokens, many work-groups do, and each writes its part of the
// tokens and pages (the sums of 96 requests again cost less than a second launch).  Where the state
// advances in place, which the other work-groups may still read, or the sums pass the LDS, one
// work-group writes sums and state, and a second kernel the tokens and pages.
// What bounds it: latency (three trips to memory one after the other, and the launch): 256 requests of
// a token each 5.0 us, 96 with 78000 tokens 5.3 (in two launches 8.4).
#include <string.h>

#include <initializer_list>

#include "common.hpp"
#include "page_math.hpp"
#include "page_spans.hpp"

namespace pa {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanRequests = 2048;  // requests whose sums fit the scan's LDS

struct TablesK {
  const int32_t* before;
  const int32_t* fresh;
  const int32_t* free_list;
  const int32_t* free_count;
  int32_t* tables;
  int64_t pitch, n_pages;
  int32_t R, page_lg, cols, tokens;
  int32_t* lengths;
  int32_t* q_start;
  int32_t* slots;
  int32_t* positions;
  int32_t* free_left;
  int32_t* status;
  // workspace: tokens before each request's (R + 1), new pages before each request's (R + 1;
  // the last entry is the count of the pages taken), tokens cached before (R)
  int32_t* row0;
  int32_t* page0;
  int32_t* held;
};

// What a thread needs to write one token or one new page: the sums, from LDS or memory.
struct TablesView {
  const int32_t* row0;
  const int32_t* page0;
  const int32_t* held;
};

// Largest r with start[r] <= x (start ascending, start[0] = 0 <= x; empty requests are passed).
__device__ __forceinline__ int request_at(const int32_t* start, int R, int x) {
  int lo = 0, hi = R;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Item i of the step's tokens (first `tokens` items) and new pages.
__device__ __forceinline__ void write_item(const TablesK& a, const TablesView& v, int64_t i, int64_t taken, int32_t top) {
  const int one = (1 << a.page_lg) - 1;
  if (i < a.tokens) {
    int32_t slot = -1, pos = -1;
    if (i < v.row0[a.R]) {
      const int r = request_at(v.row0, a.R, (int)i);
      pos = v.held[r] + (int32_t)i - v.row0[r];
      const int32_t col = pos >> a.page_lg, first = (v.held[r] + one) >> a.page_lg;
      const int32_t page = col < first ? a.tables[(int64_t)r * a.pitch + col]
                                       : a.free_list[top - 1 - (v.page0[r] + col - first)];
      slot = slot_of(page, pos, a.page_lg, a.n_pages);
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = pos;
  } else if (i - a.tokens < taken) {
    const int32_t j = (int32_t)(i - a.tokens);
    const int r = request_at(v.page0, a.R, j);
    const int32_t col = ((v.held[r] + one) >> a.page_lg) + j - v.page0[r];
    a.tables[(int64_t)r * a.pitch + col] = a.free_list[top - 1 - j];
  }
}

__device__ __forceinline__ int64_t shfl_up64(int64_t x, int o) {
  const int lo = __shfl_up((int)(uint32_t)x, o), hi = __shfl_up((int)(x >> 32), o);
  return (int64_t)((uint64_t)(uint32_t)lo | ((uint64_t)(uint32_t)hi << 32));
}

// The sums; FUSED: the tokens and pages too (R <= kScanRequests; one work-group alone where the state
// advances in place).
template <bool FUSED>
__global__ __launch_bounds__(kScanThreads) void tables_scan_kernel(const TablesK a) {
  constexpr int NW = kScanThreads / 64;
  __shared__ int64_t wave_t[NW], wave_p[NW];
  __shared__ int32_t bad_s;
  __shared__ int32_t sums[FUSED ? 3 * kScanRequests + 2 : 1];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int one = (1 << a.page_lg) - 1;
  const int32_t top = *a.free_count;  // (first, beside the other loads)
  const int64_t max_len = (int64_t)a.cols << a.page_lg;
  int32_t* row0 = FUSED ? sums : a.row0;
  int32_t* page0 = FUSED ? sums + a.R + 1 : a.page0;
  int32_t* held = FUSED ? sums + 2 * a.R + 2 : a.held;
  if (tid == 0) bad_s = 0;
  __syncthreads();

  int64_t t_sum = 0, p_sum = 0;  // of the requests before this pass's (the same in every thread)
  int32_t bad = 0;
  for (int r0 = 0; r0 < a.R; r0 += kScanThreads) {
    const int r = r0 + tid;
    int64_t t = 0, p = 0;
    int32_t b = 0;
    if (r < a.R) {
      b = a.before[r];
      const int32_t f = a.fresh[r];
      if (b < 0 || f < 0 || (int64_t)b + f > max_len) {
        bad |= 2;
        b = 0;
      } else {
        t = f;
        p = ((b + f + one) >> a.page_lg) - ((b + one) >> a.page_lg);
      }
    }
    int64_t ti = t, pi = p;  // inclusive sums of the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t tu = shfl_up64(ti, o), pu = shfl_up64(pi, o);
      if (lane >= o) {
        ti += tu;
        pi += pu;
      }
    }
    if (lane == 63) {
      wave_t[w] = ti;
      wave_p[w] = pi;
    }
    __syncthreads();
    int64_t t_at = t_sum, p_at = p_sum;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      if (x < w) {
        t_at += wave_t[x];
        p_at += wave_p[x];
      }
      t_sum += wave_t[x];
      p_sum += wave_p[x];
    }
    if (r < a.R) {
      // (a sum past the limits is an error below, and is not used)
      row0[r] = (int32_t)(t_at + ti - t);
      page0[r] = (int32_t)(p_at + pi - p);
      held[r] = b;
    }
    __syncthreads();
  }
  if (t_sum > a.tokens) bad |= 4;
  if (top < 0 || top > a.n_pages || p_sum > top) bad |= 1;
  if (bad) atomicOr(&bad_s, bad);
  __syncthreads();
  bad = bad_s;
  if (bad) t_sum = p_sum = 0;
  if (tid == 0) {
    row0[a.R] = (int32_t)t_sum;
    page0[a.R] = (int32_t)p_sum;
    if (blockIdx.x == 0) {
      *a.status = bad;
      *a.free_left = top - (int32_t)p_sum;
      a.q_start[a.R] = (int32_t)t_sum;
    }
  }
  if (blockIdx.x == 0)
    for (int r = tid; r < a.R; r += kScanThreads) {
      a.lengths[r] = bad ? a.before[r] : a.before[r] + a.fresh[r];
      a.q_start[r] = bad ? 0 : row0[r];
    }
  if constexpr (FUSED) {
    __syncthreads();  // the last entries
    const TablesView v{row0, page0, held};
    for (int64_t i = (int64_t)blockIdx.x * kScanThreads + tid; i < a.tokens + p_sum; i += (int64_t)gridDim.x * kScanThreads)
      write_item(a, v, i, p_sum, top);
  }
}

// (free_left may be free_count itself: the pages that were free are those left and those taken)
__global__ __launch_bounds__(256) void tables_fill_kernel(const TablesK a) {
  const int64_t taken = a.page0[a.R];
  const int32_t top = *a.free_left + (int32_t)taken;
  const TablesView v{a.row0, a.page0, a.held};
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.tokens + taken; i += (int64_t)gridDim.x * 256)
    write_item(a, v, i, taken, top);
}

// One work-group, a wave per request in turn: count, sum, write.  Its work is the columns of the ranges,
// whether they hold pages or not, each read twice, 64 at a time with one trip to memory after the other:
// the whole row of a finished request, and where a window leaves pages behind, all columns between the
// sinks and the window at every call, so it grows with the lengths.  8 of 64 requests of 32768 tokens
// finished in pages of 64 take 13 us; a page each of 128 such requests 30 us, in pages of 16 92 us (of 4096
// tokens 16 us), and as long where no page goes back.
__global__ __launch_bounds__(kScanThreads) void release_kernel(const int32_t* first, const int32_t* last, int32_t R,
                                                               int32_t* tables, int64_t pitch, int32_t cols,
                                                               int32_t* free_list, const int32_t* free_count,
                                                               int64_t n_pages, int32_t* free_left, int32_t* status,
                                                               int32_t* counts) {
  constexpr int NW = kScanThreads / 64;
  __shared__ int64_t wave_n[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto valid = [&](int64_t at) { return checked_page(tables[at], n_pages) >= 0; };
  for (int r = w; r < R; r += NW) {
    const int32_t lo = imax(first[r], 0), hi = imin(last[r], cols);
    int n = 0;
    for (int c = lo; c < hi; c += 64)
      n += (int)__builtin_popcountll(__ballot(c + lane < hi && valid((int64_t)r * pitch + c + lane)));
    if (lane == 0) counts[r] = n;
  }
  __syncthreads();
  // exclusive sums, in place
  int64_t total = 0;
  for (int r0 = 0; r0 < R; r0 += kScanThreads) {
    const int r = r0 + tid;
    const int64_t n = r < R ? counts[r] : 0;
    int64_t in = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t up = shfl_up64(in, o);
      if (lane >= o) in += up;
    }
    if (lane == 63) wave_n[tid >> 6] = in;
    __syncthreads();
    int64_t at = total;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      if (x < (tid >> 6)) at += wave_n[x];
      total += wave_n[x];
    }
    if (r < R) counts[r] = (int32_t)(at + in - n);
    __syncthreads();
  }
  const int32_t top = *free_count;
  const bool bad = top < 0 || top + total > n_pages;
  __syncthreads();  // every thread has the old count
  if (tid == 0) {
    *status = bad ? 1 : 0;
    *free_left = bad ? top : top + (int32_t)total;
  }
  if (bad) return;
  for (int r = w; r < R; r += NW) {
    const int32_t lo = imax(first[r], 0), hi = imin(last[r], cols);
    int64_t at = top + counts[r];
    for (int c = lo; c < hi; c += 64) {
      const int64_t e = (int64_t)r * pitch + c + lane;
      const bool in = c + lane < hi && valid(e);
      const uint64_t all = __ballot(in);
      if (in) {
        const int before = (int)__builtin_popcountll(all & ((1ull << lane) - 1ull));
        free_list[at + before] = tables[e];
        tables[e] = -1;
      }
      at += (int64_t)__builtin_popcountll(all);
    }
  }
}

// A thread per 16-byte unit of the tokens' K and V rows: units of a row, then heads, then tokens,
// so a wave reads whole rows; what bounds it is HBM (the rows read and written once: 21000 tokens of 8
// heads of 128 bytes, 87 MB, 15 to 17 us, 5.2 to 5.9 TB/s, where a copy of 2 GiB reaches 5.0).  A few
// tokens: the launch and two trips to memory (256 tokens 5.5 us).
template <typename Index>
__global__ __launch_bounds__(256) void append_kernel(const char* k_new, const char* v_new, int64_t n_st, int64_t n_sh,
                                                     const int32_t* slots, Index units, char* k, char* v,
                                                     int64_t c_sp, int64_t c_sh, int64_t c_sn, uint32_t n_slots,
                                                     int32_t page_lg, int32_t upr_lg, uint32_t Hkv) {
  const char* src = blockIdx.y ? v_new : k_new;
  char* dst = blockIdx.y ? v : k;
  const int32_t one = (1 << page_lg) - 1;
  for (Index i = (Index)blockIdx.x * 256 + threadIdx.x; i < units; i += (Index)gridDim.x * 256) {
    const uint32_t u = (uint32_t)i & ((1u << upr_lg) - 1u);
    const Index th = i >> upr_lg;
    const Index t = th / Hkv;
    const uint32_t h = (uint32_t)(th - t * Hkv);
    const uint32_t slot = (uint32_t)slots[t];
    if (slot >= n_slots) continue;
    *reinterpret_cast<uint4*>(dst + (int64_t)(slot >> page_lg) * c_sp + h * c_sh + (int64_t)(slot & one) * c_sn + 16 * u) =
        *reinterpret_cast<const uint4*>(src + (int64_t)t * n_st + h * n_sh + 16 * u);
  }
}

int page_lg_of(int32_t ps) {
  for (int lg = 4; lg <= 8; ++lg)
    if (ps == 1 << lg) return lg;
  return -1;
}

struct Named {
  const char* name;
  Strided<1> at;
  const char* same = "";  // an input that this output may be
};
Strided<1> tables_span(const int32_t* tables, int32_t R, int64_t pitch, int32_t cols) {
  return strided<1>(tables, 4ll * cols, {cols ? R : 0}, {pitch}, 4);
}
int check_apart(const char* who, std::initializer_list<Named> in, std::initializer_list<Named> out) {
  for (const Named& o : out) {
    for (const Named& i : in)
      PA_CHECK_ARG(!overlap(o.at, i.at) || (!strcmp(o.same, i.name) && o.at.at == i.at.at && span(o.at) == span(i.at)),
                   "%s: %s and %s overlap", who, o.name, i.name);
    for (const Named& i : out)
      PA_CHECK_ARG(&i == &o || !overlap(o.at, i.at), "%s: %s and %s overlap", who, o.name, i.name);
  }
  return PA_OK;
}

}  // namespace

// The cache's shape as every entry point checks it; page_lg is set.
int check_pages(const char* who, int64_t n_pages, int32_t page_size, int* page_lg) {
  *page_lg = page_lg_of(page_size);
  PA_CHECK_ARG(*page_lg >= 0, "%s: page_size=%d (16, 32, 64, 128 or 256)", who, page_size);
  PA_CHECK_ARG(n_pages >= 0 && n_pages < (1ll << 31) && n_pages * page_size < (1ll << 31), "%s: n_pages=%lld (slots stay below 2^31)", who,
               (long long)n_pages);
  return PA_OK;
}

}  // namespace pa

extern "C" int pa_page_tables(const pa_tables_args* x, void* stream) {
  using namespace pa;
  PA_CHECK_ARG(x, "pa_page_tables: null arguments");
  int lg;
  if (int rc = check_pages("pa_page_tables", x->n_pages, x->page_size, &lg)) return rc;
  PA_CHECK_ARG(x->R >= 0, "pa_page_tables: R=%d", x->R);
  PA_CHECK_ARG(x->cols >= 0 && ((int64_t)x->cols << lg) <= kMaxPosition && x->pitch >= x->cols,
               "pa_page_tables: %d columns of %d, pitch %lld", x->cols, x->page_size, (long long)x->pitch);
  PA_CHECK_ARG(x->tokens >= 0 && x->tokens <= kMaxPosition, "pa_page_tables: tokens=%lld", (long long)x->tokens);
  PA_CHECK_ARG(x->free_count && x->q_start && x->free_left && x->status && x->workspace,
               "pa_page_tables: null free_count / q_start / free_left / status / workspace");
  PA_CHECK_ARG(x->R == 0 || (x->before && x->fresh && x->lengths), "pa_page_tables: null before / fresh / lengths");
  PA_CHECK_ARG(x->R == 0 || x->cols == 0 || x->tables, "pa_page_tables: null tables");
  PA_CHECK_ARG(x->n_pages == 0 || x->free_list, "pa_page_tables: null free_list");
  PA_CHECK_ARG(x->tokens == 0 || x->slots, "pa_page_tables: null slots");
  // (outputs are written beside reads of the inputs, by other work-groups too)
  const int64_t R = x->R;
  if (int rc = check_apart("pa_page_tables", {{"before", flat(x->before, 4 * R)}, {"fresh", flat(x->fresh, 4 * R)},
                                              {"free_list", flat(x->free_list, 4 * x->n_pages)}, {"free_count", flat(x->free_count, 4)}},
                           {{"lengths", flat(x->lengths, 4 * R), "before"}, {"q_start", flat(x->q_start, 4 * (R + 1))},
                            {"slots", flat(x->slots, 4 * x->tokens)},
                            {"positions", flat(x->positions, x->positions ? 4 * x->tokens : 0)},
                            {"free_left", flat(x->free_left, 4), "free_count"}, {"status", flat(x->status, 4)},
                            {"workspace", flat(x->workspace, 4 * (3 * R + 2))},
                            {"tables", tables_span(x->tables, x->R, x->pitch, x->cols)}}))
    return rc;
  TablesK a;
  a.before = x->before;
  a.fresh = x->fresh;
  a.free_list = x->free_list;
  a.free_count = x->free_count;
  a.tables = x->tables;
  a.pitch = x->pitch;
  a.n_pages = x->n_pages;
  a.R = x->R;
  a.page_lg = lg;
  a.cols = x->cols;
  a.tokens = (int32_t)x->tokens;
  a.lengths = x->lengths;
  a.q_start = x->q_start;
  a.slots = x->slots;
  a.positions = x->positions;
  a.free_left = x->free_left;
  a.status = x->status;
  a.row0 = x->workspace;
  a.page0 = x->workspace + x->R + 1;
  a.held = x->workspace + 2 * (int64_t)x->R + 2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // (new pages: at most one per page_size tokens and one per request)
  const int64_t items = x->tokens + (x->tokens >> lg) + x->R;
  const bool few = x->tokens <= 4 * kScanThreads;
  if (x->R <= kScanRequests && (few || (x->lengths != x->before && x->free_left != x->free_count))) {
    const int64_t groups = few ? 1 : (items + kScanThreads - 1) / kScanThreads;
    hipLaunchKernelGGL(tables_scan_kernel<true>, dim3((unsigned)(groups < 512 ? groups : 512)), dim3(kScanThreads), 0, s, a);
    PA_LAUNCH_CHECK("tables_scan_kernel");
    return PA_OK;
  }
  hipLaunchKernelGGL(tables_scan_kernel<false>, dim3(1), dim3(kScanThreads), 0, s, a);
  PA_LAUNCH_CHECK("tables_scan_kernel");
  const int64_t blocks = (items + 255) / 256;
  hipLaunchKernelGGL(tables_fill_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, a);
  PA_LAUNCH_CHECK("tables_fill_kernel");
  return PA_OK;
}

extern "C" int pa_page_release(const int32_t* first, const int32_t* last, int32_t R, int32_t* tables, int64_t pitch,
                               int32_t cols, int32_t* free_list, const int32_t* free_count, int64_t n_pages,
                               int32_t* free_left, int32_t* status, int32_t* workspace, void* stream) {
  using namespace pa;
  PA_CHECK_ARG(R >= 0 && cols >= 0 && pitch >= cols && n_pages >= 0 && n_pages < (1ll << 31),
               "pa_page_release: R=%d cols=%d pitch=%lld n_pages=%lld", R, cols, (long long)pitch, (long long)n_pages);
  PA_CHECK_ARG(free_count && free_left && status, "pa_page_release: null free_count / free_left / status");
  PA_CHECK_ARG(R == 0 || (first && last && workspace && (cols == 0 || tables)),
               "pa_page_release: null first / last / tables / workspace");
  PA_CHECK_ARG(n_pages == 0 || free_list, "pa_page_release: null free_list");
  // (what is written shares no memory with anything else, but for the count that advances in place)
  const int64_t n = R;
  if (int rc = check_apart("pa_page_release", {{"first", flat(first, 4 * n)}, {"last", flat(last, 4 * n)},
                                               {"free_count", flat(free_count, 4)}},
                           {{"tables", tables_span(tables, R, pitch, cols)}, {"free_list", flat(free_list, 4 * n_pages)},
                            {"free_left", flat(free_left, 4), "free_count"}, {"status", flat(status, 4)},
                            {"workspace", flat(workspace, 4 * n)}}))
    return rc;
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kScanThreads), 0, static_cast<hipStream_t>(stream), first, last, R,
                     tables, pitch, cols, free_list, free_count, n_pages, free_left, status, workspace);
  PA_LAUNCH_CHECK("release_kernel");
  return PA_OK;
}

extern "C" int pa_paged_append(const void* k_new, const void* v_new, int64_t n_st, int64_t n_sh, const int32_t* slots,
                               int64_t T, void* k, void* v, int64_t c_sp, int64_t c_sh, int64_t c_sn, int64_t n_pages,
                               int32_t page_size, int32_t Hkv, int32_t D, int32_t dtype, void* stream) {
  using namespace pa;
  int lg;
  if (int rc = check_pages("pa_paged_append", n_pages, page_size, &lg)) return rc;
  PA_CHECK_ARG(dtype == PA_BF16 || dtype == PA_F16 || dtype == PA_F32, "pa_paged_append: dtype %d", dtype);
  PA_CHECK_ARG(D == 64 || D == 128, "pa_paged_append: D=%d (64 or 128)", D);
  PA_CHECK_ARG(Hkv >= 1 && Hkv <= 65535, "pa_paged_append: Hkv=%d", Hkv);
  PA_CHECK_ARG(T >= 0 && T <= kMaxPosition, "pa_paged_append: T=%lld", (long long)T);
  if (T == 0 || n_pages == 0) return PA_OK;
  PA_CHECK_ARG(k_new && v_new && slots && k && v, "pa_paged_append: null pointer");
  const int64_t esz = dtype == PA_F32 ? 4 : 2;
  auto al = [&](const void* p, int64_t a, int64_t b, int64_t c) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a * esz) % 16 == 0 && (b * esz) % 16 == 0 && (c * esz) % 16 == 0;
  };
  PA_CHECK_ARG(al(k_new, n_st, n_sh, 0) && al(v_new, n_st, n_sh, 0) && al(k, c_sp, c_sh, c_sn) && al(v, c_sp, c_sh, c_sn),
               "pa_paged_append: rows must be 16-byte aligned");
  PA_CHECK_ARG(n_st >= 0 && n_sh >= 0 && c_sp >= 0 && c_sh >= 0 && c_sn >= D, "pa_paged_append: negative strides, or rows closer than D");
  PA_CHECK_ARG((n_pages == 1 || c_sp >= D) && (Hkv == 1 || c_sh >= D), "pa_paged_append: pages or heads closer than D");
  // K and V are written by different work-groups, a row by one: no two rows share a byte, within K, within
  // V or between the two (which nest as one more dimension where they lie in one buffer, by the places in
  // a page's pitch where pages lie outermost and these are some pages apart; k may be v where k_new is
  // v_new)
  Strided<4> kv = strided<4>(k, D * esz, {n_pages, Hkv, page_size, 2}, {c_sp, c_sh, c_sn, 0}, (int)esz);
  const wide apart = strided<1>(v, 0, {1}, {0}).at - kv.at;
  kv.s[3] = apart < 0 ? -apart : apart;
  if (apart == 0 && k_new == v_new) kv.n[3] = 1;
  bool ok = nested(kv);
  if (!ok && kv.s[0] > 0 && (Hkv == 1 || kv.s[0] >= kv.s[1]) && kv.s[0] >= kv.s[2]) {
    kv.s[3] %= kv.s[0];
    ok = nested(kv);
  }
  PA_CHECK_ARG(ok, "pa_paged_append: rows of k and v overlap");
  const int upr_lg = (D * esz == 128) ? 3 : (D * esz == 256) ? 4 : 5;
  const int64_t units = (T * Hkv) << upr_lg, blocks = (units + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384), 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel, auto n) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, static_cast<const char*>(k_new), static_cast<const char*>(v_new),
                       n_st * esz, n_sh * esz, slots, n, static_cast<char*>(k), static_cast<char*>(v),
                       c_sp * esz, c_sh * esz, c_sn * esz, (uint32_t)(n_pages << lg), lg, upr_lg, (uint32_t)Hkv);
  };
  if (units < (1ll << 31))
    go(append_kernel<uint32_t>, (uint32_t)units);
  else
    go(append_kernel<uint64_t>, (uint64_t)units);
  PA_LAUNCH_CHECK("append_kernel");
  return PA_OK;
}
