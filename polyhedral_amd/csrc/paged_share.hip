// Which tokens of a step share a prefix (gfx950): the plan of pa_shared_attn, once for all layers.
//
// With own(r) the holder of request r where it has one, tokens in this step and whole pages to share,
// a group is the requests of one holder, if they are two or more; its prefix is the least that they
// share.  Each request sums over the others (R^2 comparisons, spread over the work-group: 64 requests
// are 4 a thread), so no atomic gives an order, and the same step has the same plan always.  More than 1024 are
// taken 1024 at a time, each compared with those of its own time alone, so the work grows as their number.
//
// What bounds it: latency, three trips to memory, the exchanges over the LDS and the launch: 5.0 us for 65 requests of
// 64 tokens, 5.5 for 45 of 110; for many the comparisons: 256 requests 12 us, 1024 127, 4096 290 (all with all: 2.6 ms),
// 2^20 73 ms.
#include "page_checks.hpp"
#include "paged_attn.hpp"

namespace pa {
namespace {

constexpr int kShareThreads = 1024;
constexpr int kShareRequests = 1024;  // requests whose state fits the LDS

struct ShareK {
  const int32_t* lengths;
  const int32_t* q_start;
  const int32_t* holders;
  const int32_t* shared;
  int32_t R, T, page_lg;
  int32_t* start;
  int32_t* rows;
  int32_t* positions;
  int32_t* prefix;
  int32_t* low;
  int32_t* high;
  int32_t* first;
  int32_t* workspace;
};

template <bool LDS>
__global__ __launch_bounds__(kShareThreads) void share_kernel(const ShareK a) {
  constexpr int NW = kShareThreads / 64;
  __shared__ int32_t lds[LDS ? 8 * kShareRequests : 2 * kShareThreads];
  __shared__ int32_t wave_n[NW];
  int32_t* at = LDS ? lds : a.workspace;
  int32_t *s0 = at, *n = at + a.R, *len = at + 2 * (int64_t)a.R, *own = at + 3 * (int64_t)a.R, *some = at + 4 * (int64_t)a.R,
          *off = at + 5 * (int64_t)a.R, *cut = at + 6 * (int64_t)a.R, *tot = at + 7 * (int64_t)a.R;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;

  // ---- the requests: starts that fall back are taken as the largest before (as in pa_paged_attn) ------
  bool falls = false;
  for (int r = tid; r < a.R; r += kShareThreads) {
    const int32_t x = imin(imax(a.q_start[r], 0), a.T), y = imin(imax(a.q_start[r + 1], 0), a.T);
    const int32_t o = a.holders[r], l = imin(imax(a.lengths[r], 0), kMaxPosition);
    const int32_t m = imin(imax(a.shared[r], 0), l) >> a.page_lg << a.page_lg;
    s0[r] = x;
    n[r] = y - x;
    len[r] = l;
    some[r] = m;
    own[r] = (uint32_t)o < (uint32_t)a.R && y != x && m > 0 ? o : -1;
    falls |= y < x;
  }
  if (__syncthreads_or(falls)) {
    int32_t top = 0;
    for (int r0 = 0; r0 < a.R; r0 += kShareThreads) {
      const int r = r0 + tid;
      const bool in = r < a.R;
      const int32_t y = in ? s0[r] + n[r] : 0;
      int32_t x = in ? s0[r] : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int32_t u = __shfl_up(x, o);
        x = lane >= o ? imax(x, u) : x;
      }
      if (lane == 63) wave_n[w] = x;
      __syncthreads();
      x = imax(x, top);
#pragma unroll
      for (int z = 0; z < NW; ++z) {
        const int32_t u = wave_n[z];
        x = z < w ? imax(x, u) : x;
        top = imax(top, u);
      }
      if (in) {
        const int32_t o = a.holders[r];
        s0[r] = x;
        n[r] = imax(y, x) - x;
        own[r] = (uint32_t)o < (uint32_t)a.R && n[r] > 0 && some[r] > 0 ? o : -1;
      }
      __syncthreads();
    }
  }

  // ---- a request among those of its holder, and as a holder: `per` lanes to a request --------------------
  int per = 1;
  while (per < 64 && 2 * per * a.R <= kShareThreads) per *= 2;
  const int sub = tid & (per - 1);
  if constexpr (LDS) {
    for (int r0 = 0; r0 < a.R; r0 += kShareThreads / per) {
      const int r = r0 + tid / per;
      const int32_t mine = r < a.R ? own[r] : -1;
      int32_t count = 0, before = 0, least = kMaxPosition;
      int32_t members = 0, sum = 0, lo = kMaxPosition, hi = 0, pre = kMaxPosition;
      for (int x = sub; x < a.R; x += per) {
        const int32_t o = own[x], nx = n[x], sx = some[x], lx = len[x];
        if (o >= 0 && o == mine) {
          ++count;
          before += x < r ? nx : 0;
          least = imin(least, sx);
        }
        if (o == r) {
          ++members;
          sum += nx;
          lo = imin(lo, lx - nx);
          hi = imax(hi, lx - 1);
          pre = imin(pre, sx);
        }
      }
      for (int o = 1; o < per; o <<= 1) {
        count += __shfl_xor(count, o);
        before += __shfl_xor(before, o);
        least = imin(least, __shfl_xor(least, o));
        members += __shfl_xor(members, o);
        sum += __shfl_xor(sum, o);
        lo = imin(lo, __shfl_xor(lo, o));
        hi = imax(hi, __shfl_xor(hi, o));
        pre = imin(pre, __shfl_xor(pre, o));
      }
      if (r < a.R && sub == 0) {
        const bool in = count > 1, group = members > 1;
        off[r] = before;
        cut[r] = in ? least : 0;
        tot[r] = group ? sum : 0;
        a.first[r] = in ? least : 0;
        a.prefix[r] = group ? pre : 0;
        a.low[r] = group ? lo : 0;
        a.high[r] = group ? hi : 0;
      }
    }
  } else {
    // Many requests, in order, as many at a time as there are threads: a request's rows come after those that its
    // holder's earlier ones have, which are the sum so far and what the LDS shows of these.  (Whole numbers, whose
    // sums and least ones do not depend on the order of the atomics; these pass the L1, so the loads do too.)
    int32_t *count = a.first, *sum = a.start, *pre = a.prefix, *lo = a.low, *hi = a.high;
    int32_t *by = lds, *of = lds + kShareThreads;
    auto get = [](const int32_t* p) __attribute__((always_inline)) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    for (int g = tid; g < a.R; g += kShareThreads) {
      count[g] = sum[g] = hi[g] = 0;
      pre[g] = lo[g] = kMaxPosition;
    }
    for (int r0 = 0; r0 < a.R; r0 += kShareThreads) {
      const int r = r0 + tid;
      const int32_t o = r < a.R ? own[r] : -1, m = r < a.R ? n[r] : 0;
      by[tid] = o;
      of[tid] = m;
      __threadfence();
      __syncthreads();
      int32_t before = o >= 0 ? get(sum + o) : 0;
#pragma unroll 8
      for (int x = 0; x < 64 * (w + 1); ++x) before += by[x] == o && x < tid ? of[x] : 0;
      if (r < a.R) off[r] = before;
      __syncthreads();
      if (o >= 0) {
        atomicAdd(count + o, 1);
        atomicAdd(sum + o, m);
        atomicMin(pre + o, some[r]);
        atomicMin(lo + o, len[r] - m);
        atomicMax(hi + o, len[r] - 1);
      }
    }
    __threadfence();
    __syncthreads();
    for (int r = tid; r < a.R; r += kShareThreads) {
      const int32_t o = own[r];
      cut[r] = o >= 0 && get(count + o) > 1 ? get(pre + o) : 0;
    }
    __syncthreads();
    for (int g = tid; g < a.R; g += kShareThreads) {
      const bool group = get(count + g) > 1;
      tot[g] = group ? get(sum + g) : 0;
      pre[g] = group ? get(pre + g) : 0;
      lo[g] = group ? get(lo + g) : 0;
      hi[g] = group ? get(hi + g) : 0;
      a.first[g] = cut[g];
    }
  }
  __syncthreads();
  // ---- exclusive sums of the groups' rows, in place (at most T in all) ---------------------------------
  int32_t total = 0;
  for (int r0 = 0; r0 < a.R; r0 += kShareThreads) {
    const int g = r0 + tid;
    const int32_t x = g < a.R ? tot[g] : 0, in = wave_scan(x);
    if (lane == 63) wave_n[w] = in;
    __syncthreads();
    int32_t base = total;
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const int32_t z = wave_n[y];
      base += y < w ? z : 0;
      total += z;
    }
    if (g < a.R) {
      tot[g] = base + in - x;
      a.start[g] = base + in - x;
    }
    __syncthreads();
  }
  if (tid == 0) a.start[a.R] = total;
  // ---- the rows ----------------------------------------------------------------------------------------
  for (int r0 = 0; r0 < a.R; r0 += kShareThreads / per) {
    const int r = r0 + tid / per;
    if (r >= a.R || cut[r] == 0) continue;
    const int32_t to = tot[own[r]] + off[r], from = s0[r], m = n[r], p0 = len[r] - m;
    for (int i = sub; i < m; i += per) {
      a.rows[to + i] = from + i;
      a.positions[to + i] = p0 + i;
    }
  }
  for (int i = total + tid; i < a.T; i += kShareThreads) a.rows[i] = a.positions[i] = -1;
}

// Which requests give their pages back: one work-group marks the holders of requests that go on, then a thread per
// request says what becomes of it, then a wave per request clears what its table names of its holder's pages.  What
// bounds it: latency, two trips to memory and the launch.
struct FinishK {
  const uint8_t* done;
  int32_t* holders;
  int32_t* shared;
  int32_t* lengths;
  int32_t R, page_lg;
  int32_t* tables;
  int64_t pitch;
  int32_t cols, refused_bits;
  int32_t* refused;
  int32_t* first;
  int32_t* last;
  int32_t* busy;
};

__global__ __launch_bounds__(kShareThreads) void finish_kernel(const FinishK a) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int r = tid; r < a.R; r += kShareThreads) a.busy[r] = 0;
  __syncthreads();
  for (int r = tid; r < a.R; r += kShareThreads) {
    const int32_t h = a.holders[r];
    if ((uint32_t)h < (uint32_t)a.R && h != r && !a.done[r]) a.busy[h] = 1;
  }
  __syncthreads();
  bool kept = false;
  for (int r = tid; r < a.R; r += kShareThreads) {
    const bool done = a.done[r], busy = a.busy[r];
    const int32_t h = a.holders[r];
    const bool member = (uint32_t)h < (uint32_t)a.R && h != r, go = done && !busy;
    kept |= done && busy;
    a.first[r] = go && member ? imin(imax(a.shared[r], 0) >> a.page_lg, a.cols) : 0;
    a.last[r] = go ? a.cols : 0;
    if (go) {
      a.lengths[r] = a.shared[r] = 0;
      a.holders[r] = -1;
    }
  }
  if (__syncthreads_or(kept) && tid == 0) *a.refused |= a.refused_bits;
  for (int r = w; r < a.R; r += kShareThreads / 64)
    for (int32_t c = lane; c < a.first[r]; c += 64) a.tables[r * a.pitch + c] = -1;
}

}  // namespace
}  // namespace pa

extern "C" int pa_page_finish(const pa_finish_args* x, void* stream) {
  using namespace pa;
  PA_CHECK_ARG(x, "pa_page_finish: null arguments");
  int lg;
  if (int rc = check_pages("pa_page_finish", 0, x->page_size, &lg)) return rc;
  PA_CHECK_ARG(x->R >= 0 && x->R < (1 << 24), "pa_page_finish: R=%d (below 2^24)", x->R);
  PA_CHECK_ARG(x->cols >= 0 && ((int64_t)x->cols << lg) <= kMaxPosition && x->pitch >= x->cols,
               "pa_page_finish: %d columns of %d, pitch %lld", x->cols, x->page_size, (long long)x->pitch);
  if (x->R == 0) return PA_OK;
  PA_CHECK_ARG(x->done && x->holders && x->shared && x->lengths && x->refused && x->first && x->last && x->workspace &&
                   (x->cols == 0 || x->tables),
               "pa_page_finish: null pointer");
  const int64_t n = 4ll * x->R;
  if (int rc = check_apart("pa_page_finish", {{"done", flat(x->done, x->R)}},
                           {{"holders", flat(x->holders, n)}, {"shared", flat(x->shared, n)}, {"lengths", flat(x->lengths, n)},
                            {"tables", tables_span(x->tables, x->R, x->pitch, x->cols)}, {"refused", flat(x->refused, 4)},
                            {"first", flat(x->first, n)}, {"last", flat(x->last, n)}, {"workspace", flat(x->workspace, n)}}))
    return rc;
  const FinishK a{x->done, x->holders, x->shared, x->lengths, x->R, lg, x->tables, x->pitch, x->cols, x->refused_bits, x->refused,
                  x->first, x->last, x->workspace};
  hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(kShareThreads), 0, static_cast<hipStream_t>(stream), a);
  PA_LAUNCH_CHECK("finish_kernel");
  return PA_OK;
}

extern "C" int pa_share_rows(const pa_share_args* x, void* stream) {
  using namespace pa;
  PA_CHECK_ARG(x, "pa_share_rows: null arguments");
  int lg;
  if (int rc = check_pages("pa_share_rows", 0, x->page_size, &lg)) return rc;
  PA_CHECK_ARG(x->R >= 0 && x->R < (1 << 24), "pa_share_rows: R=%d (below 2^24)", x->R);
  PA_CHECK_ARG(x->T >= 0 && x->T <= kMaxPosition, "pa_share_rows: T=%lld", (long long)x->T);
  PA_CHECK_ARG(x->start && x->q_start, "pa_share_rows: null start / q_start");
  PA_CHECK_ARG(x->R == 0 || (x->lengths && x->holders && x->shared && x->prefix && x->low && x->high && x->first && x->workspace),
               "pa_share_rows: null lengths / holders / shared / prefix / low / high / first / workspace");
  PA_CHECK_ARG(x->T == 0 || (x->rows && x->positions), "pa_share_rows: null rows / positions");
  const int64_t R = x->R;
  if (int rc = check_apart("pa_share_rows",
                           {{"lengths", flat(x->lengths, 4 * R)}, {"q_start", flat(x->q_start, 4 * (R + 1))},
                            {"holders", flat(x->holders, 4 * R)}, {"shared", flat(x->shared, 4 * R)}},
                           {{"start", flat(x->start, 4 * (R + 1))}, {"rows", flat(x->rows, 4 * x->T)},
                            {"positions", flat(x->positions, 4 * x->T)}, {"prefix", flat(x->prefix, 4 * R)},
                            {"low", flat(x->low, 4 * R)}, {"high", flat(x->high, 4 * R)}, {"first", flat(x->first, 4 * R)},
                            {"workspace", flat(x->workspace, 32 * R)}}))
    return rc;
  const ShareK a{x->lengths, x->q_start, x->holders, x->shared, x->R, (int32_t)x->T, lg, x->start, x->rows, x->positions,
                 x->prefix, x->low, x->high, x->first, x->workspace};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (x->R <= kShareRequests)
    hipLaunchKernelGGL(share_kernel<true>, dim3(1), dim3(kShareThreads), 0, s, a);
  else
    hipLaunchKernelGGL(share_kernel<false>, dim3(1), dim3(kShareThreads), 0, s, a);
  PA_LAUNCH_CHECK("share_kernel");
  return PA_OK;
}
