// Pages, slots and positions of a forward's new tokens, and pages given back: the bookkeeping of a
// paged KV cache on the device, so that a step needs no host read and can be captured.
//
// The free pages are a stack: free_pages[0 .. free_count). Row b holds have = ceil(len / P) pages
// (P = page_size) and needs need = ceil((len + new) / P), so it takes need - have off the stack, the
// rows in order: with upto the inclusive sum of the takes,
//   table[b][have + i] = free_pages[free_count - 1 - (upto_b - take_b) - i].
// A row whose pages the stack no longer holds, or that would outgrow the table, or whose lengths are
// negative, takes none and its tokens get slot and position -1 (`refused` counts such rows). Token i
// of row b is at position len + i, slot table[b][position / P] * P + position % P; tokens past the
// last row's get -1, and so do tokens whose page, taken now or before, is none of the pool (`refused`
// counts those taken now).
//
// reserve: one workgroup sums over the rows (integer sums: the same pages whatever the timing), then
// tokens are dealt to threads. A page that is taken begins at its first new token, which writes its
// number into the table. Up to kOneLaunchTokens tokens the same workgroup does both; more take a
// second launch. Rows' offsets, lengths and first pages are searched in LDS (up to kThreads rows), the page
// numbers of all of a thread's tokens asked for before any is used. 64 rows of a token: 6.4 us (8.8 with the
// search in memory), three scans and two round trips; 512 rows of a million tokens, 12.6 MB written: 4.5 + 9.0,
// 1.4 TB/s: 2.2 are every workgroup's copy of the rows' numbers and a thread's four searches among them (8 rows
// of as many tokens take 6.8), the rest the launch, a round trip for the page numbers, and stores of 4 and 8 bytes.
//
// release: one workgroup; 128 rows of up to 32 pages 7.8 us, 512 rows of 8000 pages 20.
#include "paged.h"

namespace mcamd {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kOneLaunchTokens = 4096;
constexpr int kTokens = 4;  // tokens of a thread

struct PlanParams {
  int32_t *table;
  const int32_t *seqlens, *new_lens;
  const int32_t *free_pages;
  int32_t *free_count, *refused, *cu;
  int32_t *first;  // per row: the stack index of its first page, or -1 (refused)
  int64_t *slots;
  int32_t *positions;
  int64_t table_stride;
  int n_rows, max_pages, n_pages, shift, total;
};

// Inclusive sum over the wave.
__device__ __forceinline__ int64_t wave_scan(int64_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

// Inclusive sum of x over the workgroup, after `carry`; carry becomes the whole sum.
__device__ __forceinline__ int64_t group_scan(int64_t x, int64_t &carry, int64_t *s_sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t y = wave_scan(x, lane);
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 63) s_sum[wave] = y;
  __syncthreads();
  int64_t all = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += s_sum[w];
    all += s_sum[w];
  }
  y += carry + before;
  carry += all;
  return y;
}

// What the tokens need to know of the rows: in LDS where kThreads rows are the most, else where it lies.
struct SharedRows {
  int cu[kThreads + 1], first[kThreads], len[kThreads];
};
struct GlobalRows {
  const int32_t *cu, *first, *len;
};

// kTokens tokens, `step` apart from t0 on; returns how many of the pages taken for them are no pages, whose
// tokens get no slot.
template <class Rows>
__device__ __forceinline__ int write_tokens(const PlanParams &P, const Rows &rows, int t0, int step) {
  int row[kTokens];
#pragma unroll
  for (int u = 0; u < kTokens; ++u) {
    // The row of the token: the last one that begins at or before it (those before it may be empty).
    int lo = 0, hi = P.n_rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (rows.cu[mid] <= t0 + u * step)
        lo = mid;
      else
        hi = mid;
    }
    row[u] = lo;
  }
  // The numbers of all of its pages are asked for before any is used; a token without one asks for the
  // stack's first.
  const int page_mask = (1 << P.shift) - 1;
  int pos[kTokens], id[kTokens];
  int32_t *named[kTokens];  // where a page that is taken goes
#pragma unroll
  for (int u = 0; u < kTokens; ++u) {
    const int t = t0 + u * step, b = row[u];
    const int first = rows.first[b], len = rows.len[b], begin = rows.cu[b];
    const bool planned = t < rows.cu[b + 1] && first >= 0;
    pos[u] = planned ? len + t - begin : -1;
    const int have = int((int64_t(len) + page_mask) >> P.shift), page = pos[u] >> P.shift;
    int32_t *const line = P.table + b * P.table_stride + page;
    id[u] = *(!planned ? P.free_pages : page < have ? line : P.free_pages + (first - (page - have)));
    named[u] = planned && page >= have && (pos[u] & page_mask) == 0 ? line : nullptr;
  }
  int lost = 0;
#pragma unroll
  for (int u = 0; u < kTokens; ++u) {
    const int t = t0 + u * step;
    if (t >= P.total) break;
    const bool page = uint32_t(id[u]) < uint32_t(P.n_pages);
    if (named[u]) {
      *named[u] = page ? id[u] : -1;
      lost += !page;
    }
    P.slots[t] = pos[u] < 0 || !page ? -1 : (int64_t(id[u]) << P.shift) + (pos[u] & page_mask);
    P.positions[t] = pos[u];
  }
  return lost;
}

__global__ __launch_bounds__(kThreads) void reserve_kernel(PlanParams P, int with_tokens) {
  __shared__ SharedRows s_rows;
  __shared__ int64_t s_sum[kWaves];
  __shared__ int s_refused;
  const int tid = threadIdx.x;
  if (tid == 0) s_refused = 0;
  const int64_t stack = min(max(P.free_count[0], 0), P.n_pages);
  const int64_t page = int64_t(1) << P.shift;
  int64_t taken = 0, tokens = 0, kept = 0;  // pages asked for, tokens, pages given so far
  int64_t given = 0;                        // of this thread's rows
  for (int b0 = 0; b0 < P.n_rows; b0 += kThreads) {
    const int b = b0 + tid;
    const bool here = b < P.n_rows;
    const int64_t len = here ? P.seqlens[b] : 0;
    const int64_t asked = here ? P.new_lens[b] : 0;
    // Tokens past `total` are not planned, and get no pages.
    const int64_t all = group_scan(max(asked, int64_t(0)), tokens, s_sum);
    const int64_t end = min(all, int64_t(P.total));
    const int64_t fresh = end - min(all - max(asked, int64_t(0)), int64_t(P.total));
    const int64_t have = (max(len, int64_t(0)) + page - 1) >> P.shift;
    const int64_t need = (max(len, int64_t(0)) + fresh + page - 1) >> P.shift;
    const bool fits = len >= 0 && asked >= 0 && need <= P.max_pages;
    const int64_t take = fits ? need - have : 0;
    const int64_t upto = group_scan(take, taken, s_sum);
    const bool ok = fits && (take == 0 || upto <= stack);
    if (here) {
      // A row that takes none has no first page; any index but -1 will do.
      const int first = !ok ? -1 : take == 0 ? 0 : int(stack - 1 - (upto - take));
      P.first[b] = first;
      P.cu[b + 1] = int(end);
      if (b < kThreads) {
        s_rows.first[b] = first;
        s_rows.cu[b + 1] = int(end);
        s_rows.len[b] = int(len);
      }
      if (!ok) atomicAdd(&s_refused, 1);
      given += ok ? take : 0;
    }
  }
  group_scan(given, kept, s_sum);
  if (tid == 0) {
    P.cu[0] = s_rows.cu[0] = 0;
    P.free_count[0] = int(stack - kept);
  }
  __syncthreads();  // the rows' numbers are written
  if (with_tokens) {
    int lost = 0;
    for (int t = tid; t < P.total; t += kThreads * kTokens) {
      if (P.n_rows <= kThreads)
        lost += write_tokens(P, s_rows, t, kThreads);
      else
        lost += write_tokens(P, GlobalRows{P.cu, P.first, P.seqlens}, t, kThreads);
    }
    if (lost > 0) atomicAdd(&s_refused, lost);
    __syncthreads();
  }
  if (tid == 0) P.refused[0] = s_refused;
}

__global__ __launch_bounds__(256) void tokens_kernel(PlanParams P) {
  __shared__ SharedRows s_rows;
  const int t = int(blockIdx.x) * 256 * kTokens + int(threadIdx.x);
  int lost;
  if (P.n_rows > kThreads) {
    lost = write_tokens(P, GlobalRows{P.cu, P.first, P.seqlens}, t, 256);
  } else {
    for (int b = threadIdx.x; b < P.n_rows; b += 256) {
      s_rows.cu[b + 1] = P.cu[b + 1];
      s_rows.first[b] = P.first[b];
      s_rows.len[b] = P.seqlens[b];
    }
    if (threadIdx.x == 0) s_rows.cu[0] = 0;
    __syncthreads();
    lost = write_tokens(P, s_rows, t, 256);
  }
  if (lost > 0) atomicAdd(P.refused, lost);  // whole numbers: the same in any order
}

// Rows rows[0 .. n) give their pages back, in order, and are empty then. A row that is named twice
// gives them where it is named first; a row outside the batch is passed over, and so is a number in the
// table that is no page.
__global__ __launch_bounds__(kThreads) void release_kernel(int32_t *table, int64_t table_stride,
                                                           int32_t *seqlens, const int32_t *rows,
                                                           int n, int n_rows, int32_t *free_pages,
                                                           int32_t *free_count, int max_pages,
                                                           int n_pages, int shift) {
  __shared__ int64_t s_sum[kWaves], s_end[kThreads];
  __shared__ __attribute__((aligned(16))) int s_row[kThreads];
  const int tid = threadIdx.x;
  int64_t top = min(max(free_count[0], 0), n_pages);
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + tid;
    int row = i < n ? rows[i] : -1;
    if (row < 0 || row >= n_rows) row = -1;
    s_row[tid] = row;
    __syncthreads();
    int again = 0;  // names of the same row before this one
#pragma unroll 8
    for (int j = 0; j < (row < 0 ? 0 : tid >> 2); ++j) {
      const int4 x = reinterpret_cast<const int4 *>(s_row)[j];
      again |= int(x.x == row) | int(x.y == row) | int(x.z == row) | int(x.w == row);
    }
    for (int j = tid & ~3; j < tid; ++j) again |= int(s_row[j] == row);
    if (again) row = -1;
    const int len = row >= 0 ? seqlens[row] : 0;
    if (row >= 0) seqlens[row] = 0;
    const int64_t held =
        min((max(int64_t(len), int64_t(0)) + (1 << shift) - 1) >> shift, int64_t(max_pages));
    int64_t all = 0;
    s_end[tid] = group_scan(held, all, s_sum);
    __syncthreads();
    auto entry = [&](int64_t p) {  // of page p of these rows, in the table
      int lo = 0, hi = kThreads - 1;  // the first row whose pages end past p
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > p)
          hi = mid;
        else
          lo = mid + 1;
      }
      return s_row[lo] * table_stride + p - (lo ? s_end[lo - 1] : 0);
    };
    auto taken_from = [&](int64_t p) {
      const int64_t at = entry(p);
      const int id = table[at];
      table[at] = -1;
      return id;
    };
    auto is_page = [&](int id) { return uint32_t(id) < uint32_t(n_pages); };
    const int64_t base = top;
    bool odd = false;  // an entry is no page, or there are more than the stack has room for
    for (int64_t p = tid; p < all; p += kThreads) {
      if (base + p < n_pages) {
        const int id = taken_from(p);
        free_pages[base + p] = id;
        odd = odd || !is_page(id);
      } else {
        odd = true;
      }
    }
    top += all;
    if (__syncthreads_or(odd)) {
      // What is no page of the pool, as in a row that was refused and moved on all the same, is not one to
      // give: the pages behind it move up, none past where its own thread has read it.
      top = base;
      for (int64_t p0 = 0; p0 < all; p0 += kThreads) {
        const int64_t p = p0 + tid;
        const int id = p >= all ? -1 : base + p < n_pages ? free_pages[base + p] : taken_from(p);
        const int64_t to = group_scan(int64_t(is_page(id)), top, s_sum) - 1;
        if (is_page(id) && to < n_pages) free_pages[to] = id;
      }
    }
    __syncthreads();  // s_row and s_end have been read
  }
  if (tid == 0) free_count[0] = int(min(top, int64_t(n_pages)));
}

constexpr int64_t kMax31 = 0x7fffffff;

}  // namespace
}  // namespace mcamd

using namespace mcamd;

extern "C" int mcamd_paged_reserve(int32_t *block_table, int64_t table_stride,
                                   const int32_t *cache_seqlens, const int32_t *new_lens,
                                   const int32_t *free_pages, int32_t *free_count,
                                   int32_t *row_scratch, int32_t *cu_seqlens, int64_t *slots,
                                   int32_t *positions, int32_t *refused, int64_t n_rows,
                                   int64_t max_pages, int64_t n_pages, int64_t page_size,
                                   int64_t total, void *stream) {
  PlanParams P{};
  if (n_rows < 0 || total < 0 || max_pages <= 0 || n_pages <= 0)
    return fail(MCAMD_EINVAL, "paged_reserve: sizes must be positive (n_rows, total may be 0)");
  if (!page_shift(page_size, P.shift))
    return fail(MCAMD_EINVAL, "paged_reserve: page_size must be a power of two from 16 to 2^30");
  if (table_stride < max_pages)
    return fail(MCAMD_EINVAL, "paged_reserve: table_stride smaller than max_pages");
  if (n_rows >= kMax31 - kThreads || total > kMax31 - kThreads * kTokens ||
      n_pages > kMax31 / page_size || max_pages > kMax31 / page_size)
    return fail(MCAMD_EUNSUPPORTED, "paged_reserve: sizes beyond 31 bits");
  if (!free_count || !cu_seqlens || !refused ||
      (n_rows > 0 && (!block_table || !cache_seqlens || !new_lens || !free_pages || !row_scratch)) ||
      (total > 0 && (!slots || !positions)))
    return fail(MCAMD_EINVAL, "paged_reserve: null pointer");
  if (n_rows == 0 && total > 0)
    return fail(MCAMD_EINVAL, "paged_reserve: tokens without a row");
  P.table = block_table;
  P.table_stride = table_stride;
  P.seqlens = cache_seqlens;
  P.new_lens = new_lens;
  P.free_pages = free_pages;
  P.free_count = free_count;
  P.refused = refused;
  P.cu = cu_seqlens;
  P.first = row_scratch;
  P.slots = slots;
  P.positions = positions;
  P.n_rows = int(n_rows);
  P.max_pages = int(max_pages);
  P.n_pages = int(n_pages);
  P.total = int(total);
  const bool one = total <= kOneLaunchTokens;
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), P, int(one));
  const int st = launch_status("paged_reserve");
  if (st != MCAMD_OK || one) return st;
  const int64_t threads = (total + kTokens - 1) / kTokens;
  hipLaunchKernelGGL(tokens_kernel, dim3(unsigned((threads + 255) / 256)), dim3(256), 0,
                     as_stream(stream), P);
  return launch_status("paged_reserve");
}

extern "C" int mcamd_paged_release(int32_t *block_table, int64_t table_stride,
                                   int32_t *cache_seqlens, const int32_t *rows, int64_t n_release,
                                   int64_t n_rows, int32_t *free_pages, int32_t *free_count,
                                   int64_t max_pages, int64_t n_pages, int64_t page_size,
                                   void *stream) {
  int shift = 0;
  if (n_rows < 0 || n_release < 0 || max_pages <= 0 || n_pages <= 0)
    return fail(MCAMD_EINVAL, "paged_release: sizes must be positive (n_rows, n_release may be 0)");
  if (!page_shift(page_size, shift))
    return fail(MCAMD_EINVAL, "paged_release: page_size must be a power of two from 16 to 2^30");
  if (table_stride < max_pages)
    return fail(MCAMD_EINVAL, "paged_release: table_stride smaller than max_pages");
  if (n_rows >= kMax31 - kThreads || n_release >= kMax31 - kThreads ||
      n_pages > kMax31 / page_size || max_pages > kMax31 / page_size)
    return fail(MCAMD_EUNSUPPORTED, "paged_release: sizes beyond 31 bits");
  if (n_release == 0 || n_rows == 0) {
    clear_error();
    return MCAMD_OK;
  }
  if (!block_table || !cache_seqlens || !rows || !free_pages || !free_count)
    return fail(MCAMD_EINVAL, "paged_release: null pointer");
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), block_table,
                     table_stride, cache_seqlens, rows, int(n_release), int(n_rows), free_pages,
                     free_count, int(max_pages), int(n_pages), shift);
  return launch_status("paged_release");
}
