// Sums over a workgroup's rows, and pages that go back onto the stack of free ones: what the plan of a paged
// cache's step and the end of one share. One workgroup of kThreads.
#pragma once

#include "paged.h"

namespace mcamd {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

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

// The pages of up to kThreads rows go onto the stack from `top` on, the rows in order; returns the new top.
// Row i's, thread i's, are the table's entries from first(i) on, s_end[i] being the sum of how many over the
// rows up to it and `all` that over all of them. Their entries become -1. What is no page of the pool is
// passed over.
template <class First>
__device__ __forceinline__ int64_t push_pages(int32_t *table, const int64_t *s_end, int64_t all, int64_t top,
                                              int32_t *free_pages, int n_pages, int64_t *s_sum,
                                              const First &first) {
  const int tid = threadIdx.x;
  auto taken_from = [&](int64_t p) {
    int lo = 0, hi = kThreads - 1;  // the first row whose pages end past p
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > p)
        hi = mid;
      else
        lo = mid + 1;
    }
    const int64_t at = first(lo) + p - (lo ? s_end[lo - 1] : 0);
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
  return top;
}

}  // namespace
}  // namespace mcamd
