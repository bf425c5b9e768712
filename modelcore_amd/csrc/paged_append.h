// New tokens' K and V into their pages, bit for bit: kAppendTokens tokens a workgroup, whose places its
// first threads find, then 16-byte pieces by all of them. A row that does not fit its line of the
// table, and a token whose page is outside the pool, are passed over. Bound by latency in small calls, by
// HBM in large ones: 16384 tokens of 4 heads of 128 in bf16, 67 MB in and out, 13.4 us (5.0 TB/s).
//
// A launch of its own, or the last workgroups of the streaming kernel's, which appends for its own rows by
// itself and comes before the other rows' launch.
#pragma once

#include "paged.h"

namespace mcamd {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 8;

struct PagedAppend {
  const uint4 *k, *v;
  uint4 *k_pages, *v_pages;
  PagedKv kv;  // page_stride in pieces
  const int32_t *seqlens, *cu;
  int n_rows, t_new, total, units;
  int G, skip;  // rows of few_pairs() by it append by themselves
};

__device__ __forceinline__ void append_tokens(const PagedAppend &A, int block) {
  __shared__ int64_t s_at[kAppendTokens];
  const int t0 = block * kAppendTokens;
  if (threadIdx.x < kAppendTokens) {
    const int t = t0 + threadIdx.x;
    int64_t at = -1;
    if (t < A.total) {
      int b, tok0, T;
      if (A.cu) {
        int lo = 0, hi = A.n_rows;  // the last row that begins at or before t
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (A.cu[mid] <= t)
            lo = mid;
          else
            hi = mid;
        }
        b = lo;
      } else {
        b = t / A.t_new;
      }
      row_tokens(A.cu, A.t_new, A.total, b, tok0, T);
      const int64_t s0 = A.seqlens[b], pos = s0 + (t - tok0);
      if (t >= tok0 && t < tok0 + T && s0 >= 0 && s0 + T <= int64_t(A.kv.max_pages) << A.kv.shift &&
          !few_pairs(T, A.G, A.skip)) {
        const int id = A.kv.table[b * A.kv.table_stride + (pos >> A.kv.shift)];
        if (A.kv.is_page(id)) at = A.kv.offset(id, A.kv.in_page(int(pos)), A.units);
      }
    }
    s_at[threadIdx.x] = at;
  }
  __syncthreads();
  const int n = min(kAppendTokens, A.total - t0) * A.units;
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const int t = i / A.units, u = i - t * A.units;
    const int64_t at = s_at[t], from = (int64_t(t0) + t) * A.units + u;
    if (at < 0) continue;
    const uint4 x = A.k[from], y = A.v[from];
    A.k_pages[at + u] = x;
    A.v_pages[at + u] = y;
  }
}

inline PagedAppend paged_append(const PagedArgs &a, int64_t skip) {
  const int64_t elem = a.dtype == MCAMD_F32 ? 4 : 2;
  PagedAppend A;
  A.k = static_cast<const uint4 *>(a.k_new);
  A.v = static_cast<const uint4 *>(a.v_new);
  A.k_pages = static_cast<uint4 *>(a.k_pages);
  A.v_pages = static_cast<uint4 *>(a.v_pages);
  A.kv = a.kv;
  A.kv.page_stride = a.kv.page_stride * elem / 16;
  A.seqlens = a.seqlens;
  A.cu = a.cu;
  A.n_rows = int(a.n_rows);
  A.t_new = int(a.t_new);
  A.total = int(a.total);
  A.units = int(a.n_kv_head * a.head_dim * elem / 16);
  A.G = int(a.n_head / a.n_kv_head);
  A.skip = int(skip);
  return A;
}
inline int64_t paged_append_blocks(const PagedArgs &a) {
  return (a.total + kAppendTokens - 1) / kAppendTokens;
}

}  // namespace
}  // namespace mcamd
