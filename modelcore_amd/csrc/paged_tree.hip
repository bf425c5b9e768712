// Drafted trees over a paged cache: where their nodes stand and whom they see, and what becomes of them in
// the cache once it is known how many are accepted.
//
// tree: node i of a row (its index among the row's new tokens) follows parents[i], a node before it, or none
// (-1). Bit j of its mask says that j is i or an ancestor, its position is the row's length plus its depth. A
// workgroup a row, a wave for each 64 of its nodes: six doublings among the lanes give a node's ancestors of the
// same 64 and the first one before them, and with those of all nodes in LDS it has the rest in at most 15 steps, a
// word each. Latency: 2.4 us for a chain of 8, 2.6 for 64 rows with chains of 64, 3.1 for 20 with chains of 200, 11
// for one of 1024; with every node climbing to its root by itself 3.6, 15, 42 and 203.
//
// keep: the row's accepted nodes kept[0] < kept[1] < .. (kept[j] >= j) become its tokens s, s + 1, ..: in every
// slot the key and value of node kept[j] move to where node j's are. A thread moves 16 bytes of all of a
// row's nodes, in order, so that every place is read before it is written and threads share nothing. Then one
// workgroup moves the lengths on and gives back the pages that no token is left in.
#include "paged_stack.h"

namespace mcamd {
namespace {

constexpr int64_t kMax31 = 0x7fffffff;

struct TreeParams {
  const int32_t *parents, *cu, *seqlens;
  int32_t *positions;
  uint64_t *masks;
  int n_rows, total, words;
};

constexpr int kRoot = -1, kNone = -2;  // what a node follows: the row's tokens; nothing that is there

__global__ __launch_bounds__(1024) void tree_kernel(TreeParams P) {
  __shared__ uint64_t s_near[64 * kMaxTreeWords];  // a node's ancestors among its 64, and itself
  __shared__ int s_up[64 * kMaxTreeWords];         // and the first one before them
  const int tid = threadIdx.x, threads = 64 * P.words;
  if (int(blockIdx.x) >= P.n_rows) {  // tokens that are no row's, or past its last word
    const int t = (int(blockIdx.x) - P.n_rows) * threads + tid;
    if (t >= P.total) return;
    int lo = 0, hi = P.n_rows;  // the last row that begins at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (P.cu[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    int begin, n;
    row_tokens(P.cu, threads, P.total, lo, begin, n);
    if (t >= begin && t < begin + n) return;
    for (int w = 0; w < P.words; ++w) P.masks[int64_t(t) * P.words + w] = 0;
    P.positions[t] = -1;
    return;
  }
  int begin, n;
  row_tokens(P.cu, threads, P.total, int(blockIdx.x), begin, n);
  const int lane = tid & 63, base = tid - lane;
  if (base < n) {
    int up = kNone;
    uint64_t near = 0;
    if (tid < n) {
      up = P.parents[begin + tid];
      if (up >= tid || up < kRoot) up = kNone;
      near = uint64_t(1) << lane;
    }
#pragma unroll
    for (int step = 0; step < 6; ++step) {  // near: of the nodes from here to `up`, which is left out
      const int from = up >= base ? up - base : lane;
      const uint64_t its = __shfl(near, from, 64);
      const int next = __shfl(up, from, 64);
      near |= up >= base ? its : 0;
      up = up >= base ? next : up;
    }
    s_near[tid] = near;
    s_up[tid] = up;
  }
  __syncthreads();
  if (tid >= n) return;
  const int64_t s0 = P.seqlens[blockIdx.x];
  int a = tid, depth = -1;
  for (; a >= 0; a = s_up[a]) depth += __popcll(s_near[a]);
  const bool ok = a == kRoot && s0 >= 0 && s0 + depth <= kMax31;
  a = ok ? tid : kRoot;
  uint64_t *const line = P.masks + int64_t(begin + tid) * P.words;
  for (int w = P.words - 1; w >= 0; --w) {
    const bool here = a >= 64 * w;  // and before the word past it
    line[w] = here ? s_near[a] : 0;
    a = here ? s_up[a] : a;
  }
  P.positions[begin + tid] = ok ? int(s0 + depth) : -1;
}

struct KeepParams {
  uint4 *k_pages, *v_pages;
  PagedKv kv;  // page_stride in pieces of 16 bytes
  int64_t slot_stride;
  int32_t *table;
  int32_t *seqlens;
  const int32_t *new_lens, *kept, *counts;
  int64_t kept_stride;
  int32_t *free_pages, *free_count;
  int n_rows, units, most;  // most: entries of a line of kept
};

// A row's tokens, its nodes and how many of them it keeps; none where it does not fit its line of the table, or
// where the page of its last node is none of the pool (its nodes were refused).
struct KeptRow {
  int s0, nodes, n;
};
__device__ __forceinline__ KeptRow kept_row(const KeepParams &P, int b) {
  KeptRow r;
  r.s0 = P.seqlens[b];
  r.nodes = max(P.new_lens[b], 0);
  r.n = 0;
  const int64_t end = int64_t(r.s0) + r.nodes;
  if (r.s0 < 0 || end > int64_t(P.kv.max_pages) << P.kv.shift) {
    r.s0 = r.nodes = 0;
    return r;
  }
  if (r.nodes > 0 && P.kv.is_page(P.table[b * P.kv.table_stride + ((end - 1) >> P.kv.shift)]))
    r.n = max(0, min(min(P.counts[b], P.most), r.nodes));
  return r;
}

__global__ __launch_bounds__(256) void keep_kernel(KeepParams P) {
  const int b = blockIdx.y, u = int(blockIdx.x) * 256 + int(threadIdx.x);
  const KeptRow r = kept_row(P, b);
  if (u >= P.units) return;
  uint4 *const pool = (blockIdx.z & 1 ? P.v_pages : P.k_pages) + int64_t(blockIdx.z >> 1) * P.slot_stride + u;
  const int32_t *const line = P.table + b * P.kv.table_stride;
  const int32_t *const kept = P.kept + b * P.kept_stride;
  auto at = [&](int id, int t) { return P.kv.offset(id, P.kv.in_page(t), P.units); };
  for (int j = 0; j < r.n; ++j) {
    const int from = kept[j];
    if (from <= j || from >= r.nodes) continue;
    const int src = line[(r.s0 + from) >> P.kv.shift], dst = line[(r.s0 + j) >> P.kv.shift];
    if (P.kv.is_page(src) && P.kv.is_page(dst)) pool[at(dst, r.s0 + j)] = pool[at(src, r.s0 + from)];
  }
}

__global__ __launch_bounds__(kThreads) void keep_tables_kernel(KeepParams P) {
  __shared__ int64_t s_sum[kWaves], s_end[kThreads], s_first[kThreads];
  const int tid = threadIdx.x;
  const int64_t page = int64_t(1) << P.kv.shift;
  int64_t top = min(max(P.free_count[0], 0), P.kv.n_pages);
  for (int b0 = 0; b0 < P.n_rows; b0 += kThreads) {
    const int b = b0 + tid;
    int64_t back = 0;
    if (b < P.n_rows) {
      const KeptRow r = kept_row(P, b);
      const int64_t has = (int64_t(r.s0) + r.n + page - 1) >> P.kv.shift;
      back = ((int64_t(r.s0) + r.nodes + page - 1) >> P.kv.shift) - has;
      s_first[tid] = b * P.kv.table_stride + has;
      if (r.n > 0) P.seqlens[b] = r.s0 + r.n;
    }
    int64_t all = 0;
    s_end[tid] = group_scan(back, all, s_sum);
    __syncthreads();
    top = push_pages(P.table, s_end, all, top, P.free_pages, P.kv.n_pages, s_sum,
                     [&](int i) { return s_first[i]; });
    __syncthreads();  // s_first and s_end have been read
  }
  if (tid == 0) P.free_count[0] = int(min(top, int64_t(P.kv.n_pages)));
}

}  // namespace
}  // namespace mcamd

using namespace mcamd;

extern "C" int mcamd_paged_tree(const int32_t *parents, const int32_t *cu_seqlens,
                                const int32_t *cache_seqlens, int32_t *positions, uint64_t *masks,
                                int64_t n_rows, int64_t total, int64_t mask_words, void *stream) {
  if (n_rows < 0 || total < 0) return fail(MCAMD_EINVAL, "paged_tree: negative size");
  if (mask_words < 1 || mask_words > kMaxTreeWords)
    return fail(MCAMD_EINVAL, "paged_tree: a node has a mask of 1 to 16 words, 64 of a row's nodes a word");
  if (n_rows >= kMax31 || total > kMax31 - 256)
    return fail(MCAMD_EUNSUPPORTED, "paged_tree: sizes beyond 31 bits");
  if (total == 0) {
    clear_error();
    return MCAMD_OK;
  }
  if (n_rows == 0) return fail(MCAMD_EINVAL, "paged_tree: nodes without a row");
  if (!parents || !cu_seqlens || !cache_seqlens || !positions || !masks)
    return fail(MCAMD_EINVAL, "paged_tree: null pointer");
  if (!aligned(masks, 8)) return fail(MCAMD_EINVAL, "paged_tree: the masks must be 8-byte aligned");
  const TreeParams P{parents, cu_seqlens, cache_seqlens, positions, masks, int(n_rows), int(total), int(mask_words)};
  const int64_t threads = 64 * mask_words, blocks = n_rows + (total + threads - 1) / threads;
  if (blocks > kMax31 / threads) return fail(MCAMD_EUNSUPPORTED, "paged_tree: sizes beyond 31 bits");
  hipLaunchKernelGGL(tree_kernel, dim3(unsigned(blocks)), dim3(unsigned(threads)), 0, as_stream(stream), P);
  return launch_status("paged_tree");
}

extern "C" int mcamd_paged_keep(void *k_pages, void *v_pages, int64_t n_slots, int64_t slot_stride,
                                int32_t *block_table, int64_t table_stride, int32_t *cache_seqlens,
                                const int32_t *new_lens, const int32_t *kept, int64_t max_kept,
                                const int32_t *counts, int32_t *free_pages, int32_t *free_count,
                                int64_t n_rows, int64_t max_pages, int64_t n_pages, int64_t page_size,
                                int64_t page_stride, int64_t row_elems, int dtype, void *stream) {
  KeepParams P{};
  if (dtype != MCAMD_F32 && dtype != MCAMD_BF16)
    return fail(MCAMD_EINVAL, "paged_keep: dtype must be MCAMD_F32 or MCAMD_BF16");
  if (n_slots < 0 || n_rows < 0 || max_kept < 0 || max_pages <= 0 || n_pages <= 0 || row_elems <= 0)
    return fail(MCAMD_EINVAL, "paged_keep: sizes must be positive (n_slots, n_rows, max_kept may be 0)");
  if (!page_shift(page_size, P.kv.shift))
    return fail(MCAMD_EINVAL, "paged_keep: page_size must be a power of two from 16 to 2^30");
  if (table_stride < max_pages) return fail(MCAMD_EINVAL, "paged_keep: table_stride smaller than max_pages");
  if (n_rows > 65535 || n_slots > 32767 || max_kept > kMax31 || n_pages > kMax31 / page_size ||
      max_pages > kMax31 / page_size || row_elems > kMax31 / page_size)
    return fail(MCAMD_EUNSUPPORTED, "paged_keep: more than 65535 rows or 32767 slots, or sizes beyond 31 bits");
  const int64_t elem = dtype == MCAMD_F32 ? 4 : 2;
  const int64_t page_elems = page_size * row_elems;
  if (page_stride < page_elems ||  // the pages before a slot's last one: by a quotient, which stays within 64 bits
      (n_slots > 1 && (slot_stride < page_elems || (slot_stride - page_elems) / page_stride < n_pages - 1)))
    return fail(MCAMD_EINVAL, "paged_keep: page_stride or slot_stride smaller than what it steps over");
  if (n_rows == 0) {
    clear_error();
    return MCAMD_OK;
  }
  if ((n_slots > 0 && (!k_pages || !v_pages)) || !block_table || !cache_seqlens || !new_lens ||
      (max_kept > 0 && !kept) || !counts || !free_pages || !free_count)
    return fail(MCAMD_EINVAL, "paged_keep: null pointer");
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || row_elems * elem % 16 != 0 ||
      page_stride * elem % 16 != 0 || (n_slots > 1 && slot_stride * elem % 16 != 0))
    return fail(MCAMD_EINVAL, "paged_keep: tokens, pages and slots must be 16-byte aligned");
  P.k_pages = static_cast<uint4 *>(k_pages);
  P.v_pages = static_cast<uint4 *>(v_pages);
  P.slot_stride = slot_stride * elem / 16;
  P.kv.table = P.table = block_table;
  P.kv.table_stride = table_stride;
  P.kv.page_stride = page_stride * elem / 16;
  P.kv.n_pages = int(n_pages);
  P.kv.max_pages = int(max_pages);
  P.seqlens = cache_seqlens;
  P.new_lens = new_lens;
  P.kept = kept;
  P.kept_stride = max_kept;
  P.counts = counts;
  P.free_pages = free_pages;
  P.free_count = free_count;
  P.n_rows = int(n_rows);
  P.units = int(row_elems * elem / 16);
  P.most = int(max_kept);
  if (n_slots > 0 && max_kept > 0) {
    const dim3 grid{unsigned((P.units + 255) / 256), unsigned(n_rows), unsigned(2 * n_slots)};
    hipLaunchKernelGGL(keep_kernel, grid, dim3(256), 0, as_stream(stream), P);
    const int st = launch_status("paged_keep");
    if (st != MCAMD_OK) return st;
  }
  hipLaunchKernelGGL(keep_tables_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), P);
  return launch_status("paged_keep");
}
