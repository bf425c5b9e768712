// The attention operator over a paged cache: its argument checks, the append of new tokens into
// their pages, and which kernels a call takes.
#include "paged_append.h"

#include <algorithm>
#include <cmath>

namespace mcamd {
namespace {

__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(PagedAppend A) {
  append_tokens(A, blockIdx.x);
}

int check(const PagedArgs &a) {
  if (a.dtype != MCAMD_F32 && a.dtype != MCAMD_BF16)
    return fail(MCAMD_EINVAL, "paged attention: dtype must be MCAMD_F32 or MCAMD_BF16");
  if (a.n_rows < 0 || a.t_new < 0 || a.total < 0 || a.n_head <= 0 || a.n_kv_head <= 0 ||
      a.head_dim <= 0)
    return fail(MCAMD_EINVAL, "paged attention: sizes must be positive (rows and tokens may be 0)");
  if (a.n_kv_head > a.n_head || a.n_head % a.n_kv_head != 0)
    return fail(MCAMD_EINVAL, "paged attention: n_head must be a multiple of n_kv_head");
  const int64_t elem = a.dtype == MCAMD_F32 ? 4 : 2;
  if (a.head_dim > 256 || a.head_dim * elem % 16 != 0)
    return fail(MCAMD_EUNSUPPORTED,
                "paged attention: head_dim must be at most 256, its bytes a multiple of 16");
  if (a.n_head / a.n_kv_head > 64)
    return fail(MCAMD_EUNSUPPORTED, "paged attention: more than 64 query heads per KV head");
  if (!a.q || !a.out || !a.k_pages || !a.v_pages || !a.kv.table || !a.seqlens)
    return a.n_rows > 0 && a.total > 0 ? fail(MCAMD_EINVAL, "paged attention: null pointer") : MCAMD_OK;
  if ((int64_t(a.n_kv_head) << a.kv.shift) * a.head_dim * elem > 0x7fffffff)
    return fail(MCAMD_EUNSUPPORTED, "paged attention: a page of more than 2 GiB");
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || !aligned(a.k_pages, 16) ||
      !aligned(a.v_pages, 16) || (a.k_new && !aligned(a.k_new, 16)) ||
      (a.v_new && !aligned(a.v_new, 16)) || a.kv.page_stride * elem % 16 != 0 ||
      !aligned(a.scratch, 16))
    return fail(MCAMD_EINVAL, "paged attention: tensors must be 16-byte aligned");
  return MCAMD_OK;
}

// Pairs per KV head up to which a row counts as one of few pairs (few_pairs()): one block of the bf16
// streaming kernel, and single tokens for the fp32 one.
int64_t few_of(const PagedArgs &a) { return a.dtype == MCAMD_BF16 ? 32 : 1; }

struct Kernels {
  bool stream, tiles;
};
Kernels kernels_of(const PagedArgs &a) {
  const int64_t G = a.n_head / a.n_kv_head;
  const bool few = a.t_new == 1 || a.t_new * G <= few_of(a);  // of every row
  return {few || a.cu != nullptr, !few};
}

// New tokens of a mixed call up to which the streaming kernel's launch appends those of the long rows too.
// Three rows of 97 tokens 12.6 us in two launches, 10.4 in one; 60 single tokens beside four chunks, 2100
// tokens, 171 and 179, eight prompts of 16384 18 and 23: more workgroups stand in the way of ranges that
// are all to be on the chip at once.
constexpr int64_t kAppendWithin = 512;

int launch(PagedArgs a) {
  const Kernels k = kernels_of(a);
  const bool within = k.stream && (!k.tiles || a.total <= kAppendWithin);
  if (a.k_new && !within) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(unsigned(paged_append_blocks(a))), dim3(kAppendThreads), 0,
                       a.stream, paged_append(a, 0));
    const int st = launch_status("paged_append");
    if (st != MCAMD_OK) return st;
    a.k_new = a.v_new = nullptr;
  }
  if (k.stream) {
    const int st = a.dtype == MCAMD_BF16 ? launch_paged_stream(a, few_of(a), k.tiles)
                                         : launch_paged_stream_f32(a, k.tiles);
    if (st != MCAMD_OK || !k.tiles) return st;
  }
  const int64_t skip = k.stream ? few_of(a) : 0;
  return paged_mfma_supported(a) ? launch_paged_mfma(a, skip) : launch_paged_tiled(a, skip);
}

}  // namespace
}  // namespace mcamd

using namespace mcamd;

extern "C" size_t mcamd_paged_scratch_bytes(int64_t n_rows, int64_t total, int64_t max_seqlen,
                                            int64_t n_head, int64_t n_kv_head, int64_t head_dim,
                                            int64_t max_pages, int64_t page_size, int64_t window,
                                            int dtype) {
  if (n_rows <= 0 || total <= 0 || max_seqlen <= 0 || n_kv_head <= 0 || n_head < n_kv_head ||
      head_dim <= 0 || head_dim > 256 || max_pages <= 0 || n_head > 65535 || n_rows > 65535 ||
      total > (int64_t(1) << 30) / n_head)
    return 0;
  PagedArgs a{};
  if (!page_shift(page_size, a.kv.shift) || max_pages > (int64_t(1) << 30) / page_size) return 0;
  a.kv.max_pages = int(max_pages);
  a.n_rows = n_rows;
  a.t_new = std::min(max_seqlen, total);  // no row has more, and 31 bits hold it
  a.total = total;
  a.n_head = n_head;
  a.n_kv_head = n_kv_head;
  a.head_dim = head_dim;
  a.window = std::min(window, int64_t(1) << 30);  // no position is past it
  a.dtype = dtype;
  // The sizes do not tell packed rows from uniform ones: room for both.
  const int32_t packed = 0;
  size_t most = 0;
  for (const int32_t *cu : {(const int32_t *)nullptr, &packed}) {
    a.cu = cu;
    const Kernels k = kernels_of(a);
    const int64_t skip = k.stream ? few_of(a) : 0;
    if (k.stream)
      most = std::max(most, a.dtype == MCAMD_BF16 ? paged_stream_bytes(a, few_of(a)) : paged_stream_f32_bytes(a));
    if (k.tiles)
      most = std::max(most, paged_mfma_supported(a) ? paged_mfma_bytes(a, skip) : paged_tiled_bytes(a, skip));
  }
  return most;
}

extern "C" int mcamd_flash_attn_paged_with_kvcache(
    const void *q, const void *k, const void *v, void *k_pages, void *v_pages,
    const int32_t *block_table, int64_t table_stride, const int32_t *cache_seqlens,
    const int32_t *cu_seqlens, void *out, int64_t n_rows, int64_t total, int64_t max_seqlen,
    int64_t n_head, int64_t n_kv_head, int64_t head_dim, int64_t n_pages, int64_t page_size,
    int64_t page_stride, int64_t max_pages, int64_t window, int causal, int dtype, void *scratch,
    size_t scratch_bytes, void *stream) {
  (void)causal;
  if ((k == nullptr) != (v == nullptr))
    return fail(MCAMD_EINVAL, "flash_attn_paged_with_kvcache: pass both k and v, or neither");
  PagedArgs a{};
  if (!page_shift(page_size, a.kv.shift))
    return fail(MCAMD_EINVAL, "paged attention: page_size must be a power of two from 16 to 2^30");
  if (n_pages <= 0 || max_pages <= 0 || max_seqlen < 0)
    return fail(MCAMD_EINVAL, "paged attention: empty pool or block table, or negative max_seqlen");
  if (n_pages > 0x7fffffff / page_size || max_pages > (int64_t(1) << 30) / page_size ||
      n_rows > 65535 || n_head > 65535 || n_kv_head > 65535 || head_dim > 65535 ||
      total > (int64_t(1) << 30) / (n_head > 0 ? n_head : 1) ||
      (!cu_seqlens && max_seqlen > int64_t(1) << 30))
    return fail(MCAMD_EUNSUPPORTED, "paged attention: sizes beyond the 32-bit index range of the kernels");
  if (page_stride < page_size * n_kv_head * head_dim)
    return fail(MCAMD_EINVAL, "paged attention: page_stride smaller than page_size*H_kv*D");
  if (table_stride < max_pages)
    return fail(MCAMD_EINVAL, "paged attention: table_stride smaller than max_pages");
  if (!cu_seqlens && total != n_rows * max_seqlen)
    return fail(MCAMD_EINVAL, "paged attention: without cu_seqlens every row has max_seqlen tokens");
  a.q = q;
  a.k_new = k;
  a.v_new = v;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.kv.table = block_table;
  a.kv.table_stride = table_stride;
  a.kv.page_stride = page_stride;
  a.kv.n_pages = int(n_pages);
  a.kv.max_pages = int(max_pages);
  a.seqlens = cache_seqlens;
  a.cu = cu_seqlens;
  a.out = out;
  a.n_rows = n_rows;
  a.t_new = std::min(max_seqlen, total);  // no row has more, and 31 bits hold it
  a.total = total;
  a.n_head = n_head;
  a.n_kv_head = n_kv_head;
  a.head_dim = head_dim;
  a.window = std::min(window, int64_t(1) << 30);  // no position is past it
  a.dtype = dtype;
  a.scratch = scratch;
  a.scratch_bytes = scratch_bytes;
  a.stream = as_stream(stream);
  const int st = check(a);
  if (st != MCAMD_OK) return st;
  if (n_rows == 0 || total == 0 || max_seqlen == 0) {
    clear_error();
    return MCAMD_OK;
  }
  return launch(a);
}
