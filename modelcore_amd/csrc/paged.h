// The paged KV cache as the kernels see it: a pool of pages and, per row, a line of a block table.
//
// Position t of row b lies in page table[b][t >> shift] at token t & (page_size - 1) of it; a page
// holds page_size tokens of (H_kv, D) and pages are page_stride elements apart, so an address is 64
// bits wide in any pool. Page sizes are powers of two from 16 on: a group of 16 keys aligned to 16
// lies in one page, which is what lets a wave take a page per load instead of one per lane.
//
// A number in the table that is no page of the pool (-1 where no page was given) is never followed:
// its keys are read from page 0 and the outputs that see them become NaN.
#pragma once

#include "kernels.h"
#include "prefill_split.h"

namespace mcamd {

constexpr int64_t kMinPageSize = 16, kMaxPageSize = int64_t(1) << 30;

// The power of two that a page size is; false where it is none that the kernels take.
inline bool page_shift(int64_t page_size, int &shift) {
  if (page_size < kMinPageSize || page_size > kMaxPageSize || (page_size & (page_size - 1)) != 0) return false;
  for (shift = 0; (int64_t(1) << shift) < page_size;) ++shift;
  return true;
}

struct PagedKv {
  const int32_t *table;
  int64_t table_stride;  // numbers between rows of the table
  int64_t page_stride;   // elements between pages
  int shift, n_pages, max_pages;

  __device__ __forceinline__ bool is_page(int id) const {
    return uint32_t(id) < uint32_t(n_pages);
  }
  // Elements from the pool's start to token `at` (of page_size) of a page, tok elements a token.
  __device__ __forceinline__ int64_t offset(int id, int at, int64_t tok) const {
    return int64_t(is_page(id) ? id : 0) * page_stride + at * tok;
  }
  __device__ __forceinline__ int in_page(int t) const { return t & ((1 << shift) - 1); }
};

struct PagedArgs {
  const void *q, *k_new, *v_new;  // k_new, v_new: appended (NULL = they are in the pages)
  void *k_pages, *v_pages;
  PagedKv kv;
  const int32_t *seqlens, *cu;  // cu: packed rows of their own lengths; NULL = t_new tokens each
  void *out;
  int64_t n_rows, t_new, total, n_head, n_kv_head, head_dim, window;
  int dtype;
  void *scratch;
  size_t scratch_bytes;
  hipStream_t stream;
};

// The new tokens of row b: [tok0, tok0 + T) of q, and no more than t_new, by which grids and scratch are
// sized, whatever cu holds.
__device__ __forceinline__ void row_tokens(const int32_t *cu, int t_new, int total, int b, int &tok0,
                                           int &T) {
  tok0 = cu ? max(cu[b], 0) : b * t_new;
  T = cu ? min(max(min(cu[b + 1], total) - tok0, 0), t_new) : t_new;
}

// Whether a row of T new tokens is one of few pairs, which the streaming kernels take: a single token, or
// at most `most` (token, head) pairs per KV head; most = 0: none is.
__device__ __forceinline__ bool few_pairs(int T, int G, int most) {
  return most > 0 && (T == 1 || T * G <= most);  // a call's pairs per KV head fit 30 bits
}

// A block of queries of a row: its block qt, the row's tokens and its position.
struct PagedBlock {
  int b, qt, tok0, T, s0;
  int n_blocks;    // of the whole call, its KV heads counted
  int part, most;  // which key range of the block, of how many at most
  bool noted;      // blocks of the call may be cut: the merge is told what each has become
  int half;        // the block is cut in two, whose second range is number `half` of the call; else -1
};

// Inclusive sum over the wave.
__device__ __forceinline__ int wave_upto(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

// Block i of a call, blocks with the most keys first: by their number within their row, last first,
// and rows in order within a number, so that long rows do not fall to one XCD. `pairs` (position,
// head) pairs make a block; rows of few_pairs() by `skip` have none. Each wave does this by itself: the
// rows' lengths and positions are loaded at once and stay in registers, R a lane (rows past 64 R are read
// again), and the number is found by bisection over how many blocks there are from it on. (With the
// found row's numbers read again from memory, and R = 4 for eight rows too, eight prompts of 37 to 4001
// tokens took 2% longer.)
//
// Where the partials of `slots` blocks have room, at most half as many blocks may be cut into key
// ranges: the first ranges of all blocks come first, then the second ones, and so on. With more blocks, of
// packed rows without a window, the deepest ones are cut in two, as many as there are slots left, none of
// half the deepest's keys or less: their second ranges come after all first ones, without gaps, since
// workgroups are dealt to the chip's parts in turn and one that finds no room in its part holds up all
// behind it.
constexpr int kMaxPagedSplits = 32;

struct PagedCall {
  const int32_t *cu, *seqlens;
  int n_rows, t_new, total, G, H_kv, pairs, skip, slots, room, halve;
  // The keys of a row's last block, and of its block qt; 0 for a row that does not fit its line.
  __device__ __forceinline__ int depth_of(int T, int s0) const { return s0 >= 0 && s0 <= room - T ? s0 + T : 0; }
  __device__ __forceinline__ int depth_of(int T, int s0, int qt) const {
    return depth_of(T, s0) == 0 ? 0 : s0 + min(int(uint32_t(qt + 1) * uint32_t(pairs) / uint32_t(G)), T);
  }
  // Blocks of a row, its last ones, that have more than `keys` keys.
  __device__ __forceinline__ int deeper(int T, int s0, int blocks, int keys) const {
    if (blocks == 0 || depth_of(T, s0) <= keys) return 0;
    const int from = max(keys - s0 + 1, 0);  // at most T
    const int shallow = int((uint32_t(from) * uint32_t(G) + uint32_t(pairs) - 1) / uint32_t(pairs)) - 1;
    return blocks - max(shallow, 0);
  }
  __device__ __forceinline__ int blocks_of(int T) const {
    return few_pairs(T, G, skip) ? 0 : int((uint32_t(T * G) + uint32_t(pairs) - 1) / uint32_t(pairs));
  }
  // The key range that i is of, and i's block; false past the last.
  __device__ __forceinline__ bool range_of(int blocks, int &i, PagedBlock &v) const {
    v.n_blocks = blocks * H_kv;
    v.part = 0, v.most = 1, v.half = -1, v.noted = false;
    if (blocks > 0 && slots >= 2 * v.n_blocks) {
      v.most = min(slots / v.n_blocks, kMaxPagedSplits);
      v.part = i / blocks;
      i -= v.part * blocks;
      v.noted = true;
    }
    return i < blocks && v.part < v.most;
  }
};

template <int R>
__device__ __forceinline__ bool find_packed_block(const PagedCall &c, int i, int lane, PagedBlock &v) {
  int tok0[R], T[R], s0[R], mine[R], deepest = 0;
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int b = min(64 * u + lane, c.n_rows - 1);
    row_tokens(c.cu, c.t_new, c.total, b, tok0[u], T[u]);
    s0[u] = c.seqlens[b];
  }
#pragma unroll
  for (int u = 0; u < R; ++u) {
    mine[u] = 64 * u + lane < c.n_rows ? c.blocks_of(T[u]) : 0;
    deepest = max(deepest, mine[u]);
  }
  auto far = [&](int b) {  // of a row past the registers
    if (b >= c.n_rows) return 0;
    int tok, n;
    row_tokens(c.cu, c.t_new, c.total, b, tok, n);
    return c.blocks_of(n);
  };
  // Blocks numbered k or more.
  auto from = [&](int k) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < R; ++u) n += max(mine[u] - k, 0);
    for (int b = 64 * R + lane; b < c.n_rows; b += 64) n += max(far(b) - k, 0);
    return wave_total(n);
  };
  const int blocks = from(0);
  const int spare = c.halve > 0 && c.n_rows <= 64 * R && c.slots < 2 * blocks * c.H_kv
                        ? (c.slots - blocks * c.H_kv) / c.H_kv : 0;
  const bool fits = c.range_of(blocks, i, v);
  int keys = 0, cut[R];  // blocks of more keys are cut in two: so many of each row
  if (spare > 0) {
    v.noted = true;
    int deep = 0;
#pragma unroll
    for (int u = 0; u < R; ++u) deep = max(deep, mine[u] > 0 ? c.depth_of(T[u], s0[u]) : 0);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) deep = max(deep, __shfl_xor(deep, o, 64));
    deep = __builtin_amdgcn_readfirstlane(deep);
    auto all = [&](int k) {
      int n = 0;
#pragma unroll
      for (int u = 0; u < R; ++u) n += cut[u] = c.deeper(T[u], s0[u], mine[u], k);
      return wave_total(n);
    };
    int under = max(deep >> 1, c.halve - 1);
    keys = max(deep, under);
    for (int step = 0; step < 5 && keys - under > 1; ++step) {
      const int mid = (under + keys) >> 1;
      if (all(mid) <= spare)
        keys = mid;
      else
        under = mid;
    }
    const int halves = all(keys);
    if (!fits) {  // the second range of one of them
      int nth = i - blocks;
      if (nth >= halves) return false;
      v.part = 1, v.most = 2, v.half = i;
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const int upto = wave_upto(cut[u], lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > nth);
        if (past == 0) {
          nth -= __builtin_amdgcn_readlane(upto, 63);
          continue;
        }
        const int l = __builtin_ctzll(past);
        v.b = 64 * u + l;
        v.tok0 = __builtin_amdgcn_readlane(tok0[u], l);
        v.T = __builtin_amdgcn_readlane(T[u], l);
        v.s0 = __builtin_amdgcn_readlane(s0[u], l);
        v.qt = __builtin_amdgcn_readlane(mine[u], l) - 1 - (nth - __builtin_amdgcn_readlane(upto - cut[u], l));
        return true;
      }
      return false;
    }
  }
  if (!fits) return false;
  for (int b = 64 * R + lane; b < c.n_rows; b += 64) deepest = max(deepest, far(b));
  int lo = 0, hi = 1;  // more than i blocks from lo on; at most i from hi on
  while (__builtin_amdgcn_ballot_w64(deepest > hi) != 0 && from(hi) > i) lo = hi, hi *= 2;
  while (hi - lo > 1) {
    const int k = (lo + hi) >> 1;
    if (from(k) > i)
      lo = k;
    else
      hi = k;
  }
  v.qt = lo;
  int nth = i - from(lo + 1);  // among the rows that have a block lo
  v.b = -1;
  auto look = [&](int n) {  // the lane of that row among 64, or -1
    uint64_t has = __builtin_amdgcn_ballot_w64(n > lo);
    const int count = __builtin_popcountll(has);
    if (nth >= count) {
      nth -= count;
      return -1;
    }
    for (; nth > 0; --nth) has &= has - 1;
    return int(__builtin_ctzll(has));
  };
#pragma unroll
  for (int u = 0; u < R; ++u) {
    if (v.b >= 0) continue;
    const int l = look(mine[u]);
    if (l < 0) continue;
    v.b = 64 * u + l;
    v.tok0 = __builtin_amdgcn_readlane(tok0[u], l);
    v.T = __builtin_amdgcn_readlane(T[u], l);
    v.s0 = __builtin_amdgcn_readlane(s0[u], l);
  }
  if (v.b >= 0) {
    if (spare > 0 && c.depth_of(v.T, v.s0, v.qt) > keys) {
      int before = 0;  // halves of rows before it
#pragma unroll
      for (int u = 0; u < R; ++u) before += 64 * u + lane < v.b ? cut[u] : 0;
      v.most = 2;
      v.half = blocks + wave_total(before) + c.blocks_of(v.T) - 1 - v.qt;
    }
    return true;
  }
  for (int b0 = 64 * R; b0 < c.n_rows; b0 += 64) {
    const int l = look(far(b0 + lane));
    if (l < 0) continue;
    v.b = b0 + l;
    row_tokens(c.cu, c.t_new, c.total, v.b, v.tok0, v.T);
    v.s0 = c.seqlens[v.b];
    return true;
  }
  return false;
}

__device__ __forceinline__ bool find_paged_block(const int32_t *cu, const int32_t *seqlens, int n_rows,
                                                 int t_new, int total, int G, int H_kv, int pairs,
                                                 int skip, int slots, int room, int halve, int i,
                                                 int lane, PagedBlock &v) {
  const PagedCall c{cu, seqlens, n_rows, t_new, total, G, H_kv, pairs, skip, slots, room, halve};
  if (cu) {
    const bool found =
        n_rows <= 64 ? find_packed_block<1>(c, i, lane, v) : find_packed_block<4>(c, i, lane, v);
    for (int *x : {&v.b, &v.qt, &v.tok0, &v.T, &v.s0, &v.n_blocks, &v.part, &v.most, &v.half})
      *x = __builtin_amdgcn_readfirstlane(*x);  // so the compiler knows as well
    v.noted = __builtin_amdgcn_readfirstlane(v.noted);
    return __builtin_amdgcn_readfirstlane(found);
  }
  const int each = c.blocks_of(t_new);
  if (!c.range_of(each * n_rows, i, v)) return false;
  v.qt = each - 1 - i / n_rows;
  v.b = i % n_rows;
  row_tokens(cu, t_new, total, v.b, v.tok0, v.T);
  v.s0 = seqlens[v.b];
  return true;
}

// At most so many blocks of `pairs` pairs in a call's rows that are not of few_pairs(.., skip).
inline int64_t paged_blocks_bound(const PagedArgs &a, int64_t pairs, int64_t skip) {
  const int64_t G = a.n_head / a.n_kv_head;
  if (!a.cu) return a.n_rows * ((a.t_new * G + pairs - 1) / pairs);
  const int64_t shortest = skip > 0 ? (skip / G > 1 ? skip / G : 1) + 1 : 1;  // tokens of such a row
  const int64_t rows = a.total / shortest < a.n_rows ? a.total / shortest : a.n_rows;
  return a.total * G / pairs + rows;
}

// What the tiled kernels of long rows share beyond their own parameters.
struct PagedTiles {
  PagedKv kv;
  int n_rows, total;
  int skip;         // rows of few_pairs() by it are another launch's
  int kt;           // keys of a tile
  int groups;       // of 32 pairs, of a block
  int slots;        // blocks for whose partials there is room, or 0: no block is cut
  float ratio;      // prefill_split.h's, times the blocks of the call
  int min_tiles;    // of a range, about
  int halve;        // keys from which on a block may be cut in two, or 0: none is
  float *part_o;    // [slot][groups of 32 pairs][md][4][64][4], as SplitGeo lays them out
  float *part_ml;   // [slot][groups][32][2]
  struct Cut {      // a block, for the merge
    int b, qt, tok0, T, s0, ranges, second, unused;  // second: the slot of its second range
  };
  Cut *cuts;        // [slots]: the blocks of a call that may be cut, by their number
  int *n_cuts;      // and how many

  // Ranges of a block of n tiles: what pays for their partials, by the cost rule of prefill_split.h, none
  // much shorter than what starting it takes.
  __device__ __forceinline__ int ranges_of(const PagedBlock &v, int n) const {
    if (v.half >= 0) return 2;
    const int most = min(v.most, n / min_tiles), s = int(sqrtf(float(n) * ratio / float(v.n_blocks)));
    return max(1, min(s, most));
  }
  // Left for the merge by a call's first workgroup, and by the first range of each block.
  __device__ __forceinline__ void note_call(bool found, const PagedBlock &v) const {
    if (slots > 0) *n_cuts = found && v.noted ? v.n_blocks : 0;
  }
  __device__ __forceinline__ void note_block(int id, const PagedBlock &v, int ranges, int H_kv) const {
    cuts[id] = Cut{v.b, v.qt, v.tok0, v.T, v.s0, ranges,
                   v.half >= 0 ? v.half * H_kv + id % H_kv : id + v.n_blocks, 0};
  }
};

// Keys of a block, at most: by the width of the table's lines, since the rows' lengths are the device's.
inline int64_t paged_keys(const PagedArgs &a) {
  const int64_t room = int64_t(a.kv.max_pages) << a.kv.shift;
  return a.window < 0 ? room : std::min<int64_t>(room, a.window + 256 + 64);
}

// Room for the partials of `per_cu` workgroups per compute unit, where a call of at most `blocks` blocks can
// have so few that ranges of some run side by side, and a block keys for two of min_keys. Uniform rows have
// that many blocks, packed ones about as many as their tokens fill, or more.
inline int paged_slots(const PagedArgs &a, int64_t blocks, int64_t pairs, int per_cu, int64_t min_keys) {
  const int64_t slots = int64_t(per_cu) * device_cus();
  const int64_t least = (a.cu ? a.total * (a.n_head / a.n_kv_head) / pairs : 2 * blocks) * a.n_kv_head;
  return least <= slots && paged_keys(a) >= 2 * min_keys ? int(slots) : 0;
}

inline size_t paged_tiles_bytes(int64_t slots, int64_t slot_floats) {
  return slots == 0 ? 0 : size_t(slots) * size_t(slot_floats) * 4 + size_t(slots) * sizeof(PagedTiles::Cut) + 16;
}
// Lays out the scratch of a call with so many slots, if it is large enough; else no block is cut.
inline void paged_tiles_buffers(const PagedArgs &a, PagedTiles &t, int64_t slots, int64_t slot_floats,
                                int64_t ml_floats) {
  t.slots = a.scratch && a.scratch_bytes >= paged_tiles_bytes(slots, slot_floats) ? int(slots) : 0;
  t.part_o = static_cast<float *>(a.scratch);
  t.part_ml = t.part_o + t.slots * (slot_floats - ml_floats);
  t.cuts = reinterpret_cast<PagedTiles::Cut *>(t.part_o + t.slots * slot_floats);
  t.n_cuts = reinterpret_cast<int *>(t.cuts + t.slots);
  t.halve = a.window < 0 ? 2 * t.min_tiles * t.kt : 0;
}

// Rows of few pairs (few_pairs(.., most)) of a bf16 call: append where k_new is given, with `others` of the
// other rows too, and attention.
int launch_paged_stream(const PagedArgs &a, int64_t most, bool others);
size_t paged_stream_bytes(const PagedArgs &a, int64_t most);  // of scratch, to cut long rows' keys
// Single tokens of an fp32 call, the same.
int launch_paged_stream_f32(const PagedArgs &a, bool others);
size_t paged_stream_f32_bytes(const PagedArgs &a);
// Every row but those, whose new tokens are in their pages.
int launch_paged_tiled(const PagedArgs &a, int64_t skip);
size_t paged_tiled_bytes(const PagedArgs &a, int64_t skip);
// The same for bf16 and head_dim 128.
bool paged_mfma_supported(const PagedArgs &a);
int launch_paged_mfma(const PagedArgs &a, int64_t skip);
size_t paged_mfma_bytes(const PagedArgs &a, int64_t skip);
// The ranges of cut blocks (of `pairs` pairs) added up.
int launch_paged_tiles_merge(const PagedArgs &a, const PagedTiles &t, int pairs, int64_t bound);

}  // namespace mcamd
