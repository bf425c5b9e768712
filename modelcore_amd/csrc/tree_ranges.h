// How a call over drafted trees is dealt to the workgroups of tree_stream.hip and paged_tiled.hip: each takes a key
// range of one block of a row's (node, head) pairs.
//
// A row's nodes all see its tokens, so its blocks have the same tiles, and rows differ in how many. All ranges are
// to be on the chip at once, none longer than it must be: `len`, the most tiles of a range, is the least for
// which there are no more ranges than `target` workgroups (a KV head each), found by bisection over the sum of the
// rows' ceil(tiles / len). With more blocks than that, or more rows than a wave has lanes, it is the work over what
// is left, which is at most twice that. Every wave does this sum by itself, 64 rows at a time. 32 rows of 16 nodes
// after 512 to 8191 tokens, 16 / 4 heads of 128, on the kernel of 256 pairs: 104 us, 133 by the rule for sequences
// (paged.h), which cuts by what each row has to give. Equal shares of all rows' tiles, of which a workgroup may have
// the end of one block and the beginning of another, took 8 us for each such change and gave nothing: 77 us for
// 76 in tree_stream.hip.
#pragma once

#include "paged.h"

#include <algorithm>

namespace mcamd {

// Inclusive sum over the wave, by moves between lanes.
__device__ __forceinline__ int wave_scan32(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
// ceil(x / y) of x up to 2^26, y > 0: the quotient of floats is off by at most two.
__device__ __forceinline__ int ceil_of(int x, int y) {
  int q = int(float(x) * __builtin_amdgcn_rcpf(float(y)));
  const int r = x - q * y;  // of -2 y to 3 y
  q += (r > 0) + (r > y) + (r > 2 * y);
  q -= (r <= -y) + (r <= -2 * y);
  return q;
}

struct TreeRanges {
  const int32_t *cu, *seqlens;
  int n_rows, t_new, total, G, H_kv, pairs, skip, room, window, kt;
  int target, min_tiles;  // target 0: no row is cut

  struct Row {
    int tok0, T, s0, blocks, tiles;
  };
  __device__ __forceinline__ Row row_of(int b) const {
    Row r;
    row_tokens(cu, t_new, total, b, r.tok0, r.T);
    r.s0 = seqlens[b];
    r.blocks = few_pairs(r.T, G, skip) ? 0 : ceil_of(r.T * G, pairs);
    const bool ok = r.s0 >= 0 && r.s0 <= room - r.T;
    const int lo = window >= 0 ? max(0, r.s0 - 1 - window) : 0;
    r.tiles = ok ? int((uint32_t(r.s0 + r.T - lo) + uint32_t(kt) - 1) / uint32_t(kt)) : 1;  // a shift
    return r;
  }
  static __device__ __forceinline__ int ranges_of(const Row &r, int len) {
    return len >= r.tiles ? 1 : ceil_of(r.tiles, len);
  }
  static __device__ __forceinline__ int64_t wave_total64(int64_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
  }

  // Tiles of a range, at most. first: row `lane`.
  __device__ __forceinline__ int len_of(int lane, const Row &first) const {
    if (target == 0) return 0x7fffffff;
    const int slots = max(target / H_kv, 1);
    if (n_rows <= 64) {
      const int blocks = lane < n_rows ? first.blocks : 0, units = wave_total(blocks);
      if (units <= slots && __builtin_amdgcn_ballot_w64(blocks > 0 && first.tiles > 1 << 14) == 0) {
        const int work = wave_total(blocks * first.tiles);  // at most 1024 blocks of 2^14 tiles
        int less = max(ceil_of(work, slots), min_tiles) - 1;  // has more ranges, or is too short
        // work / len whole ranges and up to one more a block are no more than that.
        int len = slots > units ? max(ceil_of(work, slots - units), min_tiles) : 1 << 14;
        for (int step = 0; step < 8 && len - less > 1; ++step) {
          const int mid = less + (len - less) / 2;
          if (wave_total(blocks * ranges_of(first, mid)) <= slots)
            len = mid;
          else
            less = mid;
        }
        return __builtin_amdgcn_readfirstlane(len);
      }
    }
    int64_t work = 0, units = 0;
    for (int b = lane; b < n_rows; b += 64) {
      const Row r = b == lane ? first : row_of(b);
      work += int64_t(r.blocks) * r.tiles;
      units += r.blocks;
    }
    work = wave_total64(work);
    units = wave_total64(units);
    const int64_t most = units < slots / 2 ? slots - units : (slots + 1) / 2;
    return __builtin_amdgcn_readfirstlane(int(max((work + most - 1) / most, int64_t(min_tiles))));
  }
};

// A workgroup's range. `slot`: the first of its block's partials, of which there are ranges (times H_kv); `cut`:
// the number of its block among those that are cut. n_blocks: how many those are, of the whole call.
struct TreeRange : PagedBlock {
  int ranges, slot, cut;
};

// Range `id` of a call; false past the last.
__device__ __forceinline__ bool find_tree_range(const TreeRanges &c, int id, int lane, TreeRange &v) {
  const TreeRanges::Row mine = c.row_of(min(lane, c.n_rows - 1));
  const int len = c.len_of(lane, mine);
  v.b = -1;
  v.n_blocks = 0;
  int slots = 0;
  for (int b0 = 0; b0 < c.n_rows; b0 += 64) {
    TreeRanges::Row r = mine;
    if (b0 > 0) r = c.row_of(min(b0 + lane, c.n_rows - 1));
    const int blocks = b0 + lane < c.n_rows ? r.blocks : 0;
    const int ranges = c.target == 0 ? 1 : TreeRanges::ranges_of(r, len);
    const int n = ranges * blocks, n_cut = ranges > 1 ? n : 0, cuts = ranges > 1 ? blocks : 0;
    const int upto = wave_scan32(n), cut_upto = wave_scan32(n_cut), cuts_upto = wave_scan32(cuts);
    const uint64_t past = v.b < 0 ? __builtin_amdgcn_ballot_w64(upto > id) : 0;
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      v.b = b0 + l;
      id -= __builtin_amdgcn_readlane(upto - n, l);
      v.ranges = __builtin_amdgcn_readlane(ranges, l);
      v.tok0 = __builtin_amdgcn_readlane(r.tok0, l);
      v.T = __builtin_amdgcn_readlane(r.T, l);
      v.s0 = __builtin_amdgcn_readlane(r.s0, l);
      v.qt = int(uint32_t(id) / uint32_t(v.ranges));
      v.part = id - v.qt * v.ranges;
      v.slot = slots + __builtin_amdgcn_readlane(cut_upto - n_cut, l) + v.qt * v.ranges;
      v.cut = v.n_blocks + __builtin_amdgcn_readlane(cuts_upto - cuts, l) + v.qt;
    } else {
      id -= v.b < 0 ? __builtin_amdgcn_readlane(upto, 63) : 0;
    }
    slots += __builtin_amdgcn_readlane(cut_upto, 63);
    v.n_blocks += __builtin_amdgcn_readlane(cuts_upto, 63);
  }
  v.noted = v.b >= 0 && v.ranges > 1;
  v.most = v.noted ? v.ranges : 1;
  v.half = -1;
  return v.b >= 0;
}

// Where cut blocks of a tree call have their partials, and what the merge is told of them.
__device__ __forceinline__ void note_tree_range(const PagedTiles &t, const TreeRange &v, int kvh, int H_kv, int ranges) {
  t.cuts[int64_t(v.cut) * H_kv + kvh] =
      PagedTiles::Cut{v.b, v.qt, v.tok0, v.T, v.s0, ranges, v.slot * H_kv + kvh, 0};
}

// Ranges that the cut blocks of such a call have at most, KV heads counted: those of all blocks where they are
// bisected or few; else a cut one's ceil(tiles / len) is less than twice tiles / len, and the work over len
// half of the target and one.
inline int64_t tree_slots(int64_t target, int64_t n_kv_head) {
  return std::max(target, n_kv_head) + n_kv_head;
}
// Workgroups of a call of at most `bound` blocks.
inline int64_t tree_blocks(int64_t bound, int64_t target, int64_t n_kv_head) {
  return (bound + std::max<int64_t>(target / n_kv_head, 1)) * n_kv_head;
}

}  // namespace mcamd
