// Which keys a node of a drafted tree sees.
//
// The T new tokens of a row that holds s0 are nodes 0 .. T - 1, in its pages at s0 + i. Bit j of node i's
// mask (64 a word) says that j is i itself or an ancestor; bits past i do not count. Node i stands at position
// s0 + depth, depth being the number of its bits less one. It sees the row's tokens c < s0 and the
// nodes of its bits, with a window only those at most `window` positions before it: of the tokens the last
// ones, of its bits the window + 1 highest, since an ancestor's index and its depth rise together.
//
// The word with a node's own bit is kept, the others are read from memory where they are needed, which is in
// tiles that hold nodes or the window's edge: a handful of a row's tiles.
#pragma once

#include "common.h"

namespace mcamd {

constexpr int64_t kMaxTreeWords = 16;  // of 64 nodes

struct TreeMasks {
  const uint64_t *masks;  // (tokens, words)
  int words;
};

struct TreeNode {
  const uint64_t *line;
  uint64_t mine;  // the word with the node's own bit, less the bits past it
  int words, node, s0, window, pos;

  // That word as it stands, to be asked for early.
  static __device__ __forceinline__ uint64_t own_word(const TreeMasks &m, int64_t token, int node) {
    return node >> 6 < m.words ? m.masks[token * m.words + (node >> 6)] : 0;
  }
  __device__ __forceinline__ TreeNode() {}
  __device__ __forceinline__ TreeNode(const TreeMasks &m, int64_t token, int node_, int s0_, int window_)
      : TreeNode(m, token, node_, s0_, window_, own_word(m, token, node_)) {}
  __device__ __forceinline__ TreeNode(const TreeMasks &m, int64_t token, int node_, int s0_, int window_, uint64_t own)
      : line(m.masks + token * m.words),
        mine(own & ~uint64_t(0) >> (63 - (node_ & 63))),
        words(m.words),
        node(node_),
        s0(s0_),
        window(window_) {
    int n = __popcll(mine);
    for (int k = 0; k < node >> 6; ++k) n += __popcll(word(k));
    pos = s0 + n - 1;
  }
  // Word k, less the bits past the node's own.
  __device__ __forceinline__ uint64_t word(int k) const {
    const int own = node >> 6;
    if (k < 0 || k > own || k >= words) return 0;
    return k == own ? mine : line[k];
  }
  // The first key that may be seen.
  __device__ __forceinline__ int first() const { return window >= 0 ? max(0, min(s0, pos - window)) : 0; }
  // Bit x: key k0 + x is seen.
  __device__ __forceinline__ uint64_t seen(int k0) const {
    const int n = s0 - k0;  // keys of the row's tokens from k0 on
    uint64_t bits = 0;
    if (n < 64) {
      const int k = -n >> 6, r = -n & 63;
      bits = word(k) >> r | (r ? word(k + 1) << (64 - r) : 0);
      if (window >= 0 && window < node) {
        int keep = window + 1;  // bits, the highest first
        for (int j = (node >> 6) + 1; j > k + 1; --j) keep -= __popcll(word(j));
        keep -= __popcll(word(k + 1) >> r);  // those past the tile's 64
        for (int over = __popcll(bits) - max(keep, 0); over > 0; --over) bits &= bits - 1;
      }
    }
    uint64_t tokens = n >= 64 ? ~uint64_t(0) : n > 0 ? ~(~uint64_t(0) << n) : 0;
    if (window >= 0) {
      const int skip = pos - window - k0;
      tokens &= skip >= 64 ? 0 : skip > 0 ? ~uint64_t(0) << skip : ~uint64_t(0);
    }
    return tokens | bits;
  }
};

}  // namespace mcamd
