// The redo of a (position, head) pair whose result is not finite, over a paged cache.
//
// The matrix-core kernels multiply masked keys' values by a weight of zero, so an infinity or NaN in V
// would reach pairs that may not see it. Such a pair is computed again here over the keys it sees alone,
// with the formula as it stands: an infinity or NaN it does see reaches it, a NaN key makes it NaN, and so
// does a key in a page outside the pool.
#pragma once

#include "paged.h"

namespace mcamd {
namespace {

struct CarefulParams {
  const void *q, *k_pages, *v_pages;
  PagedKv kv;
  void *out;
  int H_kv, window, D;
  float scale_log2;
  TreeMasks tree;  // of calls over trees
  const void *k_new, *v_new;  // theirs: the nodes, which need not be in their pages yet; or null
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Dims [d0, d1) of one pair redone by a wave over the keys it sees alone, for pairs whose result is not
// finite: 64 keys a step, a key per lane for its score, then a dim per lane (l, l + 64, ..) for the sums.
template <class E, int DP, int LOADS = 32, bool TREE = false>  // LOADS: values (and 16-byte pieces of keys) in flight
__device__ void careful_pair(const CarefulParams &P, int row, int kvh, int64_t at, int p, int lane,
                             int d0, int d1, int64_t token = 0, int node = 0) {
  constexpr int N = (DP + 63) / 64, VEC = Vec<E>::N, U = N == 3 ? LOADS / 4 : LOADS / N;
  static_assert(64 % U == 0, "whole batches per step");
  const int D = P.D;
  const E *q = static_cast<const E *>(P.q) + at;
  E *out = static_cast<E *>(P.out) + at;
  const int64_t tok = int64_t(P.H_kv) * D;
  const E *kc = static_cast<const E *>(P.k_pages) + int64_t(kvh) * D;
  const E *vc = static_cast<const E *>(P.v_pages) + int64_t(kvh) * D;
  const int32_t *pages = P.kv.table + row * P.kv.table_stride;
  // Where key t has its key, from kc on, or its value, from vc on.
  auto from = [&](const E *cache, const void *fresh, int t) {
    if constexpr (TREE)
      if (fresh && t >= p - node)
        return static_cast<const E *>(fresh) + (token - p + t) * tok + int64_t(kvh) * D;
    return cache + P.kv.offset(pages[t >> P.kv.shift], P.kv.in_page(t), tok);
  };
  float o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;  // l: of this lane's keys
  int first = key_lo(p, P.window);
  TreeNode N_;  // TREE: node `node` of its row, token `token` of the call
  if constexpr (TREE) {
    N_ = TreeNode(P.tree, token, node, p - node, P.window);
    first = N_.first();
  }
  for (int t0 = first; t0 <= p; t0 += 64) {
    const int t = min(t0 + lane, p);
    const E *k_at = from(kc, P.k_new, t);
    float s = 0.f;
    constexpr int KU = DP / VEC < LOADS / 4 ? DP / VEC : LOADS / 4;
    for (int c0 = 0; c0 < D; c0 += KU * VEC) {
      uint4 y[KU];
#pragma unroll
      for (int c = 0; c < KU; ++c)
        y[c] = *reinterpret_cast<const uint4 *>(k_at + min(c0 + c * VEC, D - VEC));
#pragma unroll
      for (int c = 0; c < KU; ++c) {
        float x[VEC], z[VEC], dot = s;
        Vec<E>::load(q + min(c0 + c * VEC, D - VEC), x);
        Vec<E>::unpack(y[c], z);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dot = fmaf(x[e] * P.scale_log2, z[e], dot);
        s = c0 + c * VEC < D ? dot : s;
      }
    }
    bool hidden = t0 + lane > p;
    if constexpr (TREE) hidden = hidden || !((N_.seen(t0) >> lane) & 1);
    if (hidden) s = -INFINITY;
    if ((!TREE || !hidden) && !P.kv.is_page(pages[t >> P.kv.shift])) s = NAN;
    if (__builtin_amdgcn_ballot_w64(s != s) != 0) {  // a NaN key makes the output NaN, as in the softmax
      l = NAN;
      break;
    }
    const float m_new = fmaxf(m, wave_max<64>(s));
    if (m_new == -INFINITY) continue;
    const float corr = fast_exp2(m - m_new), w = fast_exp2(s - m_new);
    m = m_new;
    l = fmaf(l, corr, s == -INFINITY ? 0.f : w);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= corr;
    const uint64_t seen = __builtin_amdgcn_ballot_w64(s != -INFINITY);
    for (int k0 = 0; k0 < min(64, p - t0 + 1); k0 += U) {
      E v[U][N];  // without a branch between the loads: lanes without a dim take a neighbour's
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i)
          v[u][i] = from(vc, P.v_new, min(t0 + k0 + u, p))[max(d0, min(lane + 64 * i, d1 - 1))];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float wk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), k0 + u));
        const bool there = (seen >> (k0 + u)) & 1;  // a weight of zero must not meet an infinity
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = there ? fmaf(wk, to_f32<E>(v[u][i]), o[i]) : o[i];
      }
    }
  }
  const float all = wave_sum<64>(l);
  const float inv = TREE && all == 0.f ? 0.f : 1.f / all;  // a node that sees no key at all gets zeros
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 64 * i >= d0 && lane + 64 * i < d1) out[lane + 64 * i] = from_f32<E>(o[i] * inv);
}

}  // namespace
}  // namespace mcamd
