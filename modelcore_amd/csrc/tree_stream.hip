// Attention of drafted trees over a paged bf16 cache, for rows of more (node, head) pairs per KV head than a wave
// holds: every key and value is read once for 128 pairs (64) and put through the matrix cores for all of them.
//
// A workgroup has a key range of one block of pairs of a KV head (tree_ranges.h): 128 pairs, or 64 where no row has
// more. A wave holds 32 of them, and the waves share the keys of a tile, 16 of which each loads: straight from
// HBM to LDS (buffer loads, whole rows of a page), K and V, one tile while the one before is used; the 16 share a
// page, so that a load's page is one scalar. One barrier a tile. At the end the waves of the same pairs join their
// sums in LDS.
//   S^T (keys x pairs) = K . Q^T     v_mfma_f32_32x32x16_bf16, two independent sums of 32 keys
//   O^T (D x pairs)   += V^T . P^T   V^T by LDS transpose reads
// in the layouts of paged_stream.hip, a pair per lane. Scores, statistics and sums are fp32, q enters as it is,
// the weights as two bf16 terms, p = hi + lo, which keep them to 2^-17, as in paged_stream.hip and the tiled kernel: a
// row is as exact beside wide trees as alone, and as a tree as a sequence. With hi alone the outputs were 2.3e-3 of
// their norm off instead of the 1.7e-3 of their own rounding, for a third fewer products: one row of 64 nodes after
// 16384 tokens, 32 / 8 heads of 128, 35.2 us for 42.1; 32 rows of 16 nodes, 16 / 4 heads, bound by HBM, 73.8 for 74.2.
//
// One row of 64 nodes after 16384 tokens, 32 / 8 heads of 128: 36 us and 5.5 for the merge; of 1024 nodes 394 us, 698
// TFLOP/s of the formula's products and half as many again for the second term: 1047. 32 rows of 16 nodes after 512 to
// 8191, 16 / 4 heads: 66 us and 8.5 (4.2 TB/s). A tile of 128 keys takes eight waves of 128 pairs 3.1 us, which is what
// its LDS reads, its products and its softmax take one after another (0.85, 1.3 and 0.9 us at their full rates): the
// waves of a workgroup pass through them together. Reads ahead of the products and waves' priorities changed nothing
// when the weights had one term (2.4 us). Of the rest, finding the range takes 1.7 us, queries, pages and the first tile
// 3.7, the sums' way out 3. Blocks of 64 pairs run at 6.2 TB/s while they read; the longest range ends 9 us after the
// median one.
//
// Who sees whom: tree_bits.h, only in tiles that hold nodes or the window's edge. New nodes come from k_new and
// v_new where given, and a block's last range puts its own in their pages. A block of one range writes its
// output; otherwise (o, m, l) go to scratch in fp32 and the merge launch adds the ranges up. Pairs that are not finite
// are redone (paged_careful.h).
#include "range_tiles.h"
#include "stream_tiles.h"
#include "tree_ranges.h"

#include <type_traits>

namespace mcamd {
namespace {

constexpr int kMinRangeKeys = 256;        // of a range, unless the row is shorter
constexpr float kTileSumLimit = 32768.f;  // 2^15: a lane's weights of one tile sum to at most this
// Waves of a workgroup, and how many of those a compute unit holds. Blocks of 128 pairs have eight waves, so that
// half as many partials are written and merged (one row of 64 nodes after 16384 tokens, 32 / 8 heads of 128: 41.0 us
// for 44.3; of 1024 nodes 394 for 418; eight rows of 256 nodes, which are many blocks, in 64 dims 147 for 141); those of
// 64, of which HBM is the bound, four, so that one workgroup's loads run while the other begins or ends (32 rows of 16
// nodes, 16 / 4 heads: 77 us for 85 with one-term weights).
constexpr int waves_of(int dp, int pairs) { return dp <= 128 && pairs == 128 ? 8 : 4; }
constexpr int tree_fill(int dp, int pairs) { return dp <= 128 ? 8 / waves_of(dp, pairs) : 1; }

struct TreeParams : CarefulParams {
  const int32_t *seqlens, *cu;
  int n_rows, t_new, total, H, G;
  int target;      // workgroups a call aims at; 0: no row is cut
  float *part_o;   // [slot][pairs of a block][D]
  float *part_ml;  // [slot][pairs of a block][2]
  PagedTiles::Cut *cuts;
  int *n_cuts;
};

// A range of a block, of KV head kvh.
template <int DP, int kBlock>
__device__ __forceinline__ void attend_range(const TreeParams &P, const TreeRange R, int kvh) {
  using S_ = Shape<DP>;
  constexpr int CPR = S_::CPR, RPI = S_::RPI, NV = S_::NV, KD = S_::KD, MD = S_::MD;
  constexpr int W = waves_of(DP, kBlock), kTile = 16 * W, kThreads = 64 * W;
  constexpr int WP = kBlock / 32, WK = W / WP, MK = kTile / (32 * WK);  // waves over pairs, keys; 32 keys of a wave
  // K and V of two tiles; at the end the halves of their sums that waves of the same pairs hand each other.
  __shared__ __attribute__((aligned(1024))) uint16_t s_tiles[2][2][kTile * DP];
  __shared__ float s_ml[WK][WP][2][32];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = R.b, D = P.D;
  const int h = lane >> 5, col = lane & 31;
  const int pg = wave % WP, kg = wave / WP;  // its 32 pairs, and its part of a tile's keys
  const int pairs = R.T * P.G, p0 = R.qt * kBlock;
  const int in_block = 32 * pg + col, pair = p0 + in_block;
  const bool live = pair < pairs, busy = p0 + 32 * pg < pairs;  // this pair, any of the wave
  const int t_q = live ? pair / P.G : 0;
  const int64_t at = (int64_t(R.tok0 + t_q) * P.H + kvh * P.G + (live ? pair - t_q * P.G : 0)) * D;
  uint16_t *out = static_cast<uint16_t *>(P.out) + at;
  if (R.s0 < 0 || int64_t(R.s0) + R.T > int64_t(P.kv.max_pages) << P.kv.shift) {
    if (live && kg == 0)
      for (int d = 8 * h; d < D; d += 16)
        *reinterpret_cast<uint4 *>(out + d) =
            make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    return;
  }

  const int t_last = min(p0 + kBlock - 1, pairs - 1) / P.G;
  const int seen_from = P.window >= 0 ? max(0, R.s0 - 1 - P.window) : 0;  // keys any pair of the block sees
  const int seen_to = R.s0 + t_last;
  const int first_tile = seen_from / kTile, n_tiles = seen_to / kTile - first_tile + 1;
  const int ranges = min(R.ranges, n_tiles);
  if (R.part >= ranges) return;
  if (R.noted && R.part == 0 && tid == 0)
    P.cuts[int64_t(R.cut) * P.H_kv + kvh] =
        PagedTiles::Cut{R.b, R.qt, R.tok0, R.T, R.s0, ranges, R.slot * P.H_kv + kvh, 0};
  const int t0 = first_tile + range_tile(R.part, n_tiles, ranges);
  const int t1 = first_tile + range_tile(R.part + 1, n_tiles, ranges);

  const uint16_t *q = static_cast<const uint16_t *>(P.q) + at;
  bf16x8 qf[KD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (16 * kd + 8 * h < D) u = *reinterpret_cast<const uint4 *>(q + 16 * kd + 8 * h);
    qf[kd] = __builtin_bit_cast(bf16x8, u);
  }

  const uint64_t own_word = TreeNode::own_word(P.tree, R.tok0 + t_q, t_q);

  // This wave's loads: keys 16 wave .. of a tile, K and V. Load i covers rows RPI i + lane / CPR; its lane's chunk
  // goes to slot lane % CPR, wherever that is. (The swizzles of a row are those of the row modulo 16.)
  const int tok_bytes = P.H_kv * D * 2;
  constexpr uint32_t kNowhere = 0x80000000u;
  const int lr = lane / CPR, lc = lane % CPR;
  uint32_t off_k[NV], off_v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = RPI * i + lr, ck = lc ^ S_::k_swz(r), cv = lc ^ S_::v_swz(r);
    off_k[i] = 8 * ck < D ? uint32_t(r * tok_bytes + 16 * ck) : kNowhere;
    off_v[i] = 8 * cv < D ? uint32_t(r * tok_bytes + 16 * cv) : kNowhere;
  }
  const scalar_ints table = (scalar_ints)(P.kv.table + b * P.kv.table_stride);
  const int64_t head_at = int64_t(kvh) * D * 2;
  const uint32_t page_bytes = uint32_t(tok_bytes) << P.kv.shift;
  const bool fresh = P.k_new != nullptr;
  const char *const k_pool = static_cast<const char *>(P.k_pages), *const v_pool = static_cast<const char *>(P.v_pages);
  const int64_t k_step = static_cast<const char *>(P.k_new) - k_pool, v_step = static_cast<const char *>(P.v_new) - v_pool;
  bool lost = false;
  // The page of this wave's keys of a tile; one that no key needs is page 0.
  auto page_of = [&](int tile) __attribute__((always_inline)) {
    const int k = tile * kTile + 16 * wave;
    return tile < t1 && k + 15 >= seen_from && k <= seen_to ? table[k >> P.kv.shift] : 0;
  };
  // Into place `at`; past the range's end zeros, so that as many loads are under way in every turn.
  auto load_tile = [&](int tile, int id, int at) __attribute__((always_inline)) {
    const int k0 = tile * kTile, k = k0 + 16 * wave;
    uint16_t *const to_k = s_tiles[0][at] + wave * NV * 512, *const to_v = s_tiles[1][at] + wave * NV * 512;
    lost = lost || !P.kv.is_page(id);
    if (fresh && tile < t1 && k0 + kTile > R.s0) {
      // Nodes come from their own rows; past the last one it is read again.
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int r = RPI * i + lr, key = max(seen_from, min(k + r, seen_to));
        const bool node = key >= R.s0;
        const int64_t from = (node ? int64_t(R.tok0 + key - R.s0) * tok_bytes
                                   : 2 * P.kv.offset(id, P.kv.in_page(key), int64_t(P.H_kv) * D)) + head_at;
        const int ck = min(lc ^ S_::k_swz(r), D / 8 - 1), cv = min(lc ^ S_::v_swz(r), D / 8 - 1);
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)(k_pool + from + (node ? k_step : 0) + 16 * ck),
            (__attribute__((address_space(3))) void *)(to_k + i * 512), 16, 0, 0);
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)(v_pool + from + (node ? v_step : 0) + 16 * cv),
            (__attribute__((address_space(3))) void *)(to_v + i * 512), 16, 0, 0);
      }
      return;
    }
    const bool edge = k0 < seen_from || k0 + kTile - 1 > seen_to || tile >= t1;
    const int64_t base = (P.kv.is_page(id) ? id : 0) * P.kv.page_stride * 2 + head_at;
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(k_pool + base), 0, int(page_bytes - uint32_t(head_at)), 0x00020000);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(v_pool + base), 0, int(page_bytes - uint32_t(head_at)), 0x00020000);
    const int in_page = P.kv.in_page(k) * tok_bytes;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t ok = off_k[i], ov = off_v[i];
      if (edge) {
        const int key = k + RPI * i + lr;
        const bool there = key >= seen_from && key <= seen_to && tile < t1;
        ok = there ? ok : kNowhere;
        ov = there ? ov : kNowhere;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rk, (__attribute__((address_space(3))) void *)(to_k + i * 512), 16, int(ok), in_page, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rv, (__attribute__((address_space(3))) void *)(to_v + i * 512), 16, int(ov), in_page, 0, 0);
    }
  };

  // LDS addresses of this lane's reads, in a tile.
  uint32_t ka[KD], va[2 * MD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd)
    ka[kd] = lds_addr(s_tiles[0][0]) + 2 * (kg * 32 * MK * DP + col * DP + 8 * ((2 * kd + h) ^ S_::k_swz(col)));
  const int tr_row = (lane & 15) >> 2, tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
  for (int md = 0; md < MD; ++md)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 4 * h + tr_row + 8 * u, c = 32 * md + tr_col;
      va[2 * md + u] =
          lds_addr(s_tiles[1][0]) + 2 * (kg * 32 * MK * DP + r * DP + 8 * ((c >> 3) ^ S_::v_swz(r)) + (c & 7));
    }

  f32x16 o[MD];
#pragma unroll
  for (int md = 0; md < MD; ++md)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[md][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  if (D < DP) {  // dims past the head's are zero, whether or not a load past a page's end writes
    for (int i = tid; i < 2 * 2 * kTile * DP / 8; i += kThreads)
      reinterpret_cast<uint4 *>(s_tiles)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  {
    const int id = page_of(t0);
    load_tile(t0, id, 0);
  }
  int next = page_of(t0 + 1);
  // The queries were asked for before these: waited for here, since in the loop the compiler would wait for the
  // loads to LDS with them.
  wait_loads<0>();
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) asm volatile("" : "+v"(qf[kd]));
  const TreeNode node(P.tree, R.tok0 + t_q, t_q, R.s0, P.window, own_word);

  // One tile, in place AT.
  auto turn = [&](int tile, auto at_c) __attribute__((always_inline)) {
    constexpr int AT = decltype(at_c)::value;
    constexpr int kOff = AT * kTile * DP * 2;  // bytes
    const int k0 = tile * kTile + 32 * MK * kg;  // of this wave
    // This wave's loads of the tile have landed, and everyone's; and everyone has read the tile before, whose place
    // the next load takes.
    wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    load_tile(tile + 1, next, 1 - AT);
    next = page_of(tile + 2);
    if (!busy) return;

    f32x16 s[MK];
#pragma unroll
    for (int mk = 0; mk < MK; ++mk)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[mk][e] = 0.f;
    constexpr int KB = KD < 4 ? KD : 4;
    auto scores = [&](auto k8_c) __attribute__((always_inline)) {
      constexpr int k8 = decltype(k8_c)::value;
      bf16x8 f[MK][KB];
      uint32_t a[KB];
#pragma unroll
      for (int i = 0; i < KB; ++i) a[i] = ka[k8 + i];
      if constexpr (MK == 2)
        read_rows_two<kOff, kOff + 64 * DP, KB>(f[0], f[MK - 1], a);
      else
        read_rows_at<kOff, KB>(f[0], a);
#pragma unroll
      for (int i = 0; i < KB; ++i)
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
          s[mk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[mk][i], qf[k8 + i], s[mk], 0, 0, 0);
    };
    scores(std::integral_constant<int, 0>{});
    if constexpr (KD > 4) scores(std::integral_constant<int, 4>{});
    if constexpr (KD > 8) scores(std::integral_constant<int, 8>{});
    if constexpr (KD > 12) scores(std::integral_constant<int, 12>{});

    // Keys the pair may not see.
    if (k0 + 32 * MK - 1 >= R.s0 || (P.window >= 0 && k0 < R.s0 + t_last - P.window)) {
      const uint64_t seen = node.seen(k0) >> (4 * h);
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((seen >> (32 * mk + 8 * (e >> 2) + (e & 3))) & 1)) s[mk][e] = -INFINITY;
    }
    // Weights against the running maximum; the tile's own is taken, and the sums rescaled, only where a lane's
    // weights sum past 2^15 or are not finite, or the pair has no maximum yet.
    bf16x8 pk[2 * MK], pl[2 * MK];  // their two terms
    auto weigh = [&]() __attribute__((always_inline)) {
      const float ref = m == -INFINITY ? 0.f : m;
      float ts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2 * MK; ++ks) {
        f32x8 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = fast_exp2(fmaf(s[ks >> 1][8 * (ks & 1) + e], P.scale_log2, -ref));
          ts[e & 3] += w[e];
        }
        pk[ks] = __builtin_convertvector(w, bf16x8);
        pl[ks] = __builtin_convertvector(w - __builtin_convertvector(pk[ks], f32x8), bf16x8);
      }
      return (ts[0] + ts[1]) + (ts[2] + ts[3]);
    };
    float tl = weigh();
    if (__builtin_amdgcn_ballot_w64(!(tl <= kTileSumLimit) || m == -INFINITY) != 0) {
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int e = 0; e < 16; ++e) m4[e & 3] = fmaxf(m4[e & 3], s[mk][e]);
      const float mx = max_halves(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))) * P.scale_log2;
      const float m_new = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
      l *= alpha;
#pragma unroll
      for (int md = 0; md < MD; ++md)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[md][e] *= alpha;
      m = m_new;
      tl = weigh();
    }
    l += tl;

    constexpr int VB = 2 * MD < 8 ? 2 * MD : 8;
    auto add_dims = [&](auto ks_c, auto v8_c) __attribute__((always_inline)) {
      constexpr int ks = decltype(ks_c)::value, v8 = decltype(v8_c)::value;
      bf16x4 f[VB];
      uint32_t a[VB];
#pragma unroll
      for (int i = 0; i < VB; ++i) a[i] = va[v8 + i];
      read_columns_at<kOff + ks * 32 * DP, VB>(f, a);
#pragma unroll
      for (int i = 0; i < VB / 2; ++i) {
        const bf16x8 x = __builtin_shufflevector(f[2 * i], f[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        o[v8 / 2 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, pk[ks], o[v8 / 2 + i], 0, 0, 0);
        o[v8 / 2 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, pl[ks], o[v8 / 2 + i], 0, 0, 0);
      }
    };
    auto add_values = [&](auto ks_c) __attribute__((always_inline)) {  // of 16 keys
      add_dims(ks_c, std::integral_constant<int, 0>{});
      if constexpr (2 * MD > 8) add_dims(ks_c, std::integral_constant<int, 8>{});
    };
    add_values(std::integral_constant<int, 0>{});
    add_values(std::integral_constant<int, 1>{});
    if constexpr (MK == 2) {
      add_values(std::integral_constant<int, 2>{});
      add_values(std::integral_constant<int, 3>{});
    }
  };
  for (int tile = t0;;) {
    turn(tile, std::integral_constant<int, 0>{});
    if (++tile >= t1) break;
    turn(tile, std::integral_constant<int, 1>{});
    if (++tile >= t1) break;
  }
  wait_loads<0>();
  l = sum_halves(l);

  // The nodes whose first pair the block has, into their pages: by its last range.
  if (fresh && R.part == ranges - 1) {
    const int units = D / 8;  // of 16 bytes, of K and of V
    const int own = (p0 + P.G - 1) / P.G, end = min((p0 + kBlock + P.G - 1) / P.G, R.T);
    for (int i = tid; i < (end - own) * units; i += kThreads) {
      const int row = i / units, t = own + row, u = i - row * units, key = R.s0 + t;
      const int pid = P.kv.table[b * P.kv.table_stride + (key >> P.kv.shift)];
      if (!P.kv.is_page(pid)) continue;
      const int64_t from = int64_t(R.tok0 + t) * tok_bytes + head_at + 16 * u;
      const int64_t to = 2 * P.kv.offset(pid, P.kv.in_page(key), int64_t(P.H_kv) * D) + head_at + 16 * u;
      const uint4 x = *reinterpret_cast<const uint4 *>(static_cast<const char *>(P.k_new) + from);
      const uint4 y = *reinterpret_cast<const uint4 *>(static_cast<const char *>(P.v_new) + from);
      *reinterpret_cast<uint4 *>(static_cast<char *>(const_cast<void *>(P.k_pages)) + to) = x;
      *reinterpret_cast<uint4 *>(static_cast<char *>(const_cast<void *>(P.v_pages)) + to) = y;
    }
  }
  if (__syncthreads_or(lost)) l = NAN;  // and the tiles are read

  // The two waves of the same pairs add their sums up, each half of the dims: o[0 .. OWN) from dim d0 on. (32 dims
  // are one piece: the first wave has it.)
  constexpr bool HALVES = WK == 2 && MD > 1;
  constexpr int OWN = HALVES ? MD / 2 : MD;
  static_assert(WK <= 2 && MD <= 2 * OWN, "two waves");
  const int d0 = HALVES ? 32 * OWN * kg : 0;
  if constexpr (WK == 2) {
    static_assert(kBlock * DP * 4 <= int(sizeof(s_tiles)), "they fit the tiles");
    constexpr int GIVEN = HALVES ? OWN : 0;  // the first piece for the other
    if (HALVES && kg == 1)
#pragma unroll
      for (int md = 0; md < OWN; ++md) {
        const f32x16 x = o[md];
        o[md] = o[MD - OWN + md];
        o[MD - OWN + md] = x;
      }
    // [32 pairs][whose half][piece][8 dims][lane][4]
    float *const so = reinterpret_cast<float *>(s_tiles) + pg * 32 * DP + 4 * lane;
    if (HALVES || kg == 1)
#pragma unroll
      for (int i = 0; i < OWN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float4 *>(so + ((HALVES ? 1 - kg : 0) * OWN + i) * 1024 + j * 256) =
              make_float4(o[GIVEN + i][4 * j], o[GIVEN + i][4 * j + 1], o[GIVEN + i][4 * j + 2], o[GIVEN + i][4 * j + 3]);
    if (h == 0) s_ml[kg][pg][0][col] = m, s_ml[kg][pg][1][col] = l;
    __syncthreads();
    if (!HALVES && kg == 1) return;
    const float m2 = s_ml[1 - kg][pg][0][col], l2 = s_ml[1 - kg][pg][1][col], both = fmaxf(m, m2);
    const float a1 = m == -INFINITY ? 0.f : fast_exp2(m - both), a2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - both);
    // Without a key l = 0; a NaN l must stay.
    l = l * (m == -INFINITY ? 1.f : a1) + l2 * (m2 == -INFINITY ? 1.f : a2);
    m = both;
#pragma unroll
    for (int i = 0; i < OWN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(so + ((HALVES ? kg : 0) * OWN + i) * 1024 + j * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][4 * j + e] = fmaf(x[e], a2, o[i][4 * j + e] * a1);
      }
  }

  // o[i][4j + e] is dim d0 + 32 i + 8 j + 4 h + e of pair `col`.
  if (ranges > 1) {
    if (!live) return;
    const int64_t slot = (int64_t(R.slot + R.part) * P.H_kv + kvh) * kBlock + in_block;
    float *po = P.part_o + slot * D + d0;
#pragma unroll
    for (int i = 0; i < OWN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d0 + 32 * i + 8 * j < D)
          *reinterpret_cast<float4 *>(po + 32 * i + 8 * j + 4 * h) =
              make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
    if (h == 0 && kg == 0) *reinterpret_cast<float2 *>(P.part_ml + slot * 2) = make_float2(m, l);
    return;
  }
  const float inv = 1.f / l;
  bool ok = true;
#pragma unroll
  for (int i = 0; i < OWN; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      o[i][e] *= inv;
      ok = ok && (finite(o[i][e]) || d0 + 32 * i + 8 * (e >> 2) >= D);
    }
  const uint64_t bad64 = __builtin_amdgcn_ballot_w64(live && !ok);
  const uint32_t bad = uint32_t(bad64) | uint32_t(bad64 >> 32);
  if (live && !((bad >> col) & 1u)) {
#pragma unroll
    for (int i = 0; i < OWN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (d0 + 32 * i + 8 * j >= D) continue;
        const f32x4 x = {o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
        *reinterpret_cast<uint2 *>(out + d0 + 32 * i + 8 * j + 4 * h) =
            __builtin_bit_cast(uint2, __builtin_convertvector(x, bf16x4));
      }
  }
  for (uint32_t left = bad; __builtin_expect(left != 0, 0); left &= left - 1) {
    const int pr = p0 + 32 * pg + __builtin_ctz(left), t = pr / P.G;
    careful_pair<bf16, DP, 8, true>(P, b, kvh, (int64_t(R.tok0 + t) * P.H + kvh * P.G + (pr - t * P.G)) * D,
                                    R.s0 + t, lane, d0, min(d0 + 32 * OWN, D), R.tok0 + t, t);
  }
}

template <int DP, int kBlock>
__global__ __launch_bounds__(64 * waves_of(DP, kBlock))
    __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1))) void tree_stream_kernel(TreeParams P) {
  constexpr int kTile = 16 * waves_of(DP, kBlock);
  TreeRange R;
  const TreeRanges call{P.cu, P.seqlens, P.n_rows, P.t_new, P.total, P.G, P.H_kv, kBlock, 0,
                        P.kv.max_pages << P.kv.shift, P.window, kTile, P.target, kMinRangeKeys / kTile};
  const bool found = find_tree_range(call, int(blockIdx.x) / P.H_kv, threadIdx.x & 63, R);
  if (blockIdx.x == 0 && threadIdx.x == 0 && P.target > 0) *P.n_cuts = R.n_blocks;
  if (!found) return;
  attend_range<DP, kBlock>(P, R, int(blockIdx.x) % P.H_kv);
}

// The ranges of cut blocks added up: a workgroup has two pairs (D up to 128; one of more) of a block and KV head, half
// a wave a pair with four dims a lane, and its waves every fourth range each, eight of them under way.
template <int DP, int kBlock>
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(TreeParams P) {
  constexpr int LPP = DP <= 128 ? 32 : 64, N = 64 / LPP, U = 8;  // lanes of a pair, pairs of a wave
  __shared__ f32x4 s_o[kWaves][64];
  __shared__ float2 s_ml[kWaves][N];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.y;  // of the cut blocks, KV heads counted
  // Both asked for at once; a record past the last cut block is not used.
  const scalar_ints record = (scalar_ints)(P.cuts + id);
  const PagedTiles::Cut blk{record[0], record[1], record[2], record[3], record[4], record[5], record[6], 0};
  const int n_cuts = *(scalar_ints)P.n_cuts;
  asm volatile("" ::"s"(blk.ranges), "s"(n_cuts));
  if (id >= n_cuts * P.H_kv) return;
  const int kvh = id % P.H_kv, n = min(kBlock, blk.T * P.G - blk.qt * kBlock), ranges = blk.ranges;
  const int first = N * int(blockIdx.x);
  if (ranges == 1 || first >= n) return;  // of one range: written by the block itself
  const int in_block = first + lane / LPP, d = 4 * (lane % LPP);
  const int64_t step = int64_t(P.H_kv) * kBlock, slot = int64_t(blk.second) * kBlock + min(in_block, n - 1);
  float M = -INFINITY, L = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = wave; r0 < ranges; r0 += U * kWaves) {
    float2 x[U];
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = slot + min(r0 + u * kWaves, ranges - 1) * step;
      x[u] = *reinterpret_cast<const float2 *>(P.part_ml + at * 2);
      v[u] = *reinterpret_cast<const f32x4 *>(P.part_o + at * P.D + min(d, P.D - 4));
    }
    float m_new = M;
#pragma unroll
    for (int u = 0; u < U; ++u) m_new = r0 + u * kWaves < ranges ? fmaxf(m_new, x[u].x) : m_new;
    const float keep = M == -INFINITY ? 0.f : fast_exp2(M - m_new);
    L *= M == -INFINITY ? 1.f : keep;  // 0 then, or a NaN that must stay
    y *= keep;
    M = m_new;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u * kWaves >= ranges) break;
      const float a = x[u].x == -INFINITY ? 0.f : fast_exp2(x[u].x - M);
      L += x[u].y * (x[u].x == -INFINITY ? 1.f : a);
      y += a * v[u];
    }
  }
  s_o[wave][lane] = y;
  if (lane % LPP == 0) s_ml[wave][lane / LPP] = make_float2(M, L);
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_ml[w][lane / LPP].x);
  L = 0.f;
  y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float2 x = s_ml[w][lane / LPP];
    const float a = x.x == -INFINITY ? 0.f : fast_exp2(x.x - M);
    L += x.y * (x.x == -INFINITY ? 1.f : a);
    y += a * s_o[w][lane];
  }
  y *= 1.f / L;
  const bool there = in_block < n && d < P.D;
  const bool ok = !there || (finite(y[0]) && finite(y[1]) && finite(y[2]) && finite(y[3]));
  uint64_t bad = __builtin_amdgcn_ballot_w64(!ok);
  auto pair_at = [&](int i, int &t) {
    const int pr = blk.qt * kBlock + i;
    t = pr / P.G;
    return (int64_t(blk.tok0 + t) * P.H + int64_t(kvh) * P.G + (pr - t * P.G)) * P.D;
  };
  int t;
  const int64_t at = pair_at(min(in_block, n - 1), t);
  const bool redo = (bad >> (lane / LPP * LPP) & (N == 1 ? ~uint64_t(0) : 0xffffffffu)) != 0;
  if (there && !redo)
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(P.out) + at + d) =
        __builtin_bit_cast(uint2, __builtin_convertvector(y, bf16x4));
  if (__builtin_expect(bad == 0, 1)) return;
  for (int i = 0; i < N; ++i) {
    if (!(bad >> (i * LPP) & (N == 1 ? ~uint64_t(0) : 0xffffffffu)) || first + i >= n) continue;
    const int64_t to = pair_at(first + i, t);
    careful_pair<bf16, DP, 8, true>(P, blk.b, kvh, to, blk.s0 + t, lane, 0, P.D, int64_t(blk.tok0) + t, t);
  }
}

// Pairs of a block.
int block_of(const PagedArgs &a) { return a.t_new * (a.n_head / a.n_kv_head) <= 64 ? 64 : 128; }
// Workgroups that a call aims at: all that the chip holds at once.
int64_t target_of(const PagedArgs &a) {
  return paged_keys(a) >= 2 * kMinRangeKeys ? int64_t(tree_fill(head_pad(a.head_dim), block_of(a))) * device_cus() : 0;
}
size_t bytes_of(const PagedArgs &a, int64_t target) {
  return target == 0 ? 0 : paged_tiles_bytes(tree_slots(target, a.n_kv_head), block_of(a) * (a.head_dim + 2));
}

template <int DP, int kBlock>
int run_block(const TreeParams &P, const PagedArgs &a) {
  constexpr int threads = 64 * waves_of(DP, kBlock);
  const int64_t bound = paged_blocks_bound(a, kBlock, 0);
  const int64_t blocks = P.target > 0 ? tree_blocks(bound, P.target, P.H_kv) : bound * P.H_kv;
  if (blocks > 0x7fffffff / threads) return fail(MCAMD_EUNSUPPORTED, "paged attention: grid too large");
  if (blocks == 0) return MCAMD_OK;
  hipLaunchKernelGGL((tree_stream_kernel<DP, kBlock>), dim3(unsigned(blocks)), dim3(threads), 0, a.stream, P);
  const int st = launch_status("tree_stream");
  if (st != MCAMD_OK || P.target == 0) return st;
  // A cut block has two ranges at least.
  const int64_t cut = std::min<int64_t>(bound * P.H_kv, tree_slots(P.target, P.H_kv) / 2);
  const int64_t pairs = std::min<int64_t>(kBlock, a.t_new * P.G), each = DP <= 128 ? 2 : 1;
  if (cut > 65535) return fail(MCAMD_EUNSUPPORTED, "paged attention: grid too large");
  hipLaunchKernelGGL((tree_merge_kernel<DP, kBlock>), dim3(unsigned((pairs + each - 1) / each), unsigned(cut)),
                     dim3(kThreads), 0, a.stream, P);
  return launch_status("tree_merge");
}
template <int DP>
int run(const TreeParams &P, const PagedArgs &a) {
  return block_of(a) == 64 ? run_block<DP, 64>(P, a) : run_block<DP, 128>(P, a);
}

}  // namespace

size_t tree_stream_bytes(const PagedArgs &a) { return bytes_of(a, target_of(a)); }

int launch_tree_stream(const PagedArgs &a) {
  TreeParams P{};
  P.q = a.q;
  P.k_pages = a.k_pages;
  P.v_pages = a.v_pages;
  P.kv = a.kv;
  P.out = a.out;
  P.H_kv = int(a.n_kv_head);
  P.window = int(a.window < 0 ? -1 : a.window);
  P.D = int(a.head_dim);
  P.scale_log2 = float(kLog2e / std::sqrt(double(a.head_dim)));
  P.tree = a.tree;
  P.k_new = a.k_new;
  P.v_new = a.v_new;
  P.seqlens = a.seqlens;
  P.cu = a.cu;
  P.n_rows = int(a.n_rows);
  P.t_new = int(a.t_new);
  P.total = int(a.total);
  P.H = int(a.n_head);
  P.G = int(a.n_head / a.n_kv_head);
  const int64_t target = target_of(a);
  if (target > 0 && a.scratch && a.scratch_bytes >= bytes_of(a, target)) {
    const int64_t slots = tree_slots(target, a.n_kv_head);
    P.target = int(target);
    P.part_o = static_cast<float *>(a.scratch);
    const int64_t pairs = slots * block_of(a);
    P.part_ml = P.part_o + pairs * a.head_dim;
    P.cuts = reinterpret_cast<PagedTiles::Cut *>(P.part_ml + pairs * 2);
    P.n_cuts = reinterpret_cast<int *>(P.cuts + slots);
  }
  switch (head_pad(a.head_dim)) {
    case 32: return run<32>(P, a);
    case 64: return run<64>(P, a);
    case 128: return run<128>(P, a);
    default: return run<256>(P, a);
  }
}

}  // namespace mcamd
