// Multi-token attention over a paged cache on the matrix cores, for fp32 caches and any head dim up to
// 256 made of whole 16-byte vectors. Query t of row b sits at p = cache_seqlens[b] + t and attends
// keys col <= p with p - col <= window when window >= 0; the append runs first.
//
// The tile structure is that of prefill_tiled.hip, whose comment says why each layout is what it is:
// 32 (position, head) pairs a wave, head fastest, four waves on 128 pairs (KS = 1) or on the same 32
// pairs and a quarter of each tile's keys each (KS = 4, for calls with too few pairs to fill the
// chip), both products transposed so that a lane owns a pair, bf16 weights as two terms, fp32
// scores in four chains. What differs is where keys and blocks come from:
//  * A thread's pieces of a tile name their pages one tile ahead, so that the table's latency is not in
//    front of the tile's loads. Pages may end anywhere inside a tile.
//  * find_paged_block() deals the blocks of uniform and packed rows alike, and where a call has few of
//    them, each block's tiles are cut into key ranges as in prefill_split.h, with the device's count of
//    the call's blocks in the cost rule.
//  * Not finite: a pair whose result is not finite is redone over the keys it sees alone
//    (careful_pair()), and so is every pair of a block that met a page outside the pool, which leaves
//    NaN to those that see such a page.
// Two prompts of 512, 12 heads of 64 in fp32: 22.6 us (0.81 GFLOP), with the staged tile in registers (31 with
// half of it in scratch memory); 344 tokens after 3639, 16 / 4 heads of 256 in bf16: 56 (95).
#include "paged_careful.h"
#include "prefill_order.h"
#include "prefill_split.h"
#include "range_tiles.h"
#include "tree_ranges.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mcamd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr float kTileSumLimit = 32768.f;  // 2^15: a lane's weights of one tile sum to at most this

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 lds_bf16x4 __attribute__((__vector_size__(4 * sizeof(__bf16))));

struct TiledParams : CarefulParams {
  const int32_t *seqlens, *cu;
  int T_new, H, G;
  int deal;  // workgroups per round of dealt_block()
  PagedTiles tiles;
  int md;  // 32-dim pieces of a head
  // Four dims 32 d + 8 j + 4 (lane / 32) .. of pair lane % 32 of a group's partials.
  __device__ __forceinline__ float *part_o(int64_t group, int d, int j, int lane) const {
    return tiles.part_o + ((group * md + d) * 4 + j) * 256 + lane * 4;
  }
  __device__ __forceinline__ float *part_ml(int64_t group, int pair) const {
    return tiles.part_ml + (group * 32 + pair) * 2;
  }
};

// Tile geometry of an instantiation (elements of E; DP is head_dim rounded up).
template <class E, int DP, int KS>
struct Geo {
  static constexpr bool kBf16 = sizeof(E) == 2;
  static constexpr int VEC = Vec<E>::N;
  static constexpr int KW = kBf16 && DP <= 128 && KS == 1 ? 64 : 32;  // keys per wave and tile
  static constexpr int MK = KW / 32;
  static constexpr int KT = KW * KS;                  // keys per tile
  static constexpr int PAIRS = 32 * kWaves / KS;      // pairs per workgroup
  static constexpr int MD = DP / 32;                  // 32-row blocks of O^T
  static constexpr int KSTR = DP + VEC;               // K row stride
  // V row stride: bf16 16 or 48 dwords modulo 64 (DP / 2 is 16, 48 or a multiple of 32), fp32
  // DP + 8.
  static constexpr int VSTR = kBf16 ? (DP % 64 == 0 ? DP + 32 : DP) : DP + 8;
  static constexpr int CH = KT * DP / VEC / kThreads;  // 16-byte pieces of K (or V) per thread
  static constexpr int TILE_BYTES = (KSTR + VSTR) * KT * int(sizeof(E));
  static constexpr int OSTR = DP + 4;                 // row stride of the KS = 4 merge, floats
  static constexpr int MERGE_BYTES = KS == 1 ? 0 : (32 * OSTR + 64) * 4 * kWaves + 32 * 4;
  static constexpr int LDS_BYTES = TILE_BYTES > MERGE_BYTES ? TILE_BYTES : MERGE_BYTES;
  static_assert(KT * DP % (VEC * kThreads) == 0, "whole pieces per thread");
  static_assert(!kBf16 || VSTR / 2 % 32 == 16, "V rows on 16 or 48 banks modulo 64");
};

__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Four consecutive LDS rows of one column, transposed into a lane: lane L of each 16-lane group
// passes the address of row L / 4, columns 4 (L % 4) .. + 3 of a 4 x 16 block and receives
// column L of it.
__device__ __forceinline__ bf16x4 lds_read_tr(const uint16_t *p) {
  auto lp = (__attribute__((address_space(3))) lds_bf16x4 *)(p);
  return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(lp));
}

// Four consecutive output dims.
__device__ __forceinline__ void store4(float *p, const f32x4 &x) {
  *reinterpret_cast<f32x4 *>(p) = x;
}
__device__ __forceinline__ void store4(bf16 *p, const f32x4 &x) {
  *reinterpret_cast<uint2 *>(p) =
      __builtin_bit_cast(uint2, __builtin_convertvector(x, bf16x4));
}

template <class E, int DP, int KS, bool TREE>
__global__ __launch_bounds__(kThreads) void paged_tiled_kernel(TiledParams P) {
  using G_ = Geo<E, DP, KS>;
  constexpr bool kBf16 = G_::kBf16;
  constexpr int VEC = G_::VEC, KW = G_::KW, MK = G_::MK, KT = G_::KT, MD = G_::MD, CH = G_::CH;
  constexpr int KSTR = G_::KSTR, VSTR = G_::VSTR, OSTR = G_::OSTR;
  __shared__ __attribute__((aligned(16))) unsigned char s_raw[G_::LDS_BYTES];
  E *const sK = reinterpret_cast<E *>(s_raw);
  E *const sV = sK + KT * KSTR;

  const int id = P.cu || TREE ? int(blockIdx.x) : dealt_block(int(blockIdx.x), int(gridDim.x), P.deal);
  typename std::conditional<TREE, TreeRange, PagedBlock>::type blk;
  bool found;
  if constexpr (TREE) {
    const TreeRanges ranges{P.cu, P.seqlens, P.tiles.n_rows, P.T_new, P.tiles.total, P.G, P.H_kv, G_::PAIRS,
                            P.tiles.skip, P.kv.max_pages << P.kv.shift, P.window, KT,
                            P.tiles.slots > 0 ? P.tiles.target : 0, P.tiles.min_tiles};
    found = find_tree_range(ranges, id / P.H_kv, threadIdx.x & 63, blk);
    if (id == 0 && threadIdx.x == 0 && P.tiles.slots > 0) *P.tiles.n_cuts = blk.n_blocks;
  } else {
    found = find_paged_block(P.cu, P.seqlens, P.tiles.n_rows, P.T_new, P.tiles.total, P.G, P.H_kv, G_::PAIRS,
                             P.tiles.skip, P.tiles.slots, P.kv.max_pages << P.kv.shift, P.tiles.halve,
                             id / P.H_kv, threadIdx.x & 63, blk);
    if (id == 0 && threadIdx.x == 0) P.tiles.note_call(found, blk);
  }
  if (!found) return;
  const int kvh = id % P.H_kv, part = blk.part, row = blk.b, T_b = blk.T, s0 = blk.s0;
  const int64_t tok0 = blk.tok0;
  // This workgroup's pairs: n of them from pair p0 on, which is head r0 of position q0.
  const int64_t n_pairs = int64_t(T_b) * P.G;
  const int64_t p0 = int64_t(blk.qt) * G_::PAIRS;
  const int n = int(min(int64_t(G_::PAIRS), n_pairs - p0));
  const int q0 = int(p0 / P.G), r0 = int(p0 - int64_t(q0) * P.G);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5;    // lane half
  const int col = lane & 31;  // this lane's pair within the wave's 32
  const int D = P.D;

  const bool row_ok = s0 >= 0 && int64_t(s0) + T_b <= int64_t(P.kv.max_pages) << P.kv.shift;
  const int w0 = KS == 1 ? 32 * wave : 0;  // the wave's first pair
  const bool live = w0 + col < n;
  // Position of pair i of the workgroup, and where its query and output lie.
  auto pair_pos = [&](int i) { return q0 + (r0 + i) / P.G; };
  auto pair_at = [&](int i) {
    const int pos = (r0 + i) / P.G;
    return ((tok0 + q0 + pos) * P.H + int64_t(kvh) * P.G + (r0 + i - pos * P.G)) * D;
  };
  const int pr = live ? w0 + col : 0;  // dead pairs compute on a live one
  const int tq = pair_pos(pr);
  const int64_t at = pair_at(pr);
  E *out = static_cast<E *>(P.out) + at;
  if (!row_ok) {
    if constexpr (!TREE)
      if (blk.noted && part == 0 && tid == 0) P.tiles.note_block(id, blk, 1, P.H_kv);
    if (live && part == 0 && (KS == 1 || wave == 0))
      for (int d = h; d < D; d += 2) out[d] = from_f32<E>(NAN);
    return;
  }

  const int p_abs = s0 + tq;
  const int p_first = s0 + q0;
  const int last = s0 + pair_pos(n - 1);  // the last key any pair of the workgroup sees
  int lo = P.window >= 0 ? max(0, (TREE ? s0 - 1 : p_first) - P.window) : 0, hi = last;
  int n_tiles = (hi - lo) / KT + 1;
  bool whole = true;
  if (blk.noted) {  // this workgroup's range of the block's tiles
    int ranges;
    if constexpr (TREE)
      ranges = min(blk.ranges, n_tiles);
    else
      ranges = P.tiles.ranges_of(blk, n_tiles);
    if (part >= ranges) return;
    if (part == 0 && tid == 0) {
      if constexpr (TREE)
        note_tree_range(P.tiles, blk, kvh, P.H_kv, ranges);
      else
        P.tiles.note_block(id, blk, ranges, P.H_kv);
    }
    whole = ranges == 1;
    const int t0 = range_tile(part, n_tiles, ranges), t1 = range_tile(part + 1, n_tiles, ranges);
    hi = min(hi, lo + t1 * KT - 1);
    lo += t0 * KT;
    n_tiles = t1 - t0;
  }

  int64_t slot = id;  // of this range's partials
  if constexpr (TREE) slot = int64_t(blk.slot + part) * P.H_kv + kvh;

  // Q^T fragments, B[k = dim][n = pair]. bf16: dims 16 kd + 8h .. + 7 of step kd; fp32: dims
  // 8c + 4h .. + 3, one for each of four steps. Dims past the head_dim are zero.
  constexpr int NQ = kBf16 ? DP / 16 : DP / 8;
  using QF = typename std::conditional<kBf16, bf16x8, f32x4>::type;
  QF qf[NQ];
  {
    const E *qp = static_cast<const E *>(P.q) + at;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int d = (kBf16 ? 16 : 8) * i + VEC * h;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (d < D) u = *reinterpret_cast<const uint4 *>(qp + d);
      qf[i] = __builtin_bit_cast(QF, u);
    }
  }
  const int64_t tok = int64_t(P.H_kv) * D;
  const E *kbase = static_cast<const E *>(P.k_pages) + int64_t(kvh) * D;
  const E *vbase = static_cast<const E *>(P.v_pages) + int64_t(kvh) * D;
  const int32_t *pages = P.kv.table + row * P.kv.table_stride;

  // The pages of this thread's pieces of the next tile to load.
  int page[CH];
  bool lost = false;  // a page outside the pool
  auto load_pages = [&](int k0) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      page[i] = pages[min(k0 + (tid + kThreads * i) / (DP / VEC), hi) >> P.kv.shift];
  };

  // The next tile, on its way to LDS: piece c = tid + 256 i is 16 bytes of key c / (DP / VEC).
  // Keys past `hi` re-read key `hi` (they are masked); K's dims past the head_dim are zero, V's
  // re-read the last ones (they reach no output).
  u32x4 kr[CH], vr[CH];  // as uint4, a struct, the compiler keeps V's in scratch memory
  auto load_tile = [&](int k0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + kThreads * i;
      const int key = min(k0 + c / (DP / VEC), hi);
      const int d = (c % (DP / VEC)) * VEC;
      int64_t off = P.kv.offset(page[i], P.kv.in_page(key), tok) + min(d, D - VEC);
      lost = lost || !P.kv.is_page(page[i]);
      const E *kf = kbase, *vf = vbase;
      if constexpr (TREE)
        if (P.k_new && key >= s0) {  // the nodes from their own rows
          kf = static_cast<const E *>(P.k_new) + int64_t(kvh) * D;
          vf = static_cast<const E *>(P.v_new) + int64_t(kvh) * D;
          off = (tok0 + key - s0) * tok + min(d, D - VEC);
        }
      kr[i] = *reinterpret_cast<const u32x4 *>(kf + off);
      vr[i] = *reinterpret_cast<const u32x4 *>(vf + off);
    }
  };
  auto store_tile = [&]() {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + kThreads * i;
      const int key = c / (DP / VEC), d = (c % (DP / VEC)) * VEC;
      // The zeroes go in here and not at the load, all of which would then be waited for at once.
      *reinterpret_cast<u32x4 *>(&sK[key * KSTR + d]) = d < D ? kr[i] : u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4 *>(&sV[key * VSTR + d]) = vr[i];
    }
  };

  f32x16 o[MD];
#pragma unroll
  for (int md = 0; md < MD; ++md)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[md][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  const int wk = KS == 1 ? 0 : wave * KW;  // the wave's first key within a tile
  const int tr_row = (lane & 15) >> 2;     // bf16: this lane's part of a transpose read
  const int tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  load_pages(lo);
  load_tile(lo);
  load_pages(lo + KT);
  for (int t = 0; t < n_tiles; ++t) {
    const int k0 = lo + t * KT + wk;
    if (t > 0) __syncthreads();  // every wave has read the tile before
    store_tile();
    __syncthreads();
    if (t + 1 < n_tiles) {
      load_tile(lo + (t + 1) * KT);
      load_pages(lo + (t + 2) * KT);
    }
    if (KS > 1 && k0 > hi) continue;  // no key of this wave's quarter (barriers stay paired)

    f32x16 s[MK];
#pragma unroll
    for (int mk = 0; mk < MK; ++mk) {
      const E *kp = &sK[(wk + 32 * mk + col) * KSTR + VEC * h];
      // fp32: four interleaved chains of sums, added at the end: a quarter of one chain's rounding.
      constexpr int NC = kBf16 ? 1 : 4;
      f32x16 sc[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[j][e] = 0.f;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const QF a = __builtin_bit_cast(
            QF, *reinterpret_cast<const uint4 *>(kp + (kBf16 ? 16 : 8) * i));
        if constexpr (kBf16) {
          sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[i], sc[0], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sc[j % NC] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], qf[i][j], sc[j % NC], 0, 0, 0);
        }
      }
      s[mk] = sc[0];
      if constexpr (!kBf16) s[mk] = (sc[0] + sc[1]) + (sc[2] + sc[3]);
    }
    // Keys the pair may not see, in tiles that straddle the diagonal or the window's edge.
    if constexpr (TREE) {
      if (k0 + KW - 1 >= s0 || (P.window >= 0 && k0 < last - P.window)) {
        const uint64_t seen = TreeNode(P.tree, tok0 + tq, tq, s0, P.window).seen(k0) >> (4 * h);
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!((seen >> (32 * mk + 8 * (e >> 2) + (e & 3))) & 1)) s[mk][e] = -INFINITY;
      }
    } else if (k0 + KW - 1 > p_first || (P.window >= 0 && k0 < last - P.window)) {
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int dpos = p_abs - (k0 + 32 * mk + 8 * (e >> 2) + 4 * h + (e & 3));
          if (!(dpos >= 0 && (P.window < 0 || dpos <= P.window))) s[mk][e] = -INFINITY;
        }
    }

    float w[MK][16];
    auto weigh = [&]() {
      const float mu = m == -INFINITY ? 0.f : m;
      float ts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          w[mk][e] = fast_exp2(fmaf(s[mk][e], P.scale_log2, -mu));
          ts[e & 3] += w[mk][e];
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
      const float mx =
          max_halves(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))) * P.scale_log2;
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

    if constexpr (kBf16) {
#pragma unroll
      for (int ks = 0; ks < 2 * MK; ++ks) {  // 16 keys: the eight accumulators 8 (ks % 2) ..
        f32x8 pv;
#pragma unroll
        for (int e = 0; e < 8; ++e) pv[e] = w[ks >> 1][8 * (ks & 1) + e];
        const bf16x8 hi8 = __builtin_convertvector(pv, bf16x8);
        const bf16x8 lo8 =
            __builtin_convertvector(pv - __builtin_convertvector(hi8, f32x8), bf16x8);
        const uint16_t *vp = reinterpret_cast<const uint16_t *>(sV) +
                             (wk + 16 * ks + 4 * h + tr_row) * VSTR + tr_col;
        bf16x8 a[MD];  // the lo terms after all hi terms: no product waits for the one before it
#pragma unroll
        for (int md = 0; md < MD; ++md) {
          const bf16x4 a0 = lds_read_tr(vp + 32 * md);
          const bf16x4 a1 = lds_read_tr(vp + 8 * VSTR + 32 * md);
          a[md] = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
          o[md] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[md], hi8, o[md], 0, 0, 0);
        }
#pragma unroll
        for (int md = 0; md < MD; ++md)
          o[md] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[md], lo8, o[md], 0, 0, 0);
      }
    } else {
      const float *vp = reinterpret_cast<const float *>(sV) + (wk + 4 * h) * VSTR + col;
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int md = 0; md < MD; ++md)
            o[md] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                vp[(32 * mk + 8 * (e >> 2) + (e & 3)) * VSTR + 32 * md], w[mk][e], o[md], 0, 0, 0);
    }
  }

  // The nodes whose first pair the block has, into their pages: by its last range.
  if constexpr (TREE)
    if (P.k_new && hi == last) {
      const int units = D / VEC, own = q0 + (r0 > 0), end = pair_pos(n - 1) + 1;
      for (int i = tid; i < (end - own) * units; i += kThreads) {
        const int t = own + i / units, key = s0 + t, d = VEC * (i % units);
        const int id = pages[key >> P.kv.shift];
        if (!P.kv.is_page(id)) continue;
        const int64_t fresh = (tok0 + t) * tok + int64_t(kvh) * D + d;
        const int64_t to = P.kv.offset(id, P.kv.in_page(key), tok) + int64_t(kvh) * D + d;
        const u32x4 x = *reinterpret_cast<const u32x4 *>(static_cast<const E *>(P.k_new) + fresh);
        const u32x4 y = *reinterpret_cast<const u32x4 *>(static_cast<const E *>(P.v_new) + fresh);
        *reinterpret_cast<u32x4 *>(static_cast<E *>(const_cast<void *>(P.k_pages)) + to) = x;
        *reinterpret_cast<u32x4 *>(static_cast<E *>(const_cast<void *>(P.v_pages)) + to) = y;
      }
    }

  l = sum_halves(l);
  if (__syncthreads_or(lost)) l = NAN;
  if constexpr (KS == 1) {
    if (!whole) {
      if (!live) return;
      const int64_t g = slot * kWaves + wave;
#pragma unroll
      for (int md = 0; md < MD; ++md)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (32 * md < D)
            store4(P.part_o(g, md, j, lane), f32x4{o[md][4 * j], o[md][4 * j + 1],
                                                    o[md][4 * j + 2], o[md][4 * j + 3]});
      if (h == 0) *reinterpret_cast<float2 *>(P.part_ml(g, col)) = make_float2(m, l);
      return;
    }
    const float inv = 1.f / l;
    bool ok = true;
#pragma unroll
    for (int md = 0; md < MD; ++md)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        o[md][e] *= inv;
        ok = ok && (finite(o[md][e]) || 32 * md + 8 * (e >> 2) >= D);
      }
    const uint64_t bad64 = __builtin_amdgcn_ballot_w64(live && !ok);
    const uint32_t bad = uint32_t(bad64) | uint32_t(bad64 >> 32);
    if (live && !((bad >> col) & 1u)) {
#pragma unroll
      for (int md = 0; md < MD; ++md)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 32 * md + 8 * j + 4 * h;
          if (d < D)
            store4(out + d, f32x4{o[md][4 * j], o[md][4 * j + 1], o[md][4 * j + 2],
                                  o[md][4 * j + 3]});
        }
    }
    for (uint32_t left = bad; __builtin_expect(left != 0, 0); left &= left - 1) {
      const int c = w0 + __builtin_ctz(left);
      careful_pair<E, DP, 32, TREE>(P, row, kvh, pair_at(c), s0 + pair_pos(c), lane, 0, D,
                                    tok0 + pair_pos(c), pair_pos(c));
    }
  } else {
    // Merge the four waves' (o, m, l) of the same 32 pairs; thread t then owns an eighth of the
    // dims of pair t / 8.
    float *const so = reinterpret_cast<float *>(s_raw);
    float *const sm = so + kWaves * 32 * OSTR;  // m[4][32], then l[4][32]
    int *const s_bad = reinterpret_cast<int *>(sm + 64 * kWaves);
    __syncthreads();  // the last tile has been read
#pragma unroll
    for (int md = 0; md < MD; ++md)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4 *>(&so[(wave * 32 + col) * OSTR + 32 * md + 8 * j + 4 * h]) =
            f32x4{o[md][4 * j], o[md][4 * j + 1], o[md][4 * j + 2], o[md][4 * j + 3]};
    if (h == 0) {
      sm[wave * 32 + col] = m;
      sm[kWaves * 32 + wave * 32 + col] = l;
    }
    if (tid < 32) s_bad[tid] = 0;
    __syncthreads();
    const int c = tid >> 3;
    float M = -INFINITY, L = 0.f, a[kWaves];
#pragma unroll
    for (int u = 0; u < kWaves; ++u) M = fmaxf(M, sm[u * 32 + c]);
#pragma unroll
    for (int u = 0; u < kWaves; ++u) {
      const float mu = sm[u * 32 + c];
      a[u] = mu == -INFINITY ? 0.f : fast_exp2(mu - M);
      // A wave that saw no key has l = 0; a NaN l (a NaN score) must stay.
      L += sm[kWaves * 32 + u * 32 + c] * (mu == -INFINITY ? 1.f : a[u]);
    }
    const float inv = whole ? 1.f / L : 1.f;
    constexpr int DT = DP / 8;
    f32x4 y[DT / 4];
    bool ok = true;
#pragma unroll
    for (int i = 0; i < DT / 4; ++i) {
      const int d = 32 * i + 4 * (tid & 7);
      y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < kWaves; ++u) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(&so[(u * 32 + c) * OSTR + d]);
        y[i] += x * a[u];
      }
      y[i] *= inv;
#pragma unroll
      for (int e = 0; e < 4; ++e) ok = ok && (finite(y[i][e]) || d >= D);
    }
    const bool c_live = c < n;
    if (!whole) {
      if (!c_live) return;
      const int64_t g = slot;
      const int x = tid & 7;
#pragma unroll
      for (int i = 0; i < DT / 4; ++i)
        if (32 * i < D) store4(P.part_o(g, i, x >> 1, 32 * (x & 1) + c), y[i]);
      if (x == 0) *reinterpret_cast<float2 *>(P.part_ml(g, c)) = make_float2(M, L);
      return;
    }
    if (c_live && !ok) s_bad[c] = 1;
    __syncthreads();
    if (c_live && s_bad[c] == 0) {
      E *co = static_cast<E *>(P.out) + pair_at(c);
#pragma unroll
      for (int i = 0; i < DT / 4; ++i) {
        const int d = 32 * i + 4 * (tid & 7);
        if (d < D) store4(co + d, y[i]);
      }
    }
    for (int x = wave; x < 32; x += kWaves) {
      if (__builtin_expect(s_bad[x] == 0, 1)) continue;
      careful_pair<E, DP, 32, TREE>(P, row, kvh, pair_at(x), s0 + pair_pos(x), lane, 0, D,
                                    tok0 + pair_pos(x), pair_pos(x));
    }
  }
}

// Merges the partials of key ranges, in the partials' own layout: a workgroup per 32 pairs and 32 dims of
// a block, a wave per step j of them, eight ranges' loads in flight. What the blocks are, and whether any is
// cut, the kernel before has left (each workgroup finding its block again took 10.4 us where none was cut:
// 17 rows of up to 10 tokens, 32 / 8 heads).
template <class E, bool TREE>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(TiledParams P, int pairs) {
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int j = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = P.tiles.groups;
  int id = blockIdx.x;
  const int md = id % P.md;
  id /= P.md;
  const int w = id % groups;
  id /= groups;  // the block
  const int d = 32 * md + 8 * j;  // this wave's dims d .. d + 7, lane half h d + 4h ..
  const int n_blocks = *P.tiles.n_cuts;
  const PagedTiles::Cut blk = P.tiles.cuts[id];
  const int ranges = blk.ranges;
  if (d >= P.D || id >= (TREE ? n_blocks * P.H_kv : n_blocks) || ranges == 1) return;  // of one range: written by the block itself
  const int kvh = id % P.H_kv;
  const int64_t n_pairs = int64_t(blk.T) * P.G, p0 = int64_t(blk.qt) * pairs;
  const int n = int(min(int64_t(pairs), n_pairs - p0));
  const int in_block = 32 * w + col;
  if (TREE && 32 * w >= n) return;  // no pair of the 32
  const bool live = in_block < n;
  const int t = live ? int((p0 + in_block) / P.G) : 0;
  auto pair_at = [&](int i) {
    const int tt = int((p0 + i) / P.G);
    return ((int64_t(blk.tok0) + tt) * P.H + int64_t(kvh) * P.G + int(p0 + i - int64_t(tt) * P.G)) * P.D;
  };

  constexpr int U = 8;
  int64_t group = int64_t(id) * groups + w, step = int64_t(n_blocks) * groups;
  int64_t second = int64_t(blk.second) * groups + w;
  if constexpr (TREE) {  // the ranges one after another, KV heads between them
    group = second;
    step = int64_t(P.H_kv) * groups;
    second += step;
  }
  float M = -INFINITY, L = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < ranges; r0 += U) {
    float2 x[U];
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = min(r0 + u, ranges - 1);
      const int64_t g = r == 0 ? group : second + (r - 1) * step;
      x[u] = *reinterpret_cast<const float2 *>(P.part_ml(g, col));
      v[u] = *reinterpret_cast<const f32x4 *>(P.part_o(g, md, j, lane));
    }
    float m_new = M;
#pragma unroll
    for (int u = 0; u < U; ++u) m_new = fmaxf(m_new, x[u].x);
    const float keep = M == -INFINITY ? 0.f : fast_exp2(M - m_new);
    L *= M == -INFINITY ? 1.f : keep;  // 0 then, or a NaN that must stay
    y *= keep;
    M = m_new;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u >= ranges) break;
      const float a = x[u].x == -INFINITY ? 0.f : fast_exp2(x[u].x - M);
      L += x[u].y * (x[u].x == -INFINITY ? 1.f : a);
      y += a * v[u];
    }
  }
  y *= 1.f / L;
  const bool ok = (finite(y[0]) && finite(y[1]) && finite(y[2]) && finite(y[3])) || d + 4 * h >= P.D;
  const uint64_t bad64 = __builtin_amdgcn_ballot_w64(live && !ok);
  const uint32_t bad = uint32_t(bad64) | uint32_t(bad64 >> 32);
  if (live && !((bad >> col) & 1u) && d + 4 * h < P.D)
    store4(static_cast<E *>(P.out) + pair_at(in_block) + d + 4 * h, y);
  for (uint32_t left = bad; __builtin_expect(left != 0, 0); left &= left - 1) {
    const int c = __builtin_ctz(left);
    const int t_c = __builtin_amdgcn_readlane(t, c);
    careful_pair<E, 256, 4, TREE>(P, blk.b, kvh, pair_at(32 * w + c), blk.s0 + t_c, lane, d, min(d + 8, P.D),
                                  int64_t(blk.tok0) + t_c, t_c);
  }
}

// What a call runs: the waves over pairs (KS = 1) or keys (KS = 4), and room for the partials of cut
// blocks.
struct TiledPlan {
  int ks, pairs, kt, slots, min_tiles, target;
  int64_t bound;  // of blocks
  float tile_us;
};
constexpr float kShortUs = 30.f;
// Of a range, at least: starting one takes about as long. Two chunks of 94, 16 / 4 heads of 64 in bf16, up to 864
// keys: 15.8 us, with ranges of 6 us 26.2.
constexpr float kRangeUs = 3.f;
TiledPlan tiled_plan(const PagedArgs &a, int64_t skip) {
  const bool bf = a.dtype == MCAMD_BF16;
  auto plan = [&](int ks) {
    TiledPlan t;
    t.ks = ks;
    t.pairs = 128 / ks;
    t.kt = ks == 4 ? 128 : bf && a.head_dim <= 128 ? 64 : 32;
    t.bound = paged_blocks_bound(a, t.pairs, skip);
    // Measured time of a tile on a compute unit of its own, per head dim (prefill_tiled.hip).
    t.tile_us = float(a.head_dim) * (ks == 4 ? (bf ? 0.027f : 0.085f) : (bf ? 0.012f : 0.035f));
    t.min_tiles = std::max(1, int(kRangeUs / t.tile_us));
    // Trees: workgroups of four waves on the keys, and those of wide heads, one a compute unit, with two of which the
    // ranges are shorter than it takes to begin one (one row of 5 nodes after 4000 tokens, 12 heads of 64: 19.7 us for
    // 26.0; two rows of 256 after 4000, 12 / 4 heads of 128: 146 and 159; eight rows of 256 in 64 dims 335 for 244).
    t.target = (ks == 1 && a.head_dim <= 64 ? 2 : 1) * device_cus();
    if (a.tree.masks)
      t.slots = paged_keys(a) >= 2 * int64_t(t.min_tiles) * t.kt ? int(tree_slots(t.target, a.n_kv_head)) : 0;
    else
      t.slots = paged_slots(a, t.bound, t.pairs, a.head_dim <= 128 ? 2 : 1, int64_t(t.min_tiles) * t.kt);
    return t;
  };
  const TiledPlan whole = plan(1);
  if (a.head_dim > 128) return whole;  // a tile of four waves' keys outgrows the LDS
  // KS = 4 takes twice to four times as long for the same pairs and keys, and is for calls that cannot fill
  // the chip otherwise: fewer blocks of 128 pairs than compute units, and rows of so few pairs that half of
  // such a block would be empty, or too few keys for ranges that are worth their merge (kShortUs). The keys
  // are those that the table has room for: the lengths are not known here, and the same prompts under a
  // table of 2048 positions are cut. Four waves on the keys against ranges with their merge: two prompts of
  // 512, 12 heads of 64 in fp32 (24 us by that count, in a table of 576) 22.6 and 33.1; two prompts of 830, 12 / 4 heads of 128 in fp32 (71) 93 and 86; two chunks of 512
  // after 2000, 12 heads of 64 in bf16 (55) 37 and 33.
  const TiledPlan four = plan(4);
  // Trees of at most 64 pairs always take it: most waves of a block of 128 pairs would have none, however many blocks
  // there are. 64 rows of 2 nodes after 1000 to 3000 tokens, 8 heads of 64: 191 us for 410; 20 rows of 60 after 300
  // to 1000, 12 heads of 64: 75 and 87; 30 rows of 50, 8 heads of 128: 119 and 148.
  if (a.tree.masks && a.t_new * (a.n_head / a.n_kv_head) <= 64) return four;
  const bool fills = whole.bound * a.n_kv_head >= device_cus();
  const bool few = a.t_new * (a.n_head / a.n_kv_head) <= 64;
  const bool brief = float(paged_keys(a)) / float(four.kt) * four.tile_us <= kShortUs;
  return !fills && (few || brief || whole.slots == 0) ? four : whole;
}
int64_t slot_floats(const PagedArgs &a, int pairs) {
  return int64_t(pairs) * ((a.head_dim + 31) / 32 * 32 + 2);
}

TiledParams tiled_params(const PagedArgs &a, const PagedTiles &tiles) {
  TiledParams P;
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
  P.k_new = a.tree.masks ? a.k_new : nullptr;  // of other calls they are in their pages
  P.v_new = a.tree.masks ? a.v_new : nullptr;
  P.seqlens = a.seqlens;
  P.cu = a.cu;
  P.T_new = int(a.t_new);
  P.H = int(a.n_head);
  P.G = int(a.n_head / a.n_kv_head);
  P.deal = device_cus();
  P.tiles = tiles;
  P.md = int((a.head_dim + 31) / 32);
  return P;
}

template <class E, int DP, int KS>
int run(const TiledParams &P, const PagedArgs &a, const TiledPlan &t) {
  using G_ = Geo<E, DP, KS>;
  if (t.pairs != G_::PAIRS || t.kt != G_::KT)
    return fail(MCAMD_EINVAL, "paged attention: plan and kernel disagree");
  const int64_t blocks = a.tree.masks && P.tiles.slots > 0 ? tree_blocks(t.bound, t.target, P.H_kv)
                                                           : std::max<int64_t>(t.bound * P.H_kv, P.tiles.slots);
  if (blocks > 0x7fffffff / kThreads) return fail(MCAMD_EUNSUPPORTED, "paged attention: grid too large");
  if (blocks == 0) return MCAMD_OK;
  auto kernel = paged_tiled_kernel<E, DP, KS, false>;
  if constexpr (std::is_same<E, float>::value)  // trees in bf16: tree_stream.hip, paged_stream.hip
    if (a.tree.masks) kernel = paged_tiled_kernel<E, DP, KS, true>;
  hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kThreads), 0, a.stream, P);
  const int st = launch_status("paged_tiled");
  if (st != MCAMD_OK || P.tiles.slots == 0) return st;
  return launch_paged_tiles_merge(a, P.tiles, t.pairs, t.bound);
}

template <class E, int DP>
int run_ks(const TiledParams &P, const PagedArgs &a, const TiledPlan &t) {
  if constexpr (DP <= 128) {
    if (t.ks == 4) return run<E, DP, 4>(P, a, t);
  }
  return run<E, DP, 1>(P, a, t);
}

template <class E>
int dispatch(const TiledParams &P, const PagedArgs &a, const TiledPlan &t) {
  if (P.D <= 32) return run_ks<E, 32>(P, a, t);
  if (P.D <= 64) return run_ks<E, 64>(P, a, t);
  if (P.D <= 96) return run_ks<E, 96>(P, a, t);
  if (P.D <= 128) return run_ks<E, 128>(P, a, t);
  if (P.D <= 192) return run_ks<E, 192>(P, a, t);
  return run_ks<E, 256>(P, a, t);
}

}  // namespace

int launch_paged_tiles_merge(const PagedArgs &a, const PagedTiles &tiles, int pairs, int64_t bound) {
  const TiledParams P = tiled_params(a, tiles);
  // Of more blocks than slots none is cut; of a tree's a cut one has two at least.
  const int64_t cut = a.tree.masks ? tiles.slots / 2 : tiles.slots;
  const int64_t blocks = std::min<int64_t>(bound * P.H_kv, cut) * tiles.groups * P.md;
  if (blocks > 0x7fffffff / kThreads) return fail(MCAMD_EUNSUPPORTED, "paged attention: grid too large");
  const dim3 grid{unsigned(blocks)}, threads{kThreads};
  const auto kernel = a.dtype == MCAMD_BF16 ? paged_merge_kernel<bf16, false>
                      : a.tree.masks        ? paged_merge_kernel<float, true>
                                            : paged_merge_kernel<float, false>;
  hipLaunchKernelGGL(kernel, grid, threads, 0, a.stream, P, pairs);
  return launch_status("paged_merge");
}

size_t paged_tiled_bytes(const PagedArgs &a, int64_t skip) {
  const TiledPlan t = tiled_plan(a, skip);
  return paged_tiles_bytes(t.slots, slot_floats(a, t.pairs));
}

int launch_paged_tiled(const PagedArgs &a, int64_t skip) {
  const TiledPlan t = tiled_plan(a, skip);
  PagedTiles T;
  T.kv = a.kv;
  T.n_rows = int(a.n_rows);
  T.total = int(a.total);
  T.skip = int(skip);
  T.kt = t.kt;
  T.groups = t.pairs / 32;
  T.min_tiles = t.min_tiles;
  T.target = t.target;
  paged_tiles_buffers(a, T, t.slots, slot_floats(a, t.pairs), t.pairs * 2);
  T.ratio = t.tile_us * MCAMD_SPLIT_BYTES_PER_US / (float(slot_floats(a, t.pairs)) * 8.f);
  const TiledParams P = tiled_params(a, T);
  return a.dtype == MCAMD_BF16 ? dispatch<bf16>(P, a, t) : dispatch<float>(P, a, t);
}

}  // namespace mcamd
