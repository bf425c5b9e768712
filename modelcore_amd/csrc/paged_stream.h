// What the streaming kernels of a paged cache (rows of few pairs) share: how a call's keys are cut into
// ranges, worked out on the device from the rows' lengths, and the merge of the ranges.
//
// A row's keys are cut into ranges of whole 32-key tiles; a workgroup of four waves owns (row, block of
// pairs, range, group of KV heads). In a large call a wave has a KV head (the four read token rows in runs of
// four heads, and nothing is shared between them); in one whose tiles are few the four waves take every
// fourth tile of one head, so that short rows are a tile deep. Ranges are of `len` tiles such that all
// ranges are on the chip at once (`target` workgroups), at least kMinTiles. Every wave does this sum by
// itself, 64 rows at a time.
#pragma once

#include "paged_append.h"
#include "paged_careful.h"

#include <algorithm>
#include <cmath>

namespace mcamd {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int KT = 32;        // keys per tile
constexpr int kMinTiles = 2;  // of a wave's range, unless the row is shorter
// A head per wave from so many tiles a wave on. One row of 16K keys, 8 KV heads (2 a wave): 27.1 us so,
// 18.8 with four waves a head; 60 rows of 4160 keys on average (15.6): 167.9 and 210.
constexpr int kDeepTiles = 4;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) int32_t *scalar_ints;  // read only, by the scalar unit

struct StreamParams : CarefulParams {
  const int32_t *seqlens, *cu;
  float *part_o, *part_ml;  // [slot][pair_slots][DP], [slot][pair_slots][2]
  int2 *where;              // per row: its first range and the ranges of a block, for the merge
  int n_rows, t_new, total, H, G;
  int most;        // pairs of a row, at most (a single token's rows are always taken)
  int head_waves;  // KV heads of a workgroup, in a large call
  int target;      // workgroups a call aims at; 0: no row is cut
  int pair_slots;  // pairs per partial slot
  int early;       // of trees 1: a node without a bit stands a position before the row's next
  PagedAppend append;
  int blocks;      // workgroups from that one on append
};

// The rows' shares of a call. A row has `blocks` blocks of PB pairs and `tiles` tiles; a range is at most
// `len` tiles. A row that does not fit its table has one block of one (empty) range, which writes NaN.
struct Row {
  int tok0, T, s0, lo, hi, blocks, tiles;
  bool ok;
};

template <int PB>
__device__ __forceinline__ Row row_of(const StreamParams &P, int b) {
  Row r;
  row_tokens(P.cu, P.t_new, P.total, b, r.tok0, r.T);
  r.s0 = P.seqlens[b];
  r.ok = r.s0 >= 0 && int64_t(r.s0) + r.T <= int64_t(P.kv.max_pages) << P.kv.shift;
  r.lo = r.ok && P.window >= 0 ? max(0, r.s0 - P.window - P.early) : 0;
  r.hi = r.ok ? r.s0 + r.T - 1 : 0;
  r.blocks = few_pairs(r.T, P.G, P.most) ? int(uint32_t(r.T * P.G + PB - 1) / PB) : 0;
  r.tiles = r.ok ? (r.hi / KT) - (r.lo / KT) + 1 : 1;
  return r;
}

__device__ __forceinline__ int64_t wave_total64(int64_t x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// How a call is cut: KV heads of a workgroup, and tiles of a range, at most.
struct Cut {
  int head_waves, len;
};
template <int PB>
__device__ __forceinline__ Cut cut_of(const StreamParams &P, int lane, const Row &first) {
  int64_t work = 0, units = 0;
  for (int b = lane; b < P.n_rows; b += 64) {
    const Row r = b == lane ? first : row_of<PB>(P, b);
    work += int64_t(r.blocks) * r.tiles;
    units += r.blocks;
  }
  if (P.target == 0) return Cut{1, 0x7fffffff};
  Cut c;
  auto cut = [&](auto work, auto units) {
    using T = decltype(work);
    c.head_waves = int64_t(work) * P.H_kv > int64_t(kDeepTiles * kWaves) * P.target ? P.head_waves : 1;
    // A row's last range may be shorter than the others: work / len ranges and up to one per block of pairs
    // more, all of which are to be on the chip at once.
    const int target = max(1, int(uint32_t(P.target * c.head_waves) / uint32_t(P.H_kv)));
    const T most = units < T(target / 2) ? T(target) - units : T((target + 1) / 2);
    c.len = int(max((work + most - 1) / most, T(kMinTiles * kWaves) / T(c.head_waves)));
  };
  if (__builtin_amdgcn_ballot_w64(work >= (1 << 24)) == 0)  // the sums fit 32 bits
    cut(uint32_t(wave_total(int(work))), uint32_t(wave_total(int(units))));
  else
    cut(uint64_t(wave_total64(work)), uint64_t(wave_total64(units)));
  c.head_waves = __builtin_amdgcn_readfirstlane(c.head_waves);  // so the compiler knows as well
  c.len = __builtin_amdgcn_readfirstlane(c.len);
  return c;
}
__device__ __forceinline__ int ranges_of(const Row &r, int len) {
  return int((uint32_t(r.tiles) + uint32_t(len) - 1) / uint32_t(len));
}

// A workgroup's range: KV heads `group` of the groups there are, row b (-1: none), its block of pairs and
// which of the row's ranges.
struct Range {
  int head_waves, n_groups, group, b, block, range, ranges;
  int t0, t1;  // its tiles, from the row's first one on
};
template <int PB>
__device__ __forceinline__ Range find_range(const StreamParams &P, int lane, Row &R) {
  const Row mine = row_of<PB>(P, min(lane, P.n_rows - 1));
  const Cut cut = cut_of<PB>(P, lane, mine);
  Range v;
  v.head_waves = cut.head_waves;
  v.n_groups = P.H_kv / cut.head_waves;
  v.group = blockIdx.x % v.n_groups;
  v.b = -1;
  v.ranges = 0;
  int id = blockIdx.x / v.n_groups;  // of the ranges of all rows
  for (int b0 = 0; b0 < P.n_rows; b0 += 64) {
    Row r = mine;
    if (b0 > 0) r = row_of<PB>(P, min(b0 + lane, P.n_rows - 1));
    const int rr = ranges_of(r, cut.len);
    const int n = b0 + lane < P.n_rows ? rr * r.blocks : 0;
    const int upto = wave_upto(n, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > id);
    if (past == 0) {
      id -= __builtin_amdgcn_readlane(upto, 63);
      continue;
    }
    const int l = __builtin_ctzll(past);
    v.b = b0 + l;
    id -= __builtin_amdgcn_readlane(upto - n, l);
    v.ranges = __builtin_amdgcn_readlane(rr, l);
    R.tok0 = __builtin_amdgcn_readlane(r.tok0, l);
    R.T = __builtin_amdgcn_readlane(r.T, l);
    R.s0 = __builtin_amdgcn_readlane(r.s0, l);
    R.lo = __builtin_amdgcn_readlane(r.lo, l);
    R.hi = __builtin_amdgcn_readlane(r.hi, l);
    R.tiles = __builtin_amdgcn_readlane(r.tiles, l);
    R.ok = __builtin_amdgcn_readlane(int(r.ok), l);
    break;
  }
  if (v.b < 0) return v;
  v.block = int(uint32_t(id) / uint32_t(v.ranges));
  v.range = id - v.block * v.ranges;
  // Tiles from range * tiles / ranges on, of the row's.
  const uint32_t each = uint32_t(R.tiles) / uint32_t(v.ranges), rest = R.tiles - each * v.ranges;
  v.t0 = int(each * v.range + rest * v.range / v.ranges);
  v.t1 = int(each * (v.range + 1) + rest * (v.range + 1) / v.ranges);
  if (id == 0 && v.group == 0 && threadIdx.x == 0 && P.where)
    P.where[v.b] = make_int2(int(blockIdx.x / v.n_groups), v.ranges);
  return v;
}

// The ranges of a pair added up: a workgroup of MW waves per pair, each of which takes every MW-th range,
// lane l dims l, l + 64, .. The streaming kernel has left where a row's ranges lie. Bound by the latency of
// three round trips, and with many pairs by how many workgroups the chip holds: few pairs, whose rows are
// in many ranges, take eight waves (one row of 16K keys, 64 ranges: 4.2 us, with four 8.5), more than
// kManyPairs two (60 rows of 32 heads: 6.3 us, with four 7.9, with eight 11.0).
constexpr int64_t kManyPairs = 1024;
// Workgroups of a packed call's merge, at most, beyond one per head of each row: three rows of 8 to 57
// tokens of one head per KV head took 37 us with a workgroup a row and KV head.
constexpr int64_t kMergeGroups = 1024;
template <class E, int DP, int MW, int PB, bool TREE>
__global__ __launch_bounds__(64 * MW) void paged_stream_merge_kernel(StreamParams P) {
  constexpr int N = (DP + 63) / 64, U = 8;
  __shared__ float s_o[MW][DP], s_ml[MW][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x % P.H_kv;
  const int b = blockIdx.y;
  const int2 where = P.where[b];
  const Row R = row_of<PB>(P, b);
  if (R.blocks == 0 || !R.ok) return;
  const int ranges = where.y;
  if (ranges == 1) return;  // written already
  const int64_t step = int64_t(P.H_kv) * P.pair_slots;  // from range to range
  for (int pair = blockIdx.x / P.H_kv; pair < R.T * P.G; pair += gridDim.x / P.H_kv) {
    const int64_t unit = where.x + int64_t(pair / PB) * ranges;
    const int64_t slot = (unit * P.H_kv + kvh) * P.pair_slots + pair % PB;
    float M = -INFINITY, L = 0.f, o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.f;
    auto join = [&](float m2, float l2, const float (&o2)[N]) {
      const float m_new = fmaxf(M, m2);
      const float a1 = M == -INFINITY ? 0.f : fast_exp2(M - m_new);
      const float a2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - m_new);
      // A range without a key has l = 0; a NaN l must stay.
      L = L * (M == -INFINITY ? 1.f : a1) + l2 * (m2 == -INFINITY ? 1.f : a2);
      M = m_new;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(o2[i], a2, o[i] * a1);
    };
    for (int r0 = wave; r0 < ranges; r0 += U * MW) {
      float2 x[U];
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = slot + min(r0 + u * MW, ranges - 1) * step;
        x[u] = *reinterpret_cast<const float2 *>(P.part_ml + at * 2);
#pragma unroll
        for (int i = 0; i < N; ++i) v[u][i] = P.part_o[at * DP + min(lane + 64 * i, P.D - 1)];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r0 + u * MW < ranges) join(x[u].x, x[u].y, v[u]);
    }
    __syncthreads();  // the pair before has been added up
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < DP) s_o[wave][lane + 64 * i] = o[i];
    if (lane == 0) s_ml[wave][0] = M, s_ml[wave][1] = L;
    __syncthreads();
    if (wave > 0) continue;
#pragma unroll
    for (int w = 1; w < MW; ++w) {
      float o2[N];
#pragma unroll
      for (int i = 0; i < N; ++i) o2[i] = s_o[w][min(lane + 64 * i, DP - 1)];
      join(s_ml[w][0], s_ml[w][1], o2);
    }
    const float inv = 1.f / L;
    const int t = pair / P.G;
    const int64_t at = (int64_t(R.tok0 + t) * P.H + kvh * P.G + (pair - t * P.G)) * P.D;
    bool ok = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i] *= inv;
      ok = ok && (finite(o[i]) || lane + 64 * i >= P.D);
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!ok) != 0, 0)) {
      careful_pair<E, DP, 8, TREE>(P, b, kvh, at, R.s0 + t, lane, 0, P.D, R.tok0 + t, t);
      continue;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < P.D) static_cast<E *>(P.out)[at + lane + 64 * i] = from_f32<E>(o[i]);
  }
}

struct StreamPlan {
  int head_waves, target, pair_slots;
  int64_t units;        // blocks of pairs of all rows, at most
  int64_t merge_pairs;  // workgroups of the merge per (row, KV head)
  bool cut;
};

// `block`: pairs of a block; `fill`: workgroups per compute unit that a call aims at.
StreamPlan stream_plan(const PagedArgs &a, int64_t most, int64_t block, int fill) {
  StreamPlan p;
  const int64_t G = a.n_head / a.n_kv_head;
  p.head_waves = a.n_kv_head % 4 == 0 ? 4 : a.n_kv_head % 2 == 0 ? 2 : 1;
  p.target = fill * device_cus();
  const int64_t max_pairs = std::min(a.t_new * G, std::max(most, G));
  // Of a mixture most rows have one token; a workgroup of more goes round.
  p.merge_pairs = a.cu ? std::max(G, std::min(max_pairs, kMergeGroups / (a.n_rows * a.n_kv_head))) : max_pairs;
  p.units = a.n_rows * ((max_pairs + block - 1) / block);
  p.pair_slots = int(std::min<int64_t>(block, max_pairs));
  const int64_t room = int64_t(a.kv.max_pages) << a.kv.shift;
  const int64_t keys = std::min(room, a.window >= 0 ? a.window + 2 * KT + most : room);
  p.cut = (keys + KT - 1) / KT > kMinTiles * kWaves;
  return p;
}

int head_pad(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }

int64_t slots_of(const PagedArgs &a, const StreamPlan &p) {
  // unit ids * H_kv: a call's ranges, at most target * head_waves / H_kv and one per unit.
  return ((p.units + 1) * a.n_kv_head + int64_t(p.target) * p.head_waves) * p.pair_slots;
}

size_t stream_bytes(const PagedArgs &a, const StreamPlan &p) {
  return p.cut ? size_t(slots_of(a, p)) * (head_pad(a.head_dim) + 2) * 4 + size_t(a.n_rows) * 8 : 0;
}

StreamParams stream_params(const PagedArgs &a, const StreamPlan &p, int64_t most) {
  StreamParams P;
  P.q = a.q;
  P.k_pages = a.k_pages;
  P.v_pages = a.v_pages;
  P.kv = a.kv;
  P.out = a.out;
  P.H_kv = int(a.n_kv_head);
  P.window = int(a.window < 0 ? -1 : a.window);
  P.D = int(a.head_dim);
  P.scale_log2 = float(kLog2e / std::sqrt(double(a.head_dim)));
  P.k_new = a.k_new;
  P.v_new = a.v_new;
  P.seqlens = a.seqlens;
  P.cu = a.cu;
  P.part_o = static_cast<float *>(a.scratch);
  P.part_ml = P.part_o + slots_of(a, p) * head_pad(a.head_dim);
  P.where = p.cut ? reinterpret_cast<int2 *>(P.part_ml + slots_of(a, p) * 2) : nullptr;
  P.n_rows = int(a.n_rows);
  P.t_new = int(a.t_new);
  P.total = int(a.total);
  P.H = int(a.n_head);
  P.G = int(a.n_head / a.n_kv_head);
  P.most = int(most);
  P.head_waves = p.head_waves;
  P.target = p.cut ? p.target : 0;
  P.pair_slots = p.pair_slots;
  P.tree = a.tree;
  P.early = a.tree.masks ? 1 : 0;
  P.append = paged_append(a, most);
  // A KV head at a time, or up to the target.
  P.blocks = int(std::min<int64_t>(
      p.units * a.n_kv_head + (p.cut ? std::max<int64_t>(p.target, a.n_kv_head) : 0), 0x7fffffff));
  return P;
}

// kernel: the launch of a call's ranges, by E, DP (head dims, rounded up) and blocks of PB pairs.
template <class E, int DP, int PB, bool TREE = false, class K>
int launch_stream(K kernel, const StreamParams &P, const PagedArgs &a, const StreamPlan &p, bool others) {
  const int64_t blocks = P.blocks + (a.k_new && others ? paged_append_blocks(a) : 0);
  if (blocks > 0x7fffffff / kThreads || a.n_rows > 65535)
    return fail(MCAMD_EUNSUPPORTED, "paged attention: grid too large");
  hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kThreads), 0, a.stream, P);
  const int st = launch_status("paged_stream");
  if (st != MCAMD_OK || !p.cut) return st;
  const dim3 grid{unsigned(a.n_kv_head * p.merge_pairs), unsigned(a.n_rows)};
  if ((a.cu ? a.n_rows * a.n_head : int64_t(grid.x) * grid.y) > kManyPairs)  // of a mixture, the single tokens
    hipLaunchKernelGGL((paged_stream_merge_kernel<E, DP, 2, PB, TREE>), grid, dim3(128), 0, a.stream, P);
  else
    hipLaunchKernelGGL((paged_stream_merge_kernel<E, DP, 8, PB, TREE>), grid, dim3(512), 0, a.stream, P);
  return launch_status("paged_stream_merge");
}

}  // namespace
}  // namespace mcamd
