// Single tokens over a paged fp32 cache: the streaming kernel without matrix cores, whose fp32 products
// would wait for their operands' way through LDS.
//
// How a call is cut into ranges of keys, a workgroup's: paged_stream.h. A wave walks its tiles by halves of
// 16 keys, which share a page. A lane has 16 bytes of a row, dims 4 c .. + 3, so that DP / 4 lanes have a key
// and a load takes 64 / (DP / 4) of them; K of the next half is under way from the moment V of this one is
// asked for. A key's score is summed over its lanes (cross-lane adds within 16 lanes, two swaps beyond), and
// the groups of lanes keep a running (o, m, l) each, over the keys they have seen: nothing crosses them
// before the end of the range. GP query heads of a KV head share its keys; more of them are blocks of their
// own. All arithmetic is fp32; weights are exp2 of fp32 scores.
//
// Bound by the stream from HBM: 32 rows of 512 to 8191 keys, 16 / 4 heads of 128, 571 MB in 98 us with the
// append (5.8 TB/s; the tiled kernel 547), 64 rows of 512 to 1023 keys, 12 heads of 64, 302 MB in 55. Two rows of 80
// keys take 6.6, start-up, and where the table has room for more than 256 keys a merge of nothing (1.9 traced, 3.5 us
// of the call). Registers set how many workgroups a compute unit holds: four instead of three at
// head dim 64 spill with four heads (50.9 -> 77.0 us) and gain 3% with one.
//
#include "paged_stream.h"

namespace mcamd {
namespace {

constexpr int kNonTemporal = 2;  // cache policy of the pages' loads
// Workgroups per compute unit that a call aims at: as many as its registers let run.
constexpr int fill_of(int dp) { return dp <= 32 ? 4 : dp <= 64 ? 3 : dp <= 128 ? 2 : 1; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// x of the lanes of a key added up, in each of them (LPK consecutive lanes).
template <int LPK>
__device__ __forceinline__ float key_sum(float x) {
  auto add = [&](auto ctrl) {
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xB1>{});  // quad_perm 1 0 3 2
  add(std::integral_constant<int, 0x4E>{});  // quad_perm 2 3 0 1
  add(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (LPK >= 16) add(std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (LPK >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LPK >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// (o, m, l) joined with (o2, m2, l2). Without a key l = 0; a NaN l must stay.
__device__ __forceinline__ void join(f32x4 &o, float &m, float &l, f32x4 o2, float m2, float l2) {
  const float m_new = fmaxf(m, m2);
  const float a1 = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
  const float a2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - m_new);
  l = l * (m == -INFINITY ? 1.f : a1) + l2 * (m2 == -INFINITY ? 1.f : a2);
  o = o * a1 + o2 * a2;
  m = m_new;
}

template <int DP, int GP>
__global__ __launch_bounds__(kThreads)
    __attribute__((amdgpu_waves_per_eu(fill_of(DP)))) void paged_stream_f32_kernel(StreamParams P) {
  constexpr int LPK = DP / 4, KPI = 64 / LPK, NV = 16 / KPI;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][GP][DP];
  __shared__ float s_ml[kWaves][GP][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (int(blockIdx.x) >= P.blocks) return append_tokens(P.append, int(blockIdx.x) - P.blocks);
  Row R;
  const Range mine = find_range<GP>(P, lane, R);
  if (mine.b < 0) return;
  const int b = mine.b, ranges = mine.ranges, head_waves = mine.head_waves;
  const int kvh = mine.group * head_waves + wave % head_waves;
  const int kw = wave / head_waves, n_kw = kWaves / head_waves;  // this wave's share of the tiles
  const int D = P.D;
  const int g0 = mine.block * GP, n_g = min(GP, P.G - g0);  // the block's heads
  const int lr = lane / LPK, d = 4 * (lane % LPK);          // this lane's key of a load, and its dims
  const int64_t at = (int64_t(R.tok0) * P.H + kvh * P.G + g0) * D;  // of the first head's pair
  float *out = static_cast<float *>(P.out) + at;
  if (!R.ok) {
    if (kw == 0)
      for (int i = lane; i < n_g * D; i += 64) out[i] = NAN;
    return;
  }

  f32x4 q[GP];
#pragma unroll
  for (int g = 0; g < GP; ++g) {
    q[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (g < n_g && d < D)
      q[g] = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(P.q) + at + g * D + d);
  }

  const int first_tile = R.lo / KT;
  const int t0 = first_tile + mine.t0, t1 = first_tile + mine.t1;
  const int seen_from = R.lo, s0 = R.s0;  // the keys the token sees, itself the last
  const bool fresh = P.k_new != nullptr;
  const int tok_bytes = P.H_kv * D * 4;
  constexpr uint32_t kNowhere = 0x80000000u;
  const uint32_t in_row = d < D ? uint32_t(lr * tok_bytes + 4 * d) : kNowhere;
  const scalar_ints table = (scalar_ints)(P.kv.table + b * P.kv.table_stride);
  const int64_t head_at = int64_t(kvh) * D * 4;
  const uint32_t page_bytes = uint32_t(tok_bytes) << P.kv.shift;
  const int64_t new_at = int64_t(R.tok0) * tok_bytes + head_at + 4 * d;
  bool lost = false;

  auto load = [&](const void *pool, const void *new_rows, int k0, f32x4 (&x)[NV]) {
    const bool some = k0 + 15 >= seen_from && k0 <= s0;  // else no key is seen, and page 0 as good as any
    const int id = some ? table[k0 >> P.kv.shift] : 0;
    const bool ok = P.kv.is_page(id);
    lost = lost || !ok;
    const char *base = static_cast<const char *>(pool) + (ok ? id : 0) * P.kv.page_stride * 4 + head_at;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        (void *)base, 0, int(page_bytes - uint32_t(head_at)), 0x00020000);
    const int in_page = P.kv.in_page(k0) * tok_bytes;
    const bool edge = k0 < seen_from || k0 + 15 > s0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t o = in_row;
      if (edge) {
        const int key = k0 + KPI * i + lr;
        o = key >= seen_from && key <= s0 ? o : kNowhere;
      }
      o = o == kNowhere ? o : o + uint32_t(KPI * i * tok_bytes);
      x[i] = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, int(o), in_page, kNonTemporal));
    }
    if (fresh && k0 <= s0 && k0 + 15 >= s0) {  // the token's own key and value, which its page may not hold yet
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      if (d < D) y = *reinterpret_cast<const f32x4 *>(static_cast<const char *>(new_rows) + new_at);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (k0 + KPI * i + lr == s0) x[i] = y;
    }
  };

  f32x4 o[GP];
  float m[GP], l[GP];
#pragma unroll
  for (int g = 0; g < GP; ++g) o[g] = f32x4{0.f, 0.f, 0.f, 0.f}, m[g] = -INFINITY, l[g] = 0.f;

  auto attend = [&](int k0, const f32x4 (&k)[NV], const f32x4 (&v)[NV]) {
    const bool edge = k0 < seen_from || k0 + 15 > s0;
    float s[GP][NV];
#pragma unroll
    for (int g = 0; g < GP; ++g)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float x = fmaf(q[g][3], k[i][3], fmaf(q[g][2], k[i][2], fmaf(q[g][1], k[i][1], q[g][0] * k[i][0])));
        s[g][i] = key_sum<LPK>(x);
      }
    if (edge)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int key = k0 + KPI * i + lr;
        const bool seen = key >= seen_from && key <= s0;
#pragma unroll
        for (int g = 0; g < GP; ++g) s[g][i] = seen ? s[g][i] : -INFINITY;
      }
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      float mx = s[g][0];
#pragma unroll
      for (int i = 1; i < NV; ++i) mx = fmaxf(mx, s[g][i]);
      const float m_new = fmaxf(m[g], mx * P.scale_log2);
      const float alpha = m[g] == -INFINITY ? 0.f : fast_exp2(m[g] - m_new);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      m[g] = m_new;
      l[g] *= alpha;
      o[g] *= alpha;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float w = fast_exp2(fmaf(s[g][i], P.scale_log2, -ref));
        l[g] += w;
        o[g] += w * v[i];
      }
    }
  };

  int tile = t0 + kw;
  f32x4 ka[NV], kb[NV], v[NV];
  if (tile < t1) load(P.k_pages, P.k_new, tile * KT, ka);
  for (; tile < t1; tile += n_kw) {
    const int k0 = tile * KT;
    load(P.v_pages, P.v_new, k0, v);
    load(P.k_pages, P.k_new, k0 + 16, kb);
    attend(k0, ka, v);
    load(P.v_pages, P.v_new, k0 + 16, v);
    if (tile + n_kw < t1) load(P.k_pages, P.k_new, (tile + n_kw) * KT, ka);
    attend(k0 + 16, kb, v);
  }
  // The groups' sums, in all of them.
#pragma unroll
  for (int g = 0; g < GP; ++g) {
#pragma unroll
    for (int off = LPK; off < 64; off <<= 1) {
      f32x4 o2;
#pragma unroll
      for (int e = 0; e < 4; ++e) o2[e] = __shfl_xor(o[g][e], off, 64);
      join(o[g], m[g], l[g], o2, __shfl_xor(m[g], off, 64), __shfl_xor(l[g], off, 64));
    }
    if (lost) l[g] = NAN;
  }

  // The new token into its page: in the row's last range, by the wave that has the fewest tiles. In every
  // block, so that a redo below finds it whichever other block has come how far; they write the same.
  if (fresh && mine.range == ranges - 1 && kw == n_kw - 1 && lane < LPK && d < D) {
    const int id = P.kv.table[b * P.kv.table_stride + (s0 >> P.kv.shift)];
    if (P.kv.is_page(id)) {
      const int64_t to = 4 * (P.kv.offset(id, P.kv.in_page(s0), int64_t(P.H_kv) * D) + d) + head_at;
      const f32x4 x = *reinterpret_cast<const f32x4 *>(static_cast<const char *>(P.k_new) + new_at);
      const f32x4 y = *reinterpret_cast<const f32x4 *>(static_cast<const char *>(P.v_new) + new_at);
      *reinterpret_cast<f32x4 *>(static_cast<char *>(const_cast<void *>(P.k_pages)) + to) = x;
      *reinterpret_cast<f32x4 *>(static_cast<char *>(const_cast<void *>(P.v_pages)) + to) = y;
    }
  }

  // The waves of a KV head add up their sums, each for every n_kw-th query head.
  if (n_kw > 1) {
    if (lane < LPK) {
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        *reinterpret_cast<f32x4 *>(&s_o[wave][g][d]) = o[g];
        if (lane == 0) s_ml[wave][g][0] = m[g], s_ml[wave][g][1] = l[g];
      }
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      o[g] = f32x4{0.f, 0.f, 0.f, 0.f}, m[g] = -INFINITY, l[g] = 0.f;
      if (g % n_kw != kw) continue;
      for (int w = wave % head_waves; w < kWaves; w += head_waves)
        join(o[g], m[g], l[g], *reinterpret_cast<const f32x4 *>(&s_o[w][g][d]), s_ml[w][g][0], s_ml[w][g][1]);
    }
  }

  const bool writes = lane < LPK && d < D;
  if (ranges > 1) {
    const int64_t slot = (int64_t(blockIdx.x) * head_waves + wave % head_waves) * P.pair_slots;
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      if (g >= n_g || g % n_kw != kw) continue;
      if (writes) *reinterpret_cast<f32x4 *>(P.part_o + (slot + g) * DP + d) = o[g];
      if (lane == 0) *reinterpret_cast<float2 *>(P.part_ml + (slot + g) * 2) = make_float2(m[g], l[g]);
    }
    return;
  }
  uint32_t bad = 0;  // heads that are not finite
#pragma unroll
  for (int g = 0; g < GP; ++g) {
    if (g >= n_g || g % n_kw != kw) continue;
    const f32x4 y = o[g] * (1.f / l[g]);
    const bool ok = !writes || (finite(y[0]) && finite(y[1]) && finite(y[2]) && finite(y[3]));
    if (__builtin_amdgcn_ballot_w64(!ok) != 0)
      bad |= 1u << g;
    else if (writes)
      *reinterpret_cast<f32x4 *>(out + g * D + d) = y;
  }
  for (; __builtin_expect(bad != 0, 0); bad &= bad - 1) {
    const int g = __builtin_ctz(bad);
    careful_pair<float, DP, 8>(P, b, kvh, at + g * D, s0, lane, 0, D);
  }
}

template <int GP>
int run(const StreamParams &P, const PagedArgs &a, const StreamPlan &p, bool others) {
  switch (head_pad(a.head_dim)) {
    case 32: return launch_stream<float, 32, GP>(paged_stream_f32_kernel<32, GP>, P, a, p, others);
    case 64: return launch_stream<float, 64, GP>(paged_stream_f32_kernel<64, GP>, P, a, p, others);
    case 128: return launch_stream<float, 128, GP>(paged_stream_f32_kernel<128, GP>, P, a, p, others);
    default: return launch_stream<float, 256, GP>(paged_stream_f32_kernel<256, GP>, P, a, p, others);
  }
}

// Heads of a block: the fewest that take all of a KV head's at once, up to four (the registers of eight
// spill).
int64_t heads_of(const PagedArgs &a) {
  const int64_t G = a.n_head / a.n_kv_head;
  return G <= 2 ? G : 4;
}
StreamPlan plan_of(const PagedArgs &a) {
  return stream_plan(a, 1, heads_of(a), fill_of(head_pad(a.head_dim)));
}

}  // namespace

size_t paged_stream_f32_bytes(const PagedArgs &a) { return stream_bytes(a, plan_of(a)); }

int launch_paged_stream_f32(const PagedArgs &a, bool others) {
  StreamPlan p = plan_of(a);
  if (p.cut && (!a.scratch || a.scratch_bytes < stream_bytes(a, p))) p.cut = false;
  const StreamParams P = stream_params(a, p, 1);
  switch (heads_of(a)) {
    case 1: return run<1>(P, a, p, others);
    case 2: return run<2>(P, a, p, others);
    default: return run<4>(P, a, p, others);
  }
}

}  // namespace mcamd
