// Rows with few new tokens over a paged bf16 cache (single tokens, first of all): every key and value
// is read once from HBM, so the kernel is built around the stream of pages; the products, of which a
// row needs few, go to the matrix cores because they take no time there.
//
// How a call is cut into ranges of keys, a workgroup's: paged_stream.h.
//
// A wave. Its tile of 32 keys is staged in LDS by itself alone, straight from HBM (buffer loads to LDS,
// 16 bytes a lane, whole rows), so that waves never wait for one another: K of the next tile is under way
// from the moment this tile's scores are made, V from the moment its product is. Tiles begin at multiples
// of 32 keys, so 16 keys share a page and a load's page is one scalar: a buffer resource per 16 keys,
// whose bounds are the page's; lanes of keys the row does not see, and of dims past the head's, point
// past it and get zeros.
//   S^T (keys x pairs) = K . Q^T     v_mfma_f32_32x32x16_bf16, 32 (token, head) pairs
//   O^T (D x pairs)   += V^T . P^T   V^T by LDS transpose reads, P as two bf16 terms, p = hi + lo
// in the layouts of prefill_mfma.hip, a pair per lane. Scores, softmax and sums are fp32, q enters as it
// is.
// LDS rows are swizzled in 16-byte chunks, K so that 16 rows' reads of a chunk fall on all banks, V so
// that a transpose read's four rows do.
//
// The loads are marked non-temporal (the pages are read once per call): 32 rows of up to 8192 keys, 16 / 4
// heads of 128, 57.7 -> 51.0 us, 60 rows of 32 / 8 heads 196 -> 165 (6.2 TB/s).
//
// New tokens come from k_new and v_new where given, and a wave of the row's last range puts them in
// their pages. A row of one range writes its output; otherwise (o, m, l) go to scratch in fp32, a row of
// floats per pair, and the merge launch adds the ranges up. Pairs that are not finite are redone
// (paged_careful.h).
#include "paged_stream.h"

namespace mcamd {
namespace {

constexpr int kPairs = 32;  // (token, head) pairs of a block
constexpr int kFill = 2;    // workgroups per compute unit that a call aims at (LDS holds two at DP = 128)
constexpr int kNonTemporal = 2;  // cache policy of the pages' loads

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <int DP>
struct Shape {
  static constexpr int CPR = DP / 8;     // 16-byte chunks of an LDS row
  static constexpr int RPI = 64 / CPR;   // rows of a load
  static constexpr int NI = KT / RPI;    // loads of a tile
  static constexpr int NV = 16 / RPI;    // of 16 keys
  static constexpr int KD = DP / 16, MD = DP / 32;
  static constexpr int TILE = KT * DP;   // elements
  // Chunk c of row r is stored at slot c ^ k_swz(r) (K), c ^ v_swz(r) (V).
  static __device__ __forceinline__ constexpr int k_swz(int r) {
    return CPR >= 16 ? r & 15 : CPR == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  }
  static __device__ __forceinline__ constexpr int v_swz(int r) {
    return CPR >= 16 ? 4 * (r & 3) + ((r >> 2) & 3) : CPR == 8 ? 4 * ((r >> 1) & 1) : 0;
  }
};

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return uint32_t(uintptr_t((const __attribute__((address_space(3))) void *)(p)));
}

// N LDS reads and the wait for them, as one piece: the compiler would wait for the loads to LDS under way
// before any read of its own.
template <int N>
__device__ __forceinline__ void read_rows(bf16x8 (&f)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 8)
    asm volatile(
        "ds_read_b128 %0, %8\n ds_read_b128 %1, %9\n ds_read_b128 %2, %10\n ds_read_b128 %3, %11\n"
        "ds_read_b128 %4, %12\n ds_read_b128 %5, %13\n ds_read_b128 %6, %14\n ds_read_b128 %7, %15\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]),
          "=&v"(f[7])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
        : "memory");
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b128 %0, %4\n ds_read_b128 %1, %5\n ds_read_b128 %2, %6\n ds_read_b128 %3, %7\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
        : "memory");
  else
    asm volatile("ds_read_b128 %0, %2\n ds_read_b128 %1, %3\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0]), "v"(a[1])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void read_columns(bf16x4 (&f)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 8)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n ds_read_b64_tr_b16 %1, %9\n ds_read_b64_tr_b16 %2, %10\n"
        "ds_read_b64_tr_b16 %3, %11\n ds_read_b64_tr_b16 %4, %12\n ds_read_b64_tr_b16 %5, %13\n"
        "ds_read_b64_tr_b16 %6, %14\n ds_read_b64_tr_b16 %7, %15\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]),
          "=&v"(f[7])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
        : "memory");
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n ds_read_b64_tr_b16 %1, %5\n ds_read_b64_tr_b16 %2, %6\n"
        "ds_read_b64_tr_b16 %3, %7\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
        : "memory");
  else
    asm volatile("ds_read_b64_tr_b16 %0, %2\n ds_read_b64_tr_b16 %1, %3\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0]), "v"(a[1])
                 : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "");
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int DP>
__global__ __launch_bounds__(kThreads)
    __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1))) void paged_stream_kernel(StreamParams P) {
  using S_ = Shape<DP>;
  constexpr int CPR = S_::CPR, RPI = S_::RPI, NI = S_::NI, NV = S_::NV, KD = S_::KD, MD = S_::MD;
  // A wave's K tile, then its V tile; at the end its accumulators (32 pairs of DP floats).
  __shared__ __attribute__((aligned(1024))) uint16_t s_tiles[kWaves][2][S_::TILE];
  __shared__ float s_ml[kWaves][2][32];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // This workgroup's heads, row, block of pairs and range.
  if (int(blockIdx.x) >= P.blocks) return append_tokens(P.append, int(blockIdx.x) - P.blocks);
  Row R;
  const Range mine = find_range<kPairs>(P, lane, R);
  if (mine.b < 0) return;
  const int b = mine.b, block = mine.block, range = mine.range, ranges = mine.ranges;
  const int head_waves = mine.head_waves, group = mine.group;

  const int kvh = group * head_waves + wave % head_waves;
  const int kw = wave / head_waves, n_kw = kWaves / head_waves;  // this wave's share of the tiles
  const int D = P.D;
  const int h = lane >> 5, col = lane & 31;
  const int pairs = R.T * P.G;
  const int pair = block * 32 + col;
  const bool live = pair < pairs;
  const int t_q = live ? pair / P.G : 0;
  const int64_t at = (int64_t(R.tok0 + t_q) * P.H + kvh * P.G + (live ? pair - t_q * P.G : 0)) * D;
  uint16_t *out = static_cast<uint16_t *>(P.out) + at;
  if (!R.ok) {
    if (live && kw == 0)
      for (int d = 8 * h; d < D; d += 16)
        *reinterpret_cast<uint4 *>(out + d) =
            make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    return;
  }

  // The block's last key; a range's tiles past it have nothing for its pairs.
  const int t_first = block * 32 / P.G, t_last = min(block * 32 + 31, pairs - 1) / P.G;
  const int p_abs = R.s0 + t_q;
  const int first_tile = R.lo / KT;
  const int t0 = first_tile + mine.t0, t1 = first_tile + mine.t1;

  const uint16_t *q = static_cast<const uint16_t *>(P.q) + at;
  bf16x8 qf[KD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (16 * kd + 8 * h < D) u = *reinterpret_cast<const uint4 *>(q + 16 * kd + 8 * h);
    qf[kd] = __builtin_bit_cast(bf16x8, u);
  }

  // Loads to LDS. Load i of a tile covers rows RPI i + lane / CPR; its lane's chunk goes to slot
  // lane % CPR, wherever that is.
  const int tok_bytes = P.H_kv * D * 2;
  constexpr uint32_t kNowhere = 0x80000000u;
  const int lr = lane / CPR, lc = lane % CPR;
  uint32_t k_off[NV], v_off[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = RPI * i + lr;
    const int kc = lc ^ S_::k_swz(r), vc = lc ^ S_::v_swz(r);
    k_off[i] = 8 * kc < D ? uint32_t(r * tok_bytes + 16 * kc) : kNowhere;
    v_off[i] = 8 * vc < D ? uint32_t(r * tok_bytes + 16 * vc) : kNowhere;
  }
  const scalar_ints table = (scalar_ints)(P.kv.table + b * P.kv.table_stride);
  const int64_t head_at = int64_t(kvh) * D * 2;
  const uint32_t page_bytes = uint32_t(tok_bytes) << P.kv.shift;
  bool lost = false;
  uint16_t *const sK = s_tiles[wave][0], *const sV = s_tiles[wave][1];

  const int seen_from = R.lo, seen_to = R.s0 + t_last;  // keys any pair of the block sees
  const bool fresh = P.k_new != nullptr;
  // Pages of the two halves of a tile; one that no key needs is page 0.
  auto pages_of = [&](int tile, int (&id2)[2]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int k = tile * KT + 16 * half;
      id2[half] = k + 15 >= seen_from && k <= seen_to ? table[k >> P.kv.shift] : 0;
    }
  };
  auto load_tile = [&](const void *pool, const void *new_rows, const uint32_t (&off)[NV], int tile,
                       const int (&id2)[2], uint16_t *to, bool is_v) {
    const int k0 = tile * KT;
    if (fresh && k0 + KT > R.s0) {
      // Keys of the chunk itself come from its own rows; past the last one it is read again.
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = RPI * i + lr, key = max(seen_from, min(k0 + r, seen_to));
        const int c = min(lc ^ (is_v ? S_::v_swz(r) : S_::k_swz(r)), D / 8 - 1);
        const char *from;
        if (key >= R.s0) {
          from = static_cast<const char *>(new_rows) + int64_t(R.tok0 + key - R.s0) * tok_bytes;
        } else {
          const int pid = id2[i / NV];
          from = static_cast<const char *>(pool) +
                 2 * P.kv.offset(pid, P.kv.in_page(key), int64_t(P.H_kv) * D);
        }
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)(from + head_at + 16 * c),
            (__attribute__((address_space(3))) void *)(to + i * 512), 16, 0, 0);
      }
      return;
    }
    const bool edge = k0 < seen_from || k0 + KT - 1 > seen_to;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int k = k0 + 16 * half;
      const char *base = static_cast<const char *>(pool) +
                         (P.kv.is_page(id2[half]) ? id2[half] : 0) * P.kv.page_stride * 2 + head_at;
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          (void *)base, 0, int(page_bytes - uint32_t(head_at)), 0x00020000);
      const int in_page = P.kv.in_page(k) * tok_bytes;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        uint32_t o = off[i];
        if (edge) {
          const int key = k + RPI * i + lr;
          o = key >= seen_from && key <= seen_to ? o : kNowhere;
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (__attribute__((address_space(3))) void *)(to + (half * NV + i) * 512), 16, int(o),
            in_page, 0, kNonTemporal);
      }
    }
  };
  auto load_k = [&](int tile, const int (&id2)[2]) {
    load_tile(P.k_pages, P.k_new, k_off, tile, id2, sK, false);
  };
  auto load_v = [&](int tile, const int (&id2)[2]) {
    load_tile(P.v_pages, P.v_new, v_off, tile, id2, sV, true);
  };

  // LDS addresses of this lane's reads.
  uint32_t ka[KD], va[2 * MD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd)
    ka[kd] = lds_addr(sK) + 2 * (col * DP + 8 * ((2 * kd + h) ^ S_::k_swz(col)));
  const int tr_row = (lane & 15) >> 2, tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
  for (int md = 0; md < MD; ++md)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 4 * h + tr_row + 8 * u, c = 32 * md + tr_col;
      va[2 * md + u] = lds_addr(sV) + 2 * (r * DP + 8 * ((c >> 3) ^ S_::v_swz(r)) + (c & 7));
    }

  f32x16 o[MD];
#pragma unroll
  for (int md = 0; md < MD; ++md)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[md][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  if (D < DP) {  // dims past the head's are zero, whether or not a load past a page's end writes
    for (int i = lane; i < 2 * S_::TILE / 8; i += 64)
      reinterpret_cast<uint4 *>(sK)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  int tile = t0 + kw;
  int now[2], next[2];
  if (tile < t1) {
    pages_of(tile, now);
    // The queries have arrived: a wait for them behind the loads to LDS would be one for those too.
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) asm volatile("" : "+v"(qf[kd]));
    load_k(tile, now);
    load_v(tile, now);
  }
  for (; tile < t1; tile += n_kw) {
    const int k0 = tile * KT;
    const bool more = tile + n_kw < t1;
    if (more) pages_of(tile + n_kw, next);
    lost = lost || !P.kv.is_page(now[0]) || !P.kv.is_page(now[1]);

    wait_loads<NI>();  // K has landed; V may be under way
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
    constexpr int KB = KD < 8 ? KD : 8;
#pragma unroll
    for (int k8 = 0; k8 < KD; k8 += KB) {
      bf16x8 f[KB];
      uint32_t a[KB];
#pragma unroll
      for (int i = 0; i < KB; ++i) a[i] = ka[k8 + i];
      read_rows<KB>(f, a);
#pragma unroll
      for (int i = 0; i < KB; ++i)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i], qf[k8 + i], s, 0, 0, 0);
    }
    if (more) load_k(tile + n_kw, next);

    // Keys the pair may not see.
    if (k0 + KT - 1 > R.s0 + t_first || k0 < seen_from ||
        (P.window >= 0 && k0 < R.s0 + t_last - P.window)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int gap = p_abs - (k0 + 8 * (e >> 2) + 4 * h + (e & 3));
        if (!(gap >= 0 && (P.window < 0 || gap <= P.window))) s[e] = -INFINITY;
      }
    }
    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 16; ++e) m4[e & 3] = fmaxf(m4[e & 3], s[e]);
    const float mx = max_halves(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))) * P.scale_log2;
    if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
      const float m_new = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
      l *= alpha;
#pragma unroll
      for (int md = 0; md < MD; ++md)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[md][e] *= alpha;
      m = m_new;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float w[16], ts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      w[e] = fast_exp2(fmaf(s[e], P.scale_log2, -ref));
      ts[e & 3] += w[e];
    }
    l += (ts[0] + ts[1]) + (ts[2] + ts[3]);

    if (more)
      wait_loads<NI>();  // V has landed; the next K may be under way
    else
      wait_loads<0>();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f32x8 pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = w[8 * ks + e];
      const bf16x8 hi8 = __builtin_convertvector(pv, bf16x8);
      const bf16x8 lo8 = __builtin_convertvector(pv - __builtin_convertvector(hi8, f32x8), bf16x8);
      constexpr int VB = 2 * MD < 8 ? 2 * MD : 8;
#pragma unroll
      for (int v8 = 0; v8 < 2 * MD; v8 += VB) {
        bf16x4 f[VB];
        uint32_t a[VB];
#pragma unroll
        for (int i = 0; i < VB; ++i) a[i] = va[v8 + i] + ks * 32 * DP;
        read_columns<VB>(f, a);
#pragma unroll
        for (int i = 0; i < VB / 2; ++i) {
          const int md = v8 / 2 + i;
          const bf16x8 x = __builtin_shufflevector(f[2 * i], f[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
          o[md] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, hi8, o[md], 0, 0, 0);
          o[md] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, lo8, o[md], 0, 0, 0);
        }
      }
    }
    if (more) load_v(tile + n_kw, next);
    now[0] = next[0], now[1] = next[1];
  }
  l = sum_halves(l);
  if (lost) l = NAN;

  // The new tokens into their pages: in the row's last range, by the wave that has the fewest tiles. In every
  // block, so that a redo below finds them whichever other block has come how far; they write the same.
  if (fresh && range == ranges - 1 && kw == n_kw - 1) {
    const int units = D / 8;  // of 16 bytes, of K and of V
    for (int i = lane; i < R.T * units; i += 64) {
      const int t = i / units, u = i - t * units, key = R.s0 + t;
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

  // The waves of a head leave their sums in their tiles' place; each adds up the dims 32 md .. of every
  // n_kw-th md, which are its own from here on.
  if (n_kw > 1) {
    static_assert(2 * S_::TILE * 2 == 32 * DP * 4, "a wave's sums fit its tiles");
    float *so = reinterpret_cast<float *>(s_tiles[wave][0]);
#pragma unroll
    for (int md = 0; md < MD; ++md)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4 *>(so + ((md * 4 + j) * 64 + lane) * 4) =
            make_float4(o[md][4 * j], o[md][4 * j + 1], o[md][4 * j + 2], o[md][4 * j + 3]);
    if (h == 0) s_ml[wave][0][col] = m, s_ml[wave][1][col] = l;
    __syncthreads();
    const int w0 = wave % head_waves;
    float M = -INFINITY;
    for (int w = w0; w < kWaves; w += head_waves) M = fmaxf(M, s_ml[w][0][col]);
    float L = 0.f;
#pragma unroll
    for (int md = 0; md < MD; ++md)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[md][e] = 0.f;
    for (int w = w0; w < kWaves; w += head_waves) {
      const float mw = s_ml[w][0][col];
      const float a = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
      L += s_ml[w][1][col] * (mw == -INFINITY ? 1.f : a);  // without a key l = 0; a NaN l must stay
      const float *s2 = reinterpret_cast<const float *>(s_tiles[w][0]);
#pragma unroll
      for (int md = 0; md < MD; ++md) {
        if (md % n_kw != kw) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 x = *reinterpret_cast<const float4 *>(s2 + ((md * 4 + j) * 64 + lane) * 4);
          o[md][4 * j] = fmaf(x.x, a, o[md][4 * j]);
          o[md][4 * j + 1] = fmaf(x.y, a, o[md][4 * j + 1]);
          o[md][4 * j + 2] = fmaf(x.z, a, o[md][4 * j + 2]);
          o[md][4 * j + 3] = fmaf(x.w, a, o[md][4 * j + 3]);
        }
      }
    }
    m = M;
    l = L;
  }

  // o[md][4j + i] is dim 32 md + 8 j + 4 h + i of pair `col`.
  if (ranges > 1) {
    if (!live) return;
    const int64_t slot =
        (int64_t(blockIdx.x) * head_waves + wave % head_waves) * P.pair_slots + col;
    float *po = P.part_o + slot * DP;
#pragma unroll
    for (int md = 0; md < MD; ++md) {
      if (md % n_kw != kw) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * md + 8 * j < D)
          *reinterpret_cast<float4 *>(po + 32 * md + 8 * j + 4 * h) =
              make_float4(o[md][4 * j], o[md][4 * j + 1], o[md][4 * j + 2], o[md][4 * j + 3]);
    }
    if (h == 0 && kw == 0) *reinterpret_cast<float2 *>(P.part_ml + slot * 2) = make_float2(m, l);
    return;
  }
  const float inv = 1.f / l;
  uint32_t bad_of = 0;  // lane md: the pairs whose dims 32 md .. are not finite
#pragma unroll
  for (int md = 0; md < MD; ++md) {
    if (md % n_kw != kw || 32 * md >= D) continue;
    bool ok = true;
    bf16x4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = o[md][4 * j + i] * inv;
        ok = ok && (finite(x[i]) || 32 * md + 8 * j >= D);
      }
      y[j] = __builtin_convertvector(x, bf16x4);
    }
    const uint64_t bad64 = __builtin_amdgcn_ballot_w64(live && !ok);
    const uint32_t bad = uint32_t(bad64) | uint32_t(bad64 >> 32);
    if (live && !((bad >> col) & 1u)) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * md + 8 * j < D)
          *reinterpret_cast<uint2 *>(out + 32 * md + 8 * j + 4 * h) = __builtin_bit_cast(uint2, y[j]);
    }
    bad_of = lane == md ? bad : bad_of;
  }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad_of != 0) == 0, 1)) return;
  for (int md = 0; md < MD; ++md)
    for (uint32_t left = __builtin_amdgcn_readlane(bad_of, md); left != 0; left &= left - 1) {
      const int pr = block * 32 + __builtin_ctz(left), t = pr / P.G;
      careful_pair<bf16, DP, 8>(P, b, kvh,
                                (int64_t(R.tok0 + t) * P.H + kvh * P.G + (pr - t * P.G)) * D, R.s0 + t,
                                lane, 32 * md, min(32 * md + 32, D));
    }
}

}  // namespace

size_t paged_stream_bytes(const PagedArgs &a, int64_t most) {
  return stream_bytes(a, stream_plan(a, most, kPairs, kFill));
}

int launch_paged_stream(const PagedArgs &a, int64_t most, bool others) {
  StreamPlan p = stream_plan(a, most, kPairs, kFill);
  if (p.cut && (!a.scratch || a.scratch_bytes < stream_bytes(a, p))) p.cut = false;
  const StreamParams P = stream_params(a, p, most);
  switch (head_pad(a.head_dim)) {
    case 32: return launch_stream<bf16, 32, kPairs>(paged_stream_kernel<32>, P, a, p, others);
    case 64: return launch_stream<bf16, 64, kPairs>(paged_stream_kernel<64>, P, a, p, others);
    case 128: return launch_stream<bf16, 128, kPairs>(paged_stream_kernel<128>, P, a, p, others);
    default: return launch_stream<bf16, 256, kPairs>(paged_stream_kernel<256>, P, a, p, others);
  }
}

}  // namespace mcamd
