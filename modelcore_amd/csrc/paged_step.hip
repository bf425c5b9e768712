// The step before the attention over a paged cache, fused: RoPE, QK RMS-norm and scale of q and k,
// and k and v into their slots -- the form of qk_epilogue.hip whose tokens have a position and a
// slot (page * page_size + token of the page) each, packed one after another.
//
// Per token at position p, for every query head of q and KV head of k, j < D/2:
//   y[j] = x[j] c + x[j + D/2] s,  y[j + D/2] = x[j + D/2] c - x[j] s   (c, s = cos, sin[p, j])
//   out  = y * scale / sqrt(mean(y^2) + eps)
// in fp32 throughout, rounded once to the storage type (the step into contiguous caches rounds after
// every operation, as the separate ops it restates do; results differ by those roundings).
//
// LPI lanes per head: lane L holds dims VEC L .. of the first half and their partners in the second,
// so a rotation needs no exchange and the sum of squares log2(LPI) steps. VEC is 16 bytes where rows
// and tables are made of such pieces, else one element with 64 lanes a head. 4096 tokens of 32 / 8 heads
// of 128 in bf16, 102 MB: 20.9 us, 4.86 TB/s, what a copy reaches; 64 tokens 4.1, one round trip for the
// position, one for its table rows.
//
// A token whose position is outside the tables gets NaN in q and writes nothing; one whose slot is
// outside the pool writes nothing.
#include "paged.h"

#include <cmath>
#include <type_traits>

namespace mcamd {
namespace {

constexpr int kThreads = 256;

template <class T, int VEC>
__device__ __forceinline__ void load_piece(const T *p, float (&x)[VEC]) {
  if constexpr (VEC == Vec<T>::N)
    Vec<T>::load(p, x);
  else
    x[0] = to_f32<T>(*p);
}
template <class T, int VEC>
__device__ __forceinline__ void store_piece(T *p, const float (&x)[VEC]) {
  if constexpr (VEC == Vec<T>::N)
    Vec<T>::store(p, x);
  else
    *p = from_f32<T>(x[0]);
}

struct StepParams {
  const void *q, *k, *v, *cos, *sin;
  void *k_pages, *v_pages, *q_out;
  const int32_t *positions;
  const int64_t *slots;
  int64_t q_tok, k_tok, v_tok, page_stride, n_pos, n_slots, n_items_all;
  int H, H_kv, D, n_items, shift;
  float eps, scale;
};

// R pieces a lane and half (two where 64 lanes of one element do not cover half a head of 256).
template <class T, int VEC, int LPI, int R>
__global__ __launch_bounds__(kThreads) void paged_step_kernel(StepParams P) {
  const int64_t at = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / LPI;
  const int L = threadIdx.x % LPI;
  const bool here = at < P.n_items_all;
  const int64_t tok = here ? at / P.n_items : 0;
  const int item = here ? int(at - tok * P.n_items) : 0;
  const int half = P.D >> 1;
  const bool is_q = item < P.H, is_v = item >= P.H + P.H_kv;
  const int64_t pos = P.positions[tok];
  const int64_t slot = is_q ? 0 : P.slots[tok];
  const bool in_table = pos >= 0 && pos < P.n_pos;
  const bool writes = is_q || (in_table && slot >= 0 && slot < P.n_slots);

  const T *src;
  T *dst;
  if (is_q) {
    src = static_cast<const T *>(P.q) + tok * P.q_tok + int64_t(item) * P.D;
    dst = static_cast<T *>(P.q_out) + (tok * P.H + item) * P.D;
  } else {
    const int hk = item - P.H - (is_v ? P.H_kv : 0);
    src = (is_v ? static_cast<const T *>(P.v) + tok * P.v_tok
                : static_cast<const T *>(P.k) + tok * P.k_tok) + int64_t(hk) * P.D;
    const int64_t in_page = slot & ((int64_t(1) << P.shift) - 1);
    dst = static_cast<T *>(is_v ? P.v_pages : P.k_pages) + (slot >> P.shift) * P.page_stride +
          (in_page * P.H_kv + hk) * P.D;
  }
  if (is_v) {  // a plain copy
    if (!here || !writes) return;
    typedef typename std::conditional<VEC == 1, T, uint4>::type U;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = VEC * (L + LPI * r);
      if (j >= half) continue;
      const U a = *reinterpret_cast<const U *>(src + j);
      const U b = *reinterpret_cast<const U *>(src + half + j);
      *reinterpret_cast<U *>(dst + j) = a;
      *reinterpret_cast<U *>(dst + half + j) = b;
    }
    return;
  }
  float y1[R][VEC], y2[R][VEC];
  float ss = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = VEC * (L + LPI * r);
#pragma unroll
    for (int e = 0; e < VEC; ++e) y1[r][e] = y2[r][e] = 0.f;
    if (!here || j >= half || !in_table) continue;
    float x1[VEC], x2[VEC], c[VEC], s[VEC];
    load_piece<T, VEC>(src + j, x1);
    load_piece<T, VEC>(src + half + j, x2);
    load_piece<T, VEC>(static_cast<const T *>(P.cos) + pos * half + j, c);
    load_piece<T, VEC>(static_cast<const T *>(P.sin) + pos * half + j, s);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      y1[r][e] = fmaf(x1[e], c[e], x2[e] * s[e]);
      y2[r][e] = fmaf(x2[e], c[e], -x1[e] * s[e]);
      ss = fmaf(y1[r][e], y1[r][e], fmaf(y2[r][e], y2[r][e], ss));
    }
  }
  ss = wave_sum<LPI>(ss);
  if (!here || !writes) return;
  const float by = in_table ? P.scale / sqrtf(ss / float(P.D) + P.eps) : NAN;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = VEC * (L + LPI * r);
    if (j >= half) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) y1[r][e] *= by, y2[r][e] *= by;
    store_piece<T, VEC>(dst + j, y1[r]);
    store_piece<T, VEC>(dst + half + j, y2[r]);
  }
}

template <class T>
int run(const StepParams &P, hipStream_t stream) {
  constexpr int N = Vec<T>::N;
  const int half = P.D / 2;
  auto pieces = [&](const void *p, int64_t stride) {
    return aligned(p, 16) && stride * int64_t(sizeof(T)) % 16 == 0;
  };
  const bool whole = half % N == 0 && pieces(P.q, P.q_tok) && pieces(P.q_out, P.D) &&
                     pieces(P.cos, half) && pieces(P.sin, half) &&
                     (!P.k || (pieces(P.k, P.k_tok) && pieces(P.v, P.v_tok) &&
                               pieces(P.k_pages, P.page_stride) && pieces(P.v_pages, P.page_stride)));
  int lpi = 64;
  if (whole)
    for (lpi = 1; lpi * N < half;) lpi *= 2;
  if (P.n_items_all > 0x7fffffff / lpi) return fail(MCAMD_EUNSUPPORTED, "rope_norm_append_paged: grid too large");
  const int64_t blocks = (P.n_items_all * lpi + kThreads - 1) / kThreads;
  const dim3 grid{unsigned(blocks)}, threads{kThreads};
#define MCAMD_STEP(VEC, LPI, R) \
  hipLaunchKernelGGL((paged_step_kernel<T, VEC, LPI, R>), grid, threads, 0, stream, P)
  if (!whole) {
    if (half <= 64)
      MCAMD_STEP(1, 64, 1);
    else
      MCAMD_STEP(1, 64, 2);
    return launch_status("rope_norm_append_paged");
  }
  switch (lpi) {
    case 1: MCAMD_STEP(N, 1, 1); break;
    case 2: MCAMD_STEP(N, 2, 1); break;
    case 4: MCAMD_STEP(N, 4, 1); break;
    case 8: MCAMD_STEP(N, 8, 1); break;
    case 16: MCAMD_STEP(N, 16, 1); break;
    default:  // 32: fp32 past head_dim 128
      if constexpr (N == 4) MCAMD_STEP(N, 32, 1);
  }
#undef MCAMD_STEP
  return launch_status("rope_norm_append_paged");
}

}  // namespace
}  // namespace mcamd

using namespace mcamd;

extern "C" int mcamd_qk_rope_norm_append_paged(
    const void *q, int64_t q_token_stride, const void *k, int64_t k_token_stride, const void *v,
    int64_t v_token_stride, const void *cos, const void *sin, int64_t n_pos,
    const int32_t *positions, const int64_t *slots, void *k_pages, void *v_pages, void *q_out,
    int64_t total, int64_t n_head, int64_t n_kv_head, int64_t head_dim, int64_t n_pages,
    int64_t page_size, int64_t page_stride, float eps, float scale, int dtype, void *stream) {
  if (dtype != MCAMD_F32 && dtype != MCAMD_BF16)
    return fail(MCAMD_EINVAL, "rope_norm_append_paged: dtype must be MCAMD_F32 or MCAMD_BF16");
  if (total < 0 || n_head <= 0 || n_kv_head <= 0 || n_pos <= 0)
    return fail(MCAMD_EINVAL, "rope_norm_append_paged: sizes must be positive (total may be 0)");
  if (total > 0x7fffffff || n_head > 0x7fffffff / 2 || n_kv_head > 0x7fffffff / 4)
    return fail(MCAMD_EUNSUPPORTED, "rope_norm_append_paged: sizes too large");
  if (head_dim <= 0 || head_dim % 2 != 0 || head_dim > 256)
    return fail(MCAMD_EUNSUPPORTED, "rope_norm_append_paged: head_dim must be even and <= 256");
  if ((k == nullptr) != (v == nullptr))
    return fail(MCAMD_EINVAL, "rope_norm_append_paged: pass both k and v, or neither");
  if (!(eps >= 0.f) || !std::isfinite(scale))
    return fail(MCAMD_EINVAL, "rope_norm_append_paged: eps must be >= 0 and scale finite");
  const bool with_kv = k != nullptr;
  StepParams P{};
  if (with_kv) {
    if (!page_shift(page_size, P.shift))
      return fail(MCAMD_EINVAL,
                  "rope_norm_append_paged: page_size must be a power of two from 16 to 2^30");
    if (n_pages <= 0 || page_stride / page_size < n_kv_head * head_dim)
      return fail(MCAMD_EINVAL, "rope_norm_append_paged: empty pool, or page_stride smaller than "
                                "page_size*H_kv*D");
    if (n_pages > (int64_t(1) << 62) / page_size)
      return fail(MCAMD_EUNSUPPORTED, "rope_norm_append_paged: sizes too large");
  }
  if (q_token_stride < n_head * head_dim ||
      (with_kv && (k_token_stride < n_kv_head * head_dim || v_token_stride < n_kv_head * head_dim)))
    return fail(MCAMD_EINVAL, "rope_norm_append_paged: a token stride is smaller than heads * head_dim");
  if (total == 0) {
    clear_error();
    return MCAMD_OK;
  }
  if (!q || !cos || !sin || !positions || !q_out || (with_kv && (!slots || !k_pages || !v_pages)))
    return fail(MCAMD_EINVAL, "rope_norm_append_paged: null pointer");
  P.q = q;
  P.k = k;
  P.v = v;
  P.cos = cos;
  P.sin = sin;
  P.k_pages = k_pages;
  P.v_pages = v_pages;
  P.q_out = q_out;
  P.positions = positions;
  P.slots = slots;
  P.q_tok = q_token_stride;
  P.k_tok = k_token_stride;
  P.v_tok = v_token_stride;
  P.page_stride = page_stride;
  P.n_pos = n_pos;
  P.n_slots = with_kv ? n_pages * page_size : 0;
  P.H = int(n_head);
  P.H_kv = int(n_kv_head);
  P.D = int(head_dim);
  P.n_items = int(n_head + (with_kv ? 2 * n_kv_head : 0));
  P.n_items_all = total * P.n_items;
  P.eps = eps;
  P.scale = scale;
  return dtype == MCAMD_BF16 ? run<bf16>(P, as_stream(stream)) : run<float>(P, as_stream(stream));
}
