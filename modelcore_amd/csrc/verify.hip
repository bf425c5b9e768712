// How far drafted trees go: the walk from each row's root to the first node none of whose children is
// accepted, and the token drawn there, from the target's logits and one given random number a node.
//
// At node c, with p = softmax(logits[c] / t), its children are tried in the order of their indices.
//  * Drawn from q = draft_probs[c], independently: child x is accepted where u Z q(x) < (p(x) - a q(x))+, from
//    a = 0 and Z = 1 on; a refused one leaves a + Z in a's place and the sum of (p - a q)+ in Z's. (After k
//    refusals what is left of p is the k-fold remainder norm((p - q)+), and a multiple of q taken off p is
//    what that comes to.) The row's last token is drawn from (p - a q)+.
//  * Guesses (no q): accepted where u Z < p(x), Z being 1 less the p of the children refused before; the last
//    token is drawn from p without them.
//  * t = 0: accepted where x is the first of the largest logits, which is the last token too.
// Either way the accepted tokens and the last one are a draw from the target's own distribution.
//
// The draw is the smallest token whose running sum of weights passes u_0 times the whole (u_0 the root's number,
// which no test uses). It falls between neighbours of a whole vocabulary, where 32-bit sums would move
// it: weights and sums are in 64 bits, whose multiply-adds run as fast here as those of 32. A weight is
// exp2 by its series to the tenth power, within 2^-40.
//
// Two launches. The first reads every logit once, a workgroup kChunk of a node's, and leaves the largest, its
// place and the sum of the chunk's weights against it: bound by HBM. The second has a workgroup a row: a node's
// chunks are put together by a wave, the probabilities of all drafts fetched at once, and the walk then goes
// through LDS, every wave by itself; the sum (p - a q)+ over the vocabulary is taken where a further child has
// to be tried against it. The draw finds its chunk by the chunks' sums (of what is left of p and q, by a pass
// over the row) and reads that one again.
#include "kernels.h"

#include <cmath>

namespace mcamd {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxNodes = 1024;
constexpr int kChunkThreads = 256;
constexpr int kRestChunks = 64;  // whose sums of (p - a q)+ are kept
constexpr int kChunk = 16 * kChunkThreads;  // logits
static_assert(kChunk == 4 * kThreads, "the draw's threads have four each");

struct Part {  // of a chunk
  double sum;
  float top;
  int at;
};

struct VerifyParams {
  const float *logits, *probs;
  int64_t logits_stride, probs_stride;
  const int64_t *tokens;
  const int32_t *parents, *cu;
  const float *numbers;
  int32_t *kept, *counts;
  int64_t *out;
  Part *parts;  // [total][chunks]
  int total, most, vocab, chunks;
  double scale;  // log2(e) / temperature
  int greedy;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // at any float's address

// 2^y for y <= 0, to 2^-40: 2^n by the exponent, 2^f, |f| <= 1/2, by the series of e^(f ln 2).
__device__ __forceinline__ double exp2_64(double y) {
  const double n = __builtin_rint(y), r = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 3628800;
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return y > -1000.0 ? ldexp(p, int(n)) : 0.0;
}

// Logits as weights against the largest of them, which an infinite one makes 1 and all others 0. NaN has none.
struct Weigher {
  float top;
  double scale;
  __device__ __forceinline__ double operator()(float x) const {
    const double w = exp2_64((double(x) - double(top)) * scale);
    return x == top ? 1.0 : x > -INFINITY && top < INFINITY ? w : 0.0;
  }
};

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}
__device__ __forceinline__ double wave_upto64(double x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, 64));
  return x;
}

__global__ __launch_bounds__(kChunkThreads) void verify_parts_kernel(VerifyParams P) {
  constexpr int W = kChunkThreads / 64;
  __shared__ float s_top[W];
  __shared__ int s_at[W];
  __shared__ double s_sum[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int node = blockIdx.x / P.chunks, chunk = blockIdx.x - node * P.chunks;
  const float *row = P.logits + int64_t(node) * P.logits_stride;
  const int i0 = chunk * kChunk + 4 * tid;
  f32x4u x[4];
  if (chunk * kChunk + kChunk <= P.vocab) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const f32x4u *>(row + i0 + 4 * kChunkThreads * j);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + 4 * kChunkThreads * j + e;
        const float y = row[min(i, P.vocab - 1)];
        x[j][e] = i < P.vocab ? y : -INFINITY;
      }
  }
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = fmaxf(top, x[j][e]);
  top = wave_max<64>(top);
  if (lane == 0) s_top[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, s_top[w]);
  Part *const part = P.parts + int64_t(blockIdx.x);
  if (P.greedy) {
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x[j][e] == top) at = min(at, i0 + 4 * kChunkThreads * j + e);
    at = wave_min(at);
    if (lane == 0) s_at[wave] = at;
    __syncthreads();
    if (tid > 0) return;
    for (int w = 0; w < W; ++w) at = min(at, s_at[w]);
    part->top = top;
    part->at = at;
    return;
  }
  const Weigher weigh{top, P.scale};
  double sum = 0;
  if (top > -INFINITY) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += weigh(x[j][e]);
  }
  sum = wave_sum64(sum);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (tid > 0) return;
  for (int w = 1; w < W; ++w) sum += s_sum[w];
  part->sum = sum;
  part->top = top;
}

__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyParams P) {
  __shared__ double s_all[kMaxNodes], s_w[kMaxNodes];
  __shared__ float s_top[kMaxNodes], s_q[kMaxNodes], s_u[kMaxNodes];
  __shared__ int s_up[kMaxNodes], s_token[kMaxNodes], s_best[kMaxNodes];
  __shared__ double s_sum[kWaves];
  __shared__ double s_rest[kRestChunks][kWaves];
  __shared__ int s_gone[kMaxNodes], s_chunk;
  __shared__ double s_want;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int begin = max(P.cu[b], 0), n = min(max(min(P.cu[b + 1], P.total) - begin, 0), P.most);
  int32_t *const kept = P.kept + int64_t(b) * P.most;
  int64_t *const out = P.out + int64_t(b) * P.most;
  for (int j = tid; j < P.most; j += kThreads) kept[j] = -1, out[j] = -1;
  if (n == 0) {
    if (tid == 0) P.counts[b] = 0;
    return;
  }
  const int V = P.vocab, C = P.chunks;
  // Every node's draft and number, and its chunks put together.
  int up = 0, token = -1;
  if (tid < n) {
    const int64_t t = P.tokens[begin + tid];
    token = t >= 0 && t < V ? int(t) : -1;
    up = tid == 0 ? -1 : P.parents[begin + tid];
    s_up[tid] = up;
    s_token[tid] = token;
    s_u[tid] = P.numbers[begin + tid];
  }
  for (int i = wave; i < n; i += kWaves) {
    const Part *part = P.parts + int64_t(begin + i) * C;
    float top = -INFINITY;
    for (int c = lane; c < C; c += 64) top = fmaxf(top, part[c].top);
    top = wave_max<64>(top);
    if (P.greedy) {
      int best = 0x7fffffff;
      for (int c = lane; c < C; c += 64)
        if (part[c].top == top) best = min(best, part[c].at);
      best = wave_min(best);
      if (lane == 0) s_best[i] = best;
    } else {
      const Weigher weigh{top, P.scale};
      double all = 0;
      for (int c = lane; c < C; c += 64) all += part[c].sum * weigh(part[c].top);
      all = wave_sum64(all);
      if (lane == 0) s_all[i] = all;
    }
    if (lane == 0) s_top[i] = top;
  }
  __syncthreads();
  if (!P.greedy && tid > 0 && tid < n) {
    s_w[tid] = 0;
    if (up >= 0 && up < tid && token >= 0) {
      const float x = P.logits[int64_t(begin + up) * P.logits_stride + token];
      if (P.probs) s_q[tid] = P.probs[int64_t(begin + up) * P.probs_stride + token];
      s_w[tid] = Weigher{s_top[up], P.scale}(x);
    }
  }
  __syncthreads();

  int node = 0, count = 1;
  double less = 0, left = 0;  // a and Z, of guesses Z in units of the weights
  bool summed = true;         // left is the sum for this a
  const float *row = nullptr, *q_row = nullptr;
  Weigher weigh{0.f, P.scale};
  double one = 0;  // over the node's weights
  auto enter = [&]() {
    row = P.logits + int64_t(begin + node) * P.logits_stride;
    q_row = P.probs ? P.probs + int64_t(begin + node) * P.probs_stride : nullptr;
    weigh.top = s_top[node];
    less = 0;
    summed = true;
    if (P.greedy) return;
    one = 1.0 / s_all[node];
    left = q_row ? 1.0 : s_all[node];
  };
  // Four logits from token i on, or draft probabilities; past the vocabulary what has no weight.
  auto four = [&](const float *from, int i, float none) {
    f32x4u x;
    if (i + 4 <= V) {
      x = *reinterpret_cast<const f32x4u *>(from + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = i + e < V ? from[i + e] : none;
    }
    return x;
  };
  // What is left of the probabilities of four tokens.
  auto rest_of = [&](const f32x4u &x, const f32x4u &q, double (&w)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = fmax(weigh(x[e]) * one - less * double(q[e]), 0.0);
    return (w[0] + w[1]) + (w[2] + w[3]);
  };
  // The sum of it over the vocabulary, by its chunks' sums, of which the first ones are kept.
  auto rest_sum = [&]() {
    constexpr int U = 4;  // chunks whose loads are under way at once
    double sum = 0;
    __syncthreads();  // s_rest and s_sum have been read
    for (int c0 = 0; c0 < C; c0 += U) {
      f32x4u x[U], q[U];
#pragma unroll
      for (int c = 0; c < U; ++c) {
        x[c] = four(row, (c0 + c) * kChunk + 4 * tid, -INFINITY);
        q[c] = four(q_row, (c0 + c) * kChunk + 4 * tid, 0.f);
      }
#pragma unroll
      for (int c = 0; c < U; ++c) {
        double w[4];
        const double part = wave_sum64(rest_of(x[c], q[c], w));
        sum += part;
        if (lane == 0 && c0 + c < kRestChunks) s_rest[c0 + c][wave] = part;
      }
    }
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kWaves; ++w) sum += s_sum[w];
    return sum;
  };

  // The walk, by every wave alike.
  enter();
  for (;;) {
    int found = -1;
    for (int base = (node + 1) & ~63; base < n && found < 0 && weigh.top > -INFINITY; base += 64) {
      const int mine = base + lane;
      const bool kid = mine > node && mine < n && s_up[min(mine, n - 1)] == node && s_token[min(mine, n - 1)] >= 0;
      for (uint64_t left_of = __builtin_amdgcn_ballot_w64(kid); left_of != 0 && found < 0; left_of &= left_of - 1) {
        const int i = base + __builtin_ctzll(left_of), x = s_token[i];
        if (P.greedy) {
          if (x == s_best[node]) found = i;
          continue;
        }
        const double u = s_u[i];
        if (q_row) {
          if (!summed) left = rest_sum(), summed = true;
          const double q = s_q[i];
          if (u * left * q < fmax(s_w[i] * one - less * q, 0.0)) {
            found = i;
          } else {
            less += left;
            summed = false;
          }
        } else {
          double w = s_w[i];
          for (int j = node + 1; j < i; ++j)  // refused before
            if (s_up[j] == node && s_token[j] == x) w = 0;
          if (u * left < w)
            found = i;
          else
            left -= w;
        }
      }
    }
    if (found < 0) break;
    node = found;
    if (tid == 0) kept[count] = node, out[count - 1] = s_token[node];
    ++count;
    enter();
  }
  if (tid == 0) kept[0] = 0, P.counts[b] = count;
  if (P.greedy || !(weigh.top > -INFINITY)) {
    if (tid == 0) out[count - 1] = weigh.top > -INFINITY ? s_best[node] : 0;
    return;
  }

  // The draw: the chunk first. Its first wave finds it, from the sums of the chunks (the node's own, less the
  // guesses that were refused there, or of what is left of p and q).
  int n_gone = 0;  // distinct refused guesses
  const Part *parts = P.parts + int64_t(begin + node) * C;
  bool rest = q_row && less > 0;  // else all of p, or p without the refused
  if (!q_row) {
    for (int base = (node + 1) & ~63; base < n; base += 64) {
      const int mine = base + lane;
      bool kid = mine > node && mine < n && s_up[min(mine, n - 1)] == node && s_token[min(mine, n - 1)] >= 0;
      for (int j = node + 1; kid && j < mine; ++j) kid = !(s_up[j] == node && s_token[j] == s_token[mine]);
      const uint64_t kids = __builtin_amdgcn_ballot_w64(kid);
      if (wave == 0 && kid) s_gone[n_gone + __builtin_popcountll(kids & ((uint64_t(1) << lane) - 1))] = mine;
      n_gone += __builtin_popcountll(kids);
    }
  }
  __syncthreads();  // s_gone is written
  auto chunk_sum = [&](int c) {
    if (c >= C) return 0.0;
    const double all = parts[c].sum * weigh(parts[c].top);
    double sum = all;
    for (int g = 0; g < n_gone; ++g)
      if (s_token[s_gone[g]] / kChunk == c) sum -= s_w[s_gone[g]];
    return sum > all * 0x1p-45 ? sum : 0.0;  // else rounding is what is left
  };
  auto pick = [&](double whole, auto sum_of) {  // by the first wave: the chunk, and how far into it
    double want = double(s_u[0]) * whole, before = 0, in_last = 0;
    int last = 0;
    for (int c0 = 0; c0 < C; c0 += 64) {
      const double x = sum_of(c0 + lane), upto = before + wave_upto64(x, lane);
      const uint64_t past = __builtin_amdgcn_ballot_w64(x > 0 && upto > want), any = __builtin_amdgcn_ballot_w64(x > 0);
      const int l = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : 0;
      if (any) last = c0 + l, in_last = __shfl(upto - x, l, 64);
      if (past) break;
      before = __shfl(upto, 63, 64);
    }
    if (lane == 0) s_chunk = last, s_want = want - in_last;
  };
  double whole = 0;
  if (rest) {
    whole = rest_sum();
    rest = whole > 0;
  }
  if (!rest) {
    if (wave == 0) {
      for (int round = 0; round < 2; ++round) {
        whole = 0;
        for (int c = lane; c < C; c += 64) whole += chunk_sum(c);
        whole = wave_sum64(whole);
        if (whole > 0 || n_gone == 0) break;
        n_gone = 0;  // nothing is left but rounding: from all of them
      }
      pick(whole, chunk_sum);
      if (lane == 0) s_sum[0] = n_gone;
    }
    __syncthreads();
    n_gone = int(s_sum[0]);
  } else if (C <= kRestChunks) {
    if (wave == 0)
      pick(whole, [&](int c) {
        double sum = 0;
        if (c < C)
          for (int k = 0; k < kWaves; ++k) sum += s_rest[c][k];
        return sum;
      });
    __syncthreads();
  } else {
    // More chunks than are kept: one after another, until the draw's is passed.
    const double want = double(s_u[0]) * whole;
    double before = 0, in_last = 0;
    int last = 0;
    for (int c = 0; c < C; ++c) {
      double w[4];
      const int i = c * kChunk + 4 * tid;
      double sum = wave_sum64(rest_of(four(row, i, -INFINITY), four(q_row, i, 0.f), w));
      __syncthreads();
      if (lane == 0) s_sum[wave] = sum;
      __syncthreads();
      sum = 0;
      for (int k = 0; k < kWaves; ++k) sum += s_sum[k];
      if (sum > 0) last = c, in_last = before;
      before += sum;
      if (before > want) break;
    }
    __syncthreads();
    if (tid == 0) s_chunk = last, s_want = want - in_last;
    __syncthreads();
  }

  // Then the token, four of the chunk's a thread.
  const int i0 = s_chunk * kChunk + 4 * tid;
  double w[4];
  const f32x4u x = four(row, i0, -INFINITY);
  if (rest) {
    rest_of(x, four(q_row, i0, 0.f), w);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = weigh(x[e]);
      for (int g = 0; g < n_gone; ++g)
        if (s_token[s_gone[g]] == i0 + e) w[e] = 0;
    }
  }
  double upto = wave_upto64((w[0] + w[1]) + (w[2] + w[3]), lane);
  __syncthreads();  // s_sum has been read
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  upto -= (w[0] + w[1]) + (w[2] + w[3]);
  for (int k = 0; k < wave; ++k) upto += s_sum[k];
  const double want = s_want;
  int at = 0x7fffffff, last = -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    upto += w[e];
    if (w[e] > 0) {
      last = i0 + e;
      if (upto > want) at = min(at, i0 + e);
    }
  }
  // The first past it, or by rounding none: the last that has any.
  at = wave_min(at);
  last = -wave_min(-last);
  if (lane == 0) s_gone[wave] = at, s_gone[kWaves + wave] = last;
  __syncthreads();
  if (tid > 0) return;
  for (int k = 0; k < kWaves; ++k) at = min(at, s_gone[k]), last = max(last, s_gone[kWaves + k]);
  out[count - 1] = at != 0x7fffffff ? at : max(last, 0);
}

}  // namespace
}  // namespace mcamd

using namespace mcamd;

extern "C" size_t mcamd_verify_drafts_scratch_bytes(int64_t total, int64_t vocab) {
  if (total <= 0 || vocab <= 0 || total >= 0x7fffffff || vocab > (int64_t(1) << 30)) return 0;
  return size_t(total) * size_t((vocab + kChunk - 1) / kChunk) * sizeof(Part);
}

extern "C" int mcamd_verify_drafts(const float *logits, int64_t logits_stride, const float *draft_probs,
                                   int64_t draft_stride, const int64_t *tokens, const int32_t *parents,
                                   const int32_t *cu_seqlens, const float *numbers, int32_t *kept,
                                   int32_t *counts, int64_t *out_tokens, int64_t n_rows, int64_t total,
                                   int64_t max_seqlen, int64_t vocab, float temperature, void *scratch,
                                   size_t scratch_bytes, void *stream) {
  if (n_rows < 0 || total < 0 || max_seqlen < 1 || vocab <= 0 || vocab > (int64_t(1) << 30))
    return fail(MCAMD_EINVAL, "verify_drafts: need n_rows, total >= 0, max_seqlen >= 1, 0 < vocab <= 2^30");
  if (max_seqlen > kMaxNodes) return fail(MCAMD_EUNSUPPORTED, "verify_drafts: more than 1024 nodes in a row");
  if (n_rows >= 0x7fffffff || total >= 0x7fffffff)
    return fail(MCAMD_EUNSUPPORTED, "verify_drafts: sizes beyond 31 bits");
  if (!(temperature >= 0.f) || std::isinf(temperature))
    return fail(MCAMD_EINVAL, "verify_drafts: temperature must be finite and non-negative");
  if (logits_stride < vocab || (draft_probs && draft_stride < vocab))
    return fail(MCAMD_EINVAL, "verify_drafts: a row's stride smaller than the vocabulary");
  if (n_rows == 0) {
    clear_error();
    return MCAMD_OK;
  }
  if (!cu_seqlens || !kept || !counts || !out_tokens || (total > 0 && (!logits || !tokens || !parents || !numbers)))
    return fail(MCAMD_EINVAL, "verify_drafts: null pointer");
  const int64_t chunks = (vocab + kChunk - 1) / kChunk;
  if (total * chunks > 0x7fffffff / kChunkThreads)
    return fail(MCAMD_EUNSUPPORTED, "verify_drafts: grid too large");
  if (!aligned(scratch, 16)) return fail(MCAMD_EINVAL, "verify_drafts: scratch not 16-byte aligned");
  if (total > 0 && (!scratch || scratch_bytes < mcamd_verify_drafts_scratch_bytes(total, vocab)))
    return fail(MCAMD_EWORKSPACE, "verify_drafts: scratch smaller than mcamd_verify_drafts_scratch_bytes()");
  VerifyParams P;
  P.logits = logits;
  P.probs = temperature > 0.f ? draft_probs : nullptr;
  P.logits_stride = logits_stride;
  P.probs_stride = draft_stride;
  P.tokens = tokens;
  P.parents = parents;
  P.cu = cu_seqlens;
  P.numbers = numbers;
  P.kept = kept;
  P.counts = counts;
  P.out = out_tokens;
  P.total = int(total);
  P.most = int(max_seqlen);
  P.vocab = int(vocab);
  P.greedy = temperature == 0.f;
  P.scale = P.greedy ? 1.0 : 1.44269504088896340736 / double(temperature);
  P.parts = static_cast<Part *>(scratch);
  P.chunks = int(chunks);
  if (total > 0) {
    hipLaunchKernelGGL(verify_parts_kernel, dim3(unsigned(total * chunks)), dim3(kChunkThreads), 0,
                       as_stream(stream), P);
    const int st = launch_status("verify_drafts");
    if (st != MCAMD_OK) return st;
  }
  hipLaunchKernelGGL(verify_kernel, dim3(unsigned(n_rows)), dim3(kThreads), 0, as_stream(stream), P);
  return launch_status("verify_drafts");
}
