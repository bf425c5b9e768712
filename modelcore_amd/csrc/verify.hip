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
// it: weights and sums are in 64 bits.
//
// A workgroup has a row. Its sixteen waves each sum a run of the vocabulary, the run in which the draw falls is
// cut in sixteen again, until a wave's lanes hold a token each.
#include "kernels.h"

#include <cmath>

namespace mcamd {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxNodes = 1024;

struct VerifyParams {
  const float *logits, *probs;
  int64_t logits_stride, probs_stride;
  const int64_t *tokens;
  const int32_t *parents, *cu;
  const float *numbers;
  int32_t *kept, *counts;
  int64_t *out;
  int total, most, vocab;
  double inv_temp;
  int greedy;
};

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// Sums over the waves' runs, in order: what comes before run w and all.
struct Sums {
  double part[kWaves];
};
__device__ __forceinline__ double block_sum(double x, Sums &s) {
  x = wave_sum64(x);
  __syncthreads();  // the sums before have been read
  if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = x;
  __syncthreads();
  double all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += s.part[w];
  return all;
}

// A node's logits as weights against the largest of them, which an infinite one makes 1 and all others 0. NaN has none.
struct Weigher {
  float top;
  double inv_temp;
  __device__ __forceinline__ double operator()(float x) const {
    if (x == top) return 1.0;
    if (!(x > -INFINITY) || top == INFINITY) return 0.0;
    return exp((double(x) - double(top)) * inv_temp);
  }
};

__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyParams P) {
  __shared__ Sums s_sums;
  __shared__ float s_top[kWaves];
  __shared__ int s_best[kWaves];
  __shared__ int s_gone[kMaxNodes];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int begin = max(P.cu[b], 0), n = min(max(min(P.cu[b + 1], P.total) - begin, 0), P.most);
  int32_t *const kept = P.kept + int64_t(b) * P.most;
  int64_t *const out = P.out + int64_t(b) * P.most;
  for (int j = tid; j < P.most; j += kThreads) kept[j] = -1, out[j] = -1;
  __syncthreads();  // the padding is written before the tokens
  if (n == 0) {
    if (tid == 0) P.counts[b] = 0;
    return;
  }
  const int V = P.vocab;
  int node = 0, count = 1, n_gone = 0, best = 0;
  const float *row = nullptr, *q_row = nullptr;
  Weigher weigh{0.f, P.inv_temp};
  double all = 0, less = 0, left = 0;  // less, left: a and Z, of guesses Z in units of the weights

  // The node's largest logit, where it is, and the sum of its weights.
  auto enter = [&]() {
    row = P.logits + int64_t(begin + node) * P.logits_stride;
    q_row = P.probs ? P.probs + int64_t(begin + node) * P.probs_stride : nullptr;
    float top = -INFINITY;
    best = 0x7fffffff;
    for (int i = tid; i < V; i += kThreads) {
      const float x = row[i];
      if (x > top || (x == top && i < best)) top = x, best = i;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float t2 = __shfl_xor(top, o, 64);
      const int b2 = __shfl_xor(best, o, 64);
      if (t2 > top || (t2 == top && b2 < best)) top = t2, best = b2;
    }
    __syncthreads();  // of the node before
    if (lane == 0) s_top[wave] = top, s_best[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
      if (s_top[w] > top || (s_top[w] == top && s_best[w] < best)) top = s_top[w], best = s_best[w];
    weigh.top = top;
    less = 0, n_gone = 0;
    if (P.greedy) return;
    double sum = 0;
    if (top > -INFINITY)
      for (int i = tid; i < V; i += kThreads) sum += weigh(row[i]);
    all = block_sum(sum, s_sums);
    left = q_row ? 1.0 : all;
  };
  // What is left of token i's probability (q) or weight (guesses).
  auto remains = [&](int i) {
    double w = weigh(row[i]);
    if (q_row) return fmax(w / all - less * double(q_row[i]), 0.0);
    for (int g = 0; g < n_gone; ++g) w = s_gone[g] == i ? 0.0 : w;
    return w;
  };

  enter();
  for (int i = 1; i < n; ++i) {
    if (P.parents[begin + i] != node) continue;
    const int64_t x = P.tokens[begin + i];
    if (x < 0 || x >= V || !(weigh.top > -INFINITY)) continue;
    bool taken;
    const double u = P.numbers[begin + i];
    if (P.greedy) {
      taken = int(x) == best;
    } else {
      const double w = remains(int(x));
      taken = u * left * (q_row ? double(q_row[x]) : 1.0) < w;
      if (!taken) {
        if (q_row) {
          less += left;
          double sum = 0;
          for (int j = tid; j < V; j += kThreads) sum += remains(j);
          left = block_sum(sum, s_sums);
        } else {
          left -= w;
          __syncthreads();
          if (tid == 0) s_gone[n_gone] = int(x);
          ++n_gone;
          __syncthreads();
        }
      }
    }
    if (!taken) continue;
    if (tid == 0) kept[count] = i, out[count - 1] = x;
    ++count;
    node = i;
    enter();
  }
  if (tid == 0) kept[0] = 0, P.counts[b] = count;
  if (P.greedy || !(weigh.top > -INFINITY)) {
    if (tid == 0) out[count - 1] = best == 0x7fffffff ? 0 : best;
    return;
  }

  // The draw. lo .. hi: where it falls; want: how far into its weights.
  bool plain = false;  // nothing is left but rounding: from all of them
  auto weight = [&](int i) { return plain ? weigh(row[i]) : remains(i); };
  int lo = 0, hi = V;
  double want = 0;
  for (bool first = true; hi - lo > 64; first = false) {
    const int each = (hi - lo + kWaves - 1) / kWaves;
    const int from = min(lo + wave * each, hi), to = min(from + each, hi);
    auto sums = [&]() {
      double sum = 0;
      for (int i = from + lane; i < to; i += 64) sum += weight(i);
      return block_sum(sum, s_sums);
    };
    double sum = sums();
    if (first) {
      if (!(sum > 0)) {
        plain = true;
        sum = sums();
      }
      want = double(P.numbers[begin]) * sum;
    }
    double upto = 0, before = 0;
    int part = -1, last = 0;
    for (int w = 0; w < kWaves; ++w) {
      const double x = s_sums.part[w];
      if (x > 0) last = w;
      if (part < 0 && upto + x > want) part = w, before = upto;
      upto += x;
    }
    if (part < 0) {  // by rounding past them all: the last one that has any
      part = last, before = 0;
      for (int w = 0; w < last; ++w) before += s_sums.part[w];
    }
    want -= before;
    lo = min(lo + part * each, hi);
    hi = min(lo + each, hi);
  }
  if (wave > 0) return;
  const int i = lo + lane;
  double w = i < hi ? weight(i) : 0.0;
  if (V <= 64) {
    const double sum = wave_sum64(w);
    if (!(sum > 0)) {
      plain = true;
      w = i < hi ? weight(i) : 0.0;
    }
    want = double(P.numbers[begin]) * wave_sum64(w);
  }
  double upto = w;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  const uint64_t past = __builtin_amdgcn_ballot_w64(w > 0 && upto > want), any = __builtin_amdgcn_ballot_w64(w > 0);
  const int l = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : 0;
  if (lane == 0) out[count - 1] = lo + l;
}

}  // namespace
}  // namespace mcamd

using namespace mcamd;

extern "C" size_t mcamd_verify_drafts_scratch_bytes(int64_t total, int64_t vocab) {
  (void)total, (void)vocab;
  return 0;
}

extern "C" int mcamd_verify_drafts(const float *logits, int64_t logits_stride, const float *draft_probs,
                                   int64_t draft_stride, const int64_t *tokens, const int32_t *parents,
                                   const int32_t *cu_seqlens, const float *numbers, int32_t *kept,
                                   int32_t *counts, int64_t *out_tokens, int64_t n_rows, int64_t total,
                                   int64_t max_seqlen, int64_t vocab, float temperature, void *scratch,
                                   size_t scratch_bytes, void *stream) {
  (void)scratch, (void)scratch_bytes;
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
  P.inv_temp = P.greedy ? 1.0 : 1.0 / double(temperature);
  hipLaunchKernelGGL(verify_kernel, dim3(unsigned(n_rows)), dim3(kThreads), 0, as_stream(stream), P);
  return launch_status("verify_drafts");
}
