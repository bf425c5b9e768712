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
// it: weights and sums are in 64 bits, whose multiply-adds run as fast here as those of 32.
//
// Two launches. The first reads every logit once, a workgroup kChunk of a node's, and leaves the largest, its place
// and the sum of the chunk's weights against it: bound by HBM (32 trees of 32 nodes, vocabulary 32768: 134 MB in 29
// to 32 us, 4.2 to 4.6 TB/s). The second has a workgroup a row: a node's chunks are put together by a few lanes and
// the probabilities of all drafts fetched at once; its first wave then walks, out of registers and LDS, and finds
// the draw's chunk by the chunks' sums, all waves make the sums (p - a q)+ where they are wanted (before a further
// child is tried against them, and for the draw) and read that chunk again. Bound by latency: seven round trips, 12
// us for those trees, 16 with such a sum over a row (64 chains of four); with sixteen waves that all walk 19 and 21,
// since a SIMD's four wait for one another. Weights are made eight side by side or four: the ten multiply-adds of
// one wait for each other.
#include "kernels.h"

#include <cmath>

namespace mcamd {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxNodes = 1024;
constexpr int kChunkThreads = 256;
constexpr int kRestChunks = 2048;  // whose sums of (p - a q)+ have room
constexpr double kNothing = 1e-290;  // a weight up to that counts as 0; above the least that exp2_64 makes, 2^-1020
constexpr int kChunk = 16 * kChunkThreads;  // logits
static_assert(kChunk == 8 * kThreads, "the draw's threads have eight each");

struct Part {  // of a chunk
  double sum;
  float top;
  int at;
};

struct Link {  // of a node: whom it follows, and its token or -1
  int up, token;
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

// 2^y for y up to 0 (from -1020 on), to 2^-45: y + 1.5 2^52 has the nearest whole number in its low word, which
// goes into the exponent, and 2^f, |f| <= 1/2, is the polynomial that meets it in the ten Chebyshev points of the
// interval. Eighteen instructions a logit with the sum, four fewer than by the series, rint and ldexp.
// N of them side by side: alone, each multiply-add would wait for the one before.
template <int N>
__device__ __forceinline__ void exp2_64(double (&y)[N]) {
  constexpr double kWhole = 6755399441055744.0;
  constexpr double kSeries[10] = {1.0000000000000135,    0.6931471805599462,     0.2402265069564034,
                                  0.05550410866465167,   0.009618129193934313,   0.0013333558200794592,
                                  0.0001540343375125101, 1.5252672924850737e-05, 1.325964524488711e-06,
                                  1.0205905413765595e-07};
  double f[N], p[N];
  int whole[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double z = fmax(y[i], -1020.0), t = z + kWhole;
    f[i] = z - (t - kWhole);
    whole[i] = __double2loint(t) << 20;
    p[i] = kSeries[9];
  }
#pragma unroll
  for (int k = 8; k >= 0; --k)
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = fma(p[i], f[i], kSeries[k]);
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = __hiloint2double(__double2hiint(p[i]) + whole[i], __double2loint(p[i]));
}

// Logits as weights against the largest of them, which an infinite one makes 1 and all others 0. NaN has none.
// The largest is taken off before the scale is put on, so that its own weight is 1 and no exponent is above 0: one
// multiply-add with -top * scale would leave that product's rounding, which passes 1 from |top| / temperature = 6e15
// on.
struct Weigher {
  float top;
  double scale;
  __device__ __forceinline__ Weigher(float t, double s) : top(t), scale(s) {}
  // Of a finite top, those so far below it that they are 0 in 64 bits being next to nothing: for sums, in which the
  // largest is.
  template <int N>
  __device__ __forceinline__ void finite(const float (&x)[N], double (&w)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = (double(x[i]) - double(top)) * scale;
    exp2_64(w);
  }
  template <int N>
  __device__ __forceinline__ void weigh(const float (&x)[N], double (&w)[N]) const {
    finite(x, w);
    const bool inf = top == INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = inf ? (x[i] == top ? 1.0 : 0.0) : w[i] > kNothing ? w[i] : 0.0;
  }
  __device__ __forceinline__ double operator()(float x) const {
    const float x1[1] = {x};
    double w[1];
    weigh(x1, w);
    return w[0];
  }
};

// Inclusive sums over the wave, by moves between lanes on the VALU: the waves' shuffles would wait for one another
// at the LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved64(double x) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROWS, 0xf, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ double wave_upto64(double x) {
  x += moved64<0x111, 0xf>(x);  // row_shr:1
  x += moved64<0x112, 0xf>(x);  // row_shr:2
  x += moved64<0x114, 0xf>(x);  // row_shr:4
  x += moved64<0x118, 0xf>(x);  // row_shr:8
  x += moved64<0x142, 0xa>(x);  // row_bcast:15
  x += moved64<0x143, 0xc>(x);  // row_bcast:31
  return x;
}
__device__ __forceinline__ double lane64(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane),
                          __builtin_amdgcn_readlane(__double2loint(x), lane));
}
__device__ __forceinline__ double wave_sum64(double x) { return lane64(wave_upto64(x), 63); }
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
  const Weigher weigh(top, P.scale);
  double sum = 0;
  if (fabsf(top) < INFINITY) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float y[4] = {x[j][0], x[j][1], x[j][2], x[j][3]};
      double w[4];
      weigh.finite(y, w);
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
  } else if (top > 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += x[j][e] == top ? 1.0 : 0.0;
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
  __shared__ double s_all[kMaxNodes], s_one[kMaxNodes], s_w[kMaxNodes];
  __shared__ float s_top[kMaxNodes], s_q[kMaxNodes], s_u[kMaxNodes];
  __shared__ int s_best[kMaxNodes];
  __shared__ __attribute__((aligned(16))) Link s_link[kMaxNodes + 1];
  __shared__ __attribute__((aligned(16))) int s_gone[kMaxNodes];  // the tokens of refused guesses, and their weights
  __shared__ double s_gone_w[kMaxNodes];
  __shared__ double s_rest[kRestChunks];  // sums of (p - a q)+, by runs of tokens
  __shared__ double s_sum[kWaves];
  __shared__ struct {  // the first wave's word to the others
    int what, node, count, chunk, n_gone;
    bool rest;
    double less, want;
  } s_say;
  enum { kDone, kSum, kDraw };
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
  auto link_of = [&](int i) {
    Link x{-1, -1};
    if (i < n) {
      const int64_t t = P.tokens[begin + i];
      const float u = P.numbers[begin + i];
      if (i > 0) x.up = P.parents[begin + i];
      if (x.up >= i) x.up = -1;
      if (t >= 0 && t < V) x.token = int(t);
      s_u[i] = u;
    }
    if (i <= n) s_link[i] = x;  // and one behind them that follows none
    return x;
  };
  auto logit_of = [&](int i, const Link &x) {  // of the draft, behind its parent
    if (P.greedy || x.up < 0 || x.token < 0) return -INFINITY;
    if (P.probs) s_q[i] = P.probs[int64_t(begin + x.up) * P.probs_stride + x.token];
    return P.logits[int64_t(begin + x.up) * P.logits_stride + x.token];
  };
  const Link own = link_of(tid);
  for (int i = tid + kThreads; i <= n; i += kThreads) link_of(i);
  const float own_logit = logit_of(tid, own);
  int lanes = 1;  // of a node, as many as its chunks
  while (lanes < C && lanes < 64) lanes *= 2;
  for (int i0 = wave * (64 / lanes); i0 < n; i0 += kThreads / lanes) {
    const int i = i0 + lane / lanes, first = lane & (lanes - 1);
    const Part *part = P.parts + int64_t(begin + min(i, n - 1)) * C;
    float top = -INFINITY;
    for (int c = first; c < C; c += lanes) top = fmaxf(top, part[c].top);
    for (int o = lanes >> 1; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (P.greedy) {
      int best = 0x7fffffff;
      for (int c = first; c < C; c += lanes)
        if (part[c].top == top) best = min(best, part[c].at);
      for (int o = lanes >> 1; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
      if (first == 0 && i < n) s_best[i] = best;
    } else {
      const Weigher weigh(top, P.scale);
      double all = 0;
      for (int c = first; c < C; c += lanes) all += part[c].sum * weigh(part[c].top);
      for (int o = lanes >> 1; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
      if (first == 0 && i < n) s_all[i] = all, s_one[i] = 1.0 / all;
    }
    if (first == 0 && i < n) s_top[i] = top;
  }
  __syncthreads();
  for (int i = tid; !P.greedy && i < n; i += kThreads) {
    const Link x = i == tid ? own : s_link[i];
    const float logit = i == tid ? own_logit : logit_of(i, x);
    double w = logit > -INFINITY ? Weigher(s_top[x.up], P.scale)(logit) : 0.0;
    // A guess that a sibling before it has made has nothing left.
    if (!P.probs) {
      int again = 0;
      if (n <= 64) {
        for (int j0 = 0; j0 < n; j0 += 8)
#pragma unroll
          for (int j = j0; j < j0 + 8; ++j)
            again |= int(__builtin_amdgcn_readlane(x.up, j) == x.up) &
                     int(__builtin_amdgcn_readlane(x.token, j) == x.token) & int(j < lane);
      } else {
        const int4 *links = reinterpret_cast<const int4 *>(s_link);  // two nodes each
#pragma unroll 8
        for (int j = 0; j < min((i | 63) + 1, n) >> 1; ++j) {
          const int4 y = links[j];
          again |= int(y.x == x.up) & int(y.y == x.token) & int(2 * j < i);
          again |= int(y.z == x.up) & int(y.w == x.token) & int(2 * j + 1 < i);
        }
      }
      w = again ? 0.0 : w;
    }
    s_w[i] = w;
  }
  __syncthreads();

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
  // What is left of the probabilities of four tokens: p - a q, where more than next to nothing is.
  auto rest_of = [&](const Weigher &weigh, double one, double less, const f32x4u &x, const f32x4u &q,
                     double (&w)[4]) {
    const float y[4] = {x[0], x[1], x[2], x[3]};
    weigh.finite(y, w);
    if (weigh.top == INFINITY)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = y[e] == INFINITY ? 1.0 : 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = fmax(fma(w[e], one, fma(-less, double(q[e]), -kNothing)), 0.0);
    return (w[0] + w[1]) + (w[2] + w[3]);
  };
  // A chunk is `runs` runs of tokens, so that all waves have some.
  int runs = 1;
  while (runs * 2 * C <= kWaves) runs *= 2;
  // s_rest of a node, run by run: by all waves.
  auto rest_sums = [&](int node, double less) {
    constexpr int U = 8;  // loads of each under way at once
    const float *row = P.logits + int64_t(begin + node) * P.logits_stride;
    const float *q_row = P.probs + int64_t(begin + node) * P.probs_stride;
    const Weigher weigh(s_top[node], P.scale);
    const double one = s_one[node];
    const int each = kChunk / runs;
    for (int r = wave; r < C * runs; r += kWaves) {
      double sum = 0;
      for (int i0 = 0; i0 < each; i0 += 256 * U) {
        f32x4u x[U], q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + 256 * u < each ? r * each + i0 + 256 * u + 4 * lane : V;
          x[u] = four(row, i, -INFINITY);
          q[u] = four(q_row, i, 0.f);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          double w[4];
          sum += rest_of(weigh, one, less, x[u], q[u], w);
        }
      }
      sum = wave_sum64(sum);
      if (lane == 0) s_rest[r] = sum;
    }
  };

  // The walk, by the first wave. The others wait for it (and would only be in its way), but for the sums of what
  // is left and the draw. The first 64 nodes are in registers, a node a lane.
  int node = 0, count = 1, base = 0;
  double less = 0, left = 0;  // a and Z, of guesses Z in units of the weights
  bool summed = true;         // left is the sum for this a
  uint64_t kids = 0;          // that are left to try, among nodes base ..
  const double my_w = P.greedy ? 0.0 : s_w[min(lane, n - 1)];
  const float my_u = s_u[min(lane, n - 1)], my_q = P.probs ? s_q[min(lane, n - 1)] : 1.f;
  auto kids_of = [&](int base) {  // the node's children among 64, bit by bit
    const Link x = base == 0 ? own : s_link[min(base + lane, n)];
    return __builtin_amdgcn_ballot_w64(x.up == node && x.token >= 0 && base + lane < n);
  };
  auto uniform = [](bool x) { return __builtin_amdgcn_ballot_w64(x) != 0; };  // x is the same in all lanes
  auto lane32 = [&](float x, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l)); };
  auto enter = [&]() {
    less = 0;
    summed = true;
    if (!P.greedy) left = P.probs ? 1.0 : s_all[node];
    base = node & ~63;
    kids = s_top[node] > -INFINITY ? kids_of(base) : 0;
  };
  auto walk = [&]() {  // false where a sum is wanted first
    for (;;) {
      if (kids == 0) {
        if (base + 64 >= n || !(s_top[node] > -INFINITY)) return true;
        base += 64;
        kids = kids_of(base);
        continue;
      }
      const int l = __builtin_ctzll(kids), i = base + l;
      bool taken;
      if (P.greedy) {
        taken = uniform(s_link[i].token == s_best[node]);
      } else {
        const double u = base == 0 ? lane32(my_u, l) : s_u[i], w = base == 0 ? lane64(my_w, l) : s_w[i];
        if (P.probs) {
          if (!summed) return false;
          const double q = base == 0 ? lane32(my_q, l) : s_q[i];
          taken = uniform(u * left * q < fmax(w * s_one[node] - less * q, 0.0));
          if (!taken) less += left, summed = false;
        } else {
          taken = uniform(u * left < w);
          if (!taken) left -= w;
        }
      }
      kids &= kids - 1;
      if (!taken) continue;
      node = i;
      if (lane == 0) kept[count] = node, out[count - 1] = s_link[node].token;
      ++count;
      enter();
    }
  };

  // The draw's chunk: by the first wave, from the sums of the chunks, of which it is the one in which want falls.
  auto pick = [&](double whole, auto sum_of) {
    double want = double(s_u[0]) * whole, before = 0, in_last = 0;
    int last = 0;
    for (int c0 = 0; c0 < C; c0 += 64) {
      const double x = sum_of(c0 + lane), upto = before + wave_upto64(x);
      const uint64_t past = __builtin_amdgcn_ballot_w64(x > 0 && upto > want), any = __builtin_amdgcn_ballot_w64(x > 0);
      const int l = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : 0;
      if (any) last = c0 + l, in_last = lane64(upto - x, l);
      if (past) break;
      before = lane64(upto, 63);
    }
    if (lane == 0) s_say.chunk = last, s_say.want = want - in_last;
  };
  // Where nothing is left of p - a q, or there is no q: p without the guesses that were refused.
  auto pick_guesses = [&]() {
    int n_gone = 0;
    for (int base = node & ~63; !P.probs && base < n; base += 64) {
      const double w = base == 0 ? my_w : s_w[min(base + lane, n - 1)];
      const bool kid = ((kids_of(base) >> lane) & 1) && w > 0;  // distinct
      const uint64_t all = __builtin_amdgcn_ballot_w64(kid);
      if (kid) {
        const int at = n_gone + __builtin_popcountll(all & ((uint64_t(1) << lane) - 1));
        s_gone[at] = s_link[base + lane].token;
        s_gone_w[at] = w;
      }
      n_gone += __builtin_popcountll(all);
    }
    // All waves look through the list, four at a time.
    if (lane < 4 && n_gone + lane < kMaxNodes) s_gone[n_gone + lane] = -1, s_gone_w[n_gone + lane] = 0;
    __builtin_amdgcn_wave_barrier();
    const Part *parts = P.parts + int64_t(begin + node) * C;
    const Weigher weigh(s_top[node], P.scale);
    auto chunk_sum = [&](int c) {
      if (c >= C) return 0.0;
      const double all = parts[c].sum * weigh(parts[c].top);
      double sum = all;
#pragma unroll 4
      for (int g = 0; g < n_gone; ++g) sum -= s_gone[g] / kChunk == c ? s_gone_w[g] : 0.0;
      return sum > all * 0x1p-40 ? sum : 0.0;  // else rounding is what is left
    };
    double mine = 0, whole = 0;  // mine: the last of this lane's chunks
    for (int round = 0; round < 2; ++round) {
      whole = 0;
      for (int c = lane; c < C; c += 64) whole += mine = chunk_sum(c);
      whole = wave_sum64(whole);
      if (whole > 0 || n_gone == 0) break;
      n_gone = 0;  // nothing is left but rounding: from all of them
    }
    pick(whole, [&](int c) { return C <= 64 ? mine : chunk_sum(c); });
    if (lane == 0) s_say.n_gone = n_gone, s_say.rest = false;
  };

  bool walked = false;
  for (bool first = true;; first = false) {
    if (wave == 0) {
      if (first) {
        enter();
      } else {  // the sum is there
        left = 0;
        for (int r = lane; r < C * runs; r += 64) left += s_rest[r];
        left = wave_sum64(left);
        summed = true;
      }
      walked = walked || walk();
      int what = kSum;
      if (walked) {
        const bool none = P.greedy || !(s_top[node] > -INFINITY);
        if (none) {
          if (lane == 0) out[count - 1] = s_top[node] > -INFINITY ? s_best[node] : 0;
          what = kDone;
        } else if (!P.probs || less == 0 || (summed && !(left > 0))) {
          pick_guesses();
          what = kDraw;
        } else if (summed) {
          pick(left, [&](int c) {
            double sum = 0;
            if (c < C)
              for (int r = 0; r < runs; ++r) sum += s_rest[c * runs + r];
            return sum;
          });
          if (lane == 0) s_say.n_gone = 0, s_say.rest = true;
          what = kDraw;
        }
        if (what != kSum && lane == 0) kept[0] = 0, P.counts[b] = count;
      }
      if (lane == 0) s_say.what = what, s_say.node = node, s_say.count = count, s_say.less = less;
    }
    __syncthreads();
    if (s_say.what != kSum) break;
    rest_sums(s_say.node, s_say.less);
    __syncthreads();
  }
  if (s_say.what == kDone) return;

  // Then the token, eight of the chunk's a thread.
  const int at = s_say.node, i0 = s_say.chunk * kChunk + 8 * tid;
  const float *row = P.logits + int64_t(begin + at) * P.logits_stride;
  const f32x4u x0 = four(row, i0, -INFINITY), x1 = four(row, i0 + 4, -INFINITY);
  const Weigher weigh(s_top[at], P.scale);
  double w[8];
  if (s_say.rest) {
    const float *q_row = P.probs + int64_t(begin + at) * P.probs_stride;
    const f32x4u q0 = four(q_row, i0, 0.f), q1 = four(q_row, i0 + 4, 0.f);
    double w0[4], w1[4];
    rest_of(weigh, s_one[at], s_say.less, x0, q0, w0);
    rest_of(weigh, s_one[at], s_say.less, x1, q1, w1);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = w0[e], w[4 + e] = w1[e];
  } else {
    const float y[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    weigh.weigh(y, w);
    for (int g = 0; g < s_say.n_gone; g += 4) {
      const int4 gone = *reinterpret_cast<const int4 *>(&s_gone[g]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = i0 + e;
        w[e] = (int(gone.x == i) | int(gone.y == i) | int(gone.z == i) | int(gone.w == i)) ? 0.0 : w[e];
      }
    }
  }
  const double mine_all = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  double upto = wave_upto64(mine_all);
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  // The first wave that passes it, or by rounding none: the last that has any.
  const double want = s_say.want;
  const double of_wave = lane < kWaves ? s_sum[lane] : 0.0, upto_wave = wave_upto64(of_wave);
  const uint64_t past_waves = __builtin_amdgcn_ballot_w64(of_wave > 0 && upto_wave > want),
                 any_waves = __builtin_amdgcn_ballot_w64(of_wave > 0);
  if (wave != (past_waves ? __builtin_ctzll(past_waves) : any_waves ? 63 - __builtin_clzll(any_waves) : 0)) return;
  upto += lane64(upto_wave - of_wave, wave) - mine_all;
  uint32_t past = 0, any = 0;  // of this lane's eight
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    upto += w[e];
    any |= w[e] > 0 ? 1u << e : 0u;
    past |= w[e] > 0 && upto > want ? 1u << e : 0u;
  }
  const uint64_t pasts = __builtin_amdgcn_ballot_w64(past != 0), anys = __builtin_amdgcn_ballot_w64(any != 0);
  const int l = pasts ? __builtin_ctzll(pasts) : anys ? 63 - __builtin_clzll(anys) : 0;
  if (lane != l) return;
  out[s_say.count - 1] = i0 + (past ? __builtin_ctz(past) : any ? 31 - __builtin_clz(any) : 0);
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
  if (draft_probs && temperature > 0.f && chunks > kRestChunks)
    return fail(MCAMD_EUNSUPPORTED, "verify_drafts: with draft_probs a vocabulary of at most 2^23");
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
