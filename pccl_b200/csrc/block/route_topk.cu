// Expert routing: scores, group-limited top-k with a balance bias, weights, and the rows of the choices in
// expert order; and the gradient of the weights.
//
//   p = softmax(l) or sigmoid(l);  s = p + bias;  the best `top_groups` groups of experts stay;
//   idx = the top_k largest s of what stays, ties to the lowest number;
//   w_k = scale * p_k / sum p  (or scale * p_k);
//   rows[t][k] = offsets[idx] + number of earlier tokens that chose the same expert.
//
// With few experts one thread takes a token (by_threads() has the rule), else one warp,
// expert e in lane e / NE, so that the lowest lane holds the lowest number and a tie is decided by the first set bit of
// a ballot.  Scores are compared as unsigned keys of the same order (one redux.sync a round); a lane keeps its keys
// sorted, so that a round costs the winner a shift.  Many tokens are bound by instructions, not by the 4 bytes a
// score that they read.
//
// The order of two scores is part of the answer, and 32 bits cannot tell scores apart that differ by less than
// their rounding.  Without a bias the order is that of the logits and needs no arithmetic.  With one, the choice
// is made in 32 bits together with the runner-up; where any two neighbours of the sorted choice (or the last
// group kept and the first dropped) are nearer than the error bound of the arithmetic, the token is chosen again
// in 64 bits.  Equal logits with equal biases are a true tie and need no repeat.
//
// Rows in expert order need no atomics whose order matters: a block of consecutive tokens marks its choices as
// bits in shared memory ([expert][token]), a choice's rank is a population count, and the blocks' counts
// per expert are summed by the second kernel in block order.
#include <math.h>

#include <algorithm>

#include "../common/util.h"
#include "../engine/cuda_driver.h"
#include "vec.cuh"

namespace pccl {
namespace block {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMostThreads = 1024;
constexpr int kThreadExperts = 8;             // up to so many experts a thread takes a token,
constexpr int kThreadExpertsFlat = 32;        // up to so many where the logits alone decide

struct RouteParams {
  RouteArgs a;
  const float* dweights;
  void* dlogits;
  uint16_t* counts;           // [blocks][pitch]: choices per expert of one block's tokens
  int pitch;                  // experts, rounded up to a multiple of four
  int tokens_per_block, words;
  int vec;                    // rows of logits can be read a lane's (or thread's) share at once
  int lanes;                  // lanes that share a group, a power of two; 0: groups do not divide so
  int block_words;            // 32-bit words of shared memory before the warps' decks
  uint32_t per_choice;        // 2^32 / top_k, rounded up: a choice's token without a division
};

// Unsigned keys in the order of the values; 0 stands below every value, infinities included.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(uint64_t k) {
  return __longlong_as_double(static_cast<int64_t>(k ^ ((k >> 63) ? 0x8000000000000000ull : 0xffffffffffffffffull)));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ float warp_max(float v) { return value_of(warp_max(key_of(v))); }
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <typename K> __device__ __forceinline__ K larger(K a, K b) { return a > b ? a : b; }
template <typename K> __device__ __forceinline__ K smaller(K a, K b) { return a > b ? b : a; }

// NaN counts as the lowest logit; +infinity as the largest finite one, so that no score is a NaN.  The sum with
// zero turns -0 into +0: the two are equal and their keys have to be.
__device__ __forceinline__ float clean(float l) { return fminf(fmaxf(l, -INFINITY), 3.402823466e38f) + 0.f; }

__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }
// For the choice alone.
__device__ __forceinline__ float quick_exp(float l) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(l * 1.44269504f));
  return r;
}
__device__ __forceinline__ float quick_sigmoid(float l) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + quick_exp(-l)));
  return r;
}

// Bound of the difference of two scores' errors; quick_exp(x) is off by (2 + 0.63 |x|) 2^-23 of itself (the instruction's
// 2^-22, the product's rounding and the constant's).  Sigmoid: p (1 - p) times that is at most 0.52 * 2^-23, the sum adds
// p 2^-24 and the reciprocal p 2^-23: below 1.7 * 2^-23 for one, 2^-21 for two.  Softmax: of the row's largest probability,
// the exponential 4 * 2^-24 ((2 + 0.63 |x|) e^-|x| is largest at 0), the sum over a lane and the warp (n + 5) 2^-24 and its
// terms' own 10 * 2^-24 (1023 terms at |x| = 5.5 beside one at 0 are the worst), quotient and product 3 * 2^-24.
__device__ __forceinline__ float score_error(bool sigmoid_scores, int n, float largest) {
  return sigmoid_scores ? 0x1.4p-21f : static_cast<float>(n + 24) * 0x1p-23f * largest;
}

// ---- a warp per token ------------------------------------------------------------------------------------------
// Largest first: Batcher's odd-even merge sort.
template <int NE>
__device__ __forceinline__ void sort_lane(uint32_t (&key)[NE]) {
#pragma unroll
  for (int p = 1; p < NE; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < NE; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < NE && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t hi = larger(key[i + j], key[i + j + k]);
            key[i + j + k] = smaller(key[i + j], key[i + j + k]);
            key[i + j] = hi;
          }
}

// Rank of this lane's group score among all, ties to the lower number; group g's score stands in lane g * lanes.
template <typename Key>
__device__ __forceinline__ int group_rank(int groups, int lanes, int group, Key mine) {
  // The lanes of a group share the comparisons.
  const int lane = threadIdx.x & 31;
  int rank = 0;
  for (int g0 = 0; g0 < groups; g0 += lanes) {
    const int g = g0 + (lane & (lanes - 1));
    const Key other = __shfl_sync(kAll, mine, g < groups ? g * lanes : 0);
    rank += g < groups && (other > mine || (other == mine && g < group)) ? 1 : 0;
  }
  for (int o = 1; o < lanes; o <<= 1) rank += __shfl_xor_sync(kAll, rank, o);
  return rank;
}

// Least and largest value that the exact score of a group can have, which is `score` in 32 bits: its parts, of sizes that
// add up to `size`, are off by half of tau each and by their own roundings, which a sum that cancels does not lose.  A
// part of minus infinity is exact, and the sum with it.
__device__ __forceinline__ float least_score(float score, float size, float tau, float step) {
  return fmaxf(score - fmaf(step, size, tau), -INFINITY);      // not a NaN
}
__device__ __forceinline__ float largest_score(float score, float size, float tau, float step) {
  return fmaxf(score + fmaf(step, size, tau), -INFINITY);
}

// Whether all that is close are pairs of choices with equal logits and equal biases, which no arithmetic can part.  (A
// choice and a runner-up that are equal are not enough: what stands behind them may be close to both.)
template <typename T>
__device__ __forceinline__ bool truly_tied(const RouteParams& p, int64_t t, int close, int pick) {
  const RouteArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  float l = 0.f, b = 0.f;
  if (lane < a.top_k) {
    const int e = min(max(pick, 0), a.experts - 1);
    l = to_f32<T>(static_cast<const T*>(a.logits)[t * a.ld + e]);
    b = a.bias != nullptr ? a.bias[e] : 0.f;
  }
  const float l1 = __shfl_down_sync(kAll, l, 1), b1 = __shfl_down_sync(kAll, b, 1);
  return !__any_sync(kAll, (close & 2) || ((close & 1) && !(lane < a.top_k - 1 && l == l1 && b == b1)));
}

// A warp's shared memory: the lanes' sorted keys, one above the other, and what was picked.
template <int NE> struct Deck {
  static constexpr int kKeys = NE <= 8 ? NE + 2 : 0;     // two rows of zeros below the last card
  uint32_t key[kKeys > 0 ? kKeys : 1][32];
  uint2 won[32];                                         // key, and lane * 8 + its lowest three bits
  uint16_t picked[32];
};

// The choice in 32 bits with up to eight experts a lane.  The lowest three bits of a key give way to the expert's
// place in the lane (lower places larger), so a lane's keys sort with two instructions a comparator and the number
// comes with the key; lanes compare with those bits set.  That moves a score by less than 2^-20 of itself.  For
// scores of 16 bits that no bias or sum has touched the bits carry nothing, and the choice is exact.
//
// A round finds the largest top card; its lane notes it and turns over the next one.  Selections, comparisons and
// logic run at half the rate of other instructions and are what many tokens wait for, so the cards lie in shared memory
// (a round of 65536 tokens took 3.7 us with the keys shifted in registers, 2.7 so).
//
// Where neighbours of the choice are close, the choices and the runner-up are ranked again by 64-bit scores, a lane
// each: enough unless something behind the runner-up is close to it as well and is not its equal in logit and bias (or is,
// and the runner-up passes more than one choice), or the scores need the whole row's sum.  Returns whether the choice has to be repeated over all experts.
template <typename T, int NE>
__device__ __forceinline__ bool choose_quick(const RouteParams& p, int64_t t, const float (&s)[NE], float tau, bool exact,
                                             const float (&l)[NE], const float (&bias)[NE], Deck<NE>& deck, int* pick) {
  const RouteArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  uint32_t key[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) key[j] = (key_of(s[j]) | 7u) ^ static_cast<uint32_t>(j);
  sort_lane<NE>(key);
  bool again = false, kept = true;
  if (a.top_groups < a.groups) {                   // p.lanes neighbouring lanes a group
    uint32_t b1 = key[0] | 7u, b2 = NE > 1 ? key[NE > 1 ? 1 : 0] | 7u : 0u;
    for (int o = 1; o < p.lanes; o <<= 1) {
      const uint32_t o1 = __shfl_xor_sync(kAll, b1, o), o2 = __shfl_xor_sync(kAll, b2, o);
      b2 = larger(smaller(b1, o1), larger(b2, o2));
      b1 = larger(b1, o1);
    }
    const int group = lane >> (__ffs(p.lanes) - 1);
    const float v1 = value_of(b1), v2 = a.top2 ? value_of(b2) : 0.f;
    const uint32_t mine = a.top2 ? key_of(v1 + v2) : b1;
    const bool real = group < a.groups;
    const int rank = group_rank(a.groups, p.lanes, group, mine);     // by the whole warp
    kept = real && rank < a.top_groups;
    if (!exact) {
      // Parts: half a unit of rounding, up to seven upwards by the keys; half a unit more for the sum.
      const float size = fabsf(v1) + fabsf(v2), score = value_of(mine), any = tau + 0x1p-140f;
      const float low = value_of(~warp_max(kept ? ~key_of(least_score(score, size, any, 0x1.4p-20f)) : 0u));
      const float high = value_of(warp_max(real && !kept ? key_of(largest_score(score, size, any, 0x1p-22f)) : 0u));
      again = !(low > high);
    }
    if (a.top2 && a.bias == nullptr) {             // the groups by their sums, the experts by their logits
#pragma unroll
      for (int j = 0; j < NE; ++j) key[j] = (key_of(l[j]) | 7u) ^ static_cast<uint32_t>(j);
      sort_lane<NE>(key);
    }
  }
#pragma unroll
  for (int j = 1; j < NE; ++j) deck.key[j][lane] = key[j];
  const uint32_t* card = &deck.key[kept ? 0 : NE][lane];
  uint32_t top = kept ? key[0] : 0u;
  const unsigned below_me = (1u << lane) - 1u;
  const int rounds = a.top_k + (exact ? 0 : 1);
  for (int i = 0; i < rounds; ++i) {
    const uint32_t best = top | 7u, m = warp_max(best);
    const bool same = best == m;
    const unsigned holders = __ballot_sync(kAll, same);
    if (same && !(holders & below_me)) {
      deck.won[i] = make_uint2(m, (top & 7u) | static_cast<uint32_t>(lane << 3));
      card += 32;
      top = *card;                                 // its own column: no other lane writes there
    }
  }
  __syncwarp();
  const uint2 won = deck.won[lane];
  // A runner-up can be missing, or be a place behind the last expert.
  const int number = static_cast<int>(won.y >> 3) * NE + static_cast<int>(~won.y & 7u);
  const bool there = lane < rounds && won.x > 7u && number < a.experts;
  *pick = there ? number : -1;
  if (exact) return false;
  if (a.bias == nullptr) tau = 0.f;                          // ranked by logits
  // Scores nearer than this may stand the other way round.  (Keys lose up to seven units, all in one direction.)
  const auto reach = [&](float score) { return tau + 0x1.4p-20f * fabsf(score) + 0x1p-140f; };
  const uint32_t below = __shfl_down_sync(kAll, won.x, 1);
  const float score = value_of(won.x);
  const bool close = lane < a.top_k && below > 7u && !(score - value_of(below) > reach(score));
  const unsigned pairs = __ballot_sync(kAll, close);
  if (again || pairs == 0) return again;

  float le = 0.f, be = 0.f;
  if (there) {
    le = clean(to_f32<T>(static_cast<const T*>(a.logits)[t * a.ld + *pick]));
    be = a.bias ? clean(a.bias[*pick]) : 0.f;
  }
  const uint32_t next = warp_max(top | 7u);
  const float edge = value_of(__shfl_sync(kAll, won.x, a.top_k));
  const bool more = (pairs >> (a.top_k - 1)) & 1u && next > 7u && !(edge - value_of(next) > reach(edge));
  if (more) {
    // Something behind the runner-up is close to it.  Only its equals may be: all that reaches it and is not its
    // equal has to be among the choices.
    const float lr = __shfl_sync(kAll, le, a.top_k), br = __shfl_sync(kAll, be, a.top_k);
    int others = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      const float v = a.bias ? s[j] : l[j];
      others += __popc(__ballot_sync(kAll, kept && !(edge - v > 2.f * reach(edge)) && !(l[j] == lr && (!a.bias || bias[j] == br))));
    }
    const unsigned chosen = __ballot_sync(kAll, lane < a.top_k && !(le == lr && be == br));
    if (others != __popc(chosen)) return true;
  }
  if (a.bias != nullptr && !a.sigmoid) {           // 64-bit scores need the row's sum, but equals need none
    const float l1 = __shfl_down_sync(kAll, le, 1), b1 = __shfl_down_sync(kAll, be, 1);
    return __any_sync(kAll, close && !(le == l1 && be == b1));
  }
  double wide = a.bias == nullptr ? static_cast<double>(le) : 1.0 / (1.0 + exp(-static_cast<double>(le))) + static_cast<double>(be);
  if (le == -INFINITY || be == -INFINITY || !there) wide = -INFINITY;
  int rank = 0;
  for (int i = 0; i < rounds; ++i) {
    const double other = __shfl_sync(kAll, wide, i);
    const int e = __shfl_sync(kAll, *pick, i);
    if (e >= 0) rank += other > wide || (other == wide && e < *pick) ? 1 : 0;
  }
  // A runner-up that passes more than one choice would take its equals along.
  if (more && __shfl_sync(kAll, rank, a.top_k) < a.top_k - 1) return true;
  if (there) deck.picked[rank] = static_cast<uint16_t>(*pick);
  __syncwarp();
  if (there) *pick = deck.picked[lane];
  return false;
}

// Choice of one token by scores s[NE]; without a bias they rank the groups and the logits rank the experts.  Lane
// i < top_k gets the i-th expert in *pick (with `check` lane top_k the runner-up).  Returns whether two scores that decide
// something differ by no more than tau (+ 2^-21 of their size): bit 0 in lane i for choices i and i + 1, bit 1 for
// the groups.
template <typename F, int NE>
__device__ __forceinline__ int choose(const RouteParams& p, const F (&s)[NE], float tau, bool check, const float (&l)[NE],
                                       uint16_t* picked, int* pick) {
  using Key = decltype(key_of(F()));
  const RouteArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  Key key[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) key[j] = key_of(s[j]);
  int close = 0;
  const bool grouped = a.top_groups < a.groups;
  const bool by_logit = a.bias == nullptr && a.top2 && grouped;   // s is not the logits here

  if (grouped) {
    const int size = a.experts / a.groups;
    Key mine = 0;                                  // the score of group `group`
    F size_of = 0;                                 // and the sizes of its parts together
    int group = lane;
    if (p.lanes) {
      // A group is p.lanes neighbouring lanes.
      Key b1 = 0, b2 = 0;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        b2 = larger(b2, smaller(b1, key[j]));
        b1 = larger(b1, key[j]);
      }
      for (int o = 1; o < p.lanes; o <<= 1) {
        const Key o1 = __shfl_xor_sync(kAll, b1, o), o2 = __shfl_xor_sync(kAll, b2, o);
        b2 = larger(smaller(b1, o1), larger(b2, o2));
        b1 = larger(b1, o1);
      }
      group = lane / p.lanes;
      const F v1 = value_of(b1), v2 = a.top2 ? value_of(b2) : F(0);
      mine = a.top2 ? key_of(v1 + v2) : b1;
      size_of = fabs(v1) + fabs(v2);
    } else {
      for (int g = 0; g < a.groups; ++g) {
        Key b1 = 0, b2 = 0;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          const int e = lane * NE + j - g * size;
          if (e >= 0 && e < size) {
            b2 = larger(b2, smaller(b1, key[j]));
            b1 = larger(b1, key[j]);
          }
        }
        const Key m1 = warp_max(b1);
        Key score = m1;
        F v2 = 0;
        if (a.top2) {
          const int owner = __ffs(__ballot_sync(kAll, b1 == m1)) - 1;
          v2 = value_of(warp_max(lane == owner ? b2 : b1));
          score = key_of(value_of(m1) + v2);
        }
        if (lane == g) {
          mine = score;
          size_of = fabs(value_of(m1)) + fabs(v2);
        }
      }
    }
    const int rank = group_rank(a.groups, p.lanes ? p.lanes : 1, group, mine);
    const bool kept = group < a.groups && rank < a.top_groups;
    if (check) {
      const float score = static_cast<float>(value_of(mine)), size = static_cast<float>(size_of);
      const float low = value_of(~warp_max(kept ? ~key_of(least_score(score, size, tau, 0x1p-22f)) : 0u));
      const float high = value_of(warp_max(group < a.groups && !kept ? key_of(largest_score(score, size, tau, 0x1p-22f)) : 0u));
      if (!(low > high)) close = 2;
    }
    if (p.lanes) {
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (!kept) key[j] = 0;
    } else {
      const unsigned keep = __ballot_sync(kAll, kept);
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (!((keep >> ((lane * NE + j) / size & 31)) & 1u)) key[j] = 0;
    }
    if (by_logit) {
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (key[j] != 0) key[j] = key_of(static_cast<F>(l[j]));
    }
  }
  check = check && a.bias != nullptr;

  Key best = 0;
#pragma unroll
  for (int j = 0; j < NE; ++j) best = larger(best, key[j]);
  Key won = 0;                                     // lane i: the key of choice i
  const int rounds = a.top_k + (check ? 1 : 0);
  for (int i = 0; i < rounds; ++i) {
    const Key m = warp_max(best);
    if (lane == i) won = m;
    if (lane == __ffs(__ballot_sync(kAll, best == m)) - 1) {
      int at = 0;
#pragma unroll
      for (int j = NE - 1; j >= 0; --j)
        if (key[j] == m) at = j;
      picked[i] = static_cast<uint16_t>(lane * NE + at);
      best = 0;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        if (j == at) key[j] = 0;
        best = larger(best, key[j]);
      }
    }
  }
  __syncwarp();
  *pick = lane < rounds ? static_cast<int>(picked[lane]) : -1;
  if (check) {
    const Key below = __shfl_down_sync(kAll, won, 1);
    if (lane < a.top_k && below != 0) {            // no runner-up: nothing to compare
      const float score = static_cast<float>(value_of(won));
      if (!(score - static_cast<float>(value_of(below)) > tau + 0x1p-21f * fabsf(score))) close |= 1;
    }
  }
  return close;
}

// Calls f with copies: arrays whose address is taken live in memory, and these are needed in registers.
template <int NE, class F>
__device__ __forceinline__ int out_of_line(const float (&x)[NE], const float (&y)[NE], F f) {
  float a[NE], b[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    a[j] = x[j];
    b[j] = y[j];
  }
  return f(a, b);
}

// choose() out of line: groups that do not fall into whole lanes are rare, and should not cost the others registers.
template <int NE>
__device__ __noinline__ int choose_ragged(const RouteParams& p, const float (&s)[NE], float tau, bool check, const float (&l)[NE],
                                          uint16_t* picked, int* pick) {
  return choose<float, NE>(p, s, tau, check, l, picked, pick);
}

// The same choice from scores in 64 bits.
template <int NE>
__device__ __noinline__ int choose_wide(const RouteParams& p, const float (&l)[NE], const float (&bias)[NE], uint16_t* picked) {
  const RouteArgs& a = p.a;
  int pick;
  double s[NE], total = 0;
  if (a.bias == nullptr && !(a.top2 && a.top_groups < a.groups)) {
#pragma unroll
    for (int j = 0; j < NE; ++j) s[j] = static_cast<double>(l[j]);
    choose<double, NE>(p, s, 0.f, false, l, picked, &pick);
    return pick;
  }
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NE; ++j) top = fmaxf(top, l[j]);
  top = warp_max(top);
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const double v = static_cast<double>(l[j]);
    s[j] = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : (l[j] == -INFINITY ? 0.0 : exp(v - static_cast<double>(top)));
    total += s[j];
  }
  if (!a.sigmoid) total = warp_sum(total);
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    if (!a.sigmoid && total > 0) s[j] /= total;
    s[j] = l[j] == -INFINITY || bias[j] == -INFINITY ? -INFINITY : s[j] + static_cast<double>(bias[j]);
  }
  choose<double, NE>(p, s, 0.f, false, l, picked, &pick);
  return pick;
}

// A lane's share of a row as it lies in memory.
constexpr bool power_of_two(int n) { return (n & (n - 1)) == 0; }
template <typename T, int NE>
struct alignas(!power_of_two(NE) ? sizeof(T) : NE * sizeof(T) > 16 ? 16 : NE * sizeof(T)) Share { T v[NE]; };

// Lanes and places beyond the last expert hold minus infinity: they have the highest numbers, so among equals every
// expert comes before them, and there are always enough experts.
template <typename T> __device__ __forceinline__ T lowest_value() { return from_f32<T>(-INFINITY); }
template <typename T, int NE> __device__ __forceinline__ Share<T, NE> empty_share() {
  Share<T, NE> r;
#pragma unroll
  for (int j = 0; j < NE; ++j) r.v[j] = lowest_value<T>();
  return r;
}
template <typename T, int NE>
__device__ __forceinline__ void load_share(const RouteParams& p, int64_t t, Share<T, NE>* to) {
  const RouteArgs& a = p.a;
  const T* row = static_cast<const T*>(a.logits) + t * a.ld;
  const int e0 = (threadIdx.x & 31) * NE;
  if (p.vec) {
    if (e0 < a.experts) *to = *reinterpret_cast<const Share<T, NE>*>(row + e0);
  } else {
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (e0 + j < a.experts) to->v[j] = row[e0 + j];
  }
}
// Cleaned logits.  Products with zero show whether there is anything to clean, at a fifth of the cost of cleaning.
// Returns whether this lane had an infinity or a NaN.
template <typename T, int NE>
__device__ __forceinline__ bool clean_share(const Share<T, NE>& from, float (&l)[NE]) {
  float odd = 0.f;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    l[j] = to_f32<T>(from.v[j]) + 0.f;
    odd = fmaf(l[j], 0.f, odd);
  }
  if (odd != 0.f) {                                // a NaN: from a NaN or an infinity
#pragma unroll
    for (int j = 0; j < NE; ++j) l[j] = clean(l[j]);
    return true;
  }
  return false;
}

// Shares of the choices among themselves, sum 1 (0 where every chosen logit is -infinity).  Scaled by the
// largest so that it holds where the scores themselves would underflow: softmax(l) over the choices, or
// sigmoid(l) / exp(m) with m = min(0, max l).
__device__ __forceinline__ float share_size(bool sigmoid_scores, float l, float top) {
  if (l == -INFINITY) return 0.f;
  if (!sigmoid_scores) return expf(l - top);
  const float e = expf(-fabsf(l));
  const float up = l > 0.f ? 1.f : top > 0.f ? e : expf(l - top);
  return __fdividef(up, 1.f + e);                  // 2 ulp, of a divisor between 1 and 2
}
__device__ __forceinline__ float share(const RouteArgs& a, float l) {
  if (static_cast<int>(threadIdx.x & 31) >= a.top_k) l = -INFINITY;
  float top = 1.f;                                 // for a sigmoid all that counts is whether one is positive
  if (!a.sigmoid || !__any_sync(kAll, l > 0.f)) top = warp_max(l);
  if (top == -INFINITY) return 0.f;
  const float q = share_size(a.sigmoid, l, top);
  return __fdividef(q, warp_sum(q));               // 2 ulp; the sum lies between 1/2 and top_k
}

// ---- rows in expert order --------------------------------------------------------------------------------------
// Exclusive sums of value[0 .. n - 1] in place (n <= kMaxExperts), the total in `part[32]`, by the whole block.
__device__ __forceinline__ void block_scan(int32_t* value, int n, int32_t* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int run = 0;
  for (int e0 = 0; e0 < n; e0 += static_cast<int>(blockDim.x)) {
    const int e = e0 + static_cast<int>(threadIdx.x);
    const int mine = e < n ? value[e] : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kAll, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      const int own = lane < warps ? part[lane] : 0;
      int all = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kAll, all, o);
        if (lane >= o) all += v;
      }
      part[lane] = all - own;
      if (lane == 31) part[32] = all;
    }
    __syncthreads();
    if (e < n) value[e] = run + part[warp] + sum - mine;
    run += part[32];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[32] = run;
  __syncthreads();
}

// Shared memory of a block: marks [experts][words], marks ahead of each word [experts][words], choices
// [tokens_per_block][top_k].
struct BlockRows {
  uint32_t* bits;
  uint16_t* ahead;
  uint16_t* chosen;
  __device__ BlockRows(const RouteParams& p, uint32_t* smem) {
    const int n = p.a.experts * p.words;
    bits = smem;
    ahead = reinterpret_cast<uint16_t*>(bits + n);
    chosen = ahead + (n + 1) / 2 * 2;
  }
  __device__ void clear(const RouteParams& p) const {
    for (int i = threadIdx.x; i < p.a.experts * p.words; i += blockDim.x) bits[i] = 0;
  }
  __device__ void mark(const RouteParams& p, int token, int e) const {
    atomicOr(bits + e * p.words + (token >> 5), 1u << (token & 31));
  }
};

// Counts and ranks of the block's marked choices.  With one block the rows are final; otherwise the counts go to
// the second kernel, and the rows start at zero for every expert.
__device__ __forceinline__ void finish_block(const RouteParams& p, const BlockRows& b, int first, int count) {
  __shared__ int32_t base[kMaxExperts];
  __shared__ int32_t part[33];
  const RouteArgs& a = p.a;
  const bool alone = gridDim.x == 1;
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    int n = 0;
    for (int w = 0; w < p.words; ++w) {
      b.ahead[e * p.words + w] = static_cast<uint16_t>(n);
      n += __popc(b.bits[e * p.words + w]);
    }
    if (!alone) p.counts[static_cast<int64_t>(blockIdx.x) * p.pitch + e] = static_cast<uint16_t>(n);
    base[e] = alone ? n : 0;
  }
  if (!alone && a.experts + static_cast<int>(threadIdx.x) < p.pitch)
    p.counts[static_cast<int64_t>(blockIdx.x) * p.pitch + a.experts + threadIdx.x] = 0;
  __syncthreads();
  if (alone) {
    block_scan(base, a.experts, part);
    for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) a.offsets[e] = e < a.experts ? base[e] : part[32];
  }
  for (int i = threadIdx.x; i < count * a.top_k; i += blockDim.x) {
    const int e = b.chosen[i], tok = a.top_k == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), p.per_choice));
    int row = -1;
    if (e != 0xffff) {
      const int at = e * p.words + (tok >> 5);
      row = base[e] + b.ahead[at] + __popc(b.bits[at] & ((1u << (tok & 31)) - 1u));
    }
    a.rows[first * a.top_k + i] = row;
  }
}

template <typename T, int NE, int kMost>
__global__ void __launch_bounds__(kMost, 1) route_warp_kernel(const RouteParams p) {
  extern __shared__ __align__(16) uint32_t smem[];
  const RouteArgs& a = p.a;
  const BlockRows mine(p, smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int first = blockIdx.x * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  Deck<NE>& deck = reinterpret_cast<Deck<NE>*>(smem + p.block_words)[warp];
  uint16_t* const picked = deck.picked;
  asm volatile("griddepcontrol.launch_dependents;");

  Share<T, NE> next = empty_share<T, NE>();
  if (warp < count) load_share<T, NE>(p, first + warp, &next);
  float bias[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) bias[j] = a.bias ? clean(a.bias[min(lane * NE + j, a.experts - 1)]) : 0.f;
  mine.clear(p);
  if constexpr (Deck<NE>::kKeys > 0) deck.key[NE][lane] = deck.key[NE + 1][lane] = 0;
  const bool grouped_sum = a.top2 && a.top_groups < a.groups;
  const bool scored = a.bias != nullptr || grouped_sum;              // the order needs the scores
  __syncthreads();

  for (int i = warp; i < count; i += warps) {
    const int64_t t = first + i;
    const Share<T, NE> raw = next;
    if (i + warps < count) load_share<T, NE>(p, t + warps, &next);
    int e = -1;
    float w = 0.f;
    if (a.mask == nullptr || a.mask[t]) {
      float l[NE], s[NE];
      const bool odd = clean_share<T, NE>(raw, l);
      float top = 0.f, total = 1.f, tau = 0.f;
      if (!a.sigmoid && (scored || !a.renormalise)) {
        top = l[0];
#pragma unroll
        for (int j = 1; j < NE; ++j) top = fmaxf(top, l[j]);
        top = warp_max(top);
        if (top == -INFINITY) top = 0.f;                             // nothing is left: every exponential is zero
        total = 0.f;
        if (a.renormalise) {
#pragma unroll
          for (int j = 0; j < NE; ++j) total += s[j] = quick_exp(l[j] - top);
        } else {
          // The weights are made of these: to the full 2^-22.
#pragma unroll
          for (int j = 0; j < NE; ++j) total += s[j] = expf(l[j] - top);
        }
        total = warp_sum(total);
      }
      if (scored) {
        const float inv = total > 0.f ? 1.f / total : 0.f;
        if (a.sigmoid) {
#pragma unroll
          for (int j = 0; j < NE; ++j) s[j] = quick_sigmoid(l[j]) + bias[j];
        } else {
#pragma unroll
          for (int j = 0; j < NE; ++j) s[j] = fmaf(s[j], inv, bias[j]);
        }
        if (odd) {                                                   // no bias brings back an expert that is out
#pragma unroll
          for (int j = 0; j < NE; ++j) s[j] = l[j] == -INFINITY ? -INFINITY : s[j];
        }
        tau = score_error(a.sigmoid, NE, inv);
      } else {
#pragma unroll
        for (int j = 0; j < NE; ++j) s[j] = l[j];
      }
      int pick;
      bool again;
      if constexpr (NE <= 8) {
        if (a.top_groups == a.groups || p.lanes) {
          again = choose_quick<T, NE>(p, t, s, tau, sizeof(T) == 2 && !scored, l, bias, deck, &pick);
        } else {
          int p1;
          const int close = out_of_line(s, l, [&](const float (&s1)[NE], const float (&l1)[NE]) {
            return choose_ragged<NE>(p, s1, tau, scored, l1, picked, &p1);
          });
          pick = p1;
          again = __any_sync(kAll, close) && !truly_tied<T>(p, t, close, pick);
        }
      } else {
        const int close = choose<float, NE>(p, s, tau, scored, l, picked, &pick);
        again = __any_sync(kAll, close) && !truly_tied<T>(p, t, close, pick);
      }
      if (again)
        pick = out_of_line(l, bias, [&](const float (&l1)[NE], const float (&b1)[NE]) { return choose_wide<NE>(p, l1, b1, picked); });
      e = lane < a.top_k ? pick : -1;
      const float le = e >= 0 ? clean(to_f32<T>(static_cast<const T*>(a.logits)[t * a.ld + e])) : -INFINITY;
      if (a.renormalise) w = share(a, le);
      else if (a.sigmoid) w = sigmoid(le);
      else w = le == -INFINITY ? 0.f : expf(le - top) / total;
      w *= a.scale;
      __syncwarp();                                                  // the deck is read
    }
    if (lane < a.top_k) {
      const int at = (first + i) * a.top_k + lane;
      a.idx[at] = e;
      a.weights[at] = w;
      mine.chosen[i * a.top_k + lane] = static_cast<uint16_t>(e);      // 0xffff: none
      if (e >= 0) mine.mark(p, i, e);
    }
  }
  __syncthreads();
  finish_block(p, mine, first, count);
}

// ---- a thread per token ----------------------------------------------------------------------------------------
// choose() by one thread over all experts; numbers go to picked[0 .. top_k - 1].  Returns whether the choice has to be
// repeated in 64 bits.
template <typename T, typename F, int NE>
__device__ __forceinline__ bool choose_alone(const RouteParams& p, const T* row, const F (&s)[NE], float tau, bool check,
                                             const float (&l)[NE], uint16_t* picked) {
  using Key = decltype(key_of(F()));
  const RouteArgs& a = p.a;
  Key key[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) key[j] = j < a.experts ? key_of(s[j]) : Key(0);
  bool close = false;
  if (NE <= kThreadExperts && a.top_groups < a.groups) {
    const int size = a.experts / a.groups;
    Key score[NE];                                 // of the group of each expert
    F size_of[NE];                                 // and the sizes of its parts together
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      Key b1 = 0, b2 = 0;
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (i / size == j / size) {
          b2 = larger(b2, smaller(b1, key[i]));
          b1 = larger(b1, key[i]);
        }
      const F v1 = value_of(b1), v2 = a.top2 ? value_of(b2) : F(0);
      score[j] = a.top2 ? key_of(v1 + v2) : b1;
      size_of[j] = fabs(v1) + fabs(v2);
    }
    float low = INFINITY, high = -INFINITY;
    unsigned keep = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      if (j >= a.experts) continue;
      int rank = 0;
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (i < a.experts && i % size == 0) rank += score[i] > score[j] || (score[i] == score[j] && i / size < j / size) ? 1 : 0;
      const float v = static_cast<float>(value_of(score[j])), size = static_cast<float>(size_of[j]);
      if (rank < a.top_groups) {
        keep |= 1u << j;
        low = fminf(low, least_score(v, size, tau, 0x1p-22f));
      } else {
        high = fmaxf(high, largest_score(v, size, tau, 0x1p-22f));
      }
    }
    close = check && !(low > high);
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      if (!((keep >> j) & 1u)) key[j] = 0;
      else if (a.bias == nullptr) key[j] = key_of(static_cast<F>(l[j]));
    }
  }
  check = check && a.bias != nullptr;
  const int rounds = a.top_k + (check ? 1 : 0);
  Key before = 0;
  float l0 = 0.f, b0 = 0.f;
  for (int i = 0; i < rounds; ++i) {
    Key best = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (key[j] > best) {
        best = key[j];
        at = j;
      }
    if (best == 0) break;                          // only the runner-up can be missing
    if (check) {
      const float l1 = clean(to_f32<T>(row[at])), b1 = clean(a.bias[at]);
      const float a0 = static_cast<float>(value_of(before));
      const bool tied = l0 == l1 && b0 == b1;
      if (i > 0 && !tied) close |= !(a0 - static_cast<float>(value_of(best)) > tau + 0x1p-21f * fabsf(a0));
      if (i > 0 && i == a.top_k && tied) {         // what stands behind the runner-up must not be close, but for its equals
#pragma unroll
        for (int j = 0; j < NE; ++j)
          if (key[j] != 0 && !(a0 - static_cast<float>(value_of(key[j])) > tau + 0x1p-21f * fabsf(a0)))
            close |= !(l[j] == l1 && clean(a.bias[min(j, a.experts - 1)]) == b1);
      }
      l0 = l1;
      b0 = b1;
    }
    if (i < a.top_k) picked[i] = static_cast<uint16_t>(at);
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (j == at) key[j] = 0;
    before = best;
  }
  return close;
}
template <typename T, int NE>
__device__ __noinline__ void choose_alone_wide(const RouteParams& p, const T* row, const float (&l)[NE], const float (&bias)[NE], uint16_t* picked) {
  const RouteArgs& a = p.a;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NE; ++j) top = fmaxf(top, l[j]);
  double s[NE], total = 0;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const double v = static_cast<double>(l[j]);
    s[j] = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : (l[j] == -INFINITY ? 0.0 : exp(v - static_cast<double>(top)));
    total += s[j];
  }
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    if (!a.sigmoid && total > 0) s[j] /= total;
    s[j] = l[j] == -INFINITY || bias[j] == -INFINITY ? -INFINITY : s[j] + static_cast<double>(bias[j]);
  }
  choose_alone<T, double, NE>(p, row, s, 0.f, false, l, picked);
}

template <typename T, int NE>
__device__ __forceinline__ void load_token(const RouteParams& p, int64_t t, float (&l)[NE]) {
  constexpr int kPiece = NE * sizeof(T) < 16 ? NE : 16 / static_cast<int>(sizeof(T));
  const RouteArgs& a = p.a;
  const T* row = static_cast<const T*>(a.logits) + t * a.ld;
  if (p.vec) {                                     // whole pieces, as many as there are experts
#pragma unroll
    for (int i = 0; i < NE; i += kPiece) {
      Share<T, kPiece> raw = empty_share<T, kPiece>();
      if (i < a.experts) raw = *reinterpret_cast<const Share<T, kPiece>*>(row + i);
#pragma unroll
      for (int j = 0; j < kPiece; ++j) l[i + j] = clean(to_f32<T>(raw.v[j]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < NE; ++j) l[j] = j < a.experts ? clean(to_f32<T>(row[j])) : -INFINITY;
  }
}

template <typename T, int NE>
__global__ void __launch_bounds__(NE <= 8 ? kMostThreads : 256, 1) route_thread_kernel(const RouteParams p) {
  extern __shared__ __align__(16) uint32_t smem[];
  const RouteArgs& a = p.a;
  const BlockRows mine(p, smem);
  const int first = blockIdx.x * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  asm volatile("griddepcontrol.launch_dependents;");
  mine.clear(p);
  const bool scored = NE <= kThreadExperts && (a.bias != nullptr || (a.top2 && a.top_groups < a.groups));
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const int64_t t = first + i;
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    uint16_t* const picked = mine.chosen + i * a.top_k;
    const bool live = a.mask == nullptr || a.mask[t];
    float top = 0.f, total = 1.f;
    if (live) {
      float l[NE], s[NE], bias[NE];
      load_token<T, NE>(p, t, l);
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        bias[j] = NE <= kThreadExperts && a.bias ? clean(a.bias[min(j, a.experts - 1)]) : 0.f;
        s[j] = l[j];
      }
      if (!a.sigmoid && (scored || !a.renormalise)) {
        top = l[0];
#pragma unroll
        for (int j = 1; j < NE; ++j) top = fmaxf(top, l[j]);
        total = 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          s[j] = l[j] == -INFINITY ? 0.f : expf(l[j] - top);
          total += s[j];
        }
      }
      if (NE <= kThreadExperts && scored) {
        const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          const float prob = a.sigmoid ? quick_sigmoid(l[j]) : s[j] * inv;
          s[j] = l[j] == -INFINITY ? -INFINITY : prob + bias[j];
        }
        if (choose_alone<T, float, NE>(p, row, s, score_error(a.sigmoid, NE, inv), true, l, picked))
          out_of_line(l, bias, [&](const float (&l1)[NE], const float (&b1)[NE]) {
            choose_alone_wide<T, NE>(p, row, l1, b1, picked);
            return 0;
          });
      } else {
        choose_alone<T, float, NE>(p, row, l, 0.f, false, l, picked);
      }
    }
    float best = -INFINITY, sum = 0.f;
    if (live && a.renormalise) {
      for (int k = 0; k < a.top_k; ++k) best = fmaxf(best, clean(to_f32<T>(row[picked[k]])));
      for (int k = 0; k < a.top_k; ++k) sum += share_size(a.sigmoid, clean(to_f32<T>(row[picked[k]])), best);
    }
    for (int k = 0; k < a.top_k; ++k) {
      int e = -1;
      float w = 0.f;
      if (live) {
        e = picked[k];
        const float le = clean(to_f32<T>(row[e]));
        if (a.renormalise) w = sum > 0.f ? share_size(a.sigmoid, le, best) / sum : 0.f;
        else if (a.sigmoid) w = sigmoid(le);
        else w = le == -INFINITY ? 0.f : expf(le - top) / total;
        w *= a.scale;
        mine.mark(p, i, e);
      } else {
        picked[k] = 0xffff;
      }
      a.idx[t * a.top_k + k] = e;
      a.weights[t * a.top_k + k] = w;
    }
  }
  __syncthreads();
  finish_block(p, mine, first, count);
}

// Adds to every choice the rows of earlier experts and of earlier blocks of its own expert.  A thread sums four
// neighbouring experts over a strip of the blocks, all its loads under way at once; whole numbers, so the order of the
// additions is free.
__global__ void __launch_bounds__(kMostThreads, 1) route_rows_kernel(const RouteParams p) {
  constexpr int kAtOnce = 10;                      // 148 blocks of 256 experts: 16 strips of 10
  const RouteArgs& a = p.a;
  __shared__ int32_t before[kMaxExperts], total[kMaxExperts], part[33];
  const int quads = p.pitch / 4, me = static_cast<int>(blockIdx.x), blocks = static_cast<int>(gridDim.x);
  for (int e = threadIdx.x; e < p.pitch; e += blockDim.x) before[e] = total[e] = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int width = 1;                                   // threads abreast: a power of two
  while (width < quads) width <<= 1;
  const int strips = static_cast<int>(blockDim.x) / width, strip = threadIdx.x / width, col = threadIdx.x % width;
  const uint2* counts = reinterpret_cast<const uint2*>(p.counts) + min(col, quads - 1);
  int b[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
  for (int b0 = strip; b0 < blocks; b0 += kAtOnce * strips) {
    uint2 c[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) c[u] = counts[static_cast<int64_t>(min(b0 + u * strips, blocks - 1)) * quads];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int at = b0 + u * strips;
      if (at >= blocks) break;
      const int n[4] = {static_cast<int>(c[u].x & 0xffffu), static_cast<int>(c[u].x >> 16),
                        static_cast<int>(c[u].y & 0xffffu), static_cast<int>(c[u].y >> 16)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[i] += n[i];
        b[i] += at < me ? n[i] : 0;
      }
    }
  }
  for (int o = width; o < 32; o <<= 1)             // lanes of the same column
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[i] += __shfl_xor_sync(kAll, b[i], o);
      t[i] += __shfl_xor_sync(kAll, t[i], o);
    }
  if (col < quads && (threadIdx.x & 31) < static_cast<unsigned>(width))
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      atomicAdd(before + 4 * col + i, b[i]);
      atomicAdd(total + 4 * col + i, t[i]);
    }
  __syncthreads();
  block_scan(total, a.experts, part);
  if (me == 0)
    for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) a.offsets[e] = e < a.experts ? total[e] : part[32];
  const int first = me * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  for (int i = threadIdx.x; i < count * a.top_k; i += blockDim.x) {
    const int at = first * a.top_k + i;
    const int e = a.idx[at];
    if (e >= 0) a.rows[at] += before[e] + total[e];
  }
}

// ---- gradient --------------------------------------------------------------------------------------------------
// dl from dw, idx constant.  With c = scale and a_k the shares of the choices (renormalised):
//   softmax  dl_k = c a_k (g_k - <g, a>)                 sigmoid  the same times (1 - p_k)
// else softmax  dl_e = c p_e (g_e - <g, p>)              sigmoid  dl_k = c g_k p_k (1 - p_k).
// All but the third leave the experts that were not chosen at zero: a row of zeros is stored and the choices over it.
template <typename T, int NE>
__global__ void __launch_bounds__(256) route_warp_backward_kernel(const RouteParams p) {
  const RouteArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
  const bool whole = !a.renormalise && !a.sigmoid;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); t < a.tokens; t += warps) {
    int e = lane < a.top_k ? a.idx[t * a.top_k + lane] : -1;
    if (e >= a.experts) e = -1;
    const float g = e >= 0 ? p.dweights[t * a.top_k + lane] : 0.f;
    const float le = e >= 0 ? clean(to_f32<T>(static_cast<const T*>(a.logits)[t * a.ld + e])) : -INFINITY;
    T* row = static_cast<T*>(p.dlogits) + t * a.experts;
    if (!whole) {
      const Share<T, NE> zero{};
      const int e0 = lane * NE;
      if (p.vec) {
        if (e0 < a.experts) *reinterpret_cast<Share<T, NE>*>(row + e0) = zero;
      } else {
        for (int j = lane; j < a.experts; j += 32) row[j] = from_f32<T>(0.f);
      }
      float d;
      if (a.renormalise) {
        const float q = share(a, le);
        d = a.scale * q * (g - warp_sum(g * q));
        if (a.sigmoid) d *= sigmoid(-le);
      } else {
        d = a.scale * g * sigmoid(le) * sigmoid(-le);
      }
      __syncwarp();                                // the zeros come first
      if (e >= 0 && le != -INFINITY) row[e] = from_f32<T>(d);
      continue;
    }
    Share<T, NE> raw = empty_share<T, NE>();
    load_share<T, NE>(p, t, &raw);
    float l[NE];
    clean_share<T, NE>(raw, l);
    float top = l[0], total = 0.f;
#pragma unroll
    for (int j = 1; j < NE; ++j) top = fmaxf(top, l[j]);
    top = warp_max(top);
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      l[j] = l[j] == -INFINITY ? 0.f : expf(l[j] - top);
      total += l[j];
    }
    total = warp_sum(total);
    const float inv = total > 0.f ? 1.f / total : 0.f;
    const float prob = le == -INFINITY ? 0.f : expf(le - top) * inv;
    const float rest = warp_sum(g * prob);
    const bool any = __any_sync(kAll, e >= 0);     // a masked token has no gradient
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      l[j] = any ? -a.scale * l[j] * inv * rest : 0.f;
      raw.v[j] = from_f32<T>(l[j]);
    }
    if (p.vec) {
      if (lane * NE < a.experts) *reinterpret_cast<Share<T, NE>*>(row + lane * NE) = raw;
    } else {
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (lane * NE + j < a.experts) row[lane * NE + j] = raw.v[j];
    }
    __syncwarp();
    if (e >= 0) row[e] = from_f32<T>(a.scale * prob * (g - rest));
  }
}

template <typename T, int NE>
__global__ void __launch_bounds__(128) route_thread_backward_kernel(const RouteParams p) {
  const RouteArgs& a = p.a;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (t >= a.tokens) return;
  const int32_t* idx = a.idx + t * a.top_k;
  const float* g = p.dweights + t * a.top_k;
  float l[NE], d[NE];
  load_token<T, NE>(p, t, l);
  unsigned picked = 0;                             // experts that were chosen
#pragma unroll
  for (int j = 0; j < NE; ++j) d[j] = 0.f;
  for (int k = 0; k < a.top_k; ++k) {
    const int e = idx[k];
    const float gk = g[k];
    if (e < 0 || e >= a.experts) continue;
    picked |= 1u << e;
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (j == e) d[j] = gk;                       // g by expert
  }
  const bool whole = !a.renormalise && !a.sigmoid;
  if (a.renormalise || whole) {
    // Shares of the choices (or, whole, of all experts), then c a (g - <g, a>).
    float top = -INFINITY, total = 0.f, rest = 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (whole || ((picked >> j) & 1u)) top = fmaxf(top, l[j]);
    float q[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      q[j] = picked && (whole || ((picked >> j) & 1u)) ? share_size(a.sigmoid, l[j], top) : 0.f;
      total += q[j];
      rest = fmaf(q[j], d[j], rest);
    }
    const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      d[j] = a.scale * q[j] * inv * (d[j] - rest * inv);
      if (a.sigmoid) d[j] *= sigmoid(-l[j]);
      if (q[j] == 0.f) d[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NE; ++j) d[j] = l[j] == -INFINITY ? 0.f : a.scale * d[j] * sigmoid(l[j]) * sigmoid(-l[j]);
  }
  T* row = static_cast<T*>(p.dlogits) + t * a.experts;
  constexpr int kPiece = NE * sizeof(T) < 16 ? NE : 16 / static_cast<int>(sizeof(T));
  if (p.vec) {
#pragma unroll
    for (int i = 0; i < NE; i += kPiece) {
      Share<T, kPiece> out;
#pragma unroll
      for (int j = 0; j < kPiece; ++j) out.v[j] = from_f32<T>(d[i + j]);
      if (i < a.experts) *reinterpret_cast<Share<T, kPiece>*>(row + i) = out;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (j < a.experts) row[j] = from_f32<T>(d[j]);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------
constexpr size_t kMaxRouteSmem = 96 * 1024;

size_t route_smem(int experts, int top_k, int tokens_per_block) {
  const size_t marks = static_cast<size_t>(experts) * ((tokens_per_block + 31) / 32);
  return (marks * 4 + (marks + 1) / 2 * 4 + static_cast<size_t>(tokens_per_block) * top_k * 2 + 15) / 16 * 16;
}

// Experts of a lane (or of a thread) that the kernels are compiled for.
// A thread per token or a warp per token.  Measured, thread / warp: 8 experts top 2, 16384 tokens 7.5 / 14.6 us, one token
// 4.1 / 3.3; 16 experts top 2, 16384 tokens 7.9 / 14.6, top 8 with 4096 tokens 12.9 / 10.1, 256 tokens 5.8 / 6.6.  With a bias a
// thread that has to choose again in 64 bits over all of 32 experts holds up its warp for 20 us.
bool by_threads(const RouteArgs& a) {
  if (a.experts <= kThreadExperts) return a.tokens > 8;
  return a.experts <= kThreadExpertsFlat && a.top_groups == a.groups && a.bias == nullptr && a.top_k <= 4 && a.tokens > 1024;
}
int share_of(const RouteArgs& a) {
  if (by_threads(a)) return a.experts <= 4 ? 4 : a.experts <= 8 ? 8 : a.experts <= 16 ? 16 : 32;
  const int ne = (a.experts + 31) / 32;
  return ne <= 6 ? ne : ne <= 8 ? 8 : ne <= 16 ? 16 : 32;
}
// Lanes that share a group where a lane has `ne` experts, if groups fall into whole lanes, a power of two of them.
int lanes_of(const RouteArgs& a, int ne) {
  const int size = a.experts / a.groups;
  return size % ne == 0 && power_of_two(size / ne) && a.groups * (size / ne) <= 32 ? size / ne : 0;
}

// Few tokens stay in one block, which needs no second kernel; more get about a block per SM, small ones as long as
// there are SMs left (256 tokens of 256 experts: 32 a block 22.6 us, 8 a block 17).
int tokens_per_block(const RouteArgs& a) {
  int tpb;
  if (by_threads(a)) {
    tpb = a.tokens <= 256 ? a.tokens : (a.tokens + 591) / 592;
    if (tpb < 128 && a.tokens > 256) tpb = 128;
    if (tpb > 1024) tpb = 1024;
  } else {
    tpb = a.tokens <= 24 ? a.tokens : (a.tokens + 147) / 148;
    if (tpb < 8) tpb = 8;
  }
  if (tpb > 32) tpb = (tpb + 31) / 32 * 32;
  if (tpb < 1) tpb = 1;
  while (tpb > 32 && route_smem(a.experts, a.top_k, tpb) > kMaxRouteSmem) tpb -= 32;
  return tpb;
}

int sm_count() {
  int dev = 0, sms = 0;
  PCCL_CUDA(cudaGetDevice(&dev));
  PCCL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  return sms;
}

template <class Kernel> void launch_route(Kernel kernel, const RouteParams& p, int blocks, int threads, size_t smem, cudaStream_t stream) {
  if (smem > 32 * 1024)
    PCCL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  kernel<<<blocks, threads, smem, stream>>>(p);
}

template <typename T, int NE>
void launch_warps(const RouteParams& p, bool backward, int blocks, size_t smem, cudaStream_t stream) {
  if (backward) {
    const int64_t want = (static_cast<int64_t>(p.a.tokens) + 7) / 8, most = 8ll * sm_count();
    route_warp_backward_kernel<T, NE><<<static_cast<int>(want < most ? want : most), 256, 0, stream>>>(p);
    return;
  }
  constexpr int kMost = NE <= 8 ? 1024 : 512;      // 64 or 128 registers a thread
  int threads = (p.a.tokens < p.tokens_per_block ? p.a.tokens : p.tokens_per_block) * 32;
  threads = threads < 128 ? 128 : threads > kMost ? kMost : threads;
  launch_route(route_warp_kernel<T, NE, kMost>, p, blocks, threads, smem + threads / 32 * sizeof(Deck<NE>), stream);
}

template <typename T, int NE>
void launch_threads(const RouteParams& p, bool backward, int blocks, size_t smem, cudaStream_t stream) {
  if (backward) route_thread_backward_kernel<T, NE><<<(p.a.tokens + 127) / 128, 128, 0, stream>>>(p);
  else launch_route(route_thread_kernel<T, NE>, p, blocks, std::clamp(p.tokens_per_block, 128, NE <= 8 ? kMostThreads : 256), smem, stream);
}

void launch_any(RouteParams& p, bool backward, int blocks, size_t smem, cudaStream_t stream) {
  const RouteArgs& a = p.a;
  const bool alone = by_threads(a);
  const int bytes = dtype_bytes(a.dtype);
  int ne = share_of(a);
  p.lanes = lanes_of(a, ne);
  // A few idle lanes are cheaper than groups that cross them.
  if (!alone && a.top_groups < a.groups)
    for (const int wider : {2, 3, 4, 5, 6, 8})
      if (!p.lanes && wider > ne) {
        p.lanes = lanes_of(a, wider);
        if (p.lanes) ne = wider;
      }
  const int piece = ne * bytes < 16 ? ne * bytes : 16;
  p.vec = power_of_two(ne) && (alone ? a.experts * bytes % piece == 0 : a.experts % ne == 0) &&
          reinterpret_cast<uintptr_t>(a.logits) % piece == 0 && a.ld * bytes % piece == 0 &&
          (!backward || (reinterpret_cast<uintptr_t>(p.dlogits) % piece == 0 && static_cast<int64_t>(a.experts) * bytes % piece == 0));
  PCCL_BLOCK_TYPES(a.dtype, T,
    if (alone && ne == 4) launch_threads<T, 4>(p, backward, blocks, smem, stream);
    else if (alone && ne == 8) launch_threads<T, 8>(p, backward, blocks, smem, stream);
    else if (alone && ne == 16) launch_threads<T, 16>(p, backward, blocks, smem, stream);
    else if (alone) launch_threads<T, 32>(p, backward, blocks, smem, stream);
    else if (ne == 1) launch_warps<T, 1>(p, backward, blocks, smem, stream);
    else if (ne == 2) launch_warps<T, 2>(p, backward, blocks, smem, stream);
    else if (ne == 3) launch_warps<T, 3>(p, backward, blocks, smem, stream);
    else if (ne == 4) launch_warps<T, 4>(p, backward, blocks, smem, stream);
    else if (ne == 5) launch_warps<T, 5>(p, backward, blocks, smem, stream);
    else if (ne == 6) launch_warps<T, 6>(p, backward, blocks, smem, stream);
    else if (ne == 8) launch_warps<T, 8>(p, backward, blocks, smem, stream);
    else if (ne == 16) launch_warps<T, 16>(p, backward, blocks, smem, stream);
    else launch_warps<T, 32>(p, backward, blocks, smem, stream))
  PCCL_CUDA(cudaGetLastError());
}

}  // namespace

size_t route_workspace(const RouteArgs& a) {
  const int tpb = tokens_per_block(a);
  const int blocks = (a.tokens + tpb - 1) / tpb;
  return blocks > 1 ? static_cast<size_t>(blocks) * ((a.experts + 3) / 4 * 4) * sizeof(uint16_t) : 0;
}

void route_topk(const RouteArgs& a, cudaStream_t stream) {
  RouteParams p{};
  p.a = a;
  p.tokens_per_block = tokens_per_block(a);
  p.words = (p.tokens_per_block + 31) / 32;
  p.pitch = (a.experts + 3) / 4 * 4;
  p.per_choice = static_cast<uint32_t>((0x100000000ull + a.top_k - 1) / a.top_k);
  int blocks = (a.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  if (blocks < 1) blocks = 1;
  p.block_words = static_cast<int>(route_smem(a.experts, a.top_k, p.tokens_per_block) / 4);
  p.counts = static_cast<uint16_t*>(a.workspace);
  PCCL_CHECK(blocks == 1 || p.counts != nullptr, "route_topk: no workspace");
  launch_any(p, false, blocks, route_smem(a.experts, a.top_k, p.tokens_per_block), stream);
  if (blocks > 1) {
    // Its blocks may start while the first kernel ends; they wait for its results on the device.
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(kMostThreads);
    config.stream = stream;
    config.attrs = &early;
    config.numAttrs = 1;
    PCCL_CUDA(cudaLaunchKernelEx(&config, route_rows_kernel, p));
  }
}

void route_topk_backward(const RouteArgs& a, const float* dweights, void* dlogits, cudaStream_t stream) {
  if (a.tokens == 0) return;
  RouteParams p{};
  p.a = a;
  p.dweights = dweights;
  p.dlogits = dlogits;
  launch_any(p, true, 0, 0, stream);
}

}  // namespace block
}  // namespace pccl
