// Expert routing: scores, group-limited top-k with a balance bias, weights, and the rows of the choices in
// expert order; and the gradient of the weights.
//
//   p = softmax(l) or sigmoid(l);  s = p + bias;  the best `top_groups` groups of experts stay;
//   idx = the top_k largest s of what stays, ties to the lowest number;
//   w_k = scale * p_k / sum p  (or scale * p_k);
//   rows[t][k] = offsets[idx] + number of earlier tokens that chose the same expert.
//
// One warp per token, expert e in lane e / NE, so that the lowest lane holds the lowest number and a tie is
// decided by the first set bit of a ballot.  Scores are compared as unsigned keys of the same order (one
// redux.sync a round).
//
// The order of two scores is part of the answer, and 32 bits cannot tell scores apart that differ by less than
// their rounding.  Without a bias the order is that of the logits and needs no arithmetic.  With one, the choice
// is made in 32 bits together with the runner-up; where any two neighbours of the sorted choice (or the last
// group kept and the first dropped) are nearer than the error bound of the arithmetic, the warp repeats the
// token in 64 bits.  Equal logits with equal biases are a true tie and need no repeat.
//
// Rows in expert order need no atomics whose order matters: a block of consecutive tokens marks its choices as
// bits in shared memory ([expert][token]), a choice's rank is a population count, and the blocks' counts
// per expert are summed by the second kernel in block order.
#include <math.h>

#include "../common/util.h"
#include "../engine/cuda_driver.h"
#include "vec.cuh"

namespace pccl {
namespace block {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr unsigned kAll = 0xffffffffu;

struct RouteParams {
  RouteArgs a;
  const float* dweights;
  void* dlogits;
  uint16_t* counts;           // [blocks][experts]: choices per expert of one block's tokens
  int tokens_per_block, words;
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

// NaN counts as the lowest logit; +infinity as the largest finite one, so that no score is a NaN.  The sum with
// zero turns -0 into +0: the two are equal and their keys have to be.
__device__ __forceinline__ float clean(float l) { return l != l ? -INFINITY : fminf(l, 3.402823466e38f) + 0.f; }

// Choice of one token by scores s[NE]; without a bias they rank the groups and the logits rank the experts.  Lane
// i < top_k returns the i-th expert; *near is set where two scores that decide something differ by no more than
// tau (+ 2^-21 of their size).
template <typename F, int NE>
__device__ __forceinline__ int choose(const RouteArgs& a, const F (&s)[NE], float tau, bool check, const float (&l)[NE],
                                      const float (&bias)[NE], bool* near) {
  using Key = decltype(key_of(F()));
  const int lane = threadIdx.x & 31;
  Key key[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) key[j] = lane * NE + j < a.experts ? key_of(s[j]) : Key(0);
  bool close = false;

  if (a.top_groups < a.groups) {
    const int size = a.experts / a.groups;
    Key mine = 0;                                  // lane g: the score of group g
    for (int g = 0; g < a.groups; ++g) {
      Key b1 = 0, b2 = 0;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        const int e = lane * NE + j - g * size;
        if (e >= 0 && e < size) {
          if (key[j] > b1) { b2 = b1; b1 = key[j]; }
          else if (key[j] > b2) b2 = key[j];
        }
      }
      const Key m1 = warp_max(b1);
      F score = value_of(m1);
      if (a.top2) {
        const int owner = __ffs(__ballot_sync(kAll, b1 == m1)) - 1;
        score += value_of(warp_max(lane == owner ? b2 : b1));
      }
      if (lane == g) mine = key_of(score);
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const Key other = __shfl_sync(kAll, mine, g);
      rank += other > mine || (other == mine && g < lane) ? 1 : 0;
    }
    const bool kept = lane < a.groups && rank < a.top_groups;
    const unsigned keep = __ballot_sync(kAll, kept);
    if (check) {
      const F low = value_of(static_cast<Key>(~warp_max(kept ? static_cast<Key>(~mine) : Key(0))));
      const F high = value_of(warp_max(lane < a.groups && !kept ? mine : Key(0)));
      close = !(static_cast<float>(low - high) > 2.f * tau + 0x1p-20f * fabsf(static_cast<float>(low)));
    }
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (!((keep >> ((lane * NE + j) / size & 31)) & 1u)) key[j] = 0;
      else if (a.bias == nullptr && key[j] != 0) key[j] = key_of(static_cast<F>(l[j]));
  }
  check = check && a.bias != nullptr;

  Key best = 0;
#pragma unroll
  for (int j = 0; j < NE; ++j) best = key[j] > best ? key[j] : best;
  int mine = -1;
  F score = 0;
  float my_l = 0.f, my_b = 0.f;
  const int rounds = a.top_k + (check ? 1 : 0);
  for (int i = 0; i < rounds; ++i) {
    const Key m = warp_max(best);
    if (m == 0) break;                             // only the runner-up can be missing
    const int owner = __ffs(__ballot_sync(kAll, best == m)) - 1;
    int e = 0;
    float el = 0.f, eb = 0.f;
    if (lane == owner) {
      bool found = false;
      best = 0;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        if (!found && key[j] == m) {
          found = true;
          key[j] = 0;
          e = lane * NE + j;
          el = l[j];
          eb = bias[j];
        }
        best = key[j] > best ? key[j] : best;
      }
    }
    e = __shfl_sync(kAll, e, owner);
    if (check) {
      el = __shfl_sync(kAll, el, owner);
      eb = __shfl_sync(kAll, eb, owner);
    }
    if (lane == i) { mine = e; score = value_of(m); my_l = el; my_b = eb; }
  }
  if (check) {
    const int next = __shfl_down_sync(kAll, mine, 1);
    const F below = __shfl_down_sync(kAll, score, 1);
    const float l1 = __shfl_down_sync(kAll, my_l, 1), b1 = __shfl_down_sync(kAll, my_b, 1);
    if (lane < a.top_k && next >= 0 && !(l1 == my_l && b1 == my_b))
      close |= !(static_cast<float>(score - below) > tau + 0x1p-21f * fabsf(static_cast<float>(score)));
  }
  *near = __any_sync(kAll, close);
  return lane < a.top_k ? mine : -1;
}

// The same choice from scores in 64 bits.
template <int NE>
__device__ __noinline__ int choose_wide(const RouteArgs& a, const float (&l)[NE], const float (&bias)[NE]) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NE; ++j) top = fmaxf(top, l[j]);
  top = warp_max(top);
  double s[NE], total = 0;
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
  bool near;
  return choose<double, NE>(a, s, 0.f, false, l, bias, &near);
}

// Row of a token: cleaned logits, -infinity beyond the last expert.
template <typename T, int NE>
__device__ __forceinline__ void load_row(const RouteArgs& a, int64_t t, float (&l)[NE]) {
  const T* row = static_cast<const T*>(a.logits) + t * a.ld;
  const int e0 = (threadIdx.x & 31) * NE;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const float v = to_f32<T>(row[min(e0 + j, a.experts - 1)]);
    l[j] = e0 + j < a.experts ? clean(v) : -INFINITY;
  }
}

__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }

// Shares of the choices among themselves, sum 1 (0 where every chosen logit is -infinity).  Scaled by the
// largest so that it holds where the scores themselves would underflow: softmax(l) over the choices, or
// sigmoid(l) / exp(m) with m = min(0, max l).
__device__ __forceinline__ float share(const RouteArgs& a, float l) {
  const int lane = threadIdx.x & 31;
  const bool live = lane < a.top_k && l != -INFINITY;
  const float top = warp_max(live ? l : -INFINITY);
  if (top == -INFINITY) return 0.f;
  float q;
  if (a.sigmoid) {
    q = l > 0.f ? sigmoid(l) : expf(l - fminf(top, 0.f)) / (1.f + expf(l));
  } else {
    q = expf(l - top);
  }
  if (!live) q = 0.f;
  return q / warp_sum(q);
}

template <typename T, int NE>
__global__ void __launch_bounds__(kThreads) route_topk_kernel(const RouteParams p) {
  extern __shared__ uint32_t smem[];
  const RouteArgs& a = p.a;
  uint32_t* bits = smem;                                             // [experts][words]
  uint16_t* chosen = reinterpret_cast<uint16_t*>(bits + a.experts * p.words);   // [tokens_per_block][top_k]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  for (int i = threadIdx.x; i < a.experts * p.words; i += kThreads) bits[i] = 0;

  float bias[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const int e = min(lane * NE + j, a.experts - 1);
    bias[j] = a.bias ? clean(a.bias[e]) : 0.f;
  }
  const bool scored = a.bias != nullptr || (a.top2 && a.top_groups < a.groups);   // the order needs the scores
  __syncthreads();

  for (int i = warp; i < count; i += kWarps) {
    const int64_t t = first + i;
    int e = -1;
    float w = 0.f;
    if (a.mask == nullptr || a.mask[t]) {
      float l[NE];
      load_row<T, NE>(a, t, l);
      float top = 0.f, total = 1.f;
      float s[NE];
#pragma unroll
      for (int j = 0; j < NE; ++j) s[j] = l[j];
      if (!a.sigmoid && (scored || !a.renormalise)) {
        top = l[0];
#pragma unroll
        for (int j = 1; j < NE; ++j) top = fmaxf(top, l[j]);
        top = warp_max(top);
        total = 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          s[j] = l[j] == -INFINITY ? 0.f : expf(l[j] - top);
          total += s[j];
        }
        total = warp_sum(total);
      }
      bool near = false;
      if (scored) {
        const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
        for (int j = 0; j < NE; ++j) {
          const float prob = a.sigmoid ? sigmoid(l[j]) : s[j] * inv;
          s[j] = l[j] == -INFINITY || bias[j] == -INFINITY ? -INFINITY : prob + bias[j];
        }
        // Error of one score: exp 2^-22, sum (NE + 5) 2^-24 + 2^-22, quotient and product 2^-23, each of the
        // row's largest probability 1 / total; twice that for a difference.  Sigmoid: 1.5 * 2^-22 of at most 1.
        const float tau = a.sigmoid ? 0x1p-20f : (NE + 18) * 0x1p-23f * inv;
        e = choose<float, NE>(a, s, tau, true, l, bias, &near);
        if (near) e = choose_wide<NE>(a, l, bias);
      } else {
        e = choose<float, NE>(a, l, 0.f, false, l, bias, &near);
      }
      const float le = e >= 0 ? clean(to_f32<T>(static_cast<const T*>(a.logits)[t * a.ld + e])) : -INFINITY;
      if (a.renormalise) w = share(a, le);
      else if (a.sigmoid) w = sigmoid(le);
      else w = le == -INFINITY ? 0.f : expf(le - top) / total;
      w *= a.scale;
    }
    if (lane < a.top_k) {
      a.idx[t * a.top_k + lane] = e;
      a.weights[t * a.top_k + lane] = w;
      chosen[i * a.top_k + lane] = static_cast<uint16_t>(e);           // 0xffff: none
      if (e >= 0) atomicOr(bits + e * p.words + (i >> 5), 1u << (i & 31));
    }
  }
  __syncthreads();

  // Choices per expert: to the second kernel, or (one block) straight into the offsets.
  __shared__ int32_t base[kMaxExperts + 1];
  for (int e = threadIdx.x; e < a.experts; e += kThreads) {
    int n = 0;
    for (int w = 0; w < p.words; ++w) n += __popc(bits[e * p.words + w]);
    if (gridDim.x > 1) p.counts[static_cast<int64_t>(blockIdx.x) * a.experts + e] = static_cast<uint16_t>(n);
    base[e] = gridDim.x > 1 ? 0 : n;
  }
  __syncthreads();
  if (gridDim.x == 1) {
    if (warp == 0) {
      int run = 0;
      for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int n = e0 + lane < a.experts ? base[e0 + lane] : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(kAll, sum, o);
          if (lane >= o) sum += v;
        }
        if (e0 + lane < a.experts) {
          base[e0 + lane] = run + sum - n;
          a.offsets[e0 + lane] = run + sum - n;
        }
        run += __shfl_sync(kAll, sum, 31);
      }
      if (lane == 0) a.offsets[a.experts] = run;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < count * a.top_k; i += kThreads) {
    const int e = chosen[i], tok = i / a.top_k;
    int row = -1;
    if (e != 0xffff) {
      row = base[e];
      for (int w = 0; w < tok >> 5; ++w) row += __popc(bits[e * p.words + w]);
      row += __popc(bits[e * p.words + (tok >> 5)] & ((1u << (tok & 31)) - 1u));
    }
    a.rows[static_cast<int64_t>(first) * a.top_k + i] = row;
  }
}

// Adds to every choice the rows of earlier experts and of earlier blocks of its own expert.
__global__ void __launch_bounds__(kThreads) route_rows_kernel(const RouteParams p) {
  const RouteArgs& a = p.a;
  __shared__ int32_t before[kMaxExperts], total[kMaxExperts];
  const int lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < a.experts; e += kThreads) {
    int sum = 0, mine = 0;
    for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
      if (b == static_cast<int>(blockIdx.x)) mine = sum;
      sum += p.counts[static_cast<int64_t>(b) * a.experts + e];
    }
    before[e] = mine;
    total[e] = sum;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int run = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int n = e0 + lane < a.experts ? total[e0 + lane] : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kAll, sum, o);
        if (lane >= o) sum += v;
      }
      if (e0 + lane < a.experts) {
        before[e0 + lane] += run + sum - n;
        if (blockIdx.x == 0) a.offsets[e0 + lane] = run + sum - n;
      }
      run += __shfl_sync(kAll, sum, 31);
    }
    if (blockIdx.x == 0 && lane == 0) a.offsets[a.experts] = run;
  }
  __syncthreads();
  const int first = blockIdx.x * p.tokens_per_block;
  const int count = min(p.tokens_per_block, a.tokens - first);
  for (int i = threadIdx.x; i < count * a.top_k; i += kThreads) {
    const int64_t at = static_cast<int64_t>(first) * a.top_k + i;
    const int e = a.idx[at];
    if (e >= 0) a.rows[at] += before[e];
  }
}

// dl from dw, idx constant.  With c = scale and a_k the shares of the choices (renormalised):
//   softmax  dl_k = c a_k (g_k - <g, a>)                 sigmoid  the same times (1 - p_k)
// else softmax  dl_e = c p_e (g_e - <g, p>)              sigmoid  dl_k = c g_k p_k (1 - p_k).
template <typename T, int NE>
__global__ void __launch_bounds__(kThreads) route_topk_backward_kernel(const RouteParams p) {
  const RouteArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp; t < a.tokens;
       t += static_cast<int64_t>(gridDim.x) * kWarps) {
    int e = lane < a.top_k ? a.idx[t * a.top_k + lane] : -1;
    if (e >= a.experts) e = -1;
    const float g = e >= 0 ? p.dweights[t * a.top_k + lane] : 0.f;
    const float le = e >= 0 ? clean(to_f32<T>(static_cast<const T*>(a.logits)[t * a.ld + e])) : -INFINITY;
    float d, rest = 0.f, top = 0.f, inv = 0.f;
    float l[NE];
    if (a.renormalise) {
      const float q = share(a, le);
      d = a.scale * q * (g - warp_sum(g * q));
      if (a.sigmoid) d *= sigmoid(-le);
    } else if (a.sigmoid) {
      d = a.scale * g * sigmoid(le) * sigmoid(-le);
    } else {
      load_row<T, NE>(a, t, l);
      top = l[0];
#pragma unroll
      for (int j = 1; j < NE; ++j) top = fmaxf(top, l[j]);
      top = warp_max(top);
      float total = 0.f;
#pragma unroll
      for (int j = 0; j < NE; ++j) total += l[j] == -INFINITY ? 0.f : expf(l[j] - top);
      total = warp_sum(total);
      inv = total > 0.f ? 1.f / total : 0.f;
      const float prob = le == -INFINITY ? 0.f : expf(le - top) * inv;
      rest = warp_sum(g * prob);
      d = g;
    }
    if (le == -INFINITY) d = 0.f;
    float out[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) out[j] = 0.f;
    for (int k = 0; k < a.top_k; ++k) {
      const int ek = __shfl_sync(kAll, e, k);
      const float dk = __shfl_sync(kAll, d, k);
#pragma unroll
      for (int j = 0; j < NE; ++j)
        if (ek == lane * NE + j) out[j] = dk;
    }
    if (!a.renormalise && !a.sigmoid) {
      const bool any = __any_sync(kAll, e >= 0);
#pragma unroll
      for (int j = 0; j < NE; ++j)
        out[j] = any && l[j] != -INFINITY ? a.scale * expf(l[j] - top) * inv * (out[j] - rest) : 0.f;
    }
    T* row = static_cast<T*>(p.dlogits) + t * a.experts;
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (lane * NE + j < a.experts) row[lane * NE + j] = from_f32<T>(out[j]);
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  PCCL_CUDA(cudaGetDevice(&dev));
  PCCL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  return sms;
}

constexpr int kMinTokensPerBlock = 32;
constexpr size_t kMaxRouteSmem = 96 * 1024;

size_t route_smem(int experts, int top_k, int tokens_per_block) {
  return static_cast<size_t>(experts) * (tokens_per_block / 32) * 4 + static_cast<size_t>(tokens_per_block) * top_k * 2;
}

// A block per SM, as many tokens as its bit marks have room for.
int tokens_per_block(int tokens, int experts, int top_k) {
  const int sms = 148;
  int tpb = (tokens + sms - 1) / sms;
  tpb = (tpb + 31) / 32 * 32;
  if (tpb < kMinTokensPerBlock) tpb = kMinTokensPerBlock;
  while (tpb > 32 && route_smem(experts, top_k, tpb) > kMaxRouteSmem) tpb -= 32;
  return tpb;
}

template <typename T, int NE>
void launch_route(const RouteParams& p, bool backward, int blocks, size_t smem, cudaStream_t stream) {
  if (backward) {
    route_topk_backward_kernel<T, NE><<<blocks, kThreads, 0, stream>>>(p);
    return;
  }
  if (smem > 40 * 1024)
    PCCL_CUDA(cudaFuncSetAttribute(route_topk_kernel<T, NE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(smem)));
  route_topk_kernel<T, NE><<<blocks, kThreads, smem, stream>>>(p);
}

void launch_route_any(const RouteParams& p, bool backward, int blocks, size_t smem, cudaStream_t stream) {
  const int per_lane = (p.a.experts + 31) / 32;
  PCCL_BLOCK_TYPES(p.a.dtype, T,
    if (per_lane <= 1) launch_route<T, 1>(p, backward, blocks, smem, stream);
    else if (per_lane <= 2) launch_route<T, 2>(p, backward, blocks, smem, stream);
    else if (per_lane <= 4) launch_route<T, 4>(p, backward, blocks, smem, stream);
    else if (per_lane <= 8) launch_route<T, 8>(p, backward, blocks, smem, stream);
    else if (per_lane <= 16) launch_route<T, 16>(p, backward, blocks, smem, stream);
    else launch_route<T, 32>(p, backward, blocks, smem, stream))
  PCCL_CUDA(cudaGetLastError());
}

}  // namespace

size_t route_workspace(int tokens, int experts, int top_k) {
  const int tpb = tokens_per_block(tokens, experts, top_k);
  const int blocks = (tokens + tpb - 1) / tpb;
  return blocks > 1 ? static_cast<size_t>(blocks) * experts * sizeof(uint16_t) : 0;
}

void route_topk(const RouteArgs& a, cudaStream_t stream) {
  RouteParams p{};
  p.a = a;
  p.tokens_per_block = tokens_per_block(a.tokens, a.experts, a.top_k);
  p.words = p.tokens_per_block / 32;
  int blocks = (a.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  if (blocks < 1) blocks = 1;
  p.counts = static_cast<uint16_t*>(a.workspace);
  PCCL_CHECK(blocks == 1 || p.counts != nullptr, "route_topk: no workspace");
  launch_route_any(p, false, blocks, route_smem(a.experts, a.top_k, p.tokens_per_block), stream);
  if (blocks > 1) {
    route_rows_kernel<<<blocks, kThreads, 0, stream>>>(p);
    PCCL_CUDA(cudaGetLastError());
  }
}

void route_topk_backward(const RouteArgs& a, const float* dweights, void* dlogits, cudaStream_t stream) {
  if (a.tokens == 0) return;
  RouteParams p{};
  p.a = a;
  p.dweights = dweights;
  p.dlogits = dlogits;
  const int64_t want = (static_cast<int64_t>(a.tokens) + kWarps - 1) / kWarps, most = 4ll * sm_count();
  launch_route_any(p, true, static_cast<int>(want < most ? want : most), 0, stream);
}

}  // namespace block
}  // namespace pccl
