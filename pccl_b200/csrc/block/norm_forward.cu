// The norms around a block with its gate and residual scale, one pass over the rows.
//
//   n1 = x * r1, r1 = 1 / sqrt(mean x^2 + eps);  v = n1 * post_gamma           (v = x without a norm behind)
//   h  = scale * residual + gate * v
//   n2 = h * r2, r2 = 1 / sqrt(mean h^2 + eps);  y = n2 * gamma
//
// y is formed from h as it stands in 32 bits, before its rounding to the stream's type.  post_gamma and gate wait in
// shared memory as their product g1.
#include <type_traits>

#include "norm_common.cuh"

namespace pccl {
namespace block {
namespace norm {
namespace {

// Slots of a thread, in bytes: gamma (the first), g1 (kFull: a norm behind the block or a gate), its share of the ring.
template <typename TX, typename TR, bool kFull> struct ForwardSlots {
  static constexpr int kG1 = kBytes<float>, kWeights = kBytes<float> * (kFull ? 2 : 1);
  static constexpr int kX = kBytes<TR>, kShare = kBytes<TR> + kBytes<TX>;
};

template <typename TX, typename TR, int kMode, bool kFull, bool kSplit, int kMost>
__global__ void __launch_bounds__(kMost, 1) norm_forward_kernel(const NormParams p) {
  using Slots = ForwardSlots<TX, TR, kFull>;
  constexpr bool kVec = kMode == kRing;
  constexpr int G = kGroup<TX, TR>, kGroups = kHeld / G;
  __shared__ RowSums sums;
  extern __shared__ __align__(128) char smem[];
  const NormArgs& a = p.a;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  const int rank = kSplit ? cluster_rank() : 0, worker = static_cast<int>(blockIdx.x) / (kSplit ? kSplitBlocks : 1);
  const Columns<kVec, G> c(n, rank);
  row_sum_clear<kSplit>(sums);
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);

  char* const gammas = smem;
  char* const g1 = smem + Slots::kG1 * width;
  char* const ring = smem + Slots::kWeights * width;
  const int stage = kMode == kRing ? Slots::kShare * width : window_bytes<TR>(width) + window_bytes<TX>(width);
  const int off_x = kMode == kRing ? Slots::kX * width : window_bytes<TR>(width);
  const TR* const residual = static_cast<const TR*>(a.residual);
  const TX* const x_rows = static_cast<const TX*>(a.x);
  const auto fetch = [&](int64_t row, int s) {
    if (row < end) {
      char* to = ring + s * stage;
      if constexpr (kMode == kRing) {
        fetch_share<TR, G>(to, residual + row * a.ldr, c);
        if (a.x) fetch_share<TX, G>(to + off_x, x_rows + row * a.ldx, c);
      } else {
        fetch_window(to, residual + row * a.ldr, c);
        if (a.x) fetch_window(to + off_x, x_rows + row * a.ldx, c);
      }
    }
    copies_commit();
  };
  for (int s = 0; s < p.ring - 1; ++s) fetch(begin + s, s);

  if (a.gamma.ptr) {
    float2 w[kHeld / 2];
    load_weight<TX, kVec, G>(a.gamma, 0, c, w);
    slots_store(gammas, w);
  }
  int64_t group = 0, left = 0;                     // rows left of the present group of rows that share a gate
  if constexpr (kFull) {
    group = a.gate.ptr ? begin / a.gate_rows : 0;
    left = a.gate.ptr ? (group + 1) * a.gate_rows - begin : a.rows;
    form_g1<TX, kVec, G>(a, group, g1, c);
  }

  int turn = 0, s = 0;
  for (int64_t t = begin; t < end; ++t) {
    const char* held = ring + s * stage;
    const int last = s == 0 ? p.ring - 1 : s - 1;
    if constexpr (kMode == kRing) {
      fetch(t + p.ring - 1, last);
      copies_wait(p.ring - 1);
    } else if (p.ring > 1) {
      copies_wait(p.ring - 2);
      __syncthreads();                             // everybody's copies of this row, and the last one's readers
      fetch(t + p.ring - 1, last);
    } else {
      __syncthreads();
      fetch(t, 0);
      copies_wait(0);
      __syncthreads();
    }
    s = s + 1 == p.ring ? 0 : s + 1;
    float2 x[kHeld / 2], h[kHeld / 2];
    float r1 = 1.f;
    if (kFull || a.x) {
      float2 ss = both(0.f);
#pragma unroll
      for (int v = 0; v < kGroups; ++v) {
        take<TX, kMode, G>(held + off_x, x_rows + t * a.ldx, v, c, x + v * (G / 2));
        if (kFull)
#pragma unroll
          for (int j = 0; j < G / 2; ++j) ss = fma2(x[v * (G / 2) + j], x[v * (G / 2) + j], ss);
      }
      if constexpr (kFull) {
        if (a.post_gamma.ptr) {
          r1 = rsqrtf(row_sum<kSplit>(ss.x + ss.y, sums, &turn) * inv_n + a.eps);
          if (p.r1 && tid == 0 && rank == 0) p.r1[t] = r1;
        }
        if (left == 0) {
          form_g1<TX, kVec, G>(a, ++group, g1, c);
          left = a.gate_rows;
        }
        --left;
      }
    }
    float2 ss = both(0.f);
#pragma unroll
    for (int v = 0; v < kGroups; ++v) {
      float2* const hv = h + v * (G / 2);
      float2* const xv = x + v * (G / 2);
      take<TR, kMode, G>(held, residual + t * a.ldr, v, c, hv);
      if constexpr (kFull) {
        float2 w[G / 2];
        slots_load<G>(g1, v, w);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) hv[j] = fma2(both(a.scale), hv[j], mul2(mul2(xv[j], both(r1)), w[j]));
      } else if (a.x) {
#pragma unroll
        for (int j = 0; j < G / 2; ++j) hv[j] = fma2(both(a.scale), hv[j], xv[j]);
      }
#pragma unroll
      for (int j = 0; j < G / 2; ++j) ss = fma2(hv[j], hv[j], ss);
      if (p.h) store_group<TR, kVec, G>(static_cast<TR*>(p.h) + t * n, v, c, hv);
    }
    if (a.gamma.ptr) {
      const float r2 = rsqrtf(row_sum<kSplit>(ss.x + ss.y, sums, &turn) * inv_n + a.eps);
      if (p.r2 && tid == 0 && rank == 0) p.r2[t] = r2;
#pragma unroll
      for (int v = 0; v < kGroups; ++v) {
        float2 w[G / 2];
        slots_load<G>(gammas, v, w);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) w[j] = mul2(mul2(h[v * (G / 2) + j], both(r2)), w[j]);
        store_group<TX, kVec, G>(static_cast<TX*>(p.y) + t * n, v, c, w);
      }
    }
  }
  copies_wait(0);
}

template <typename TX, typename TR, int kMode, bool kFull, bool kSplit, int kMost>
void forward_launch(NormParams& p, const Layout& l, cudaStream_t stream) {
  // One wave of blocks: a block's later rows are on their way while it works.
  const auto kernel = norm_forward_kernel<TX, TR, kMode, kFull, kSplit, kMost>;
  allow_smem(kernel, l);
  const int64_t most = static_cast<int64_t>(max_coresident(kernel, l.threads, l.smem)) / l.split;
  PCCL_CHECK(most > 0, "block norm: the kernel does not fit on this device");
  p.workers = static_cast<int>(p.a.rows < most ? p.a.rows : most);
  p.ring = l.ring;
  launch(kernel, p, l, stream);
}

template <typename TX, typename TR, bool kFull>
void forward_mode(NormParams& p, bool vec, cudaStream_t stream) {
  using Slots = ForwardSlots<TX, TR, kFull>;
  // One block a row as long as it fits (12288 columns of bf16: 5.3 TB/s so, 3.5 split over two).
  const Layout l = layout_of(p.a.hidden, vec, Slots::kWeights, Slots::kShare, 2, 1024, true);
  const auto go = [&](auto mode) {
    constexpr int kMode = decltype(mode)::value;
    if (l.split > 1) forward_launch<TX, TR, kMode, kFull, true, 512>(p, l, stream);
    else if (l.threads > 512) forward_launch<TX, TR, kMode, kFull, false, 1024>(p, l, stream);
    else forward_launch<TX, TR, kMode, kFull, false, 512>(p, l, stream);
  };
  if (vec) go(std::integral_constant<int, kRing>());
  else go(std::integral_constant<int, kWindow>());
}

template <typename TX, typename TR>
void forward_typed(NormParams& p, bool vec, cudaStream_t stream) {
  if (has_g1(p.a)) forward_mode<TX, TR, true>(p, vec, stream);
  else forward_mode<TX, TR, false>(p, vec, stream);
}

}  // namespace
}  // namespace norm

void norm_forward(const NormArgs& a, void* h, void* y, float* r1, float* r2, cudaStream_t stream) {
  if (a.rows == 0) return;
  norm::NormParams p{};
  p.a = a;
  p.h = h;
  p.y = y;
  p.r1 = r1;
  p.r2 = r2;
  const bool vec = norm::inputs_aligned(a) && norm::aligned(h, a.hidden, dtype_bytes(a.rt)) &&
                   norm::aligned(y, a.hidden, dtype_bytes(a.xt));
  PCCL_BLOCK_TYPES(a.xt, T,
    if (a.rt == a.xt) norm::forward_typed<T, T>(p, vec, stream);
    else norm::forward_typed<T, float>(p, vec, stream))
  PCCL_CUDA(cudaGetLastError());
}

}  // namespace block
}  // namespace pccl
