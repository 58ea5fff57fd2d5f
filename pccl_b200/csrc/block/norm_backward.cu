// The gradients of the norms around a block (norm_forward.cu has the formulas), one pass over the rows.
//
// With mean over a row:
//   d  = dh + r2 * (dy gamma - n2 * mean(dy gamma n2));   dresidual = scale * d;   dgamma = sum_rows dy n2
//   dgate = sum_rows d v;  dv = gate d;  dpost_gamma = sum_rows dv n1;  dx = r1 * (dv post_gamma - n1 mean(..))
// h is computed again from x and the residual: a 16-bit h has lost what dgamma needs, a 32-bit one is read.
//
// post_gamma and gate wait in shared memory as their product g1, which is all that a row needs:
// h = scale * residual + n1 g1 and dx = r1 * (d g1 - n1 mean(d g1 n1)).  Their gradients both follow from one sum per
// group of rows that share a gate, S = sum d n1: dgate = post_gamma S, dpost_gamma = sum over groups of gate S.
//
// A block takes a run of consecutive rows and sums the weights' gradients in registers; a second kernel adds the
// blocks' sums in their order, so results do not depend on timing.
#include <type_traits>

#include "norm_common.cuh"

namespace pccl {
namespace block {
namespace norm {
namespace {

// Slots of a thread, in bytes: gamma (the first), g1 (kFull: a norm behind the block or a gate), its share of the ring.  x is read where h is formed again (16-bit streams) or its norm is undone.
template <typename TX, typename TR, bool kFull> struct BackwardSlots {
  static constexpr bool kReadsX = kFull || sizeof(TR) == 2;
  static constexpr int kG1 = kBytes<float>, kWeights = kBytes<float> * (kFull ? 2 : 1);
  static constexpr int kDy = kBytes<TR>, kH = kDy + kBytes<TX>, kX = kH + kBytes<TR>;
  static constexpr int kShare = kX + (kReadsX ? kBytes<TX> : 0);
  static constexpr int kWindows = kReadsX ? 4 : 3;
};

template <typename T, bool kVec, int G>
__device__ __forceinline__ void store_weight_grad(void* out, int f32, int64_t first, const Columns<kVec, G>& c,
                                                  const float2* f) {
  if (f32) store_row<float, kVec, G>(static_cast<float*>(out) + first, c, f);
  else store_row<T, kVec, G>(static_cast<T*>(out) + first, c, f);
}

template <typename TX, typename TR, int kMode, bool kFull, bool kSplit>
__global__ void __launch_bounds__(512, 1) norm_backward_kernel(const NormParams p) {
  using Slots = BackwardSlots<TX, TR, kFull>;
  constexpr bool kVec = kMode == kRing;
  constexpr int G = kGroup<TX, TR>, kGroups = kHeld / G;
  __shared__ RowSums sums;
  extern __shared__ __align__(128) char smem[];         // rows of the ring begin with a line: 154 us instead of 168
  const NormArgs& a = p.a;
  const NormGrads& g = p.g;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  asm volatile("griddepcontrol.launch_dependents;");
  const int rank = kSplit ? cluster_rank() : 0, worker = static_cast<int>(blockIdx.x) / (kSplit ? kSplitBlocks : 1);
  const Columns<kVec, G> c(n, rank);
  row_sum_clear<kSplit>(sums);
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);

  char* const gammas = smem;
  char* const g1 = smem + Slots::kG1 * width;
  char* const ring = smem + Slots::kWeights * width;
  const int wx = window_bytes<TX>(width), wr = window_bytes<TR>(width);
  const int stage = kMode == kRing ? Slots::kShare * width : 2 * wr + (Slots::kReadsX ? 2 : 1) * wx;
  const int off_dy = kMode == kRing ? Slots::kDy * width : wr;
  const int off_h = kMode == kRing ? Slots::kH * width : wr + wx;
  const int off_x = kMode == kRing ? Slots::kX * width : 2 * wr + wx;
  // The stream to read: as it was stored (32 bits), or the residual that it is formed from.
  const TR* const stream = static_cast<const TR*>(g.h ? g.h : a.residual);
  const int64_t lds = g.h ? n : a.ldr;
  const TX* const x_rows = static_cast<const TX*>(a.x);
  const TX* const dy_rows = static_cast<const TX*>(g.dy);
  const TR* const dh_rows = static_cast<const TR*>(g.dh);
  const bool reads_x = Slots::kReadsX && a.x != nullptr;
  const auto fetch = [&](int64_t row, int s) {
    if (row < end) {
      char* to = ring + s * stage;
      if constexpr (kMode == kRing) {
        if (g.dh) fetch_share<TR, G>(to, dh_rows + row * g.lddh, c);
        if (g.dy) {
          fetch_share<TX, G>(to + off_dy, dy_rows + row * g.lddy, c);
          fetch_share<TR, G>(to + off_h, stream + row * lds, c);
        }
        if (reads_x) fetch_share<TX, G>(to + off_x, x_rows + row * a.ldx, c);
      } else {
        if (g.dh) fetch_window(to, dh_rows + row * g.lddh, c);
        if (g.dy) {
          fetch_window(to + off_dy, dy_rows + row * g.lddy, c);
          fetch_window(to + off_h, stream + row * lds, c);
        }
        if (reads_x) fetch_window(to + off_x, x_rows + row * a.ldx, c);
      }
    }
    copies_commit();
  };
  for (int s = 0; s < p.ring - 1; ++s) fetch(begin + s, s);

  float2 acc_gamma[kHeld / 2], acc_s[kFull ? kHeld / 2 : 1];
#pragma unroll
  for (int i = 0; i < kHeld / 2; ++i) {
    acc_gamma[i] = both(0.f);
    if (kFull) acc_s[i] = both(0.f);
  }
  if (a.gamma.ptr) {
    float2 w[kHeld / 2];
    load_weight<TX, kVec, G>(a.gamma, 0, c, w);
    slots_store(gammas, w);
  }
  bool first = true;                               // no group has ended yet
  int64_t group = 0, left = 0;                     // rows left of the present group of rows that share a gate
  if constexpr (kFull) {
    group = a.gate.ptr ? begin / a.gate_rows : 0;
    left = a.gate.ptr ? (group + 1) * a.gate_rows - begin : a.rows;
    form_g1<TX, kVec, G>(a, group, g1, c);
  }
  float next_r1 = kFull && a.post_gamma.ptr ? g.r1[begin] : 1.f;
  float next_r2 = g.dy ? g.r2[begin] : 0.f;

  int turn = 0, s = 0;
  for (int64_t t = begin; t < end; ++t) {
    const float r1 = next_r1, r2 = next_r2;
    if (t + 1 < end) {
      if (kFull && a.post_gamma.ptr) next_r1 = g.r1[t + 1];
      if (g.dy) next_r2 = g.r2[t + 1];
    }
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
    const TX* const row_x = x_rows + t * a.ldx;
    // The row is gone through in groups of columns, and inputs are read again rather than kept: what stays in
    // registers over a barrier are the two sums of the weights' gradients and two values a column.
    float2 d[kHeld / 2], n2[kHeld / 2];
    if (g.dy) {
      float2 dot = both(0.f);
#pragma unroll
      for (int v = 0; v < kGroups; ++v) {
        float2 f[G / 2], w[G / 2];
        float2* const h = n2 + v * (G / 2);
        take<TR, kMode, G>(held + off_h, stream + t * lds, v, c, h);
        if (Slots::kReadsX && reads_x && !g.h) {
          take<TX, kMode, G>(held + off_x, row_x, v, c, f);
          if (kFull) {
            slots_load<G>(g1, v, w);
#pragma unroll
            for (int j = 0; j < G / 2; ++j) f[j] = mul2(mul2(f[j], both(r1)), w[j]);
          }
#pragma unroll
          for (int j = 0; j < G / 2; ++j) h[j] = fma2(both(a.scale), h[j], f[j]);
        }
        take<TX, kMode, G>(held + off_dy, dy_rows + t * g.lddy, v, c, f);
        slots_load<G>(gammas, v, w);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) {
          h[j] = mul2(h[j], both(r2));
          acc_gamma[v * (G / 2) + j] = fma2(f[j], h[j], acc_gamma[v * (G / 2) + j]);
          d[v * (G / 2) + j] = mul2(f[j], w[j]);
          dot = fma2(d[v * (G / 2) + j], h[j], dot);
        }
      }
      const float pull = -r2 * inv_n * row_sum<kSplit>(dot.x + dot.y, sums, &turn);
#pragma unroll
      for (int i = 0; i < kHeld / 2; ++i) d[i] = fma2(both(r2), d[i], mul2(both(pull), n2[i]));
    } else {
#pragma unroll
      for (int i = 0; i < kHeld / 2; ++i) d[i] = both(0.f);
    }
    float2 dot = both(0.f);
#pragma unroll
    for (int v = 0; v < kGroups; ++v) {
      float2 f[G / 2], w[G / 2];
      if (g.dh) {
        take<TR, kMode, G>(held, dh_rows + t * g.lddh, v, c, f);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) d[v * (G / 2) + j] = add2(d[v * (G / 2) + j], f[j]);
      }
      if (g.dresidual) {
#pragma unroll
        for (int j = 0; j < G / 2; ++j) f[j] = mul2(both(a.scale), d[v * (G / 2) + j]);
        store_group<TR, kVec, G>(static_cast<TR*>(g.dresidual) + t * n, v, c, f);
      }
      if constexpr (kFull) {
        take<TX, kMode, G>(held + off_x, row_x, v, c, f);
        slots_load<G>(g1, v, w);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) {
          f[j] = mul2(f[j], both(r1));
          acc_s[v * (G / 2) + j] = fma2(d[v * (G / 2) + j], f[j], acc_s[v * (G / 2) + j]);
          d[v * (G / 2) + j] = mul2(d[v * (G / 2) + j], w[j]);
          dot = fma2(d[v * (G / 2) + j], f[j], dot);
        }
      }
    }
    if (kFull && a.post_gamma.ptr) {
      // n1 = r1 * x once more
      const float pull = -r1 * r1 * inv_n * row_sum<kSplit>(dot.x + dot.y, sums, &turn);
      if (g.dx) {
#pragma unroll
        for (int v = 0; v < kGroups; ++v) {
          float2 f[G / 2];
          take<TX, kMode, G>(held + off_x, row_x, v, c, f);
#pragma unroll
          for (int j = 0; j < G / 2; ++j) f[j] = fma2(both(r1), d[v * (G / 2) + j], mul2(both(pull), f[j]));
          store_group<TX, kVec, G>(static_cast<TX*>(g.dx) + t * n, v, c, f);
        }
      }
    } else if (g.dx) {
#pragma unroll
      for (int v = 0; v < kGroups; ++v) store_group<TX, kVec, G>(static_cast<TX*>(g.dx) + t * n, v, c, d + v * (G / 2));
    }
    if constexpr (kFull) {
      if (--left == 0 || t + 1 == end) {
        if (a.gate.ptr) {
          // The group's last row here: dgate is whole if this run held all of the group, else a part.
          if (a.post_gamma.ptr) {
            float2 w[kHeld / 2];
            if (p.part_post) {
              // Added up in this thread's own columns of the block's part: once a group, so not worth registers.
              float* const part = p.part_post + static_cast<int64_t>(worker) * n;
              load_weight<TX, kVec, G>(a.gate, group * n, c, w);
#pragma unroll
              for (int v = 0; v < kGroups; ++v) {
                float2 sum[G / 2];
                if (first) {
#pragma unroll
                  for (int j = 0; j < G / 2; ++j) sum[j] = both(0.f);
                } else {
                  load_group<float, kVec, G>(part, v, c, sum);
                }
#pragma unroll
                for (int j = 0; j < G / 2; ++j) sum[j] = fma2(w[v * (G / 2) + j], acc_s[v * (G / 2) + j], sum[j]);
                store_group<float, kVec, G>(part, v, c, sum);
              }
              first = false;
            }
            load_weight<TX, kVec, G>(a.post_gamma, 0, c, w);
#pragma unroll
            for (int i = 0; i < kHeld / 2; ++i) acc_s[i] = mul2(acc_s[i], w[i]);
          }
          if (g.dgate) {
            if (group * a.gate_rows >= begin && (group + 1) * a.gate_rows <= end) {
              store_weight_grad<TX, kVec, G>(g.dgate, a.gate.f32, group * n, c, acc_s);
            } else {
              const int slot = group * a.gate_rows <= begin ? 0 : 1;
              store_row<float, kVec, G>(p.part_gate + (static_cast<int64_t>(worker) * 2 + slot) * n, c, acc_s);
            }
          }
#pragma unroll
          for (int i = 0; i < kHeld / 2; ++i) acc_s[i] = both(0.f);
          if (t + 1 < end) form_g1<TX, kVec, G>(a, ++group, g1, c);
          left = a.gate_rows;
        }
      }
    }
  }
  copies_wait(0);
  if (p.part_gamma) store_row<float, kVec, G>(p.part_gamma + static_cast<int64_t>(worker) * n, c, acc_gamma);
  if constexpr (kFull) {
    if (p.part_post && !a.gate.ptr) {
      store_row<float, kVec, G>(p.part_post + static_cast<int64_t>(worker) * n, c, acc_s);
    }
  }
}

// Adds the blocks' parts in their order, a strip of them to each warp: blockIdx.y 0 gamma, 1 post_gamma, 2.. the
// groups of gate rows.  C columns a thread (four where rows of parts are aligned).
template <typename T, int C>
__global__ void __launch_bounds__(512) norm_reduce_kernel(const NormParams p) {
  struct alignas(C * 4) Part { float v[C]; };
  __shared__ Part part[16][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const NormArgs& a = p.a;
  const int lane = threadIdx.x & 31, strip = threadIdx.x >> 5, strips = blockDim.x >> 5, n = a.hidden;
  const int col = (blockIdx.x * 32 + lane) * C;
  for (int64_t what = blockIdx.y; what < 2 + (p.part_gate ? a.rows / a.gate_rows : 0); what += gridDim.y) {
    const float* src;
    int first = 0, last = p.workers;
    int64_t step = n, group = 0;
    void* out;
    int f32;
    if (what == 0) {
      src = p.part_gamma; out = p.g.dgamma; f32 = a.gamma.f32;
    } else if (what == 1) {
      src = p.part_post; out = p.g.dpost_gamma; f32 = a.post_gamma.f32;
    } else {
      group = what - 2;
      src = p.part_gate; out = p.g.dgate; f32 = a.gate.f32;
      step = 2 * static_cast<int64_t>(n);
      // The runs that hold the group's first and last row: runs have rows / workers rows, the first ones one more.
      const int64_t each = a.rows / p.workers, longer = a.rows % p.workers;
      const int64_t r0 = group * a.gate_rows, r1 = r0 + a.gate_rows - 1;
      first = static_cast<int>(r0 < longer * (each + 1) ? r0 / (each + 1) : longer + (r0 - longer * (each + 1)) / each);
      last = static_cast<int>(r1 < longer * (each + 1) ? r1 / (each + 1) : longer + (r1 - longer * (each + 1)) / each) + 1;
      if (last - first == 1) src = nullptr;                  // written whole by its only worker
    }
    if (src == nullptr || out == nullptr) continue;
    Part sum{};
    const auto add = [&](const float* at) {
      const Part q = *reinterpret_cast<const Part*>(at);
#pragma unroll
      for (int i = 0; i < C; ++i) sum.v[i] += q.v[i];
    };
    if (col < n) {
      // Only the first of them can have begun with another group: its part stands in the second place.
      if (what >= 2) {
        if (strip == 0) add(src + first * step + (group * a.gate_rows > run_start(a.rows, p.workers, first) ? n : 0) + col);
        ++first;
      }
      const float* at = src + (first + strip) * step + col;
#pragma unroll 8
      for (int w = first + strip; w < last; w += strips, at += strips * step) add(at);
    }
    part[strip][lane] = sum;
    __syncthreads();
    if (strip == 0 && col < n) {
      for (int s = 1; s < strips; ++s)
#pragma unroll
        for (int i = 0; i < C; ++i) sum.v[i] += part[s][lane].v[i];
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (f32) static_cast<float*>(out)[group * n + col + i] = sum.v[i];
        else static_cast<T*>(out)[group * n + col + i] = from_f32<T>(sum.v[i]);
      }
    }
    __syncthreads();
  }
}

template <typename T, int C> void reduce_launch(const NormParams& p, cudaStream_t stream) {
  // Its blocks may start while the first kernel ends; they wait for its results on the device.
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  const int64_t targets = 2 + (p.part_gate ? p.a.rows / p.a.gate_rows : 0);
  config.gridDim = dim3((p.a.hidden + 32 * C - 1) / (32 * C), static_cast<unsigned>(targets < 1024 ? targets : 1024));
  config.blockDim = dim3(512);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  PCCL_CUDA(cudaLaunchKernelEx(&config, norm_reduce_kernel<T, C>, p));
}

// How rows are laid out, and how many clusters share them: what the SMs hold, each with at least one row.
template <typename TX, typename TR, bool kFull> Layout backward_layout(const NormArgs& a, bool vec, int* workers) {
  using Slots = BackwardSlots<TX, TR, kFull>;
  const Layout l = layout_of(a.hidden, vec, Slots::kWeights, Slots::kShare, Slots::kWindows, 512, false);
  const int64_t most = static_cast<int64_t>(blocks_per_sm(l.threads)) * sm_count() / l.split;
  *workers = static_cast<int>(a.rows < most ? a.rows : most);
  return l;
}

template <typename TX, typename TR, bool kFull>
void backward_mode(NormParams& p, bool vec, cudaStream_t stream) {
  const Layout l = backward_layout<TX, TR, kFull>(p.a, vec, &p.workers);
  p.ring = l.ring;
  const auto go = [&](auto kernel) {
    allow_smem(kernel, l);
    launch(kernel, p, l, stream);
  };
  if (vec && l.split > 1) go(norm_backward_kernel<TX, TR, kRing, kFull, true>);
  else if (vec) go(norm_backward_kernel<TX, TR, kRing, kFull, false>);
  else if (l.split > 1) go(norm_backward_kernel<TX, TR, kWindow, kFull, true>);
  else go(norm_backward_kernel<TX, TR, kWindow, kFull, false>);
}

// Calls f(TX(), TR(), kFull) for the types and weights of these arguments.
template <class F> void with_types(const NormArgs& a, F f) {
  PCCL_BLOCK_TYPES(a.xt, T,
    if (a.rt == a.xt && has_g1(a)) f(T(), T(), std::true_type());
    else if (a.rt == a.xt) f(T(), T(), std::false_type());
    else if (has_g1(a)) f(T(), float(), std::true_type());
    else f(T(), float(), std::false_type()))
}

bool all_aligned(const NormArgs& a, const NormGrads& g) {
  const int xb = dtype_bytes(a.xt), rb = dtype_bytes(a.rt);
  return inputs_aligned(a) && aligned(g.dy, g.lddy, xb) && aligned(g.dh, g.lddh, rb) && aligned(g.h, a.hidden, 4) &&
         aligned(g.dx, a.hidden, xb) && aligned(g.dresidual, a.hidden, rb) &&
         aligned(g.dgate, a.hidden, a.gate.f32 ? 4 : xb) && aligned(g.workspace, a.hidden, 4);
}

}  // namespace
}  // namespace norm

size_t norm_workspace(const NormArgs& a, const NormGrads& g) {
  // Either way of reading rows may be taken: the larger count of workers.
  int most = 0;
  norm::with_types(a, [&](auto x, auto r, auto full) {
    for (const bool vec : {true, false}) {
      int workers = 0;
      norm::backward_layout<decltype(x), decltype(r), decltype(full)::value>(a, vec, &workers);
      most = workers > most ? workers : most;
    }
  });
  const size_t row = static_cast<size_t>(most) * a.hidden * sizeof(float);
  return row * ((g.dgamma ? 1 : 0) + (g.dpost_gamma ? 1 : 0) + (g.dgate ? 2 : 0));
}

void norm_backward(const NormArgs& a, const NormGrads& g, cudaStream_t stream) {
  if (a.rows == 0) return;
  norm::NormParams p{};
  p.a = a;
  p.g = g;
  const bool vec = norm::all_aligned(a, g);
  norm::with_types(a, [&](auto x, auto r, auto full) {
    norm::backward_layout<decltype(x), decltype(r), decltype(full)::value>(a, vec, &p.workers);
  });
  const int64_t row = static_cast<int64_t>(p.workers) * a.hidden;
  float* at = static_cast<float*>(g.workspace);
  if (g.dgamma) { p.part_gamma = at; at += row; }
  if (g.dpost_gamma) { p.part_post = at; at += row; }
  if (g.dgate) p.part_gate = at;
  norm::with_types(a, [&](auto x, auto r, auto full) {
    norm::backward_mode<decltype(x), decltype(r), decltype(full)::value>(p, vec, stream);
  });
  PCCL_CUDA(cudaGetLastError());
  if (g.dgamma || g.dpost_gamma || g.dgate) {
    PCCL_BLOCK_TYPES(a.xt, T,
      if (a.hidden % 4 == 0) norm::reduce_launch<T, 4>(p, stream);
      else norm::reduce_launch<T, 1>(p, stream))
  }
}

}  // namespace block
}  // namespace pccl
