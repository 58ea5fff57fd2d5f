// The norms around a block with its gate and residual scale, one pass over the rows, and their gradients.
//
//   n1 = x * r1, r1 = 1 / sqrt(mean x^2 + eps);  v = n1 * post_gamma           (v = x without a norm behind)
//   h  = scale * residual + gate * v
//   n2 = h * r2, r2 = 1 / sqrt(mean h^2 + eps);  y = n2 * gamma
//
// y is formed from h as it stands in 32 bits, before its rounding to the stream's type.  Backwards, with
// mean over a row:
//   d  = dh + r2 * (dy gamma - n2 * mean(dy gamma n2));   dresidual = scale * d;   dgamma = sum_rows dy n2
//   dgate = sum_rows d v;  dv = gate d;  dpost_gamma = sum_rows dv n1;  dx = r1 * (dv post_gamma - n1 mean(..))
// h is computed again from x and the residual: a 16-bit h has lost what dgamma needs, a 32-bit one is read.
//
// A row belongs to a warp (short rows) or to a block of threads (long ones) that holds it in registers.  In the
// backward kernel each of these workers takes a run of consecutive rows and sums the weights' gradients in
// registers; a second kernel adds the workers' sums in their order, so results do not depend on timing.
//
// Both passes are bound by memory, and what keeps memory waiting is a row's own chain: load, sum over the row,
// barrier, use, perhaps a second sum.  So every thread copies the columns it will use of the coming rows into
// its own slots of a ring in shared memory (cp.async: no registers, and no barrier, since nobody else reads
// them) while it works on the present one.  Rows that are not aligned to 16 bytes (odd sizes) and rows too long for
// the ring are loaded directly.
//
// The weights wait in such slots as 32-bit values, post_gamma and gate as their product g1, which is all that
// a row needs: h = scale * residual + n1 g1, and dx = r1 * (d g1 - n1 mean(d g1 n1)).  Their gradients both follow
// from one sum per group of rows that share a gate, S = sum d n1: dgate = post_gamma S, dpost_gamma = sum gate S.
#include "../common/launch.h"
#include "../common/util.h"
#include "../engine/cuda_driver.h"
#include "vec.cuh"

namespace pccl {
namespace block {

namespace {

constexpr int kVecs = 2;                       // groups of eight values a thread holds of its row
constexpr int kHeld = 8 * kVecs;

struct NormParams {
  NormArgs a;
  NormGrads g;
  void* h;
  void* y;
  float* r1;
  float* r2;
  float* part_gamma;          // [workers][hidden]
  float* part_post;           // [workers][hidden]
  float* part_gate;           // [workers][2][hidden]: the run's first group of rows, its last one
  int workers;
};

// Column of value j of group v held by a thread: eight in a row where rows are aligned, else a thread's values
// stand a whole row of threads apart, so that neighbours read neighbours.
template <bool kVec> __device__ __forceinline__ int column(int v, int j, int tid, int width) {
  return kVec ? (v * width + tid) * 8 + j : (v * 8 + j) * width + tid;
}

template <typename T, bool kVec>
__device__ __forceinline__ void load_row(const T* row, int hidden, int tid, int width, float* f) {
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    if constexpr (kVec) {
      const int at = (v * width + tid) * 8;
      if (at < hidden) {
        unpack8<T>(load_raw8<T>(row + at), f + 8 * v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[8 * v + j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = column<false>(v, j, tid, width);
        f[8 * v + j] = at < hidden ? to_f32<T>(row[at]) : 0.f;
      }
    }
  }
}
template <typename T, bool kVec>
__device__ __forceinline__ void store_row(T* row, int hidden, int tid, int width, const float* f) {
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    if constexpr (kVec) {
      const int at = (v * width + tid) * 8;
      if (at < hidden) store_raw8<T>(row + at, pack8<T>(f + 8 * v));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = column<false>(v, j, tid, width);
        if (at < hidden) row[at] = from_f32<T>(f[8 * v + j]);
      }
    }
  }
}
// A weight vector is of the activations' type or of 32 bits.
template <typename T, bool kVec>
__device__ __forceinline__ void load_weight(const Weight& w, int64_t first, int hidden, int tid, int width, float* f) {
  if (w.f32) load_row<float, kVec>(static_cast<const float*>(w.ptr) + first, hidden, tid, width, f);
  else load_row<T, kVec>(static_cast<const T*>(w.ptr) + first, hidden, tid, width, f);
}

// ---- ring ------------------------------------------------------------------------------------------------
// A plane holds 16 bytes per thread of a row; an input of T takes kVecs * sizeof(T) / 2 planes.
template <typename T> constexpr int kPlanes = kVecs * static_cast<int>(sizeof(T)) / 2;

__device__ __forceinline__ void copy_async(uint4* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

template <typename T>
__device__ __forceinline__ void fetch_row(uint4* plane, const T* row, int hidden, int tid, int width) {
  constexpr int kQ = sizeof(T) / 2;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int at = (v * width + tid) * 8;
    if (at < hidden)
#pragma unroll
      for (int q = 0; q < kQ; ++q)
        copy_async(plane + (v * kQ + q) * width + tid, reinterpret_cast<const uint4*>(row + at) + q);
  }
}
template <typename T>
__device__ __forceinline__ void held_row(const uint4* plane, int hidden, int tid, int width, float* f) {
  constexpr int kQ = sizeof(T) / 2;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    if ((v * width + tid) * 8 < hidden) {
      Raw8<T> r;
#pragma unroll
      for (int q = 0; q < kQ; ++q) r.v[q] = plane[(v * kQ + q) * width + tid];
      unpack8<T>(r, f + 8 * v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[8 * v + j] = 0.f;
    }
  }
}
// The eight values of group v: from a ring plane, or from the row itself.
template <typename T, bool kVec, bool kHeldRow>
__device__ __forceinline__ void take8(const uint4* plane, const T* row, int v, int hidden, int tid, int width, float* f) {
  if constexpr (kHeldRow) {
    constexpr int kQ = sizeof(T) / 2;
    Raw8<T> r;
#pragma unroll
    for (int q = 0; q < kQ; ++q) r.v[q] = plane[(v * kQ + q) * width + tid];
    unpack8<T>(r, f);
    if ((v * width + tid) * 8 >= hidden) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
  } else if constexpr (kVec) {
    const int at = (v * width + tid) * 8;
    if (at < hidden) {
      unpack8<T>(load_raw8<T>(row + at), f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = column<false>(v, j, tid, width);
      f[j] = at < hidden ? to_f32<T>(row[at]) : 0.f;
    }
  }
}
template <typename T, bool kVec>
__device__ __forceinline__ void put8(T* row, int v, int hidden, int tid, int width, const float* f) {
  if constexpr (kVec) {
    const int at = (v * width + tid) * 8;
    if (at < hidden) store_raw8<T>(row + at, pack8<T>(f));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = column<false>(v, j, tid, width);
      if (at < hidden) row[at] = from_f32<T>(f[j]);
    }
  }
}
__device__ __forceinline__ void slots_load8(const uint4* plane, int v, int tid, int width, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 q = reinterpret_cast<const float4*>(plane)[(2 * v + i) * width + tid];
    f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
  }
}

// Sum over the threads of a row; `sums` alternates between two sets so that one barrier a call is enough.  Sets
// are cleared once (row_sum_clear), so that whole groups of four can be read.
struct __align__(16) RowSums { float set[2][32]; };
__device__ __forceinline__ void row_sum_clear(RowSums& sums) {
  if (blockDim.x == 32) return;
  if (threadIdx.x < 64) (&sums.set[0][0])[threadIdx.x] = 0.f;
  __syncthreads();
}
__device__ __forceinline__ float row_sum(float v, RowSums& sums, int* turn) {
  v = warp_sum(v);
  if (blockDim.x == 32) return v;
  float* s = sums.set[*turn];
  *turn ^= 1;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); w += 4) {
    const float4 q = *reinterpret_cast<const float4*>(s + w);
    v += (q.x + q.y) + (q.z + q.w);
  }
  return v;
}

// A thread's slots of one weight: kHeld 32-bit values.
constexpr int kWeightPlanes = kHeld / 4;
__device__ __forceinline__ void slots_store(uint4* plane, int tid, int width, const float* f) {
#pragma unroll
  for (int i = 0; i < kWeightPlanes; ++i) reinterpret_cast<float4*>(plane)[i * width + tid] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}
__device__ __forceinline__ void slots_load(const uint4* plane, int tid, int width, float* f) {
#pragma unroll
  for (int i = 0; i < kWeightPlanes; ++i) {
    const float4 q = reinterpret_cast<const float4*>(plane)[i * width + tid];
    f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
  }
}

// g1 = post_gamma * gate of one group of rows into its slots (what is absent counts as 1).
template <typename T, bool kVec>
__device__ __forceinline__ void form_g1(const NormArgs& a, int64_t group, uint4* plane, int tid, int width) {
  float f[kHeld], w[kHeld];
  if (a.post_gamma.ptr) load_weight<T, kVec>(a.post_gamma, 0, a.hidden, tid, width, f);
  if (a.gate.ptr) {
    load_weight<T, kVec>(a.gate, group * a.hidden, a.hidden, tid, width, w);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) f[i] = a.post_gamma.ptr ? f[i] * w[i] : w[i];
  }
  slots_store(plane, tid, width, f);
}

// First row of worker w's run; w = workers gives the number of rows.
__device__ __forceinline__ int64_t run_start(int64_t rows, int workers, int w) {
  return rows / workers * w + min(static_cast<int64_t>(w), rows % workers);
}

// Slots of a worker, in planes: gamma, g1, (backward) the sum that becomes dpost_gamma, then the rows of the ring.
__host__ __device__ __forceinline__ bool has_g1(const NormArgs& a) { return a.post_gamma.ptr || a.gate.ptr; }
__host__ __device__ __forceinline__ int weight_planes(const NormArgs& a, bool backward) {
  return kWeightPlanes * ((a.gamma.ptr ? 1 : 0) + (has_g1(a) ? 1 : 0) + (backward && a.post_gamma.ptr && a.gate.ptr ? 1 : 0));
}
template <typename TX, typename TR> __host__ __device__ __forceinline__ int forward_planes(const NormArgs& a) {
  return kPlanes<TR> + (a.x ? kPlanes<TX> : 0);
}
template <typename TX, typename TR> __host__ __device__ __forceinline__ int backward_planes(const NormArgs& a, const NormGrads& g) {
  int planes = 0;
  if (g.dh) planes += kPlanes<TR>;
  if (g.dy) planes += kPlanes<TX> + (g.h ? kPlanes<float> : kPlanes<TR>);
  if (a.x) planes += kPlanes<TX>;
  return planes;
}

template <typename TX, typename TR, bool kVec, int kRing, int kMost>
__global__ void __launch_bounds__(kMost, 1) norm_forward_kernel(const NormParams p) {
  __shared__ RowSums sums;
  extern __shared__ uint4 slots[];
  const NormArgs& a = p.a;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  row_sum_clear(sums);
  const int worker = blockIdx.x * blockDim.y + threadIdx.y;
  if (worker >= p.workers) return;                 // whole warps of a block of warps
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);

  const int stage = kRing ? forward_planes<TX, TR>(a) * width : 0, weights = weight_planes(a, false) * width;
  uint4* const gammas = slots + (weights + kRing * stage) * threadIdx.y;
  uint4* const g1 = gammas + (a.gamma.ptr ? kWeightPlanes * width : 0);
  uint4* const ring = gammas + weights;
  const auto fetch = [&](int64_t row, int s) {
    if (row < end) {
      fetch_row<TR>(ring + s * stage, static_cast<const TR*>(a.residual) + row * a.ldr, n, tid, width);
      if (a.x) fetch_row<TX>(ring + s * stage + kPlanes<TR> * width, static_cast<const TX*>(a.x) + row * a.ldx, n, tid, width);
    }
    copies_commit();
  };
  if constexpr (kRing > 0) {
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) fetch(begin + s, s);
  }
  if (a.gamma.ptr) {
    float w[kHeld];
    load_weight<TX, kVec>(a.gamma, 0, n, tid, width, w);
    slots_store(gammas, tid, width, w);
  }
  int64_t group = 0, left = 0;                     // rows left of the present group of rows that share a gate
  if (has_g1(a)) {
    group = a.gate.ptr ? begin / a.gate_rows : 0;
    left = a.gate.ptr ? (group + 1) * a.gate_rows - begin : a.rows;
    form_g1<TX, kVec>(a, group, g1, tid, width);
  }

  int turn = 0, s = 0;
  for (int64_t t = begin; t < end; ++t) {
    float v[kHeld], h[kHeld];
    if constexpr (kRing > 0) {
      fetch(t + kRing - 1, s == 0 ? kRing - 1 : s - 1);
      const uint4* held = ring + s * stage;
      s = s + 1 == kRing ? 0 : s + 1;
      copies_wait<kRing - 1>();
      held_row<TR>(held, n, tid, width, h);
      if (a.x) held_row<TX>(held + kPlanes<TR> * width, n, tid, width, v);
    } else {
      load_row<TR, kVec>(static_cast<const TR*>(a.residual) + t * a.ldr, n, tid, width, h);
      if (a.x) load_row<TX, kVec>(static_cast<const TX*>(a.x) + t * a.ldx, n, tid, width, v);
    }
    if (a.x) {
      if (a.post_gamma.ptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) ss = fmaf(v[i], v[i], ss);
        const float r1 = rsqrtf(row_sum(ss, sums, &turn) * inv_n + a.eps);
        if (p.r1 && tid == 0) p.r1[t] = r1;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) v[i] *= r1;
      }
      if (has_g1(a)) {
        if (left == 0) {
          form_g1<TX, kVec>(a, ++group, g1, tid, width);
          left = a.gate_rows;
        }
        --left;
        float w[kHeld];
        slots_load(g1, tid, width, w);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) h[i] = fmaf(a.scale, h[i], v[i] * w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) h[i] = fmaf(a.scale, h[i], v[i]);
      }
    }
    if (p.h) store_row<TR, kVec>(static_cast<TR*>(p.h) + t * n, n, tid, width, h);
    if (a.gamma.ptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) ss = fmaf(h[i], h[i], ss);
      const float r2 = rsqrtf(row_sum(ss, sums, &turn) * inv_n + a.eps);
      if (p.r2 && tid == 0) p.r2[t] = r2;
      slots_load(gammas, tid, width, v);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) v[i] *= h[i] * r2;
      store_row<TX, kVec>(static_cast<TX*>(p.y) + t * n, n, tid, width, v);
    }
  }
  if constexpr (kRing > 0) copies_wait<0>();
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_weight_grad(void* out, int f32, int64_t first, int n, int tid, int width,
                                                  const float* f) {
  if (f32) store_row<float, kVec>(static_cast<float*>(out) + first, n, tid, width, f);
  else store_row<T, kVec>(static_cast<T*>(out) + first, n, tid, width, f);
}

// kRing: rows in shared memory (0: loaded directly).  kFull: a gate or a norm behind the block.
template <typename TX, typename TR, bool kVec, int kRing, bool kFull, int kMost>
__global__ void __launch_bounds__(kMost, 1) norm_backward_kernel(const NormParams p) {
  __shared__ RowSums sums;
  extern __shared__ uint4 slots[];
  const NormArgs& a = p.a;
  const NormGrads& g = p.g;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  row_sum_clear(sums);
  const int worker = blockIdx.x * blockDim.y + threadIdx.y;
  if (worker >= p.workers) return;                 // whole warps of a block of warps
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);

  const int stage = kRing ? backward_planes<TX, TR>(a, g) * width : 0, weights = weight_planes(a, true) * width;
  uint4* const gammas = slots + (weights + kRing * stage) * threadIdx.y;
  uint4* const g1 = gammas + (a.gamma.ptr ? kWeightPlanes * width : 0);
  uint4* const acc_post = g1 + kWeightPlanes * width;        // where there are a gate and a norm behind
  uint4* const ring = gammas + weights;
  const int off_dy = g.dh ? kPlanes<TR> * width : 0;
  const int off_h = off_dy + (g.dy ? kPlanes<TX> * width : 0);
  const int off_x = off_h + (g.dy ? (g.h ? kPlanes<float> : kPlanes<TR>) * width : 0);
  const auto fetch = [&](int64_t row, int s) {
    if (row < end) {
      uint4* to = ring + s * stage;
      if (g.dh) fetch_row<TR>(to, static_cast<const TR*>(g.dh) + row * g.lddh, n, tid, width);
      if (g.dy) {
        fetch_row<TX>(to + off_dy, static_cast<const TX*>(g.dy) + row * g.lddy, n, tid, width);
        if (g.h) fetch_row<float>(to + off_h, static_cast<const float*>(g.h) + row * n, n, tid, width);
        else fetch_row<TR>(to + off_h, static_cast<const TR*>(a.residual) + row * a.ldr, n, tid, width);
      }
      if (a.x) fetch_row<TX>(to + off_x, static_cast<const TX*>(a.x) + row * a.ldx, n, tid, width);
    }
    copies_commit();
  };
  if constexpr (kRing > 0) {
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) fetch(begin + s, s);
  }

  float acc_gamma[kHeld], acc_s[kFull ? kHeld : 1];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    acc_gamma[i] = 0.f;
    if (kFull) acc_s[i] = 0.f;
  }
  if (a.gamma.ptr) {
    float w[kHeld];
    load_weight<TX, kVec>(a.gamma, 0, n, tid, width, w);
    slots_store(gammas, tid, width, w);
  }
  int64_t group = 0, left = 0;                     // rows left of the present group of rows that share a gate
  if (kFull) {
    group = a.gate.ptr ? begin / a.gate_rows : 0;
    left = a.gate.ptr ? (group + 1) * a.gate_rows - begin : a.rows;
    form_g1<TX, kVec>(a, group, g1, tid, width);
    if (a.post_gamma.ptr && a.gate.ptr) slots_store(acc_post, tid, width, acc_gamma);
  }
  float next_r1 = kFull && a.post_gamma.ptr && begin < end ? g.r1[begin] : 1.f;
  float next_r2 = g.dy && begin < end ? g.r2[begin] : 0.f;

  int turn = 0, s = 0;
  for (int64_t t = begin; t < end; ++t) {
    float d[kHeld];
    const float r1 = next_r1, r2 = next_r2;
    if (t + 1 < end) {
      if (kFull && a.post_gamma.ptr) next_r1 = g.r1[t + 1];
      if (g.dy) next_r2 = g.r2[t + 1];
    }
    const uint4* held = ring + s * stage;
    if constexpr (kRing > 0) {
      fetch(t + kRing - 1, s == 0 ? kRing - 1 : s - 1);
      s = s + 1 == kRing ? 0 : s + 1;
      copies_wait<kRing - 1>();
    }
    constexpr bool kHeldRow = kRing > 0;
    const TX* const row_x = static_cast<const TX*>(a.x) + t * a.ldx;
    const TX* const row_dy = static_cast<const TX*>(g.dy) + t * g.lddy;
    const TR* const row_dh = static_cast<const TR*>(g.dh) + t * g.lddh;
    // The row is gone through in groups of eight values, and inputs are read again rather than kept: what stays in
    // registers over a barrier are the two sums of the weights' gradients and two values a column.
    float n2[kHeld];
    if (g.dy) {
      float dot = 0.f;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        float f[8], w[8];
        float* const h = n2 + 8 * v;
        if (g.h) {
          take8<float, kVec, kHeldRow>(held + off_h, static_cast<const float*>(g.h) + t * n, v, n, tid, width, h);
        } else {
          take8<TR, kVec, kHeldRow>(held + off_h, static_cast<const TR*>(a.residual) + t * a.ldr, v, n, tid, width, h);
          if (a.x) {
            take8<TX, kVec, kHeldRow>(held + off_x, row_x, v, n, tid, width, f);
            if (kFull) {
              slots_load8(g1, v, tid, width, w);
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] *= r1 * w[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = fmaf(a.scale, h[j], f[j]);
          }
        }
        take8<TX, kVec, kHeldRow>(held + off_dy, row_dy, v, n, tid, width, f);
        slots_load8(gammas, v, tid, width, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          h[j] *= r2;
          acc_gamma[8 * v + j] = fmaf(f[j], h[j], acc_gamma[8 * v + j]);
          d[8 * v + j] = f[j] * w[j];
          dot = fmaf(d[8 * v + j], h[j], dot);
        }
      }
      const float pull = -r2 * inv_n * row_sum(dot, sums, &turn);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) d[i] = fmaf(r2, d[i], pull * n2[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) d[i] = 0.f;
    }
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      float f[8], w[8];
      if (g.dh) {
        take8<TR, kVec, kHeldRow>(held, row_dh, v, n, tid, width, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[8 * v + j] += f[j];
      }
      if (g.dresidual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = a.scale * d[8 * v + j];
        put8<TR, kVec>(static_cast<TR*>(g.dresidual) + t * n, v, n, tid, width, f);
      }
      if constexpr (kFull) {
        take8<TX, kVec, kHeldRow>(held + off_x, row_x, v, n, tid, width, f);
        slots_load8(g1, v, tid, width, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[j] *= r1;
          acc_s[8 * v + j] = fmaf(d[8 * v + j], f[j], acc_s[8 * v + j]);
          d[8 * v + j] *= w[j];
          dot = fmaf(d[8 * v + j], f[j], dot);
        }
      }
    }
    if (kFull && a.post_gamma.ptr) {
      // n1 = r1 * x once more
      const float pull = -r1 * r1 * inv_n * row_sum(dot, sums, &turn);
      if (g.dx) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          float f[8];
          take8<TX, kVec, kHeldRow>(held + off_x, row_x, v, n, tid, width, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = fmaf(r1, d[8 * v + j], pull * f[j]);
          put8<TX, kVec>(static_cast<TX*>(g.dx) + t * n, v, n, tid, width, f);
        }
      }
    } else if (g.dx) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) put8<TX, kVec>(static_cast<TX*>(g.dx) + t * n, v, n, tid, width, d + 8 * v);
    }
    if constexpr (kFull) {
      if (--left == 0 || t + 1 == end) {
        if (a.gate.ptr) {
          // The group's last row here: dgate is whole if this run held all of the group, else a part.
          if (a.post_gamma.ptr) {
            float w[kHeld];
            load_weight<TX, kVec>(a.gate, group * n, n, tid, width, w);
            slots_load(acc_post, tid, width, d);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) d[i] = fmaf(w[i], acc_s[i], d[i]);
            slots_store(acc_post, tid, width, d);
            load_weight<TX, kVec>(a.post_gamma, 0, n, tid, width, w);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) acc_s[i] *= w[i];
          }
          if (g.dgate) {
            if (group * a.gate_rows >= begin && (group + 1) * a.gate_rows <= end) {
              store_weight_grad<TX, kVec>(g.dgate, a.gate.f32, group * n, n, tid, width, acc_s);
            } else {
              const int slot = group * a.gate_rows <= begin ? 0 : 1;
              store_row<float, kVec>(p.part_gate + (static_cast<int64_t>(worker) * 2 + slot) * n, n, tid, width, acc_s);
            }
          }
#pragma unroll
          for (int i = 0; i < kHeld; ++i) acc_s[i] = 0.f;
          if (t + 1 < end) form_g1<TX, kVec>(a, ++group, g1, tid, width);
          left = a.gate_rows;
        }
      }
    }
  }
  if constexpr (kRing > 0) copies_wait<0>();
  if (p.part_gamma) store_row<float, kVec>(p.part_gamma + static_cast<int64_t>(worker) * n, n, tid, width, acc_gamma);
  if constexpr (kFull) {
    if (p.part_post) {
      if (a.gate.ptr) slots_load(acc_post, tid, width, acc_s);
      store_row<float, kVec>(p.part_post + static_cast<int64_t>(worker) * n, n, tid, width, acc_s);
    }
  }
}

// Adds the workers' parts in their order: blockIdx.y 0 gamma, 1 post_gamma, 2.. the groups of gate rows.
template <typename T>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const NormParams p) {
  __shared__ float part[32][33];
  const NormArgs& a = p.a;
  const int lane = threadIdx.x & 31, strip = threadIdx.x >> 5, n = a.hidden;
  const int col = blockIdx.x * 32 + lane;
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
    float sum = 0.f;
    if (col < n) {
#pragma unroll 4
      for (int w = first + strip; w < last; w += 32) {
        const float* at = src + w * step;
        if (what >= 2 && group * a.gate_rows > run_start(a.rows, p.workers, w)) at += n;
        sum += at[col];
      }
    }
    part[strip][lane] = sum;
    __syncthreads();
    if (strip == 0 && col < n) {
#pragma unroll
      for (int s = 1; s < 32; ++s) sum += part[s][lane];
      if (f32) static_cast<float*>(out)[group * n + col] = sum;
      else static_cast<T*>(out)[group * n + col] = from_f32<T>(sum);
    }
    __syncthreads();
  }
}

struct Shape {
  dim3 block;
  int rows_per_block;
};
Shape shape_of(int hidden) {
  const int threads = ((hidden + kHeld - 1) / kHeld + 31) / 32 * 32;
  if (threads == 32) return Shape{dim3(32, 4), 4};
  return Shape{dim3(threads, 1), 1};
}

int sm_count() {
  int dev = 0, sms = 0;
  PCCL_CUDA(cudaGetDevice(&dev));
  PCCL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  return sms;
}

bool aligned(const void* p, int64_t ld, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * bytes % 16 == 0);
}
bool aligned(const Weight& w, int64_t hidden, DType t) { return aligned(w.ptr, hidden, w.f32 ? 4 : dtype_bytes(t)); }

bool inputs_aligned(const NormArgs& a) {
  return a.hidden % 8 == 0 && aligned(a.x, a.ldx, dtype_bytes(a.xt)) && aligned(a.residual, a.ldr, dtype_bytes(a.rt)) &&
         aligned(a.gamma, a.hidden, a.xt) && aligned(a.post_gamma, a.hidden, a.xt) && aligned(a.gate, a.hidden, a.xt);
}

// Workers of the backward kernel: 512 threads' worth per SM (128 registers each), each with at least one row.
int worker_count(const NormArgs& a) {
  const Shape s = shape_of(a.hidden);
  const int threads = static_cast<int>(s.block.x * s.block.y);
  const int64_t most = static_cast<int64_t>(threads < 512 ? 512 / threads : 1) * sm_count() * s.rows_per_block;
  return static_cast<int>(a.rows < most ? a.rows : most);
}

// Shared memory of an SM, and of one block (less what the kernel itself and the driver keep).
constexpr size_t kSmemSm = 228 * 1024, kSmemBlock = 226 * 1024, kSmemKept = 1024 + sizeof(RowSums);

template <class Kernel> void launch_norm(Kernel kernel, NormParams& p, bool forward, size_t smem, cudaStream_t stream) {
  const Shape s = shape_of(p.a.hidden);
  const int threads = static_cast<int>(s.block.x * s.block.y);
  if (smem > 40 * 1024)
    PCCL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  if (forward) {
    // One wave of blocks: a worker's later rows are on their way while it works.
    const int64_t most = static_cast<int64_t>(max_coresident(kernel, threads, smem)) * s.rows_per_block;
    PCCL_CHECK(most > 0, "block norm: the kernel does not fit on this device");
    p.workers = static_cast<int>(p.a.rows < most ? p.a.rows : most);
  }
  kernel<<<(p.workers + s.rows_per_block - 1) / s.rows_per_block, s.block, smem, stream>>>(p);
}

// Rows in the ring: as many as leave `blocks` blocks on an SM, down to two; none where two do not fit.
int ring_rows(size_t weights, size_t row, int most, int blocks) {
  for (int r = most; r > 2; --r)
    if ((weights + r * row + kSmemKept) * blocks <= kSmemSm && weights + r * row <= kSmemBlock) return r;
  return weights + 2 * row <= kSmemBlock ? 2 : 0;
}

template <typename TX, typename TR, int kMost>
void forward_typed(NormParams& p, bool vec, cudaStream_t stream) {
  const Shape s = shape_of(p.a.hidden);
  const int threads = static_cast<int>(s.block.x * s.block.y);
  const size_t weights = static_cast<size_t>(weight_planes(p.a, false)) * 16 * threads;
  const size_t row = static_cast<size_t>(forward_planes<TX, TR>(p.a)) * 16 * threads;
  const int ring = vec ? ring_rows(weights, row, 3, threads < 512 ? 768 / threads : 1) : 0;
  if (ring == 3) launch_norm(norm_forward_kernel<TX, TR, true, 3, kMost>, p, true, weights + 3 * row, stream);
  else if (ring == 2) launch_norm(norm_forward_kernel<TX, TR, true, 2, kMost>, p, true, weights + 2 * row, stream);
  else if (vec) launch_norm(norm_forward_kernel<TX, TR, true, 0, kMost>, p, true, weights, stream);
  else launch_norm(norm_forward_kernel<TX, TR, false, 0, kMost>, p, true, weights, stream);
}

template <typename TX, typename TR, bool kFull, int kMost>
void backward_full(NormParams& p, bool vec, cudaStream_t stream) {
  const Shape s = shape_of(p.a.hidden);
  const int threads = static_cast<int>(s.block.x * s.block.y);
  const size_t weights = static_cast<size_t>(weight_planes(p.a, true)) * 16 * threads;
  const size_t row = static_cast<size_t>(backward_planes<TX, TR>(p.a, p.g)) * 16 * threads;
  const int ring = vec ? ring_rows(weights, row, 3, threads < 512 ? 512 / threads : 1) : 0;
  if (ring == 3) launch_norm(norm_backward_kernel<TX, TR, true, 3, kFull, kMost>, p, false, weights + 3 * row, stream);
  else if (ring == 2) launch_norm(norm_backward_kernel<TX, TR, true, 2, kFull, kMost>, p, false, weights + 2 * row, stream);
  else if (vec) launch_norm(norm_backward_kernel<TX, TR, true, 0, kFull, kMost>, p, false, weights, stream);
  else launch_norm(norm_backward_kernel<TX, TR, false, 0, kFull, kMost>, p, false, weights, stream);
}

template <typename TX, typename TR, int kMost>
void backward_typed(NormParams& p, bool vec, cudaStream_t stream) {
  if (has_g1(p.a)) backward_full<TX, TR, true, kMost>(p, vec, stream);
  else backward_full<TX, TR, false, kMost>(p, vec, stream);
}

template <typename TX, typename TR>
void sized(NormParams& p, bool vec, bool backward, cudaStream_t stream) {
  const bool many = shape_of(p.a.hidden).block.x > 512;      // 64 registers a thread instead of 128
  if (backward && many) backward_typed<TX, TR, 1024>(p, vec, stream);
  else if (backward) backward_typed<TX, TR, 512>(p, vec, stream);
  else if (many) forward_typed<TX, TR, 1024>(p, vec, stream);
  else forward_typed<TX, TR, 512>(p, vec, stream);
}

// TR is TX or 32 bits.
template <typename TX>
void any_typed(NormParams& p, bool vec, bool backward, cudaStream_t stream) {
  if (p.a.rt == p.a.xt) sized<TX, TX>(p, vec, backward, stream);
  else sized<TX, float>(p, vec, backward, stream);
  PCCL_CUDA(cudaGetLastError());
}

}  // namespace

void norm_forward(const NormArgs& a, void* h, void* y, float* r1, float* r2, cudaStream_t stream) {
  if (a.rows == 0) return;
  NormParams p{};
  p.a = a;
  p.h = h;
  p.y = y;
  p.r1 = r1;
  p.r2 = r2;
  const bool vec = inputs_aligned(a) && aligned(h, a.hidden, dtype_bytes(a.rt)) && aligned(y, a.hidden, dtype_bytes(a.xt));
  PCCL_BLOCK_TYPES(a.xt, T, any_typed<T>(p, vec, false, stream))
}

size_t norm_workspace(const NormArgs& a, const NormGrads& g) {
  const size_t row = static_cast<size_t>(worker_count(a)) * a.hidden * sizeof(float);
  return row * ((g.dgamma ? 1 : 0) + (g.dpost_gamma ? 1 : 0) + (g.dgate ? 2 : 0));
}

void norm_backward(const NormArgs& a, const NormGrads& g, cudaStream_t stream) {
  if (a.rows == 0) return;
  NormParams p{};
  p.a = a;
  p.g = g;
  p.workers = worker_count(a);
  const int64_t row = static_cast<int64_t>(p.workers) * a.hidden;
  float* at = static_cast<float*>(g.workspace);
  if (g.dgamma) { p.part_gamma = at; at += row; }
  if (g.dpost_gamma) { p.part_post = at; at += row; }
  if (g.dgate) p.part_gate = at;
  const int xb = dtype_bytes(a.xt), rb = dtype_bytes(a.rt);
  const bool vec = inputs_aligned(a) && aligned(g.dy, g.lddy, xb) && aligned(g.dh, g.lddh, rb) &&
                   aligned(g.h, a.hidden, 4) && aligned(g.dx, a.hidden, xb) && aligned(g.dresidual, a.hidden, rb) &&
                   (!g.dgate || aligned(g.dgate, a.hidden, a.gate.f32 ? 4 : xb)) && aligned(g.workspace, a.hidden, 4);
  PCCL_BLOCK_TYPES(a.xt, T, any_typed<T>(p, vec, true, stream))
  if (g.dgamma || g.dpost_gamma || g.dgate) {
    const int64_t targets = 2 + (g.dgate ? a.rows / a.gate_rows : 0);
    const dim3 grid((a.hidden + 31) / 32, static_cast<unsigned>(targets < 1024 ? targets : 1024));
    PCCL_BLOCK_TYPES(a.xt, T, norm_reduce_kernel<T><<<grid, 1024, 0, stream>>>(p))
    PCCL_CUDA(cudaGetLastError());
  }
}

}  // namespace block
}  // namespace pccl
