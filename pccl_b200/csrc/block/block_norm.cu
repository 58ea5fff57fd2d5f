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

constexpr int kHeld = 16;                      // values a thread holds of its row

// They stand in groups of consecutive columns, as many as 16 bytes of the widest type hold: a warp then touches
// whole 32-byte sectors in every access.  (Eight columns of 32 bits a thread, as two accesses 32 bytes apart from
// lane to lane, moved every sector twice.)
template <typename TX, typename TR> constexpr int kGroup = sizeof(TX) == 4 || sizeof(TR) == 4 ? 4 : 8;

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

// Column of value j of group v held by a thread: G in a row where rows are aligned, else a thread's values stand a
// whole row of threads apart, so that neighbours read neighbours.
template <bool kVec, int G> __device__ __forceinline__ int column(int v, int j, int tid, int width) {
  return kVec ? (v * width + tid) * G + j : (v * G + j) * width + tid;
}

// G values as they lie in memory.
template <typename T, int G> struct alignas(G * sizeof(T) > 16 ? 16 : G * sizeof(T)) Raw { uint32_t w[G * sizeof(T) / 4]; };

template <typename T, int G> __device__ __forceinline__ void unpack(const Raw<T, G>& r, float2* f) {
#pragma unroll
  for (int i = 0; i < G / 2; ++i) {
    if constexpr (sizeof(T) == 4) f[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else unpack2(r.w[i], &f[i].x, T());
  }
}
template <typename T, int G> __device__ __forceinline__ Raw<T, G> pack(const float2* f) {
  Raw<T, G> r;
#pragma unroll
  for (int i = 0; i < G / 2; ++i) {
    if constexpr (sizeof(T) == 4) {
      r.w[2 * i] = __float_as_uint(f[i].x);
      r.w[2 * i + 1] = __float_as_uint(f[i].y);
    } else {
      r.w[i] = pack2(f[i].x, f[i].y, T());
    }
  }
  return r;
}

// The values of group v, from the row itself.
template <typename T, bool kVec, int G>
__device__ __forceinline__ void load_group(const T* row, int v, int hidden, int tid, int width, float2* to) {
  if constexpr (kVec) {
    const int at = (v * width + tid) * G;
    if (at < hidden) {
      unpack<T, G>(*reinterpret_cast<const Raw<T, G>*>(row + at), to);
    } else {
#pragma unroll
      for (int j = 0; j < G / 2; ++j) to[j] = make_float2(0.f, 0.f);
    }
  } else {
    float* f = reinterpret_cast<float*>(to);
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int at = column<false, G>(v, j, tid, width);
      f[j] = at < hidden ? to_f32<T>(row[at]) : 0.f;
    }
  }
}
template <typename T, bool kVec, int G>
__device__ __forceinline__ void store_group(T* row, int v, int hidden, int tid, int width, const float2* from) {
  if constexpr (kVec) {
    const int at = (v * width + tid) * G;
    if (at < hidden) *reinterpret_cast<Raw<T, G>*>(row + at) = pack<T, G>(from);
  } else {
    const float* f = reinterpret_cast<const float*>(from);
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int at = column<false, G>(v, j, tid, width);
      if (at < hidden) row[at] = from_f32<T>(f[j]);
    }
  }
}
template <typename T, bool kVec, int G>
__device__ __forceinline__ void store_row(T* row, int hidden, int tid, int width, const float2* f) {
#pragma unroll
  for (int v = 0; v < kHeld / G; ++v) store_group<T, kVec, G>(row, v, hidden, tid, width, f + v * (G / 2));
}
// A weight vector is of the activations' type or of 32 bits.
template <typename T, bool kVec, int G>
__device__ __forceinline__ void load_weight(const Weight& w, int64_t first, int hidden, int tid, int width, float2* f) {
#pragma unroll
  for (int v = 0; v < kHeld / G; ++v) {
    if (w.f32) load_group<float, kVec, G>(static_cast<const float*>(w.ptr) + first, v, hidden, tid, width, f + v * (G / 2));
    else load_group<T, kVec, G>(static_cast<const T*>(w.ptr) + first, v, hidden, tid, width, f + v * (G / 2));
  }
}

// ---- ring ------------------------------------------------------------------------------------------------
// A thread's share of a row of T in the ring: kHeld values.
template <typename T> constexpr int kBytes = kHeld * static_cast<int>(sizeof(T));

// `kSize` bytes (8 or 16), or as many zeros.
template <int kSize> __device__ __forceinline__ void copy_async(void* to, const void* from, bool zeros) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  const int size = zeros ? 0 : kSize;
  if constexpr (kSize == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(size) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

template <typename T, int G>
__device__ __forceinline__ void fetch_row(char* slot, const T* row, int hidden, int tid, int width) {
#pragma unroll
  for (int v = 0; v < kHeld / G; ++v) {
    const int at = (v * width + tid) * G;
    const bool beyond = at >= hidden;
    copy_async<G * sizeof(T)>(slot + (v * width + tid) * (G * sizeof(T)), row + (beyond ? 0 : at), beyond);
  }
}

// The values of group v: from the ring, or from the row itself.
template <typename T, bool kVec, bool kHeldRow, int G>
__device__ __forceinline__ void take(const char* slot, const T* row, int v, int hidden, int tid, int width, float2* to) {
  if constexpr (kHeldRow) unpack<T, G>(*reinterpret_cast<const Raw<T, G>*>(slot + (v * width + tid) * (G * sizeof(T))), to);
  else load_group<T, kVec, G>(row, v, hidden, tid, width, to);
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

// A thread's slots of one weight: kHeld 32-bit values, four to an access.
__device__ __forceinline__ void slots_store(char* slot, int tid, int width, const float2* f) {
#pragma unroll
  for (int i = 0; i < kHeld / 4; ++i)
    reinterpret_cast<float4*>(slot)[i * width + tid] = make_float4(f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y);
}
template <int G> __device__ __forceinline__ void slots_load(const char* slot, int v, int tid, int width, float2* f) {
#pragma unroll
  for (int i = 0; i < G / 4; ++i) {
    const float4 q = reinterpret_cast<const float4*>(slot)[(v * (G / 4) + i) * width + tid];
    f[2 * i] = make_float2(q.x, q.y);
    f[2 * i + 1] = make_float2(q.z, q.w);
  }
}

// g1 = post_gamma * gate of one group of rows into its slots (what is absent counts as 1).
template <typename T, bool kVec, int G>
__device__ __forceinline__ void form_g1(const NormArgs& a, int64_t group, char* slot, int tid, int width) {
  float2 f[kHeld / 2], w[kHeld / 2];
  if (a.post_gamma.ptr) load_weight<T, kVec, G>(a.post_gamma, 0, a.hidden, tid, width, f);
  if (a.gate.ptr) {
    load_weight<T, kVec, G>(a.gate, group * a.hidden, a.hidden, tid, width, w);
#pragma unroll
    for (int i = 0; i < kHeld / 2; ++i) f[i] = a.post_gamma.ptr ? mul2(f[i], w[i]) : w[i];
  }
  slots_store(slot, tid, width, f);
}

// First row of worker w's run; w = workers gives the number of rows.
__device__ __forceinline__ int64_t run_start(int64_t rows, int workers, int w) {
  return rows / workers * w + min(static_cast<int64_t>(w), rows % workers);
}

// Slots of a worker, in bytes a thread: gamma, g1, (backward) the sum that becomes dpost_gamma, then the rows of
// the ring.
__host__ __device__ __forceinline__ bool has_g1(const NormArgs& a) { return a.post_gamma.ptr || a.gate.ptr; }
__host__ __device__ __forceinline__ int weight_bytes(const NormArgs& a, bool backward) {
  return kBytes<float> * ((a.gamma.ptr ? 1 : 0) + (has_g1(a) ? 1 : 0) + (backward && a.post_gamma.ptr && a.gate.ptr ? 1 : 0));
}
template <typename TX, typename TR> __host__ __device__ __forceinline__ int forward_bytes(const NormArgs& a) {
  return kBytes<TR> + (a.x ? kBytes<TX> : 0);
}
template <typename TX, typename TR> __host__ __device__ __forceinline__ int backward_bytes(const NormArgs& a, const NormGrads& g) {
  int bytes = 0;
  if (g.dh) bytes += kBytes<TR>;
  if (g.dy) bytes += kBytes<TX> + (g.h ? kBytes<float> : kBytes<TR>);
  if (a.x) bytes += kBytes<TX>;
  return bytes;
}

template <typename TX, typename TR, bool kVec, int kRing, int kMost>
__global__ void __launch_bounds__(kMost, 1) norm_forward_kernel(const NormParams p) {
  __shared__ RowSums sums;
  constexpr int G = kGroup<TX, TR>, kGroups = kHeld / G;
  extern __shared__ __align__(16) char slots[];
  const NormArgs& a = p.a;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  row_sum_clear(sums);
  const int worker = blockIdx.x * blockDim.y + threadIdx.y;
  if (worker >= p.workers) return;                 // whole warps of a block of warps
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);

  const int stage = kRing ? forward_bytes<TX, TR>(a) * width : 0, weights = weight_bytes(a, false) * width;
  char* const gammas = slots + (weights + kRing * stage) * threadIdx.y;
  char* const g1 = gammas + (a.gamma.ptr ? kBytes<float> * width : 0);
  char* const ring = gammas + weights;
  const auto fetch = [&](int64_t row, int s) {
    if (row < end) {
      fetch_row<TR, G>(ring + s * stage, static_cast<const TR*>(a.residual) + row * a.ldr, n, tid, width);
      if (a.x) fetch_row<TX, G>(ring + s * stage + kBytes<TR> * width, static_cast<const TX*>(a.x) + row * a.ldx, n, tid, width);
    }
    copies_commit();
  };
  if constexpr (kRing > 0) {
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) fetch(begin + s, s);
  }
  if (a.gamma.ptr) {
    float2 w[kHeld / 2];
    load_weight<TX, kVec, G>(a.gamma, 0, n, tid, width, w);
    slots_store(gammas, tid, width, w);
  }
  int64_t group = 0, left = 0;                     // rows left of the present group of rows that share a gate
  if (has_g1(a)) {
    group = a.gate.ptr ? begin / a.gate_rows : 0;
    left = a.gate.ptr ? (group + 1) * a.gate_rows - begin : a.rows;
    form_g1<TX, kVec, G>(a, group, g1, tid, width);
  }

  constexpr bool kHeldRow = kRing > 0;
  int turn = 0, s = 0;
  for (int64_t t = begin; t < end; ++t) {
    const char* held = ring + s * stage;
    if constexpr (kHeldRow) {
      fetch(t + kRing - 1, s == 0 ? kRing - 1 : s - 1);
      s = s + 1 == kRing ? 0 : s + 1;
      copies_wait<kRing - 1>();
    }
    const TX* const row_x = static_cast<const TX*>(a.x) + t * a.ldx;
    float2 x[kHeld / 2], h[kHeld / 2];
    float r1 = 1.f;
    if (a.x) {
      float2 ss = both(0.f);
#pragma unroll
      for (int v = 0; v < kGroups; ++v) {
        take<TX, kVec, kHeldRow, G>(held + kBytes<TR> * width, row_x, v, n, tid, width, x + v * (G / 2));
#pragma unroll
        for (int j = 0; j < G / 2; ++j) ss = fma2(x[v * (G / 2) + j], x[v * (G / 2) + j], ss);
      }
      if (a.post_gamma.ptr) {
        r1 = rsqrtf(row_sum(ss.x + ss.y, sums, &turn) * inv_n + a.eps);
        if (p.r1 && tid == 0) p.r1[t] = r1;
      }
      if (has_g1(a)) {
        if (left == 0) {
          form_g1<TX, kVec, G>(a, ++group, g1, tid, width);
          left = a.gate_rows;
        }
        --left;
      }
    }
    float2 ss = both(0.f);
#pragma unroll
    for (int v = 0; v < kGroups; ++v) {
      take<TR, kVec, kHeldRow, G>(held, static_cast<const TR*>(a.residual) + t * a.ldr, v, n, tid, width, h + v * (G / 2));
      if (a.x) {
        if (has_g1(a)) {
          float2 w[G / 2];
          slots_load<G>(g1, v, tid, width, w);
#pragma unroll
          for (int j = 0; j < G / 2; ++j) x[v * (G / 2) + j] = mul2(mul2(x[v * (G / 2) + j], both(r1)), w[j]);
        }
#pragma unroll
        for (int j = 0; j < G / 2; ++j) h[v * (G / 2) + j] = fma2(both(a.scale), h[v * (G / 2) + j], x[v * (G / 2) + j]);
      }
#pragma unroll
      for (int j = 0; j < G / 2; ++j) ss = fma2(h[v * (G / 2) + j], h[v * (G / 2) + j], ss);
      if (p.h) store_group<TR, kVec, G>(static_cast<TR*>(p.h) + t * n, v, n, tid, width, h + v * (G / 2));
    }
    if (a.gamma.ptr) {
      const float r2 = rsqrtf(row_sum(ss.x + ss.y, sums, &turn) * inv_n + a.eps);
      if (p.r2 && tid == 0) p.r2[t] = r2;
#pragma unroll
      for (int v = 0; v < kGroups; ++v) {
        float2 w[G / 2];
        slots_load<G>(gammas, v, tid, width, w);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) w[j] = mul2(mul2(h[v * (G / 2) + j], both(r2)), w[j]);
        store_group<TX, kVec, G>(static_cast<TX*>(p.y) + t * n, v, n, tid, width, w);
      }
    }
  }
  if constexpr (kHeldRow) copies_wait<0>();
}

template <typename T, bool kVec, int G>
__device__ __forceinline__ void store_weight_grad(void* out, int f32, int64_t first, int n, int tid, int width,
                                                  const float2* f) {
  if (f32) store_row<float, kVec, G>(static_cast<float*>(out) + first, n, tid, width, f);
  else store_row<T, kVec, G>(static_cast<T*>(out) + first, n, tid, width, f);
}

// kRing: rows in shared memory (0: loaded directly).  kFull: a gate or a norm behind the block.
template <typename TX, typename TR, bool kVec, int kRing, bool kFull, int kMost>
__global__ void __launch_bounds__(kMost, 1) norm_backward_kernel(const NormParams p) {
  __shared__ RowSums sums;
  constexpr int G = kGroup<TX, TR>, kGroups = kHeld / G;
  extern __shared__ __align__(16) char slots[];
  const NormArgs& a = p.a;
  const NormGrads& g = p.g;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  row_sum_clear(sums);
  const int worker = blockIdx.x * blockDim.y + threadIdx.y;
  if (worker >= p.workers) return;                 // whole warps of a block of warps
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);

  const int stage = kRing ? backward_bytes<TX, TR>(a, g) * width : 0, weights = weight_bytes(a, true) * width;
  char* const gammas = slots + (weights + kRing * stage) * threadIdx.y;
  char* const g1 = gammas + (a.gamma.ptr ? kBytes<float> * width : 0);
  char* const acc_post = g1 + kBytes<float> * width;        // where there are a gate and a norm behind
  char* const ring = gammas + weights;
  const int off_dy = g.dh ? kBytes<TR> * width : 0;
  const int off_h = off_dy + (g.dy ? kBytes<TX> * width : 0);
  const int off_x = off_h + (g.dy ? (g.h ? kBytes<float> : kBytes<TR>) * width : 0);
  const auto fetch = [&](int64_t row, int s) {
    if (row < end) {
      char* to = ring + s * stage;
      if (g.dh) fetch_row<TR, G>(to, static_cast<const TR*>(g.dh) + row * g.lddh, n, tid, width);
      if (g.dy) {
        fetch_row<TX, G>(to + off_dy, static_cast<const TX*>(g.dy) + row * g.lddy, n, tid, width);
        if (g.h) fetch_row<float, G>(to + off_h, static_cast<const float*>(g.h) + row * n, n, tid, width);
        else fetch_row<TR, G>(to + off_h, static_cast<const TR*>(a.residual) + row * a.ldr, n, tid, width);
      }
      if (a.x) fetch_row<TX, G>(to + off_x, static_cast<const TX*>(a.x) + row * a.ldx, n, tid, width);
    }
    copies_commit();
  };
  if constexpr (kRing > 0) {
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) fetch(begin + s, s);
  }

  float2 acc_gamma[kHeld / 2], acc_s[kFull ? kHeld / 2 : 1];
#pragma unroll
  for (int i = 0; i < kHeld / 2; ++i) {
    acc_gamma[i] = both(0.f);
    if (kFull) acc_s[i] = both(0.f);
  }
  if (a.gamma.ptr) {
    float2 w[kHeld / 2];
    load_weight<TX, kVec, G>(a.gamma, 0, n, tid, width, w);
    slots_store(gammas, tid, width, w);
  }
  int64_t group = 0, left = 0;                     // rows left of the present group of rows that share a gate
  if (kFull) {
    group = a.gate.ptr ? begin / a.gate_rows : 0;
    left = a.gate.ptr ? (group + 1) * a.gate_rows - begin : a.rows;
    form_g1<TX, kVec, G>(a, group, g1, tid, width);
    if (a.post_gamma.ptr && a.gate.ptr) slots_store(acc_post, tid, width, acc_gamma);
  }
  float next_r1 = kFull && a.post_gamma.ptr && begin < end ? g.r1[begin] : 1.f;
  float next_r2 = g.dy && begin < end ? g.r2[begin] : 0.f;

  int turn = 0, s = 0;
  for (int64_t t = begin; t < end; ++t) {
    const float r1 = next_r1, r2 = next_r2;
    if (t + 1 < end) {
      if (kFull && a.post_gamma.ptr) next_r1 = g.r1[t + 1];
      if (g.dy) next_r2 = g.r2[t + 1];
    }
    constexpr bool kHeldRow = kRing > 0;
    const char* held = ring + s * stage;
    if constexpr (kHeldRow) {
      fetch(t + kRing - 1, s == 0 ? kRing - 1 : s - 1);
      s = s + 1 == kRing ? 0 : s + 1;
      copies_wait<kRing - 1>();
    }
    const TX* const row_x = static_cast<const TX*>(a.x) + t * a.ldx;
    // The row is gone through in groups of eight values, and inputs are read again rather than kept: what stays in
    // registers over a barrier are the two sums of the weights' gradients and two values a column.
    float2 d[kHeld / 2], n2[kHeld / 2];
    if (g.dy) {
      float2 dot = both(0.f);
#pragma unroll
      for (int v = 0; v < kGroups; ++v) {
        float2 f[G / 2], w[G / 2];
        float2* const h = n2 + v * (G / 2);
        if (g.h) {
          take<float, kVec, kHeldRow, G>(held + off_h, static_cast<const float*>(g.h) + t * n, v, n, tid, width, h);
        } else {
          take<TR, kVec, kHeldRow, G>(held + off_h, static_cast<const TR*>(a.residual) + t * a.ldr, v, n, tid, width, h);
          if (a.x) {
            take<TX, kVec, kHeldRow, G>(held + off_x, row_x, v, n, tid, width, f);
            if (kFull) {
              slots_load<G>(g1, v, tid, width, w);
#pragma unroll
              for (int j = 0; j < G / 2; ++j) f[j] = mul2(mul2(f[j], both(r1)), w[j]);
            }
#pragma unroll
            for (int j = 0; j < G / 2; ++j) h[j] = fma2(both(a.scale), h[j], f[j]);
          }
        }
        take<TX, kVec, kHeldRow, G>(held + off_dy, static_cast<const TX*>(g.dy) + t * g.lddy, v, n, tid, width, f);
        slots_load<G>(gammas, v, tid, width, w);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) {
          h[j] = mul2(h[j], both(r2));
          acc_gamma[v * (G / 2) + j] = fma2(f[j], h[j], acc_gamma[v * (G / 2) + j]);
          d[v * (G / 2) + j] = mul2(f[j], w[j]);
          dot = fma2(d[v * (G / 2) + j], h[j], dot);
        }
      }
      const float pull = -r2 * inv_n * row_sum(dot.x + dot.y, sums, &turn);
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
        take<TR, kVec, kHeldRow, G>(held, static_cast<const TR*>(g.dh) + t * g.lddh, v, n, tid, width, f);
#pragma unroll
        for (int j = 0; j < G / 2; ++j) d[v * (G / 2) + j] = add2(d[v * (G / 2) + j], f[j]);
      }
      if (g.dresidual) {
#pragma unroll
        for (int j = 0; j < G / 2; ++j) f[j] = mul2(both(a.scale), d[v * (G / 2) + j]);
        store_group<TR, kVec, G>(static_cast<TR*>(g.dresidual) + t * n, v, n, tid, width, f);
      }
      if constexpr (kFull) {
        take<TX, kVec, kHeldRow, G>(held + off_x, row_x, v, n, tid, width, f);
        slots_load<G>(g1, v, tid, width, w);
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
      const float pull = -r1 * r1 * inv_n * row_sum(dot.x + dot.y, sums, &turn);
      if (g.dx) {
#pragma unroll
        for (int v = 0; v < kGroups; ++v) {
          float2 f[G / 2];
          take<TX, kVec, kHeldRow, G>(held + off_x, row_x, v, n, tid, width, f);
#pragma unroll
          for (int j = 0; j < G / 2; ++j) f[j] = fma2(both(r1), d[v * (G / 2) + j], mul2(both(pull), f[j]));
          store_group<TX, kVec, G>(static_cast<TX*>(g.dx) + t * n, v, n, tid, width, f);
        }
      }
    } else if (g.dx) {
#pragma unroll
      for (int v = 0; v < kGroups; ++v) store_group<TX, kVec, G>(static_cast<TX*>(g.dx) + t * n, v, n, tid, width, d + v * (G / 2));
    }
    if constexpr (kFull) {
      if (--left == 0 || t + 1 == end) {
        if (a.gate.ptr) {
          // The group's last row here: dgate is whole if this run held all of the group, else a part.
          if (a.post_gamma.ptr) {
            float2 w[kHeld / 2], sum[kHeld / 2];
            load_weight<TX, kVec, G>(a.gate, group * n, n, tid, width, w);
            slots_load<kHeld>(acc_post, 0, tid, width, sum);
#pragma unroll
            for (int i = 0; i < kHeld / 2; ++i) sum[i] = fma2(w[i], acc_s[i], sum[i]);
            slots_store(acc_post, tid, width, sum);
            load_weight<TX, kVec, G>(a.post_gamma, 0, n, tid, width, w);
#pragma unroll
            for (int i = 0; i < kHeld / 2; ++i) acc_s[i] = mul2(acc_s[i], w[i]);
          }
          if (g.dgate) {
            if (group * a.gate_rows >= begin && (group + 1) * a.gate_rows <= end) {
              store_weight_grad<TX, kVec, G>(g.dgate, a.gate.f32, group * n, n, tid, width, acc_s);
            } else {
              const int slot = group * a.gate_rows <= begin ? 0 : 1;
              store_row<float, kVec, G>(p.part_gate + (static_cast<int64_t>(worker) * 2 + slot) * n, n, tid, width, acc_s);
            }
          }
#pragma unroll
          for (int i = 0; i < kHeld / 2; ++i) acc_s[i] = both(0.f);
          if (t + 1 < end) form_g1<TX, kVec, G>(a, ++group, g1, tid, width);
          left = a.gate_rows;
        }
      }
    }
  }
  if constexpr (kRing > 0) copies_wait<0>();
  if (p.part_gamma) store_row<float, kVec, G>(p.part_gamma + static_cast<int64_t>(worker) * n, n, tid, width, acc_gamma);
  if constexpr (kFull) {
    if (p.part_post) {
      if (a.gate.ptr) slots_load<kHeld>(acc_post, 0, tid, width, acc_s);
      store_row<float, kVec, G>(p.part_post + static_cast<int64_t>(worker) * n, n, tid, width, acc_s);
    }
  }
}

// Adds the workers' parts in their order: blockIdx.y 0 gamma, 1 post_gamma, 2.. the groups of gate rows.
template <typename T>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const NormParams p) {
  __shared__ float part[8][32];
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
      // Only the first of them can have begun with another group: its part stands in the second place.
      if (strip == 0 && what >= 2) {
        sum = src[first * step + (group * a.gate_rows > run_start(a.rows, p.workers, first) ? n : 0) + col];
        ++first;
      } else if (what >= 2) {
        ++first;
      }
      const float* at = src + (first + strip) * step + col;
#pragma unroll 8
      for (int w = first + strip; w < last; w += 8, at += 8 * step) sum += *at;
    }
    part[strip][lane] = sum;
    __syncthreads();
    if (strip == 0 && col < n) {
#pragma unroll
      for (int s = 1; s < 8; ++s) sum += part[s][lane];
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
  const bool wide = a.xt == DType::kF32 || a.rt == DType::kF32;
  return a.hidden % (wide ? 4 : 8) == 0 && aligned(a.x, a.ldx, dtype_bytes(a.xt)) && aligned(a.residual, a.ldr, dtype_bytes(a.rt)) &&
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
  const size_t weights = static_cast<size_t>(weight_bytes(p.a, false)) * threads;
  const size_t row = static_cast<size_t>(forward_bytes<TX, TR>(p.a)) * threads;
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
  const size_t weights = static_cast<size_t>(weight_bytes(p.a, true)) * threads;
  const size_t row = static_cast<size_t>(backward_bytes<TX, TR>(p.a, p.g)) * threads;
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
    PCCL_BLOCK_TYPES(a.xt, T, norm_reduce_kernel<T><<<grid, 256, 0, stream>>>(p))
    PCCL_CUDA(cudaGetLastError());
  }
}

}  // namespace block
}  // namespace pccl
