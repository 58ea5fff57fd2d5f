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

// Sum over the threads of a row; `sums` alternates between two sets so that one barrier a call is enough.
__device__ __forceinline__ float row_sum(float v, float (*sums)[32], int* turn) {
  v = warp_sum(v);
  if (blockDim.x == 32) return v;
  float* s = sums[*turn];
  *turn ^= 1;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = static_cast<int>(threadIdx.x & 31) < warps ? s[threadIdx.x & 31] : 0.f;
  return warp_sum(v);
}

template <typename TX, typename TR, bool kVec, int kMost>
__global__ void __launch_bounds__(kMost) norm_forward_kernel(const NormParams p) {
  __shared__ float sums[2][32];
  const NormArgs& a = p.a;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  int turn = 0;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < a.rows;
       t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    float v[kHeld], h[kHeld], w[kHeld];
    load_row<TR, kVec>(static_cast<const TR*>(a.residual) + t * a.ldr, n, tid, width, h);
    if (a.x) {
      load_row<TX, kVec>(static_cast<const TX*>(a.x) + t * a.ldx, n, tid, width, v);
      if (a.post_gamma.ptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) ss = fmaf(v[i], v[i], ss);
        const float r1 = rsqrtf(row_sum(ss, sums, &turn) * inv_n + a.eps);
        if (p.r1 && tid == 0) p.r1[t] = r1;
        load_weight<TX, kVec>(a.post_gamma, 0, n, tid, width, w);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) v[i] = v[i] * r1 * w[i];
      }
      if (a.gate.ptr) {
        load_weight<TX, kVec>(a.gate, t / a.gate_rows * n, n, tid, width, w);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) v[i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < kHeld; ++i) h[i] = fmaf(a.scale, h[i], v[i]);
    }
    if (p.h) store_row<TR, kVec>(static_cast<TR*>(p.h) + t * n, n, tid, width, h);
    if (a.gamma.ptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) ss = fmaf(h[i], h[i], ss);
      const float r2 = rsqrtf(row_sum(ss, sums, &turn) * inv_n + a.eps);
      if (p.r2 && tid == 0) p.r2[t] = r2;
      load_weight<TX, kVec>(a.gamma, 0, n, tid, width, w);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) w[i] *= h[i] * r2;
      store_row<TX, kVec>(static_cast<TX*>(p.y) + t * n, n, tid, width, w);
    }
  }
}

// First row of worker w's run; w = workers gives the number of rows.
__device__ __forceinline__ int64_t run_start(int64_t rows, int workers, int w) {
  return rows / workers * w + min(static_cast<int64_t>(w), rows % workers);
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_weight_grad(void* out, int f32, int64_t first, int n, int tid, int width,
                                                  const float* f) {
  if (f32) store_row<float, kVec>(static_cast<float*>(out) + first, n, tid, width, f);
  else store_row<T, kVec>(static_cast<T*>(out) + first, n, tid, width, f);
}

template <typename TX, typename TR, bool kVec, bool kFull, int kMost>
__global__ void __launch_bounds__(kMost) norm_backward_kernel(const NormParams p) {
  __shared__ float sums[2][32];
  const NormArgs& a = p.a;
  const NormGrads& g = p.g;
  const int tid = threadIdx.x, width = blockDim.x, n = a.hidden;
  const float inv_n = 1.f / static_cast<float>(n);
  const int worker = blockIdx.x * blockDim.y + threadIdx.y;
  if (worker >= p.workers) return;                 // whole warps of a block of warps
  const int64_t begin = run_start(a.rows, p.workers, worker), end = run_start(a.rows, p.workers, worker + 1);
  int turn = 0;
  float acc_gamma[kHeld], acc_post[kFull ? kHeld : 1], acc_gate[kFull ? kHeld : 1];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    acc_gamma[i] = 0.f;
    if (kFull) { acc_post[i] = 0.f; acc_gate[i] = 0.f; }
  }

  for (int64_t t = begin; t < end; ++t) {
    float d[kHeld], w[kHeld], u[kHeld], gate[kHeld];
    float r1 = 0.f;
    if (g.dh) {
      load_row<TR, kVec>(static_cast<const TR*>(g.dh) + t * g.lddh, n, tid, width, d);
    } else {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) d[i] = 0.f;
    }
    // u: the block's output after the norm behind it (kFull) or as it came.
    const bool need_u = kFull || (g.dy && !g.h && a.x);
    if (need_u) {
      load_row<TX, kVec>(static_cast<const TX*>(a.x) + t * a.ldx, n, tid, width, u);
      if (kFull && a.post_gamma.ptr) {
        r1 = g.r1[t];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) u[i] *= r1;          // n1
      }
    }
    if (kFull && a.gate.ptr) load_weight<TX, kVec>(a.gate, t / a.gate_rows * n, n, tid, width, gate);
    if (g.dy) {
      float h[kHeld];
      if (g.h) {
        load_row<float, kVec>(static_cast<const float*>(g.h) + t * n, n, tid, width, h);
      } else {
        load_row<TR, kVec>(static_cast<const TR*>(a.residual) + t * a.ldr, n, tid, width, h);
        if (a.x) {
          if (kFull && a.post_gamma.ptr) load_weight<TX, kVec>(a.post_gamma, 0, n, tid, width, w);
#pragma unroll
          for (int i = 0; i < kHeld; ++i) {
            float v = u[i];
            if (kFull && a.post_gamma.ptr) v *= w[i];
            if (kFull && a.gate.ptr) v *= gate[i];
            h[i] = fmaf(a.scale, h[i], v);
          }
        }
      }
      const float r2 = g.r2[t];
      float dy[kHeld];
      load_row<TX, kVec>(static_cast<const TX*>(g.dy) + t * g.lddy, n, tid, width, dy);
      load_weight<TX, kVec>(a.gamma, 0, n, tid, width, w);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        h[i] *= r2;                                          // n2
        acc_gamma[i] = fmaf(dy[i], h[i], acc_gamma[i]);
        dy[i] *= w[i];
        dot = fmaf(dy[i], h[i], dot);
      }
      const float mean = row_sum(dot, sums, &turn) * inv_n;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) d[i] = fmaf(r2, dy[i] - h[i] * mean, d[i]);
    }
    if (g.dresidual) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) w[i] = a.scale * d[i];
      store_row<TR, kVec>(static_cast<TR*>(g.dresidual) + t * n, n, tid, width, w);
    }
    if constexpr (kFull) {
      if (a.post_gamma.ptr) load_weight<TX, kVec>(a.post_gamma, 0, n, tid, width, w);
      if (a.gate.ptr) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          acc_gate[i] = fmaf(d[i], a.post_gamma.ptr ? u[i] * w[i] : u[i], acc_gate[i]);
          d[i] *= gate[i];
        }
        // The group's last row: its sum is whole if this run held all of the group, else a part.
        const int64_t group = t / a.gate_rows;
        if ((t + 1) % a.gate_rows == 0 || t + 1 == end) {
          if (g.dgate) {
            const bool whole = group * a.gate_rows >= begin && (group + 1) * a.gate_rows <= end;
            if (whole) {
              store_weight_grad<TX, kVec>(g.dgate, a.gate.f32, group * n, n, tid, width, acc_gate);
            } else {
              const int slot = group * a.gate_rows <= begin ? 0 : 1;
              store_row<float, kVec>(p.part_gate + (static_cast<int64_t>(worker) * 2 + slot) * n, n, tid, width, acc_gate);
            }
          }
#pragma unroll
          for (int i = 0; i < kHeld; ++i) acc_gate[i] = 0.f;
        }
      }
      if (a.post_gamma.ptr) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          acc_post[i] = fmaf(d[i], u[i], acc_post[i]);
          d[i] *= w[i];
          dot = fmaf(d[i], u[i], dot);
        }
        const float mean = row_sum(dot, sums, &turn) * inv_n;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) d[i] = r1 * (d[i] - u[i] * mean);
      }
    }
    if (g.dx) store_row<TX, kVec>(static_cast<TX*>(g.dx) + t * n, n, tid, width, d);
  }
  if (p.part_gamma) store_row<float, kVec>(p.part_gamma + static_cast<int64_t>(worker) * n, n, tid, width, acc_gamma);
  if constexpr (kFull)
    if (p.part_post) store_row<float, kVec>(p.part_post + static_cast<int64_t>(worker) * n, n, tid, width, acc_post);
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
      for (int w = first + strip; w < last; w += 8) {
        const float* at = src + w * step;
        if (what >= 2 && group * a.gate_rows > run_start(a.rows, p.workers, w)) at += n;
        sum += at[col];
      }
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
  return a.hidden % 8 == 0 && aligned(a.x, a.ldx, dtype_bytes(a.xt)) && aligned(a.residual, a.ldr, dtype_bytes(a.rt)) &&
         aligned(a.gamma, a.hidden, a.xt) && aligned(a.post_gamma, a.hidden, a.xt) && aligned(a.gate, a.hidden, a.xt);
}

// Workers of the backward kernel: two blocks' worth per SM, each with at least one row.
int worker_count(const NormArgs& a) {
  const int64_t most = 2ll * sm_count() * shape_of(a.hidden).rows_per_block;
  return static_cast<int>(a.rows < most ? a.rows : most);
}

template <typename TX, typename TR, int kMost>
void forward_typed(const NormParams& p, bool vec, cudaStream_t stream) {
  const Shape s = shape_of(p.a.hidden);
  const int64_t want = (p.a.rows + s.rows_per_block - 1) / s.rows_per_block, most = 16ll * sm_count();
  const int grid = static_cast<int>(want < most ? want : most);
  if (vec) norm_forward_kernel<TX, TR, true, kMost><<<grid, s.block, 0, stream>>>(p);
  else norm_forward_kernel<TX, TR, false, kMost><<<grid, s.block, 0, stream>>>(p);
}

template <typename TX, typename TR, int kMost>
void backward_typed(const NormParams& p, bool vec, cudaStream_t stream) {
  const Shape s = shape_of(p.a.hidden);
  const int grid = (p.workers + s.rows_per_block - 1) / s.rows_per_block;
  const bool full = p.a.post_gamma.ptr || p.a.gate.ptr;
  if (vec && full) norm_backward_kernel<TX, TR, true, true, kMost><<<grid, s.block, 0, stream>>>(p);
  else if (vec) norm_backward_kernel<TX, TR, true, false, kMost><<<grid, s.block, 0, stream>>>(p);
  else if (full) norm_backward_kernel<TX, TR, false, true, kMost><<<grid, s.block, 0, stream>>>(p);
  else norm_backward_kernel<TX, TR, false, false, kMost><<<grid, s.block, 0, stream>>>(p);
}

template <typename TX, typename TR>
void sized(const NormParams& p, bool vec, bool backward, cudaStream_t stream) {
  const bool many = shape_of(p.a.hidden).block.x > 512;      // 64 registers a thread instead of 128
  if (backward && many) backward_typed<TX, TR, 1024>(p, vec, stream);
  else if (backward) backward_typed<TX, TR, 512>(p, vec, stream);
  else if (many) forward_typed<TX, TR, 1024>(p, vec, stream);
  else forward_typed<TX, TR, 512>(p, vec, stream);
}

// TR is TX or 32 bits.
template <typename TX>
void any_typed(const NormParams& p, bool vec, bool backward, cudaStream_t stream) {
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
