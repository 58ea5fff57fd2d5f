// Rows of tokens into expert order and back: dispatch (one row to many), combine (weighted sum of many) and the
// gradient of combine.  (The gradient of dispatch is combine without weights.)
//
// All three only move memory: a token's row is read once and kept in registers while its copies are written, or
// its sources are read side by side and summed in 32 bits in the order of the choices, so the result does not
// depend on the launch.  Row numbers outside the batch move nothing, whatever put them there.
#include "../common/util.h"
#include "../engine/cuda_driver.h"
#include "vec.cuh"

namespace pccl {
namespace block {

namespace {

constexpr int kThreads = 256;

struct MoveParams {
  MoveArgs a;
  const void* x;
  int64_t ldx;
  const void* d;
  int64_t ldd;
  void* out;
  float* dw;
};

// Eight values at element v of a row of `hidden`: 16 or 32 bytes at once, or one by one where rows are not aligned.
template <typename T, bool kVec> __device__ __forceinline__ void load8(const T* row, int v, int hidden, float* f) {
  if constexpr (kVec) {
    unpack8<T>(load_raw8<T>(row + v), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(row[min(v + i, hidden - 1)]);
  }
}
template <typename T, bool kVec> __device__ __forceinline__ void store8(T* row, int v, int hidden, const float* f) {
  if constexpr (kVec) {
    store_raw8<T>(row + v, pack8<T>(f));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v + i < hidden) row[v + i] = from_f32<T>(f[i]);
  }
}

// Rows behind the last choice become zero.
template <typename T, bool kVec> __device__ __forceinline__ void zero_tail(const MoveArgs& a, T* out) {
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  int64_t used = a.offsets[a.experts];
  used = used < 0 ? 0 : used;
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t r = used + blockIdx.x; r < total; r += gridDim.x)
    for (int v = threadIdx.x * 8; v < a.hidden; v += kThreads * 8)
      store8<T, kVec>(out + r * a.hidden, v, a.hidden, zero);
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) dispatch_rows_kernel(const MoveParams p) {
  const MoveArgs& a = p.a;
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  T* out = static_cast<T*>(p.out);
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const T* src = static_cast<const T*>(p.x) + t * p.ldx;
    for (int v = threadIdx.x * 8; v < a.hidden; v += kThreads * 8) {
      float f[8];
      load8<T, kVec>(src, v, a.hidden, f);
      for (int k = 0; k < a.top_k; ++k) {
        const int64_t r = a.rows[t * a.top_k + k];
        if (r >= 0 && r < total) store8<T, kVec>(out + r * a.hidden, v, a.hidden, f);
      }
    }
  }
  zero_tail<T, kVec>(a, out);
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) combine_rows_kernel(const MoveParams p) {
  const MoveArgs& a = p.a;
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    T* dst = static_cast<T*>(p.out) + t * a.hidden;
    for (int v = threadIdx.x * 8; v < a.hidden; v += kThreads * 8) {
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < a.top_k; ++k) {
        const int64_t r = a.rows[t * a.top_k + k];
        if (r < 0 || r >= total) continue;
        const float w = a.weights ? a.weights[t * a.top_k + k] : 1.f;
        float f[8];
        load8<T, kVec>(static_cast<const T*>(p.x) + r * p.ldx, v, a.hidden, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, f[i], acc[i]);
      }
      store8<T, kVec>(dst, v, a.hidden, acc);
    }
  }
}

// One warp per choice: its row of y and the token's dout pass through once for the product and the scaled copy.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) combine_rows_backward_kernel(const MoveParams p) {
  const MoveArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  T* out = static_cast<T*>(p.out);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); i < total; i += warps) {
    const int64_t r = a.rows[i];
    float dot = 0.f;
    if (r >= 0 && r < total) {
      const float w = a.weights[i];
      const T* y = static_cast<const T*>(p.x) + r * p.ldx;
      const T* d = static_cast<const T*>(p.d) + i / a.top_k * p.ldd;
      for (int v = lane * 8; v < a.hidden; v += 256) {
        float fy[8], fd[8];
        load8<T, kVec>(d, v, a.hidden, fd);
        if (p.dw) {
          load8<T, kVec>(y, v, a.hidden, fy);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (kVec || v + j < a.hidden) dot = fmaf(fy[j], fd[j], dot);
        }
        if (out) {
#pragma unroll
          for (int j = 0; j < 8; ++j) fd[j] *= w;
          store8<T, kVec>(out + r * a.hidden, v, a.hidden, fd);
        }
      }
    }
    if (p.dw) {
      dot = warp_sum(dot);
      if (lane == 0) p.dw[i] = dot;
    }
  }
  if (out) zero_tail<T, kVec>(a, out);
}

bool aligned(const void* p, int64_t ld, DType t) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * dtype_bytes(t) % 16 == 0;
}

int grid_for(int64_t items) {
  int dev = 0, sms = 0;
  PCCL_CUDA(cudaGetDevice(&dev));
  PCCL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int64_t most = 8ll * sms;
  return static_cast<int>(items < 1 ? 1 : items < most ? items : most);
}

}  // namespace

#define PCCL_BLOCK_MOVE(KERNEL, ITEMS, VEC)                                                      \
  PCCL_BLOCK_TYPES(a.dtype, T,                                                                   \
    if (VEC) KERNEL<T, true><<<grid_for(ITEMS), kThreads, 0, stream>>>(p);                       \
    else KERNEL<T, false><<<grid_for(ITEMS), kThreads, 0, stream>>>(p))                          \
  PCCL_CUDA(cudaGetLastError())

void dispatch_rows(const MoveArgs& a, const void* x, int64_t ldx, void* out, cudaStream_t stream) {
  if (a.tokens == 0 || a.hidden == 0) return;
  MoveParams p{a, x, ldx, nullptr, 0, out, nullptr};
  const bool vec = a.hidden % 8 == 0 && aligned(x, ldx, a.dtype) && aligned(out, a.hidden, a.dtype);
  PCCL_BLOCK_MOVE(dispatch_rows_kernel, a.tokens, vec);
}

void combine_rows(const MoveArgs& a, const void* y, int64_t ldy, void* out, cudaStream_t stream) {
  if (a.tokens == 0 || a.hidden == 0) return;
  MoveParams p{a, y, ldy, nullptr, 0, out, nullptr};
  const bool vec = a.hidden % 8 == 0 && aligned(y, ldy, a.dtype) && aligned(out, a.hidden, a.dtype);
  PCCL_BLOCK_MOVE(combine_rows_kernel, a.tokens, vec);
}

void combine_rows_backward(const MoveArgs& a, const void* y, int64_t ldy, const void* dout, int64_t ldd, void* dy,
                           float* dw, cudaStream_t stream) {
  if (a.tokens == 0 || (dy == nullptr && dw == nullptr)) return;
  MoveParams p{a, y, ldy, dout, ldd, dy, dw};
  const bool vec = a.hidden % 8 == 0 && aligned(y, ldy, a.dtype) && aligned(dout, ldd, a.dtype) &&
                   (dy == nullptr || aligned(dy, a.hidden, a.dtype));
  PCCL_BLOCK_MOVE(combine_rows_backward_kernel, static_cast<int64_t>(a.tokens) * a.top_k / 4, vec);
}

}  // namespace block
}  // namespace pccl
