// Rows of tokens into expert order and back: dispatch (one row to many), combine (weighted sum of many) and the
// gradient of combine.  (The gradient of dispatch is combine without weights.)
//
// All three only move memory: a token's row is read once for all its copies, or its sources are read side by side
// and summed in 32 bits in the order of the choices, so the result does not depend on the launch.  Row numbers
// outside the batch move nothing, whatever put them there.
//
// A batch in expert order may have rows that no choice names: the last ones, where tokens are masked, and any others,
// where a caller has left choices out.  They become zero, which takes knowing the named ones.  Up to kScan choices every
// block marks them as bits in its shared memory.  Beyond that a kernel ahead of the move notes each row's choice,
// namer[row] = choice, in memory that nobody has cleared: a row is named if its entry is a choice that names it, and what
// else stands there cannot pass for one.  It runs beside the move, which waits for it only before it looks for rows to
// clear.
//
// Work goes by chunks of 16 bytes of what is written.  Rows need not begin at 16 bytes (odd sizes, cut views): a
// chunk's values then lie in two neighbouring 16-byte blocks of the source, which are loaded whole and shifted
// together; only a row's first and last chunk go value by value.
#include "../common/util.h"
#include "../engine/cuda_driver.h"
#include "vec.cuh"

namespace pccl {
namespace block {

namespace {

constexpr int kThreads = 256, kFull = 8;          // a block, and how many times two that is
// Choices up to which blocks find the named rows by themselves (dispatch of 4096 columns of bf16, by bits / by the kernel ahead:
// 1032 choices 4.0 / 4.1 us, 2048 choices 6.9 / 5.6).
constexpr int kScan = 1024;

struct MoveParams {
  MoveArgs a;
  const void* x;
  int64_t ldx;
  const void* d;
  int64_t ldd;
  void* out;
  float* dw;
  int shift;                  // 1 << shift threads share a row (kFull: all of a block, known when compiled)
};

template <typename T> constexpr int kChunk = 16 / static_cast<int>(sizeof(T));

template <typename T> __device__ __forceinline__ void unpack_chunk(uint4 q, float* f) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(w[i]);
    else unpack2(w[i], f + 2 * i, T());
  }
}
template <typename T> __device__ __forceinline__ uint4 pack_chunk(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
    else w[i] = pack2(f[2 * i], f[2 * i + 1], T());
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes from any address: two neighbouring 16-byte blocks, and by how many bytes to shift them together.  Loading
// and shifting are apart, and neither branches, so that several loads are under way at a time.
struct Blocks {
  uint4 lo, hi;
  int off;
};
__device__ __forceinline__ uint4 shift_together(const Blocks& b) {
  uint32_t w[8] = {b.lo.x, b.lo.y, b.lo.z, b.lo.w, b.hi.x, b.hi.y, b.hi.z, b.hi.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = b.off & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = b.off & 4 ? w[i + 1] : w[i];
  const int bits = (b.off & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                    __funnelshift_r(w[3], w[4], bits));
}

// The chunks of a row that is written: chunk i holds columns [first + i * N, + N), of which those inside the row count.
// Aligned rows have first = 0 and whole chunks alone.
template <typename T, bool kVec> struct RowChunks {
  static constexpr int N = kChunk<T>;
  int hidden, first, count;
  __device__ RowChunks(const void* row, int hidden_) : hidden(hidden_) {
    first = kVec ? 0 : -static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    count = (hidden - first + N - 1) / N;
  }
  __device__ int column(int i) const { return first + i * N; }
  __device__ bool whole(int i) const { return kVec || (column(i) >= 0 && column(i) + N <= hidden); }
  // A source row at chunk i.  Only blocks that hold a value of the row are read (allocations begin at multiples of 256
  // bytes, so all of such a block is theirs): where one of the two does not, the other stands in for it, and what
  // that brings lies outside the row.
  __device__ Blocks load(const T* src, int i) const {
    Blocks b;
    const int c = column(i);
    if constexpr (kVec) {
      b.lo = __ldg(reinterpret_cast<const uint4*>(src + c));
      b.hi = b.lo;
      b.off = 0;
    } else {
      const uintptr_t row = reinterpret_cast<uintptr_t>(src), at = row + static_cast<int64_t>(c) * static_cast<int>(sizeof(T));
      const uintptr_t begin = row & ~static_cast<uintptr_t>(15);
      const uintptr_t end = (row + static_cast<uintptr_t>(hidden) * sizeof(T) - 1) & ~static_cast<uintptr_t>(15);
      const uintptr_t lo = at & ~static_cast<uintptr_t>(15);
      b.off = static_cast<int>(at & 15);
      b.lo = __ldg(reinterpret_cast<const uint4*>(lo < begin ? begin : lo));
      b.hi = __ldg(reinterpret_cast<const uint4*>(lo + 16 > end ? end : lo + 16));
    }
    return b;
  }
  __device__ static uint4 value(const Blocks& b) { return kVec ? b.lo : shift_together(b); }
  __device__ void store(T* dst, int i, uint4 q) const {
    const int c = column(i);
    if (whole(i)) {
      *reinterpret_cast<uint4*>(dst + c) = q;
      return;
    }
    float f[N];
    unpack_chunk<T>(q, f);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c + j >= 0 && c + j < hidden) dst[c + j] = from_f32<T>(f[j]);
  }
};

// What a block knows of the rows that choices name: bits, where there are few choices.
struct Named {
  uint32_t bits[kScan / 32];
  int32_t holes[kThreads];
  int count;
};
// By the whole block, before the move.
__device__ __forceinline__ void mark_named(const MoveArgs& a, Named& named) {
  if (a.workspace != nullptr) return;
  const int total = a.tokens * a.top_k;
  if (threadIdx.x < kScan / 32) named.bits[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int32_t r = a.rows[i];
    if (r >= 0 && r < total) atomicOr(named.bits + (r >> 5), 1u << (r & 31));
  }
}
// Rows that no choice names become zero, by the whole block, after the move.  A block has every gridDim.x-th row, so
// that runs of rows to clear are spread over all of them.
template <typename T, bool kVec> __device__ __forceinline__ void clear_unnamed(const MoveArgs& a, T* out, const int shift, Named& named) {
  const int32_t* const namer = static_cast<const int32_t*>(a.workspace);
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  if (namer != nullptr) asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lanes = 1 << shift, rows = kThreads >> shift;
  for (int64_t r0 = blockIdx.x; r0 < total; r0 += static_cast<int64_t>(gridDim.x) * kThreads) {
    if (threadIdx.x == 0) named.count = 0;
    __syncthreads();                               // also: everybody's marks
    const int64_t r = r0 + static_cast<int64_t>(threadIdx.x) * gridDim.x;
    if (r < total) {
      bool is;
      if (namer != nullptr) {
        const int32_t i = __ldcg(namer + r);       // written by the kernel ahead
        is = i >= 0 && i < total && a.rows[i] == r;
      } else {
        is = (named.bits[r >> 5] >> (r & 31)) & 1u;
      }
      if (!is) named.holes[atomicAdd(&named.count, 1)] = static_cast<int32_t>(r);
    }
    __syncthreads();
    for (int h = static_cast<int>(threadIdx.x) >> shift; h < named.count; h += rows) {
      T* const dst = out + static_cast<int64_t>(named.holes[h]) * a.hidden;
      const RowChunks<T, kVec> chunks(dst, a.hidden);
      for (int i = threadIdx.x & (lanes - 1); i < chunks.count; i += lanes) chunks.store(dst, i, make_uint4(0, 0, 0, 0));
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) note_namers_kernel(const MoveArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int32_t r = a.rows[i];
    if (r >= 0 && r < total) static_cast<int32_t*>(a.workspace)[r] = static_cast<int32_t>(i);
  }
}

template <typename T, bool kVec, bool kLong>
__global__ void __launch_bounds__(kThreads) dispatch_rows_kernel(const MoveParams p) {
  const MoveArgs& a = p.a;
  const int shift = kLong ? kFull : p.shift;
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  __shared__ Named named;
  mark_named(a, named);
  T* out = static_cast<T*>(p.out);
  const int lanes = 1 << shift, rows_abreast = kThreads >> shift, tid = threadIdx.x & (lanes - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * rows_abreast + (threadIdx.x >> shift); t < a.tokens;
       t += static_cast<int64_t>(gridDim.x) * rows_abreast) {
    const T* src = static_cast<const T*>(p.x) + t * p.ldx;
    const int32_t* rows = a.rows + t * a.top_k;
    if constexpr (kVec) {
      const RowChunks<T, true> chunks(src, a.hidden);
      for (int i = tid; i < chunks.count; i += lanes) {
        const uint4 q = chunks.value(chunks.load(src, i));
        for (int k = 0; k < a.top_k; ++k) {
          const int64_t r = rows[k];
          if (r >= 0 && r < total) chunks.store(out + r * a.hidden, i, q);
        }
      }
    } else {
      for (int k = 0; k < a.top_k; ++k) {        // every copy has chunks of its own; the source stays in L1
        const int64_t r = rows[k];
        if (r < 0 || r >= total) continue;
        T* const dst = out + r * a.hidden;
        const RowChunks<T, false> chunks(dst, a.hidden);
#pragma unroll 2
        for (int i = tid; i < chunks.count; i += lanes) chunks.store(dst, i, chunks.value(chunks.load(src, i)));
      }
    }
  }
  clear_unnamed<T, kVec>(a, out, shift, named);
}

// kAtOnce sources are under way at a time.
template <typename T, bool kVec, bool kLong, int kAtOnce>
__global__ void __launch_bounds__(kThreads) combine_rows_kernel(const MoveParams p) {
  constexpr int N = kChunk<T>;
  const MoveArgs& a = p.a;
  const int shift = kLong ? kFull : p.shift;
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  const T* y = static_cast<const T*>(p.x);
  const int lanes = 1 << shift, rows_abreast = kThreads >> shift, tid = threadIdx.x & (lanes - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * rows_abreast + (threadIdx.x >> shift); t < a.tokens;
       t += static_cast<int64_t>(gridDim.x) * rows_abreast) {
    T* const dst = static_cast<T*>(p.out) + t * a.hidden;
    const RowChunks<T, kVec> chunks(dst, a.hidden);
    const int32_t* rows = a.rows + t * a.top_k;
    const float* weights = a.weights ? a.weights + t * a.top_k : nullptr;
    for (int i = tid; i < chunks.count; i += lanes) {
      float acc[N];
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = 0.f;
      for (int k0 = 0; k0 < a.top_k; k0 += kAtOnce) {
        Blocks q[kAtOnce];
        float w[kAtOnce];
        bool valid[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int k = min(k0 + u, a.top_k - 1);
          const int64_t r = rows[k];
          valid[u] = k0 + u < a.top_k && r >= 0 && r < total;
          w[u] = weights ? weights[k] : 1.f;
          q[u] = chunks.load(y + (valid[u] ? r : 0) * p.ldx, i);       // row 0 is always there
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
          if (valid[u]) {
            float f[N];
            unpack_chunk<T>(chunks.value(q[u]), f);
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = fmaf(w[u], f[j], acc[j]);
          }
      }
      chunks.store(dst, i, pack_chunk<T>(acc));
    }
  }
}

// One warp (of short rows: part of one) per choice: its row of y and the token's dout pass through once for the product and the scaled copy.  The
// warps of a block take neighbouring choices, so a token's dout comes from L1 for all but the first.
template <typename T, bool kVec, bool kLong>
__global__ void __launch_bounds__(kThreads) combine_rows_backward_kernel(const MoveParams p) {
  constexpr int N = kChunk<T>, kAtOnce = kVec ? 4 : 2;
  const MoveArgs& a = p.a;
  const int shift = kLong || p.shift > 5 ? 5 : p.shift, width = 1 << shift, lane = threadIdx.x & (width - 1);
  const int64_t total = static_cast<int64_t>(a.tokens) * a.top_k;
  const int64_t abreast = static_cast<int64_t>(gridDim.x) * (kThreads >> shift);
  __shared__ Named named;
  T* out = static_cast<T*>(p.out);
  if (out) mark_named(a, named);
  // Whole warps go round together: the sum at the end is by all of their lanes.
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kThreads >> shift); i0 < total; i0 += abreast) {
    const int64_t i = i0 + (threadIdx.x >> shift);
    const int64_t r = i < total ? a.rows[i] : -1;
    float dot = 0.f;
    if (r >= 0 && r < total) {
      const float w = a.weights[i];
      const T* y = static_cast<const T*>(p.x) + r * p.ldx;
      const T* d = static_cast<const T*>(p.d) + i / a.top_k * p.ldd;
      T* const dst = out ? out + r * a.hidden : nullptr;
      const RowChunks<T, kVec> chunks(dst ? static_cast<const void*>(dst) : y, a.hidden);
      for (int c0 = lane; c0 < chunks.count; c0 += width * kAtOnce) {
        Blocks qd[kAtOnce], qy[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int c = min(c0 + width * u, chunks.count - 1);
          qd[u] = chunks.load(d, c);
          if (p.dw) qy[u] = chunks.load(y, c);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          if (c0 + width * u >= chunks.count) break;
          float fd[N], fy[N];
          unpack_chunk<T>(chunks.value(qd[u]), fd);
          if (p.dw) {
            unpack_chunk<T>(chunks.value(qy[u]), fy);
            if (!chunks.whole(c0 + width * u)) {
              const int c = chunks.column(c0 + width * u);
#pragma unroll
              for (int j = 0; j < N; ++j)
                if (c + j < 0 || c + j >= a.hidden) fd[j] = fy[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) dot = fmaf(fy[j], fd[j], dot);
          }
          if (dst) {
#pragma unroll
            for (int j = 0; j < N; ++j) fd[j] *= w;
            chunks.store(dst, c0 + width * u, pack_chunk<T>(fd));
          }
        }
      }
    }
    if (p.dw) {
      for (int o = width / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (lane == 0 && i < total) p.dw[i] = dot;
    }
  }
  if (out) clear_unnamed<T, kVec>(a, out, kLong ? kFull : p.shift, named);
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

// As many threads as a row has chunks (one more where it begins inside one), four at least.
int shift_for(const MoveArgs& a) {
  const int chunks = (a.hidden * dtype_bytes(a.dtype) + 15) / 16 + (a.hidden * dtype_bytes(a.dtype) % 16 ? 1 : 0);
  int shift = 2;
  while ((1 << shift) < chunks && (1 << shift) < kThreads) ++shift;
  return shift;
}

// After the kernel ahead where there is one: it may start while that one runs.
template <class Kernel> void launch_move(Kernel kernel, const MoveParams& p, int blocks, cudaStream_t stream) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = p.a.workspace != nullptr ? 1 : 0;
  PCCL_CUDA(cudaLaunchKernelEx(&config, kernel, p));
}

// The kernel ahead, where a call has a workspace.
void note_namers(const MoveArgs& a, cudaStream_t stream) {
  if (a.workspace == nullptr) {
    PCCL_CHECK(move_workspace(a) == 0, "dispatch / combine: no workspace");
    return;
  }
  const int64_t choices = static_cast<int64_t>(a.tokens) * a.top_k;
  note_namers_kernel<<<grid_for((choices + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
  PCCL_CUDA(cudaGetLastError());
}

}  // namespace

size_t move_workspace(const MoveArgs& a) {
  const int64_t choices = static_cast<int64_t>(a.tokens) * a.top_k;
  return choices > kScan ? static_cast<size_t>(choices) * sizeof(int32_t) : 0;
}

#define PCCL_BLOCK_MOVE(KERNEL, ITEMS, VEC, ...)                                                 \
  PCCL_BLOCK_TYPES(a.dtype, T,                                                                   \
    if (VEC && p.shift == kFull) launch_move(KERNEL<T, true, true __VA_ARGS__>, p, grid_for(ITEMS), stream);   \
    else if (VEC) launch_move(KERNEL<T, true, false __VA_ARGS__>, p, grid_for(ITEMS), stream);                 \
    else if (p.shift == kFull) launch_move(KERNEL<T, false, true __VA_ARGS__>, p, grid_for(ITEMS), stream);    \
    else launch_move(KERNEL<T, false, false __VA_ARGS__>, p, grid_for(ITEMS), stream))

void dispatch_rows(const MoveArgs& a, const void* x, int64_t ldx, void* out, cudaStream_t stream) {
  if (a.tokens == 0) return;
  MoveParams p{a, x, ldx, nullptr, 0, out, nullptr, shift_for(a)};
  const int64_t blocks = ((static_cast<int64_t>(a.tokens) << p.shift) + kThreads - 1) / kThreads;
  const bool vec = a.hidden * dtype_bytes(a.dtype) % 16 == 0 && aligned(x, ldx, a.dtype) && aligned(out, a.hidden, a.dtype);
  note_namers(a, stream);
  PCCL_BLOCK_MOVE(dispatch_rows_kernel, blocks, vec, );
}

void combine_rows(const MoveArgs& a, const void* y, int64_t ldy, void* out, cudaStream_t stream) {
  if (a.tokens == 0) return;
  MoveParams p{a, y, ldy, nullptr, 0, out, nullptr, shift_for(a)};
  p.a.workspace = nullptr;                         // every row of the result is written
  const int64_t blocks = ((static_cast<int64_t>(a.tokens) << p.shift) + kThreads - 1) / kThreads;
  const bool vec = a.hidden * dtype_bytes(a.dtype) % 16 == 0 && aligned(y, ldy, a.dtype) && aligned(out, a.hidden, a.dtype);
  // Up to four sources at a time, so many that the fewest loads go beyond the last one.
  int at_once = a.top_k < 4 ? a.top_k : 4;
  if (a.top_k > 4 && (a.top_k + 2) / 3 * 3 < (a.top_k + 3) / 4 * 4) at_once = 3;
  switch (at_once) {
    case 1: PCCL_BLOCK_MOVE(combine_rows_kernel, blocks, vec, , 1); break;
    case 2: PCCL_BLOCK_MOVE(combine_rows_kernel, blocks, vec, , 2); break;
    case 3: PCCL_BLOCK_MOVE(combine_rows_kernel, blocks, vec, , 3); break;
    default: PCCL_BLOCK_MOVE(combine_rows_kernel, blocks, vec, , 4); break;
  }
}

void combine_rows_backward(const MoveArgs& a, const void* y, int64_t ldy, const void* dout, int64_t ldd, void* dy,
                           float* dw, cudaStream_t stream) {
  if (a.tokens == 0 || (dy == nullptr && dw == nullptr)) return;
  MoveParams p{a, y, ldy, dout, ldd, dy, dw, shift_for(a)};
  const int shift = p.shift < 5 ? p.shift : 5;
  const int64_t blocks = ((static_cast<int64_t>(a.tokens) * a.top_k << shift) + kThreads - 1) / kThreads;
  const bool vec = a.hidden * dtype_bytes(a.dtype) % 16 == 0 && aligned(y, ldy, a.dtype) && aligned(dout, ldd, a.dtype) &&
                   (dy == nullptr || aligned(dy, a.hidden, a.dtype));
  if (dy == nullptr) p.a.workspace = nullptr;
  else note_namers(a, stream);
  PCCL_BLOCK_MOVE(combine_rows_backward_kernel, blocks, vec, );
}

}  // namespace block
}  // namespace pccl
