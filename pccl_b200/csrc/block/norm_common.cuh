// What the two kernels of the block norms share: columns, the ring of rows in shared memory, sums over a row.
//
// Both kernels are bound by memory, and what keeps memory waiting is a row's own chain: load, sum over the row,
// barrier, use, perhaps a second sum.  So the coming rows are on their way into a ring in shared memory (cp.async,
// which holds no registers) while a block works on the present one.  Two ways of reading a row:
//
//   kRing     rows aligned to 16 bytes: every thread copies the columns it will use into slots of its own, so no
//             barrier is needed to read them;
//   kWindow   rows that begin anywhere (odd sizes, cut views): the block copies the 16-byte blocks that cover the
//             row and picks the values out of shared memory.
//
// Rows too long for one block's registers or ring are split over a cluster of two blocks, which add up their sums
// through one another's shared memory: 12288 columns of bf16 backwards with all weights run at 2.5 TB/s so, at 1.9 in
// one block of 1024 threads, whose 64 registers each spill; over four blocks at 1.6, since a barrier of a cluster is
// most of a microsecond.  Forwards 64 registers suffice, and one block comes first (5.3 TB/s against 3.5).
#pragma once
#include "../common/launch.h"
#include "../common/util.h"
#include "../engine/cuda_driver.h"
#include "vec.cuh"

namespace pccl {
namespace block {
namespace norm {

constexpr int kHeld = 16;                      // values a thread holds of its row
enum Mode : int { kRing = 0, kWindow = 1 };
constexpr int kSplitBlocks = 2;                // of a cluster that shares a row

// A thread's values stand in groups of consecutive columns, as many as 16 bytes of the widest type hold: a warp then
// touches whole 32-byte sectors in every access.  (Eight columns of 32 bits a thread, as two accesses 32 bytes apart
// from lane to lane, moved every sector twice: 126 us instead of 84 for 4100 x 8192 backwards.)
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
  int workers;                // blocks, or clusters of them, each with a run of consecutive rows
  int ring;                   // rows in shared memory
};

// A warp holds 32 * kHeld consecutive columns: where rows are aligned a lane has G neighbours of every 32 * G of them,
// else one of every 32.  Steps from one access to the next are constants then, which matters: with a step of the
// block's width a third of all instructions were addresses.
template <bool kVec, int G> struct Columns {
  int part, columns;          // the block's first column, and how many it has
  int local;                  // this thread's first column within the block's
  int first, room;            // the same within the row, and the columns from there to the row's end
  __device__ Columns(int hidden, int rank) {
    const int held = static_cast<int>(blockDim.x) * kHeld;
    part = rank * held;
    columns = max(min(hidden - part, held), 0);
    local = static_cast<int>(threadIdx.x >> 5) * 32 * kHeld + static_cast<int>(threadIdx.x & 31) * (kVec ? G : 1);
    first = part + local;
    room = hidden - first;
  }
};

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
__device__ __forceinline__ void load_group(const T* row, int v, const Columns<kVec, G>& c, float2* to) {
  if constexpr (kVec) {
    if (v * 32 * G < c.room) {
      unpack<T, G>(*reinterpret_cast<const Raw<T, G>*>(row + c.first + v * 32 * G), to);
    } else {
#pragma unroll
      for (int j = 0; j < G / 2; ++j) to[j] = make_float2(0.f, 0.f);
    }
  } else {
    float* f = reinterpret_cast<float*>(to);
#pragma unroll
    for (int j = 0; j < G; ++j) f[j] = (v * G + j) * 32 < c.room ? to_f32<T>((row + c.first)[(v * G + j) * 32]) : 0.f;
  }
}
template <typename T, bool kVec, int G>
__device__ __forceinline__ void store_group(T* row, int v, const Columns<kVec, G>& c, const float2* from) {
  if constexpr (kVec) {
    if (v * 32 * G < c.room) *reinterpret_cast<Raw<T, G>*>(row + c.first + v * 32 * G) = pack<T, G>(from);
  } else {
    const float* f = reinterpret_cast<const float*>(from);
#pragma unroll
    for (int j = 0; j < G; ++j)
      if ((v * G + j) * 32 < c.room) (row + c.first)[(v * G + j) * 32] = from_f32<T>(f[j]);
  }
}
template <typename T, bool kVec, int G>
__device__ __forceinline__ void store_row(T* row, const Columns<kVec, G>& c, const float2* f) {
#pragma unroll
  for (int v = 0; v < kHeld / G; ++v) store_group<T, kVec, G>(row, v, c, f + v * (G / 2));
}
// A weight vector is of the activations' type or of 32 bits.
template <typename T, bool kVec, int G>
__device__ __forceinline__ void load_weight(const Weight& w, int64_t first, const Columns<kVec, G>& c, float2* f) {
#pragma unroll
  for (int v = 0; v < kHeld / G; ++v) {
    if (w.f32) load_group<float, kVec, G>(static_cast<const float*>(w.ptr) + first, v, c, f + v * (G / 2));
    else load_group<T, kVec, G>(static_cast<const T*>(w.ptr) + first, v, c, f + v * (G / 2));
  }
}

// ---- ring ------------------------------------------------------------------------------------------------
// A thread's share of a row of T: kHeld values.  In the ring a row is an image of itself, so a warp's copies fill whole
// lines of shared memory.  (With each thread's share in one piece the copies of neighbours went to different lines,
// and every kernel here took a quarter longer.)
template <typename T> constexpr int kBytes = kHeld * static_cast<int>(sizeof(T));

// The first `size` of kSize bytes (8 or 16), and zeros for the rest.
template <int kSize> __device__ __forceinline__ void copy_async(char* to, const void* from, int size) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (kSize == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(size) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until at most `left` of the groups committed last are under way.
__device__ __forceinline__ void copies_wait(int left) {
  if (left <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (left == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

template <typename T, int G>
__device__ __forceinline__ void fetch_share(char* image, const T* row, const Columns<true, G>& c) {
  constexpr int kSize = G * static_cast<int>(sizeof(T));
#pragma unroll
  for (int v = 0; v < kHeld / G; ++v) {
    const bool beyond = v * 32 * G >= c.room;
    copy_async<kSize>(image + c.local * static_cast<int>(sizeof(T)) + v * 32 * kSize, beyond ? row : row + c.first + v * 32 * G,
                      beyond ? 0 : kSize);
  }
}

// Bytes of a window for any row of T.
template <typename T> __host__ __device__ constexpr int window_bytes(int threads) { return threads * kBytes<T> + 16; }
// The 16-byte blocks that cover the block's part of the row, and zeros up to the last column that a thread holds.
// The first may begin with values in front of it: such a block holds a value of the row, and allocations begin at
// multiples of 256 bytes, so all of it is theirs.  Nothing is read behind the row.
template <typename T, int G>
__device__ __forceinline__ void fetch_window(char* window, const T* row, const Columns<false, G>& c) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(row + c.part);
  const int ahead = static_cast<int>(begin & 15), bytes = ahead + c.columns * static_cast<int>(sizeof(T));
  const char* const first = reinterpret_cast<const char*>(begin - ahead);
  const int all = window_bytes<T>(static_cast<int>(blockDim.x));
  for (int at = static_cast<int>(threadIdx.x) * 16; at < all; at += static_cast<int>(blockDim.x) * 16) {
    const int size = min(max(bytes - at, 0), 16);
    copy_async<16>(window + at, size > 0 ? first + at : first, size);
  }
}

// Group v of a row of T; `held` is the row's image in the ring, or its window.
template <typename T, int kMode, int G>
__device__ __forceinline__ void take(const char* held, const T* row, int v, const Columns<kMode == kRing, G>& c, float2* to) {
  if constexpr (kMode == kRing) {
    unpack<T, G>(*reinterpret_cast<const Raw<T, G>*>(held + c.local * static_cast<int>(sizeof(T)) + v * static_cast<int>(32 * G * sizeof(T))), to);
  } else {
    const T* at = reinterpret_cast<const T*>(held + (reinterpret_cast<uintptr_t>(row + c.part) & 15)) + c.local;
    float* f = reinterpret_cast<float*>(to);
#pragma unroll
    for (int j = 0; j < G; ++j) f[j] = to_f32<T>(at[(v * G + j) * 32]);
  }
}

// Sum over a row; `sums` alternates between two sets so that one barrier a call is enough.  Sets are cleared once
// (row_sum_clear), so that whole groups of four can be read.  Blocks that share a row send one another their sums
// and add them in the order of their ranks, so all get the same.
struct __align__(16) RowSums {
  float set[2][32];
  float block[2][kSplitBlocks];
};
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <bool kSplit> __device__ __forceinline__ void row_sum_clear(RowSums& sums) {
  if (blockDim.x == 32) return;
  if (threadIdx.x < 64) (&sums.set[0][0])[threadIdx.x] = 0.f;
  if constexpr (kSplit) cluster_barrier();         // every block has begun before one writes to it
  else __syncthreads();
}
template <bool kSplit> __device__ __forceinline__ float row_sum(float v, RowSums& sums, int* turn) {
  v = warp_sum(v);
  if (blockDim.x == 32) return v;                  // a split row has more threads
  const int now = *turn;
  *turn ^= 1;
  float* s = sums.set[now];
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); w += 4) {
    const float4 q = *reinterpret_cast<const float4*>(s + w);
    v += (q.x + q.y) + (q.z + q.w);
  }
  if constexpr (kSplit) {
    if (threadIdx.x < kSplitBlocks) {
      const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&sums.block[now][cluster_rank()]));
      uint32_t theirs;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(static_cast<int>(threadIdx.x)));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(theirs), "f"(v) : "memory");
    }
    cluster_barrier();
    v = 0.f;
#pragma unroll
    for (int r = 0; r < kSplitBlocks; ++r) v += sums.block[now][r];
  }
  return v;
}

// A weight's slots: kHeld 32-bit values, four to an access.
__device__ __forceinline__ int slot_place() { return static_cast<int>(threadIdx.x >> 5) * 8 * kHeld + static_cast<int>(threadIdx.x & 31); }
__device__ __forceinline__ void slots_store(char* slots, const float2* f) {
  float4* const at = reinterpret_cast<float4*>(slots) + slot_place();
#pragma unroll
  for (int i = 0; i < kHeld / 4; ++i) at[i * 32] = make_float4(f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y);
}
template <int G> __device__ __forceinline__ void slots_load(const char* slots, int v, float2* f) {
  const float4* const at = reinterpret_cast<const float4*>(slots) + slot_place();
#pragma unroll
  for (int i = 0; i < G / 4; ++i) {
    const float4 q = at[(v * (G / 4) + i) * 32];
    f[2 * i] = make_float2(q.x, q.y);
    f[2 * i + 1] = make_float2(q.z, q.w);
  }
}

// g1 = post_gamma * gate of one group of rows into its slots (what is absent counts as 1).
template <typename T, bool kVec, int G>
__device__ __forceinline__ void form_g1(const NormArgs& a, int64_t group, char* slots, const Columns<kVec, G>& c) {
  float2 f[kHeld / 2], w[kHeld / 2];
  if (a.post_gamma.ptr) load_weight<T, kVec, G>(a.post_gamma, 0, c, f);
  if (a.gate.ptr) {
    load_weight<T, kVec, G>(a.gate, group * a.hidden, c, w);
#pragma unroll
    for (int i = 0; i < kHeld / 2; ++i) f[i] = a.post_gamma.ptr ? mul2(f[i], w[i]) : w[i];
  }
  slots_store(slots, f);
}

// First row of worker w's run; w = workers gives the number of rows.
__device__ __forceinline__ int64_t run_start(int64_t rows, int workers, int w) {
  return rows / workers * w + min(static_cast<int64_t>(w), rows % workers);
}

// ---- host --------------------------------------------------------------------------------------------------
inline int threads_of(int hidden, int split) { return ((hidden + split * kHeld - 1) / (split * kHeld) + 31) / 32 * 32; }

inline int sm_count() {
  int dev = 0, sms = 0;
  PCCL_CUDA(cudaGetDevice(&dev));
  PCCL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  return sms;
}

inline bool has_g1(const NormArgs& a) { return a.post_gamma.ptr || a.gate.ptr; }

inline bool aligned(const void* p, int64_t ld, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * bytes % 16 == 0);
}
inline bool aligned(const Weight& w, int64_t hidden, DType t) { return aligned(w.ptr, hidden, w.f32 ? 4 : dtype_bytes(t)); }
inline bool inputs_aligned(const NormArgs& a) {
  const bool wide = a.xt == DType::kF32 || a.rt == DType::kF32;
  return a.hidden % (wide ? 4 : 8) == 0 && aligned(a.x, a.ldx, dtype_bytes(a.xt)) && aligned(a.residual, a.ldr, dtype_bytes(a.rt)) &&
         aligned(a.gamma, a.hidden, a.xt) && aligned(a.post_gamma, a.hidden, a.xt) && aligned(a.gate, a.hidden, a.xt);
}

// Shared memory of an SM, and the most of one block (less what the kernels themselves and the driver keep).
constexpr size_t kSmemSm = 228 * 1024, kSmemBlock = 226 * 1024, kSmemKept = 1024 + sizeof(RowSums);
constexpr int kMostRing = 4;

// How a row of `hidden` columns is laid out over blocks.  weights and share are bytes a thread, of its weights and of
// its share of a row; windows is how many windows a row has beyond those bytes.
struct Layout {
  int split, threads, ring;
  size_t smem;
};
// Registers let 512 threads of 128 registers (or 1024 of 64) share an SM.
inline int blocks_per_sm(int threads) { return threads < 512 ? 512 / threads : 1; }

// Tries blocks of up to `most_threads`, and where these are too few or leave no room for the ring, clusters of two;
// `alone`: a block without room for a row on its way comes before a cluster.
inline Layout layout_of(int hidden, bool vec, int weights, int share, int windows, int most_threads, bool alone) {
  Layout l{};
  const auto fits = [&](int split, int least) {
    l = Layout{split, threads_of(hidden, split), 0, 0};
    if (l.threads > most_threads) return false;
    const auto bytes = [&](int rows) {
      return static_cast<size_t>(weights + rows * share) * l.threads + (vec ? 0 : static_cast<size_t>(rows) * windows * 16);
    };
    // As many rows as leave room for the blocks that registers have room for.
    for (int r = kMostRing; r >= least && l.ring == 0; --r)
      if (bytes(r) <= kSmemBlock && (r <= 2 || (bytes(r) + kSmemKept) * blocks_per_sm(l.threads) <= kSmemSm)) l.ring = r;
    l.smem = bytes(l.ring);
    return l.ring > 0;
  };
  const bool found = fits(1, 2) || (alone && fits(1, 1)) || fits(kSplitBlocks, 2) || fits(kSplitBlocks, 1);
  PCCL_CHECK(found, "block norm: a row of " << hidden << " columns does not fit");
  return l;
}

// Before a launch, and before a question for its occupancy.
template <class Kernel> void allow_smem(Kernel kernel, const Layout& l) {
  if (l.smem > 40 * 1024)
    PCCL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(l.smem)));
}
template <class Kernel> void launch(Kernel kernel, const NormParams& p, const Layout& l, cudaStream_t stream) {
  if (l.split == 1) {
    kernel<<<p.workers, l.threads, l.smem, stream>>>(p);
    return;
  }
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = l.split;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(p.workers * l.split);
  config.blockDim = dim3(l.threads);
  config.dynamicSmemBytes = l.smem;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = 1;
  PCCL_CUDA(cudaLaunchKernelEx(&config, kernel, p));
}

}  // namespace norm
}  // namespace block
}  // namespace pccl
