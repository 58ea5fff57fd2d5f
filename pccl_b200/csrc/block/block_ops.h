// Host-side entry points of the operators around a block's matrix products (no torch dependency): expert
// routing, rows into expert order and back, and the norms around a block.  Every call is asynchronous on
// `stream`, allocates nothing and keeps nothing; workspaces belong to the caller.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace pccl {
namespace block {

enum class DType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline int dtype_bytes(DType t) { return t == DType::kF32 ? 4 : 2; }

// ---- expert routing --------------------------------------------------------------------------------
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 31;     // one lane of a warp per choice, and one for the runner-up
constexpr int kMaxGroups = 32;
constexpr int64_t kMaxChoices = (int64_t{1} << 31) - (1 << 16);   // tokens * top_k stay below: a block's tokens more, and it still fits 31 bits

struct RouteArgs {
  const void* logits;         // [tokens] rows of `experts` values, `ld` elements apart
  DType dtype;
  int64_t ld;
  const float* bias;          // [experts] or null: added to the scores for the choice alone
  const uint8_t* mask;        // [tokens] or null: tokens whose byte is 0 choose nothing
  int tokens, experts, top_k;
  int groups, top_groups;     // experts in `groups` equal groups, of which the best `top_groups` stay
  int sigmoid;                // scores: 0 softmax over the experts, 1 sigmoid
  int top2;                   // a group's score: 0 its best score, 1 the sum of its two best
  int renormalise;
  float scale;
  int32_t* idx;               // [tokens][top_k], best first; -1 for masked tokens
  float* weights;             // [tokens][top_k]
  int32_t* rows;              // [tokens][top_k]: row of this choice in expert order, -1 for masked tokens
  int32_t* offsets;           // [experts + 1]: first row of every expert
  void* workspace;            // route_workspace() bytes (null when that is 0)
};
size_t route_workspace(const RouteArgs& a);
void route_topk(const RouteArgs& a, cudaStream_t stream);

// dlogits[tokens][experts] (contiguous) from dweights[tokens][top_k]; the choice itself is constant.
void route_topk_backward(const RouteArgs& a, const float* dweights, void* dlogits, cudaStream_t stream);

// ---- rows into expert order and back ---------------------------------------------------------------
// What follows these in a kernel's parameters begins at 16 bytes: combine of 1777 x 1431 fp16 takes 10.9 us instead of 10.3
// where it does not.
struct alignas(16) MoveArgs {
  DType dtype;
  int tokens, top_k, hidden;
  const int32_t* rows;        // [tokens][top_k], no two the same; a value outside [0, tokens * top_k) moves nothing
  const float* weights;       // [tokens][top_k] (combine)
  void* workspace;            // move_workspace() bytes (null when that is 0), where rows that no choice names are cleared
};
size_t move_workspace(const MoveArgs& a);
// out[rows[t][k]] = x[t]; rows that no choice names become zero.
void dispatch_rows(const MoveArgs& a, const void* x, int64_t ldx, void* out, cudaStream_t stream);
// out[t] = sum_k w[t][k] * y[rows[t][k]] (w = 1 where a.weights is null).
void combine_rows(const MoveArgs& a, const void* y, int64_t ldy, void* out, cudaStream_t stream);
// dy[rows[t][k]] = w[t][k] * dout[t] (rows that no choice names become zero), dw[t][k] = <y[rows[t][k]], dout[t]>; either
// output may be null, and without dy no workspace is needed.
void combine_rows_backward(const MoveArgs& a, const void* y, int64_t ldy, const void* dout, int64_t ldd, void* dy,
                           float* dw, cudaStream_t stream);

// ---- norms around a block --------------------------------------------------------------------------
constexpr int kMaxNormHidden = 16384;

struct Weight {               // a vector (or matrix) of the activations' type or of 32-bit floats
  const void* ptr;
  int f32;
};
struct NormArgs {
  int64_t rows;
  int hidden;
  DType xt, rt;               // type of x / y, and of the residual stream (the same or 32 bits)
  const void* x;              // block output, or null
  const void* residual;       // residual stream
  int64_t ldx, ldr;           // elements between rows
  Weight gamma, post_gamma, gate;   // null pointers where absent
  int64_t gate_rows;          // consecutive rows that share a row of `gate`
  float scale, eps;
};
// v = x * rsqrt(mean x^2 + eps) * post_gamma (or x);  h = scale * residual + gate * v;
// y = h * rsqrt(mean h^2 + eps) * gamma.  h / y may be null; r1, r2 [rows] receive the two inverse roots
// (null where not wanted).
void norm_forward(const NormArgs& a, void* h, void* y, float* r1, float* r2, cudaStream_t stream);

struct NormGrads {
  const void* dy;             // gradients that came in; either may be null
  const void* dh;
  int64_t lddy, lddh;
  const void* h;              // the stored 32-bit stream, read instead of x and residual where given
  const float* r1;
  const float* r2;
  void* dx;                   // gradients wanted (null where not), contiguous rows
  void* dresidual;
  void* dgamma;               // in the weights' own types
  void* dpost_gamma;
  void* dgate;
  void* workspace;            // norm_workspace() bytes
};
size_t norm_workspace(const NormArgs& a, const NormGrads& g);
void norm_backward(const NormArgs& a, const NormGrads& g, cudaStream_t stream);

}  // namespace block
}  // namespace pccl
