// Torch bindings of expert routing, dispatch / combine and the block norms, with their gradients.
//
// The gradients are C++ autograd functions: a training step of a small layer is bound by the host, and a Python
// function per call costs more than these kernels.  Every call checks its arguments first and the device last,
// works on the tensors' own device and its current stream, and takes temporaries from torch's allocator, so that
// streams and graph captures need no care here.
#include "block_bindings.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <climits>
#include <sstream>
#include <stdexcept>

#include "block_ops.h"

namespace py = pybind11;

namespace pccl {
namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// Refusals are ValueErrors in Python.
#define PCCL_ARG(COND, ...)                                  \
  do {                                                       \
    if (!(COND)) {                                           \
      std::ostringstream pccl_arg_stream;                    \
      pccl_arg_stream << __VA_ARGS__;                        \
      throw std::invalid_argument(pccl_arg_stream.str());    \
    }                                                        \
  } while (0)

bool known(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
block::DType dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? block::DType::kF32
         : t.scalar_type() == at::kHalf ? block::DType::kF16 : block::DType::kBF16;
}
const char* const kTypes = "float32, float16 or bfloat16";

void on_device(const Tensor& t, const Tensor& first, const char* op, const char* what) {
  PCCL_ARG(t.is_cuda(), op << ": " << what << " must be on a CUDA device");
  PCCL_ARG(t.device() == first.device(), op << ": " << what << " must be on the device of the other tensors");
}

// Tangents of forward-mode differentiation are refused: these operators would lose them without a word.
void no_tangent(const Tensor& t, const char* op, const char* what) {
  PCCL_ARG(!t._fw_grad(0).defined(), op << ": " << what << " has a forward-mode tangent, but there are only gradients backwards");
}
void no_tangent(const OptTensor& t, const char* op, const char* what) {
  if (t.has_value()) no_tangent(*t, op, what);
}

// Rows of `cols` values with unit stride: the tensor itself where it is laid out so, else a copy.
struct Rows {
  Tensor t;
  int64_t ld;
  const void* ptr() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
Rows as_rows(const Tensor& t) {
  if (!t.defined()) return Rows{t, 0};
  const int64_t cols = t.size(-1);
  if (t.dim() == 2 && (cols == 1 || t.stride(1) == 1) && t.stride(0) >= 0)
    return Rows{t, t.size(0) > 1 ? t.stride(0) : cols};
  return Rows{t.contiguous(), cols};
}

// Saved state of a call that is not a tensor, kept by the autograd node.
template <class T> struct Kept : torch::CustomClassHolder {
  explicit Kept(const T& v) : value(v) {}
  T value;
};
template <class T> void keep(AutogradContext* ctx, const T& v) {
  ctx->saved_data["call"] = c10::IValue::make_capsule(c10::make_intrusive<Kept<T>>(v));
}
template <class T> const T& kept(AutogradContext* ctx) {
  return static_cast<Kept<T>*>(ctx->saved_data["call"].toCapsule().get())->value;
}

// These gradients have no gradients of their own: where a graph of the backward pass is built, its results
// refuse to be differentiated instead of passing for constants.
void once(variable_list& grads) {
  if (!at::GradMode::is_enabled()) return;
  std::vector<size_t> at_index;
  variable_list given;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      at_index.push_back(i);
      given.push_back(grads[i].detach().requires_grad_(true));
    }
  if (given.empty()) return;
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "the gradient of this operator cannot be differentiated again", static_cast<int64_t>(given.size()));
  variable_list out = (*refuse)(std::move(given));
  for (size_t i = 0; i < at_index.size(); ++i) grads[at_index[i]] = out[i];
}

// Contiguous and uninitialised, on the device of `like`.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// A tensor of 32-bit values in `storage`, from the offset-th on.
Tensor slice_of(const c10::Storage& storage, at::IntArrayRef sizes, at::ScalarType type, int64_t offset) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                      c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && wants_grad(*t); }
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ---- routing -------------------------------------------------------------------------------------------
struct RouteCall {
  int64_t top_k, groups, top_groups;
  bool sigmoid, top2, renormalise;
  double scale;
};

block::RouteArgs route_args(const RouteCall& c, const Rows& logits) {
  block::RouteArgs a{};
  a.logits = logits.ptr();
  a.dtype = dtype_of(logits.t);
  a.ld = logits.ld;
  a.tokens = static_cast<int>(logits.t.size(0));
  a.experts = static_cast<int>(logits.t.size(1));
  a.top_k = static_cast<int>(c.top_k);
  a.groups = static_cast<int>(c.groups);
  a.top_groups = static_cast<int>(c.top_groups);
  a.sigmoid = c.sigmoid;
  a.top2 = c.top2;
  a.renormalise = c.renormalise;
  a.scale = static_cast<float>(c.scale);
  return a;
}

variable_list route_run(const RouteCall& c, const Tensor& logits, const OptTensor& bias, const OptTensor& mask) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const Rows rows = as_rows(logits);
  block::RouteArgs a = route_args(c, rows);
  const Tensor b = bias.has_value() ? bias->contiguous() : Tensor();
  const Tensor m = mask.has_value() ? mask->contiguous() : Tensor();
  if (b.defined()) a.bias = b.const_data_ptr<float>();
  if (m.defined()) a.mask = reinterpret_cast<const uint8_t*>(m.const_data_ptr<bool>());
  // One allocation: an allocation costs the host as much as all of the arithmetic here costs the GPU for one token.
  const int64_t n = static_cast<int64_t>(a.tokens) * a.top_k, rest = (3 * n + a.experts + 1 + 3) / 4 * 4;
  const int64_t bytes = static_cast<int64_t>(block::route_workspace(a));
  const Tensor all = fresh({rest + (bytes + 3) / 4}, at::kInt, logits);
  if (bytes) a.workspace = all.mutable_data_ptr<int32_t>() + rest;
  Tensor idx = slice_of(all.storage(), {a.tokens, a.top_k}, at::kInt, 0);
  Tensor weights = slice_of(all.storage(), {a.tokens, a.top_k}, at::kFloat, n);
  Tensor to = slice_of(all.storage(), {a.tokens, a.top_k}, at::kInt, 2 * n);
  Tensor offsets = slice_of(all.storage(), {a.experts + 1}, at::kInt, 3 * n);
  a.idx = idx.mutable_data_ptr<int32_t>();
  a.weights = weights.mutable_data_ptr<float>();
  a.rows = to.mutable_data_ptr<int32_t>();
  a.offsets = offsets.mutable_data_ptr<int32_t>();
  block::route_topk(a, stream_of(logits));
  return {idx, weights, to, offsets};
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const RouteCall& c, const OptTensor& bias,
                               const OptTensor& mask) {
    variable_list out = route_run(c, logits, bias, mask);
    ctx->mark_non_differentiable({out[0], out[2], out[3]});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, out[0]});
    keep(ctx, c);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(4);
    if (!grads[1].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    const Rows rows = as_rows(saved[0]);
    block::RouteArgs a = route_args(kept<RouteCall>(ctx), rows);
    a.idx = const_cast<int32_t*>(saved[1].const_data_ptr<int32_t>());
    {
      at::NoGradGuard no_grad;
      const Tensor dw = grads[1].contiguous();
      result[0] = fresh(saved[0].sizes(), saved[0].scalar_type(), saved[0]);
      block::route_topk_backward(a, dw.const_data_ptr<float>(), result[0].mutable_data_ptr(), stream_of(saved[0]));
    }
    once(result);
    return result;
  }
};

variable_list route_topk(const Tensor& logits, int64_t top_k, const OptTensor& bias, bool sigmoid, int64_t groups,
                         int64_t top_groups, bool top2, bool renormalise, double scale, const OptTensor& mask) {
  const char* op = "route_topk";
  PCCL_ARG(logits.dim() == 2, op << ": logits must be [tokens, experts]");
  PCCL_ARG(known(logits.scalar_type()), op << ": logits must be " << kTypes);
  const int64_t t = logits.size(0), e = logits.size(1);
  PCCL_ARG(e >= 1 && e <= block::kMaxExperts, op << ": 1 to " << block::kMaxExperts << " experts, not " << e);
  PCCL_ARG(groups >= 1 && groups <= block::kMaxGroups && e % groups == 0,
           op << ": groups must divide the experts and be at most " << block::kMaxGroups);
  PCCL_ARG(top_groups >= 1 && top_groups <= groups, op << ": top_groups must be between 1 and groups");
  PCCL_ARG(top_k >= 1 && top_k <= block::kMaxTopK && top_k <= top_groups * (e / groups),
           op << ": top_k must be at least 1, at most " << block::kMaxTopK
              << " and at most the experts of the groups that stay");
  PCCL_ARG(!top2 || top_groups == groups || e / groups >= 2, op << ": the sum of a group's two best scores needs groups of two");
  PCCL_ARG(t * top_k < block::kMaxChoices, op << ": tokens * top_k must stay below 2^31 - 2^16");
  if (bias.has_value()) {
    PCCL_ARG(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == e,
             op << ": bias must be float32 [experts]");
    PCCL_ARG(!(at::GradMode::is_enabled() && bias->requires_grad()),
             op << ": the bias takes part in the choice alone and has no gradient; detach it");
  }
  if (mask.has_value())
    PCCL_ARG(mask->scalar_type() == at::kBool && mask->dim() == 1 && mask->size(0) == t, op << ": mask must be bool [tokens]");
  no_tangent(logits, op, "logits");
  no_tangent(bias, op, "bias");
  on_device(logits, logits, op, "logits");
  if (bias.has_value()) on_device(*bias, logits, op, "bias");
  if (mask.has_value()) on_device(*mask, logits, op, "mask");
  const RouteCall c{top_k, groups, top_groups, sigmoid, top2, renormalise, scale};
  if (at::GradMode::is_enabled() && logits.requires_grad()) return RouteFunction::apply(logits, c, bias, mask);
  return route_run(c, logits, bias, mask);
}

// ---- dispatch / combine ----------------------------------------------------------------------------------
block::MoveArgs move_args(const Tensor& x, const Tensor& rows) {
  block::MoveArgs a{};
  a.dtype = dtype_of(x);
  a.tokens = static_cast<int>(rows.size(0));
  a.top_k = static_cast<int>(rows.size(1));
  a.hidden = static_cast<int>(x.size(1));
  a.rows = rows.const_data_ptr<int32_t>();
  return a;
}

// Memory for finding the rows that no choice names; null where none is needed.
Tensor move_space(block::MoveArgs& a, const Tensor& like) {
  const size_t bytes = block::move_workspace(a);
  if (bytes == 0) return Tensor();
  Tensor space = fresh({static_cast<int64_t>(bytes / 4)}, at::kInt, like);
  a.workspace = space.mutable_data_ptr<int32_t>();
  return space;
}

void check_move(const char* op, const Tensor& x, const Tensor& rows, const Tensor& offsets) {
  PCCL_ARG(x.dim() == 2 && known(x.scalar_type()), op << ": rows must be a matrix of " << kTypes);
  PCCL_ARG(rows.dim() == 2 && rows.scalar_type() == at::kInt && rows.is_contiguous(),
           op << ": routing.rows must be contiguous int32 [tokens, top_k]");
  PCCL_ARG(offsets.dim() == 1 && offsets.scalar_type() == at::kInt && offsets.is_contiguous() && offsets.size(0) >= 1,
           op << ": routing.offsets must be contiguous int32 [experts + 1]");
  PCCL_ARG(rows.size(1) >= 1 && rows.numel() < INT_MAX, op << ": tokens * top_k must be below 2^31 and top_k at least 1");
  PCCL_ARG(x.size(1) >= 1 && x.size(1) <= (1 << 24), op << ": rows hold at least one value and at most 2^24");
}

Tensor dispatch_run(const Tensor& x, const Tensor& rows) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows src = as_rows(x);
  block::MoveArgs a = move_args(x, rows);
  Tensor out = fresh({rows.numel(), x.size(1)}, x.scalar_type(), x);
  const Tensor space = move_space(a, x);
  block::dispatch_rows(a, src.ptr(), src.ld, out.mutable_data_ptr(), stream_of(x));
  return out;
}

Tensor combine_run(const Tensor& y, const Tensor& weights, const Tensor& rows) {
  const c10::cuda::CUDAGuard guard(y.device());
  const Rows src = as_rows(y);
  block::MoveArgs a = move_args(y, rows);
  if (weights.defined()) a.weights = weights.const_data_ptr<float>();
  Tensor out = fresh({rows.size(0), y.size(1)}, y.scalar_type(), y);
  block::combine_rows(a, src.ptr(), src.ld, out.mutable_data_ptr(), stream_of(y));
  return out;
}

struct DispatchFunction : torch::autograd::Function<DispatchFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& rows) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({rows});
    return dispatch_run(x, rows);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(2);
    if (!grads[0].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    {
      at::NoGradGuard no_grad;
      result[0] = combine_run(grads[0], Tensor(), saved[0]);
    }
    once(result);
    return result;
  }
};

struct CombineFunction : torch::autograd::Function<CombineFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor& rows) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({y, weights, rows});
    return combine_run(y, weights, rows);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(3);
    if (!grads[0].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const Tensor &y = saved[0], &weights = saved[1], &rows = saved[2];
    {
      at::NoGradGuard no_grad;
      const c10::cuda::CUDAGuard guard(y.device());
      const Rows src = as_rows(y), d = as_rows(grads[0]);
      block::MoveArgs a = move_args(y, rows);
      a.weights = weights.const_data_ptr<float>();
      Tensor space;
      if (ctx->needs_input_grad(0)) {
        result[0] = fresh(y.sizes(), y.scalar_type(), y);
        space = move_space(a, y);
      }
      if (ctx->needs_input_grad(1)) result[1] = fresh(weights.sizes(), at::kFloat, y);
      block::combine_rows_backward(a, src.ptr(), src.ld, d.ptr(), d.ld,
                                   result[0].defined() ? result[0].mutable_data_ptr() : nullptr,
                                   result[1].defined() ? result[1].mutable_data_ptr<float>() : nullptr, stream_of(y));
    }
    once(result);
    return result;
  }
};

Tensor dispatch(const Tensor& x, const Tensor& rows, const Tensor& offsets) {
  const char* op = "dispatch";
  check_move(op, x, rows, offsets);
  PCCL_ARG(x.size(0) == rows.size(0), op << ": x has " << x.size(0) << " rows, the routing " << rows.size(0) << " tokens");
  no_tangent(x, op, "x");
  on_device(x, x, op, "x");
  on_device(rows, x, op, "routing.rows");
  on_device(offsets, x, op, "routing.offsets");
  if (at::GradMode::is_enabled() && x.requires_grad()) return DispatchFunction::apply(x, rows);
  return dispatch_run(x, rows);
}

Tensor combine(const Tensor& y, const Tensor& weights, const Tensor& rows, const Tensor& offsets) {
  const char* op = "combine";
  check_move(op, y, rows, offsets);
  PCCL_ARG(y.size(0) == rows.numel(), op << ": y has " << y.size(0) << " rows, the routing " << rows.numel() << " choices");
  PCCL_ARG(weights.scalar_type() == at::kFloat && weights.sizes() == rows.sizes() && weights.is_contiguous(),
           op << ": routing.weights must be contiguous float32 [tokens, top_k]");
  no_tangent(y, op, "y");
  no_tangent(weights, op, "routing.weights");
  on_device(y, y, op, "y");
  on_device(weights, y, op, "routing.weights");
  on_device(rows, y, op, "routing.rows");
  on_device(offsets, y, op, "routing.offsets");
  if (at::GradMode::is_enabled() && (y.requires_grad() || weights.requires_grad()))
    return CombineFunction::apply(y, weights, rows);
  return combine_run(y, weights, rows);
}

// ---- norms -------------------------------------------------------------------------------------------------
struct NormCall {
  double scale, eps;
  int64_t gate_rows;
};

block::Weight weight_of(const Tensor& t) {
  return block::Weight{t.defined() ? t.const_data_ptr() : nullptr, t.defined() && t.scalar_type() == at::kFloat ? 1 : 0};
}

// Contiguous weights and rows of one call, and the arguments that point into them.
struct NormInputs {
  Rows residual, x;
  Tensor gamma, post, gate;
  block::NormArgs a{};
  NormInputs(const NormCall& c, const Tensor& res, const Tensor& xt, const Tensor& g, const Tensor& p, const Tensor& gt)
      : residual(as_rows(res)), x(as_rows(xt)), gamma(g.defined() ? g.contiguous() : g),
        post(p.defined() ? p.contiguous() : p), gate(gt.defined() ? gt.contiguous() : gt) {
    a.hidden = static_cast<int>(res.size(-1));
    a.rows = res.numel() / a.hidden;
    a.rt = dtype_of(res);
    a.xt = xt.defined() ? dtype_of(xt) : a.rt;
    a.x = x.ptr();
    a.ldx = x.ld;
    a.residual = residual.ptr();
    a.ldr = residual.ld;
    a.gamma = weight_of(gamma);
    a.post_gamma = weight_of(post);
    a.gate = weight_of(gate);
    a.gate_rows = c.gate_rows;
    a.scale = static_cast<float>(c.scale);
    a.eps = static_cast<float>(c.eps);
  }
};

struct NormResult {
  Tensor y, h, r1, r2;
};

NormResult norm_run(const NormCall& c, const Tensor& residual, const Tensor& x, const Tensor& gamma, const Tensor& post,
                    const Tensor& gate, bool training) {
  const c10::cuda::CUDAGuard guard(residual.device());
  const NormInputs in(c, residual, x, gamma, post, gate);
  NormResult r;
  if (x.defined()) r.h = fresh(residual.sizes(), residual.scalar_type(), residual);
  if (gamma.defined()) r.y = fresh(residual.sizes(), x.defined() ? x.scalar_type() : residual.scalar_type(), residual);
  if (training && post.defined()) r.r1 = fresh({in.a.rows}, at::kFloat, residual);
  if (training && gamma.defined()) r.r2 = fresh({in.a.rows}, at::kFloat, residual);
  block::norm_forward(in.a, r.h.defined() ? r.h.mutable_data_ptr() : nullptr,
                      r.y.defined() ? r.y.mutable_data_ptr() : nullptr,
                      r.r1.defined() ? r.r1.mutable_data_ptr<float>() : nullptr,
                      r.r2.defined() ? r.r2.mutable_data_ptr<float>() : nullptr, stream_of(residual));
  return r;
}

// Outputs: [y] without x, [h] without gamma, else [y, h].
struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& residual, const OptTensor& x, const OptTensor& gamma,
                               const OptTensor& post, const OptTensor& gate, const NormCall& c) {
    const NormResult r = norm_run(c, residual, or_none(x), or_none(gamma), or_none(post), or_none(gate), true);
    ctx->set_materialize_grads(false);
    // A stream of 32 bits is read back as it stands; a 16-bit one is formed again from what made it.
    const bool keep_h = x.has_value() && residual.scalar_type() == at::kFloat && gamma.has_value();
    const bool form_h = gamma.has_value() && !keep_h;
    const bool keep_x = x.has_value() && (post.has_value() || gate.has_value() || form_h);
    ctx->save_for_backward({form_h ? residual : Tensor(), keep_x ? *x : Tensor(), or_none(gamma), or_none(post),
                            or_none(gate), keep_h ? r.h : Tensor(), r.r1, r.r2});
    keep(ctx, c);
    ctx->saved_data["x"] = x.has_value();
    ctx->saved_data["xt"] = static_cast<int64_t>(x.has_value() ? x->scalar_type() : residual.scalar_type());
    ctx->saved_data["rt"] = static_cast<int64_t>(residual.scalar_type());
    variable_list out;
    if (r.y.defined()) out.push_back(r.y);
    if (r.h.defined()) out.push_back(r.h);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(6);
    const auto saved = ctx->get_saved_variables();
    const Tensor &gamma = saved[2], &post = saved[3], &gate = saved[4];
    const bool has_x = ctx->saved_data["x"].toBool();
    const auto xt = static_cast<at::ScalarType>(ctx->saved_data["xt"].toInt());
    const auto rt = static_cast<at::ScalarType>(ctx->saved_data["rt"].toInt());
    const Tensor dy = gamma.defined() ? grads[0] : Tensor();
    const Tensor dh = has_x ? grads.back() : Tensor();
    if (!dy.defined() && !dh.defined()) return result;
    {
      at::NoGradGuard no_grad;
      const Tensor& given = dy.defined() ? dy : dh;
      const c10::cuda::CUDAGuard guard(given.device());
      // A residual that is not read again is stood in for by a tensor of its shape and type.
      const Tensor residual = saved[0].defined() ? saved[0] : saved[5].defined() ? saved[5] : dh;
      Tensor x = saved[1];
      const bool full = post.defined() || gate.defined();
      NormInputs in(kept<NormCall>(ctx), residual, x, gamma, post, gate);
      in.a.xt = xt == at::kFloat ? block::DType::kF32 : xt == at::kHalf ? block::DType::kF16 : block::DType::kBF16;
      const Rows rdy = as_rows(dy), rdh = as_rows(dh);
      block::NormGrads g{};
      g.dy = rdy.ptr();
      g.lddy = rdy.ld;
      g.dh = rdh.ptr();
      g.lddh = rdh.ld;
      if (saved[5].defined()) g.h = saved[5].const_data_ptr();
      if (saved[6].defined()) g.r1 = saved[6].const_data_ptr<float>();
      if (saved[7].defined()) g.r2 = saved[7].const_data_ptr<float>();
      size_t edge = 0;
      const bool want_res = ctx->needs_input_grad(edge++);
      const bool want_x = has_x && ctx->needs_input_grad(edge++);
      const bool want_gamma = gamma.defined() && ctx->needs_input_grad(edge++);
      const bool want_post = post.defined() && ctx->needs_input_grad(edge++);
      const bool want_gate = gate.defined() && ctx->needs_input_grad(edge++);
      // Without a gate, a norm behind or a scale both gradients are the same numbers: one is written.
      const bool same = want_res && want_x && !full && xt == rt && in.a.scale == 1.f;
      if (want_res) {
        result[0] = fresh(given.sizes(), rt, given);
        g.dresidual = result[0].mutable_data_ptr();
      }
      if (want_x) {
        result[1] = same ? result[0] : fresh(given.sizes(), xt, given);
        if (!same) g.dx = result[1].mutable_data_ptr();
      }
      const bool none = in.a.rows == 0;
      const auto weight = [&](const Tensor& w) {
        return none ? at::zeros(w.sizes(), w.options().requires_grad(false)) : fresh(w.sizes(), w.scalar_type(), w);
      };
      if (want_gamma) { result[2] = weight(gamma); g.dgamma = result[2].mutable_data_ptr(); }
      if (want_post) { result[3] = weight(post); g.dpost_gamma = result[3].mutable_data_ptr(); }
      if (want_gate) { result[4] = weight(gate); g.dgate = result[4].mutable_data_ptr(); }
      Tensor workspace;
      if (!none) {
        if (const size_t bytes = block::norm_workspace(in.a, g)) {
          workspace = fresh({static_cast<int64_t>(bytes)}, at::kByte, given);
          g.workspace = workspace.mutable_data_ptr();
        }
        block::norm_backward(in.a, g, stream_of(given));
      }
    }
    once(result);
    return result;
  }
};

void check_weight(const char* op, const OptTensor& w, int64_t hidden, at::ScalarType xt, const char* what) {
  if (!w.has_value()) return;
  PCCL_ARG(w->dim() == 1 && w->size(0) == hidden, op << ": " << what << " must be [hidden]");
  PCCL_ARG(w->scalar_type() == xt || w->scalar_type() == at::kFloat, op << ": " << what << " must have the activations' type or float32");
}

// (y or None, h or None)
std::pair<OptTensor, OptTensor> residual_rms_norm(const Tensor& residual, const OptTensor& x, const OptTensor& gamma,
                                                  const OptTensor& post_gamma, const OptTensor& gate, double scale,
                                                  double eps) {
  const char* op = x.has_value() ? "residual_rms_norm" : "rms_norm";
  const char* first = x.has_value() ? "residual" : "x";
  PCCL_ARG(residual.dim() >= 1, op << ": " << first << " must be [..., hidden]");
  PCCL_ARG(known(residual.scalar_type()), op << ": " << first << " must be " << kTypes);
  const int64_t hidden = residual.size(-1);
  PCCL_ARG(hidden >= 1 && hidden <= block::kMaxNormHidden,
           op << ": hidden must be between 1 and " << block::kMaxNormHidden << ", not " << hidden);
  at::ScalarType xt = residual.scalar_type();
  if (x.has_value()) {
    xt = x->scalar_type();
    PCCL_ARG(known(xt), op << ": x must be " << kTypes);
    PCCL_ARG(x->sizes() == residual.sizes(), op << ": x and residual must have the same shape");
    PCCL_ARG(residual.scalar_type() == xt || residual.scalar_type() == at::kFloat,
             op << ": residual must have the type of x or float32");
  }
  PCCL_ARG(x.has_value() || gamma.has_value(), op << ": gamma is missing");
  check_weight(op, gamma, hidden, xt, "gamma");
  check_weight(op, post_gamma, hidden, xt, "post_gamma");
  NormCall c{scale, eps, 1};
  const int64_t rows = residual.numel() / hidden;
  if (gate.has_value()) {
    PCCL_ARG(gate->scalar_type() == xt || gate->scalar_type() == at::kFloat, op << ": gate must have the activations' type or float32");
    PCCL_ARG((gate->dim() == 1 || gate->dim() == 2) && gate->size(-1) == hidden, op << ": gate must be [hidden] or [sequences, hidden]");
    const int64_t groups = gate->dim() == 2 ? gate->size(0) : 1;
    PCCL_ARG(groups >= 1 && rows % groups == 0, op << ": the rows must divide evenly over the gate's " << groups << " sequences");
    c.gate_rows = rows > 0 ? rows / groups : 1;
  }
  PCCL_ARG(eps >= 0, op << ": eps must not be negative");
  no_tangent(residual, op, first);
  no_tangent(x, op, "x");
  no_tangent(gamma, op, "gamma");
  no_tangent(post_gamma, op, "post_gamma");
  no_tangent(gate, op, "gate");
  on_device(residual, residual, op, first);
  if (x.has_value()) on_device(*x, residual, op, "x");
  if (gamma.has_value()) on_device(*gamma, residual, op, "gamma");
  if (post_gamma.has_value()) on_device(*post_gamma, residual, op, "post_gamma");
  if (gate.has_value()) on_device(*gate, residual, op, "gate");
  std::pair<OptTensor, OptTensor> out;
  if (at::GradMode::is_enabled() &&
      (wants_grad(residual) || wants_grad(x) || wants_grad(gamma) || wants_grad(post_gamma) || wants_grad(gate))) {
    const variable_list r = NormFunction::apply(residual, x, gamma, post_gamma, gate, c);
    if (gamma.has_value()) out.first = r.front();
    if (x.has_value()) out.second = r.back();
    return out;
  }
  const NormResult r = norm_run(c, residual, or_none(x), or_none(gamma), or_none(post_gamma), or_none(gate), false);
  if (r.y.defined()) out.first = r.y;
  if (r.h.defined()) out.second = r.h;
  return out;
}

}  // namespace

void bind_block_ops(py::module_& m) {
  auto b = m.def_submodule("block", "operators around a block's matrix products: routing, dispatch / combine, norms");
  b.def("route_topk", &route_topk, py::arg("logits"), py::arg("top_k"), py::arg("bias"), py::arg("sigmoid"),
        py::arg("groups"), py::arg("top_groups"), py::arg("top2"), py::arg("renormalise"), py::arg("scale"), py::arg("mask"));
  b.def("dispatch", &dispatch, py::arg("x"), py::arg("rows"), py::arg("offsets"));
  b.def("combine", &combine, py::arg("y"), py::arg("weights"), py::arg("rows"), py::arg("offsets"));
  b.def("residual_rms_norm", &residual_rms_norm, py::arg("residual"), py::arg("x"), py::arg("gamma"),
        py::arg("post_gamma"), py::arg("gate"), py::arg("scale"), py::arg("eps"));
}

}  // namespace pccl
