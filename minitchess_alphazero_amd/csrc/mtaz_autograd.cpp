// The logits operators for torch, over the C entries of libmtaz.so: nodes of its autograd graph where a gradient is
// required, plain calls elsewhere.
//
// Each operator is one of torch's dispatcher: an implementation on the GPU that calls the C entry, one that knows the
// results' shapes alone (Meta), and one for autograd where it has a gradient.  What records torch's operators (a tracer,
// tensors without data) so sees the operator itself, its backward pass likewise.  The stream is the current one of
// the moment of the call.
//
// A node written in Python has the engine's own thread wait for the interpreter: forward and backward of a loss of 64 x
// 554 took the host 105 us that way and takes 72 here.  A call without gradients costs it 3 us less than through ctypes.
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "mtaz.h"

// In one piece in the library, where build.py looks for it: what only a function returns, the compiler may store in parts.
extern "C" const char mtaz_autograd_built_from[] = MTAZ_AUTOGRAD_SHA256;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;
using Two = std::tuple<Tensor, Tensor>;
using Three = std::tuple<Tensor, Tensor, Tensor>;

int type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? MTAZ_F32 : t.scalar_type() == at::kHalf ? MTAZ_F16 : MTAZ_BF16;
}
// t with its last dimension dense (a copy where it is not)
Tensor unit(const Tensor& t) { return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor fresh(const Tensor& like) { return at::empty_symint(like.sym_sizes(), like.options()); }
Tensor or_none(const MaybeTensor& t) { return t ? *t : Tensor(); }
bool there(const MaybeTensor& t) { return t && t->defined(); }
void* at(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// elements from one row to the next; 0 where one row serves all
int64_t row_stride(const Tensor& t) { return !t.defined() || t.dim() == 1 || t.size(0) == 1 ? 0 : t.stride(0); }
int64_t checked(int64_t rc) {
  TORCH_CHECK(rc >= 0, "mtaz error ", rc, ": ", mtaz_last_error());
  return rc;
}
// the current stream of t's device; autograd's engine runs a backward pass on that of its forward pass
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// ---- the operators on the GPU -----------------------------------------------------------------------------------
// The loss, with the rows' statistics where stats is, and with gradients of scale * loss where dz or dv is defined
Tensor loss_of(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
               const MaybeTensor& legal, const Tensor& dz, const Tensor& dv, double scale, Tensor* stats) {
  const Tensor z = unit(logits), t = unit(target), mask = unit(or_none(legal)), v = dense(or_none(value)),
               r = dense(or_none(reward));
  const int64_t rows = z.size(0), cols = z.size(1), size = checked(mtaz_policy_loss_workspace(rows, cols));
  const auto floats = z.options().dtype(at::kFloat);
  const Tensor loss = at::empty({}, floats);
  if (stats) *stats = at::empty({rows, 4}, floats);
  // scratch memory, and the statistics behind it where nobody else wants them (on a boundary of 256 bytes)
  const int64_t floats_each = (size + 255) / 256 * 64;
  const Tensor work = at::empty({floats_each + (stats ? 0 : 4 * rows)}, floats);
  float* const w = (float*)work.data_ptr();
  checked(mtaz_policy_loss(z.get_device(), rows, cols, type_of(z), type_of(t), at(z), z.stride(0), at(t), t.stride(0),
                           (const uint32_t*)at(mask), row_stride(mask), (const float*)at(v), (const float*)at(r),
                           (float*)at(loss), stats ? (float*)at(*stats) : w + floats_each, at(dz), cols, (float*)at(dv),
                           scale, w, size, stream_of(z)));
  return loss;
}
Two loss_gpu(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
             const MaybeTensor& legal) {
  Tensor stats;
  const Tensor loss = loss_of(logits, value, target, reward, legal, Tensor(), Tensor(), 1., &stats);
  return {loss, stats};
}
Three loss_grad_gpu(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
                    const MaybeTensor& legal, double scale) {
  const Tensor dz = fresh(logits), dv = there(value) ? fresh(*value) : Tensor();
  return {loss_of(logits, value, target, reward, legal, dz, dv, scale, nullptr), dz, dv};
}
Two loss_back_gpu(const Tensor& grad, const Tensor& logits, const MaybeTensor& value, const Tensor& target,
                  const MaybeTensor& reward, const MaybeTensor& legal, const Tensor& stats, bool want_z, bool want_v) {
  const Tensor g = dense(grad), z = unit(logits), v = dense(or_none(value)), t = unit(target), r = dense(or_none(reward)),
               mask = unit(or_none(legal)), dz = want_z ? fresh(z) : Tensor(), dv = want_v ? fresh(v) : Tensor();
  checked(mtaz_policy_loss_grad(z.get_device(), z.size(0), z.size(1), type_of(z), type_of(t), at(z), z.stride(0), at(t),
                                t.stride(0), (const uint32_t*)at(mask), row_stride(mask), (const float*)at(v),
                                (const float*)at(r), (const float*)at(stats), (const float*)at(g), at(dz), z.size(1),
                                (float*)at(dv), stream_of(z)));
  return {dz, dv};
}
Tensor adjust_gpu(const Tensor& logits, const MaybeTensor& bias, const MaybeTensor& legal, const MaybeTensor& actions,
                  const MaybeTensor& lengths, const MaybeTensor& per_row, double repetition, double frequency,
                  double presence, bool) {
  const Tensor x = unit(logits), b = unit(or_none(bias)), mask = unit(or_none(legal)), a = or_none(actions), y = fresh(x);
  const double penalties[3] = {repetition, frequency, presence};
  checked(mtaz_adjust_logits(x.get_device(), x.size(0), x.size(1), type_of(x), at(x), x.stride(0), at(y), x.size(1),
                             (const uint32_t*)at(mask), row_stride(mask), (const float*)at(b), row_stride(b),
                             (const int32_t*)at(a), a.defined() ? a.stride(0) : 0, a.defined() ? (int)a.size(1) : 0,
                             (const int32_t*)at(or_none(lengths)), penalties, (const float*)at(or_none(per_row)),
                             stream_of(x)));
  return y;
}
// bias: the shape of the bias whose gradient is wanted
Two adjust_back_gpu(const Tensor& grad, const MaybeTensor& logits, const MaybeTensor& legal, const MaybeTensor& actions,
                    const MaybeTensor& lengths, const MaybeTensor& per_row, double repetition, bool want_x,
                    at::OptionalIntArrayRef bias) {
  const Tensor g = unit(grad), x = unit(or_none(logits)), mask = unit(or_none(legal)), a = or_none(actions);
  const int64_t rows = g.size(0), cols = g.size(1);
  const Tensor dx = want_x ? fresh(g) : Tensor();
  const bool shared = bias && (bias->size() == 1 || (*bias)[0] == 1);
  const int64_t size = shared ? checked(mtaz_adjust_logits_grad_workspace(rows, cols)) : 0;
  const auto floats = g.options().dtype(at::kFloat);
  const Tensor db = bias ? at::empty(*bias, floats) : Tensor(),
               work = shared ? at::empty({std::max<int64_t>(size, 4) / 4}, floats) : Tensor();
  const double penalties[3] = {repetition, 0., 0.};     // the others are constants
  checked(mtaz_adjust_logits_grad(g.get_device(), rows, cols, type_of(g), at(g), g.stride(0), at(x),
                                  x.defined() ? x.stride(0) : 0, at(dx), cols, (float*)at(db), shared ? 0 : cols,
                                  (const uint32_t*)at(mask), row_stride(mask), (const int32_t*)at(a),
                                  a.defined() ? a.stride(0) : 0, a.defined() ? (int)a.size(1) : 0,
                                  (const int32_t*)at(or_none(lengths)), penalties, (const float*)at(or_none(per_row)),
                                  at(work), size, stream_of(g)));
  return {dx, db};
}

// ---- their shapes -----------------------------------------------------------------------------------------------
Tensor floats_like(const Tensor& t, c10::SymIntArrayRef size) { return at::empty_symint(size, t.options().dtype(at::kFloat)); }

Two loss_meta(const Tensor& logits, const MaybeTensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&) {
  return {floats_like(logits, {}), floats_like(logits, {logits.sym_size(0), 4})};
}
Three loss_grad_meta(const Tensor& logits, const MaybeTensor& value, const Tensor&, const MaybeTensor&, const MaybeTensor&,
                     double) {
  return {floats_like(logits, {}), fresh(logits), there(value) ? fresh(*value) : Tensor()};
}
Two loss_back_meta(const Tensor&, const Tensor& logits, const MaybeTensor& value, const Tensor&, const MaybeTensor&,
                   const MaybeTensor&, const Tensor&, bool want_z, bool want_v) {
  return {want_z ? fresh(logits) : Tensor(), want_v ? fresh(*value) : Tensor()};
}
Tensor adjust_meta(const Tensor& logits, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&,
                   const MaybeTensor&, double, double, double, bool) {
  return fresh(logits);
}
Two adjust_back_meta(const Tensor& grad, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&,
                     const MaybeTensor&, double, bool want_x, at::OptionalIntArrayRef bias) {
  return {want_x ? fresh(grad) : Tensor(), bias ? at::empty(*bias, grad.options().dtype(at::kFloat)) : Tensor()};
}

// ---- autograd ---------------------------------------------------------------------------------------------------
// The operator `name` of F's type below autograd
template <typename F> auto operator_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
Two loss_below(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
               const MaybeTensor& legal) {
  static const auto op = operator_of<decltype(loss_gpu)>("mtaz::policy_loss");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, value, target, reward, legal);
}
Tensor adjust_below(const Tensor& logits, const MaybeTensor& bias, const MaybeTensor& legal, const MaybeTensor& actions,
                    const MaybeTensor& lengths, const MaybeTensor& per_row, double repetition, double frequency,
                    double presence, bool bends) {
  static const auto op = operator_of<decltype(adjust_gpu)>("mtaz::adjust_logits");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, bias, legal, actions, lengths, per_row, repetition, frequency, presence, bends);
}
bool wanted(const Tensor& a, const MaybeTensor& b) {
  return at::GradMode::is_enabled() && (a.requires_grad() || (there(b) && b->requires_grad()));
}

// An input that carries a tangent (forward-mode differentiation) is refused: without this the result would have none,
// which says that its derivative is 0.
template <typename... T> void no_tangent(const char* what, const T&... inputs) {
  auto has = [](const MaybeTensor& t) { return there(t) && t->_fw_grad(0).defined(); };
  TORCH_CHECK_VALUE(!(has(inputs) || ...), what, " has no forward-mode derivative");
}

// Gradients that cannot be differentiated once more: with create_graph they say so, and are no constants.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (auto& g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_());
  if (given.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is not twice differentiable", (int64_t)given.size());
  given = (*error)(std::move(given));
  size_t next = 0;
  for (auto& g : grads)
    if (g.defined()) g = given[next++];
  return grads;
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const MaybeTensor& value, const Tensor& target,
                        const MaybeTensor& reward, const MaybeTensor& legal, Tensor* stats) {
    Tensor loss;
    std::tie(loss, *stats) = loss_below(logits, value, target, reward, legal);
    ctx->save_for_backward({logits, or_none(value), target, or_none(reward), or_none(legal), *stats});
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto op = operator_of<decltype(loss_back_gpu)>("mtaz::policy_loss_back");
    const variable_list saved = ctx->get_saved_variables();
    Tensor dz, dv;
    if (grads[0].defined()) {
      no_tangent("policy_value_loss's backward pass", grads[0], saved[0], saved[1]);
      const at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dz, dv) = op.call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], saved[5],
                                 ctx->needs_input_grad(0), saved[1].defined() && ctx->needs_input_grad(1));
    }
    return once({dz, dv, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct AdjustLogits : torch::autograd::Function<AdjustLogits> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const MaybeTensor& bias, const MaybeTensor& legal,
                        const MaybeTensor& actions, const MaybeTensor& lengths, const MaybeTensor& per_row,
                        double repetition, double frequency, double presence, bool bends) {
    const Tensor y = adjust_below(logits, bias, legal, actions, lengths, per_row, repetition, frequency, presence, bends);
    // where the penalties do not bend the logits their gradient is 1, and neither these nor the actions are needed
    ctx->save_for_backward(bends ? variable_list{logits, or_none(legal), or_none(actions), or_none(lengths), or_none(per_row)}
                                 : variable_list{Tensor(), or_none(legal), Tensor(), Tensor(), Tensor()});
    ctx->saved_data["repetition"] = repetition;
    if (there(bias)) ctx->saved_data["bias"] = bias->sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto op = operator_of<decltype(adjust_back_gpu)>("mtaz::adjust_logits_back");
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(10);
    if (grads[0].defined()) {
      no_tangent("adjust_logits' backward pass", grads[0]);
      const auto bias = ctx->saved_data.find("bias");
      std::vector<int64_t> shape;
      at::OptionalIntArrayRef sizes;
      if (bias != ctx->saved_data.end() && ctx->needs_input_grad(1)) shape = bias->second.toIntVector(), sizes = shape;
      const at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1]) = op.call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4],
                                         ctx->saved_data["repetition"].toDouble(), ctx->needs_input_grad(0), sizes);
    }
    return once(std::move(out));
  }
};

Two loss_autograd(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
                  const MaybeTensor& legal) {
  no_tangent("policy_value_loss", logits, value, target, reward);
  if (!wanted(logits, value)) return loss_below(logits, value, target, reward, legal);
  Tensor stats;
  const Tensor loss = PolicyLoss::apply(logits, value, target, reward, legal, &stats);
  return {loss, stats};
}
// cut off from the graph
Three loss_grad_autograd(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
                         const MaybeTensor& legal, double scale) {
  static const auto op = operator_of<decltype(loss_grad_gpu)>("mtaz::policy_loss_grad");
  no_tangent("policy_value_loss_grad", logits, value, target, reward);
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(logits, value, target, reward, legal, scale);
}
Tensor adjust_autograd(const Tensor& logits, const MaybeTensor& bias, const MaybeTensor& legal, const MaybeTensor& actions,
                       const MaybeTensor& lengths, const MaybeTensor& per_row, double repetition, double frequency,
                       double presence, bool bends) {
  no_tangent("adjust_logits", logits, bias, per_row);
  if (!wanted(logits, bias))
    return adjust_below(logits, bias, legal, actions, lengths, per_row, repetition, frequency, presence, bends);
  return AdjustLogits::apply(logits, bias, legal, actions, lengths, per_row, repetition, frequency, presence, bends);
}
std::string built_from() { return mtaz_autograd_built_from; }

}  // namespace

TORCH_LIBRARY(mtaz, m) {
  m.def("policy_loss(Tensor logits, Tensor? value, Tensor target, Tensor? reward, Tensor? legal) -> (Tensor, Tensor)");
  m.def("policy_loss_grad(Tensor logits, Tensor? value, Tensor target, Tensor? reward, Tensor? legal, float scale) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("policy_loss_back(Tensor grad, Tensor logits, Tensor? value, Tensor target, Tensor? reward, Tensor? legal, "
        "Tensor stats, bool want_z, bool want_v) -> (Tensor, Tensor)");
  m.def("adjust_logits(Tensor logits, Tensor? bias, Tensor? legal, Tensor? actions, Tensor? lengths, Tensor? per_row, "
        "float repetition, float frequency, float presence, bool bends) -> Tensor");
  m.def("adjust_logits_back(Tensor grad, Tensor? logits, Tensor? legal, Tensor? actions, Tensor? lengths, "
        "Tensor? per_row, float repetition, bool want_x, int[]? bias) -> (Tensor, Tensor)");
  m.def("built_from() -> str", &built_from);
}
TORCH_LIBRARY_IMPL(mtaz, CUDA, m) {
  m.impl("policy_loss", &loss_gpu);
  m.impl("policy_loss_grad", &loss_grad_gpu);
  m.impl("policy_loss_back", &loss_back_gpu);
  m.impl("adjust_logits", &adjust_gpu);
  m.impl("adjust_logits_back", &adjust_back_gpu);
}
TORCH_LIBRARY_IMPL(mtaz, Meta, m) {
  m.impl("policy_loss", &loss_meta);
  m.impl("policy_loss_grad", &loss_grad_meta);
  m.impl("policy_loss_back", &loss_back_meta);
  m.impl("adjust_logits", &adjust_meta);
  m.impl("adjust_logits_back", &adjust_back_meta);
}
TORCH_LIBRARY_IMPL(mtaz, Autograd, m) {
  m.impl("policy_loss", &loss_autograd);
  m.impl("policy_loss_grad", &loss_grad_autograd);
  m.impl("adjust_logits", &adjust_autograd);
}
