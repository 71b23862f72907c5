// The logits operators for torch, over the C entries of libmtaz.so: nodes of its autograd graph where a gradient is
// required, plain calls elsewhere.
//
// A node written in Python has the engine's own thread wait for the interpreter: forward and backward of a loss of 64 x
// 554 took the host 105 us that way and takes 72 here.  A call without gradients costs it 3 us less than through ctypes.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "mtaz.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

int type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? MTAZ_F32 : t.scalar_type() == at::kHalf ? MTAZ_F16 : MTAZ_BF16;
}
// t with its last dimension dense (a copy where it is not)
Tensor unit(const Tensor& t) { return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }
Tensor or_none(const MaybeTensor& t) { return t ? *t : Tensor(); }
void* at(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// elements from one row to the next; 0 where one row serves all
int64_t row_stride(const Tensor& t) { return !t.defined() || t.dim() == 1 || t.size(0) == 1 ? 0 : t.stride(0); }
int64_t checked(int64_t rc) {
  TORCH_CHECK(rc >= 0, "mtaz error ", rc, ": ", mtaz_last_error());
  return rc;
}
void* stream_of(AutogradContext* ctx) { return (void*)ctx->saved_data["stream"].toInt(); }   // a node runs where it was made

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

// The loss and the rows' statistics; with gradients of scale * loss where dz or dv is defined.
std::pair<Tensor, Tensor> loss_of(const Tensor& logits, const Tensor& value, const Tensor& target, const Tensor& reward,
                                  const Tensor& legal, const Tensor& dz, const Tensor& dv, double scale, int64_t stream) {
  const Tensor z = unit(logits), t = unit(target), mask = unit(legal), v = dense(value), r = dense(reward);
  const int64_t rows = z.size(0), cols = z.size(1), work = checked(mtaz_policy_loss_workspace(rows, cols));
  const auto floats = z.options().dtype(at::kFloat);
  Tensor loss = at::empty({}, floats), stats = at::empty({4 * rows + work / 4}, floats);   // scratch memory behind them
  float* const s = (float*)stats.data_ptr();
  checked(mtaz_policy_loss(z.get_device(), rows, cols, type_of(z), type_of(t), at(z), z.stride(0), at(t), t.stride(0),
                           (const uint32_t*)at(mask), row_stride(mask), (const float*)at(v), (const float*)at(r),
                           (float*)at(loss), s, at(dz), cols, (float*)at(dv), scale, s + 4 * rows, work, (void*)stream));
  return {loss, stats};
}
Tensor adjusted(const Tensor& logits, const Tensor& bias, const Tensor& legal, const Tensor& a, const Tensor& n,
                const Tensor& p, const double* penalties, int64_t stream) {
  const Tensor x = unit(logits), b = unit(bias), mask = unit(legal), y = fresh(x);
  checked(mtaz_adjust_logits(x.get_device(), x.size(0), x.size(1), type_of(x), at(x), x.stride(0), at(y), x.size(1),
                             (const uint32_t*)at(mask), row_stride(mask), (const float*)at(b), row_stride(b),
                             (const int32_t*)at(a), a.defined() ? a.stride(0) : 0, a.defined() ? (int)a.size(1) : 0,
                             (const int32_t*)at(n), penalties, (const float*)at(p), (void*)stream));
  return y;
}
bool wanted(const Tensor& a, const MaybeTensor& b) {
  return at::GradMode::is_enabled() && (a.requires_grad() || (b && b->defined() && b->requires_grad()));
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const MaybeTensor& value, const Tensor& target,
                        const MaybeTensor& reward, const MaybeTensor& legal, int64_t stream) {
    const auto [loss, stats] = loss_of(logits, or_none(value), target, or_none(reward), or_none(legal), Tensor(), Tensor(), 1.,
                                       stream);
    ctx->save_for_backward({logits, or_none(value), target, or_none(reward), or_none(legal), stats});
    ctx->saved_data["stream"] = stream;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor g = dense(grads[0]), z = unit(saved[0]), v = dense(saved[1]), t = unit(saved[2]), r = dense(saved[3]),
                 mask = unit(saved[4]);
    Tensor dz, dv;
    if (g.defined()) {
      if (ctx->needs_input_grad(0)) dz = fresh(z);
      if (v.defined() && ctx->needs_input_grad(1)) dv = fresh(v);
      const int64_t rows = z.size(0), cols = z.size(1);
      checked(mtaz_policy_loss_grad(z.get_device(), rows, cols, type_of(z), type_of(t), at(z), z.stride(0), at(t), t.stride(0),
                                    (const uint32_t*)at(mask), row_stride(mask), (const float*)at(v), (const float*)at(r),
                                    (const float*)at(saved[5]), (const float*)at(g), at(dz), cols, (float*)at(dv),
                                    stream_of(ctx)));
    }
    return once({dz, dv, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct AdjustLogits : torch::autograd::Function<AdjustLogits> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const MaybeTensor& bias, const MaybeTensor& legal,
                        const MaybeTensor& actions, const MaybeTensor& lengths, const MaybeTensor& per_row,
                        double repetition, double frequency, double presence, bool bends, int64_t stream) {
    const Tensor a = or_none(actions), n = or_none(lengths), p = or_none(per_row);
    const double penalties[3] = {repetition, frequency, presence};
    const Tensor y = adjusted(logits, or_none(bias), or_none(legal), a, n, p, penalties, stream);
    // where the penalties do not bend the logits their gradient is 1, and neither these nor the actions are needed
    ctx->save_for_backward(bends ? variable_list{logits, or_none(legal), a, n, p}
                                 : variable_list{Tensor(), or_none(legal), Tensor(), Tensor(), Tensor()});
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["type"] = (int64_t)type_of(logits);
    ctx->saved_data["repetition"] = repetition;
    if (bias && bias->defined()) ctx->saved_data["bias"] = bias->sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor g = unit(grads[0]), x = unit(saved[0]), mask = unit(saved[1]), a = saved[2], n = saved[3], p = saved[4];
    Tensor dx, db, work;
    if (g.defined()) {
      const int64_t rows = g.size(0), cols = g.size(1);
      int64_t size = 0;
      bool shared = false;
      if (ctx->needs_input_grad(0)) dx = fresh(g);
      const auto bias = ctx->saved_data.find("bias");
      if (bias != ctx->saved_data.end() && ctx->needs_input_grad(1)) {
        const std::vector<int64_t> shape = bias->second.toIntVector();
        db = at::empty(shape, g.options().dtype(at::kFloat));
        shared = shape.size() == 1 || shape[0] == 1;
        if (shared) {
          size = checked(mtaz_adjust_logits_grad_workspace(rows, cols));
          work = at::empty({size > 0 ? size : 1}, g.options().dtype(at::kByte));
        }
      }
      const double penalties[3] = {ctx->saved_data["repetition"].toDouble(), 0., 0.};   // the others are constants
      checked(mtaz_adjust_logits_grad(g.get_device(), rows, cols, (int)ctx->saved_data["type"].toInt(), at(g), g.stride(0),
                                      at(x), x.defined() ? x.stride(0) : 0, at(dx), cols, (float*)at(db), shared ? 0 : cols,
                                      (const uint32_t*)at(mask), row_stride(mask), (const int32_t*)at(a),
                                      a.defined() ? a.stride(0) : 0, a.defined() ? (int)a.size(1) : 0, (const int32_t*)at(n),
                                      penalties, (const float*)at(p), at(work), size, stream_of(ctx)));
    }
    variable_list out(11);
    out[0] = dx, out[1] = db;
    return once(std::move(out));
  }
};

Tensor policy_loss(const Tensor& logits, const MaybeTensor& value, const Tensor& target, const MaybeTensor& reward,
                   const MaybeTensor& legal, int64_t stream) {
  if (wanted(logits, value)) return PolicyLoss::apply(logits, value, target, reward, legal, stream);
  return loss_of(logits, or_none(value), target, or_none(reward), or_none(legal), Tensor(), Tensor(), 1., stream).first;
}
std::tuple<Tensor, Tensor, Tensor> policy_loss_grad(const Tensor& logits, const MaybeTensor& value, const Tensor& target,
                                                    const MaybeTensor& reward, const MaybeTensor& legal, double scale,
                                                    int64_t stream) {
  const at::NoGradGuard off;
  const Tensor v = or_none(value), dz = fresh(logits), dv = v.defined() ? fresh(v) : Tensor();
  return {loss_of(logits, v, target, or_none(reward), or_none(legal), dz, dv, scale, stream).first, dz, dv};
}
Tensor adjust_logits(const Tensor& logits, const MaybeTensor& bias, const MaybeTensor& legal, const MaybeTensor& actions,
                     const MaybeTensor& lengths, const MaybeTensor& per_row, double repetition, double frequency,
                     double presence, bool bends, int64_t stream) {
  if (!wanted(logits, bias)) {
    const double penalties[3] = {repetition, frequency, presence};
    return adjusted(logits, or_none(bias), or_none(legal), or_none(actions), or_none(lengths), or_none(per_row), penalties,
                    stream);
  }
  return AdjustLogits::apply(logits, bias, legal, actions, lengths, per_row, repetition, frequency, presence, bends, stream);
}
std::string built_from() { return MTAZ_AUTOGRAD_SHA256; }

}  // namespace

TORCH_LIBRARY(mtaz, m) {
  m.def("policy_loss", &policy_loss);
  m.def("policy_loss_grad", &policy_loss_grad);
  m.def("adjust_logits", &adjust_logits);
  m.def("built_from", &built_from);
}
