// PyTorch-ROCm operators of the two ends of a network: embedding, and the softmax cross
// entropy of a linear layer over a large vocabulary (the reference has neither).
//
// As in register_block.cpp: implementations on the CUDA dispatch key, autograd kernels beside them.
#include <cmath>
#include <tuple>
#include <vector>

#include "register_parts.h"

namespace flash_hypercons {
namespace {

at::Tensor indices_of(const at::Tensor& t) {
  return (t.scalar_type() == at::kLong ? t : t.to(at::kLong)).contiguous();
}

bool index_type(const at::Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

// ---- embedding -----------------------------------------------------------------------

// [*tokens, streams, cols], without the streams where there are 0.
std::vector<int64_t> embedded(const at::Tensor& tokens, int64_t streams, int64_t cols) {
  auto shape = tokens.sizes().vec();
  if (streams > 0) shape.push_back(streams);
  shape.push_back(cols);
  return shape;
}

void check_tokens(const at::Tensor& tokens, int64_t streams) {
  TORCH_CHECK(tokens.is_cuda() && tokens.layout() == at::kStrided && index_type(tokens),
              "embedding: expected strided CUDA tokens in int64 or int32");
  TORCH_CHECK(streams >= 0 && streams < 1 << 16, "embedding: expected 1 <= streams < 2^16, or 0 for none");
}

// streams 0: no dimension of streams.
at::Tensor embedding_hip(const at::Tensor& tokens, const at::Tensor& weight, double scale, int64_t streams,
                         int64_t padding) {
  (void)padding;  // the gradient's
  check_tokens(tokens, streams);
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1 && strided_on(weight, tokens) &&
                  element_type(weight.scalar_type()),
              "embedding: expected weight [V, C], V, C >= 1, in float32, float16, or bfloat16 on the tokens' device");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(tokens.device());
  const int64_t vocab = weight.size(0), cols = weight.size(1);
  at::Tensor y = at::empty(embedded(tokens, streams, cols), weight.options());
  if (y.numel() == 0) return y;
  const at::Tensor t = indices_of(tokens), w = rows_of(weight, cols);
  check_status(fh_embedding(t.const_data_ptr<int64_t>(), w.const_data_ptr(), stride_of(w), scale,
                            static_cast<int>(std::max<int64_t>(streams, 1)), y.mutable_data_ptr(),
                            dtype_code(weight.scalar_type()), t.numel(), vocab, cols, current_stream()));
  return y;
}

at::Tensor embedding_backward_hip(const at::Tensor& grad, const at::Tensor& tokens, int64_t vocab, double scale,
                                  int64_t streams, int64_t padding) {
  check_tokens(tokens, streams);
  TORCH_CHECK(grad.dim() >= 1 && grad.size(-1) >= 1 && vocab >= 1 && strided_on(grad, tokens) &&
                  element_type(grad.scalar_type()) &&
                  grad.sizes() == at::IntArrayRef(embedded(tokens, streams, grad.size(-1))),
              "embedding: grad must match the result");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(tokens.device());
  const int64_t cols = grad.size(-1);
  at::Tensor dw = at::empty({vocab, cols}, grad.options());
  const at::Tensor t = indices_of(tokens), g = rows_of(grad, cols);
  with_workspace(grad, [&](void* workspace, int64_t* bytes) {
    return fh_embedding_backward(t.const_data_ptr<int64_t>(), g.const_data_ptr(), stride_of(g), scale,
                                 static_cast<int>(std::max<int64_t>(streams, 1)), padding, dw.mutable_data_ptr(),
                                 workspace, bytes, dtype_code(grad.scalar_type()), t.numel(), vocab, cols,
                                 current_stream());
  });
  return dw;
}

// ---- linear cross entropy --------------------------------------------------------------

void check_loss(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, const OptTensor& bias,
                int64_t reduction) {
  TORCH_CHECK(x.is_cuda() && x.layout() == at::kStrided && x.dim() >= 1 && x.size(-1) >= 1 &&
                  element_type(x.scalar_type()),
              "linear_cross_entropy: expected a strided CUDA [..., K] tensor, K >= 1, in float32, float16, or bfloat16");
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.size(0) >= 1 && strided_on(weight, x) &&
                  weight.scalar_type() == x.scalar_type(),
              "linear_cross_entropy: expected weight [V, K], V >= 1, of x's type and device");
  TORCH_CHECK(targets.sizes() == x.sizes().slice(0, x.dim() - 1) && strided_on(targets, x) && index_type(targets),
              "linear_cross_entropy: expected targets [...], x's dimensions but the last, in int64 or int32 on its device");
  TORCH_CHECK(!bias.has_value() ||
                  (bias->dim() == 1 && bias->size(0) == weight.size(0) && strided_on(*bias, x) &&
                   (bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat)),
              "linear_cross_entropy: expected bias [V] on x's device, of its type or float32");
  TORCH_CHECK(reduction >= FH_REDUCE_NONE && reduction <= FH_REDUCE_MEAN, "linear_cross_entropy: unknown reduction");
}

// (losses or their sum or mean, what the backward needs of each row).
std::tuple<at::Tensor, at::Tensor> loss_forward_hip(const at::Tensor& x, const at::Tensor& weight,
                                                    const at::Tensor& targets, const OptTensor& bias, int64_t ignore,
                                                    int64_t reduction) {
  check_loss(x, weight, targets, bias, reduction);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t cols = x.size(-1), vocab = weight.size(0), rows = x.numel() / cols;
  const auto floats = x.options().dtype(at::kFloat);
  at::Tensor lse = at::empty({rows, 2}, floats);
  if (rows == 0) {
    if (reduction == FH_REDUCE_NONE) return {at::empty(targets.sizes(), floats), lse};
    return {at::full({}, reduction == FH_REDUCE_MEAN ? NAN : 0.0, floats), lse};
  }
  at::Tensor loss = at::empty(reduction == FH_REDUCE_NONE ? targets.sizes() : at::IntArrayRef{}, floats);
  const at::Tensor xr = rows_of(x, cols), w = rows_of(weight, cols), b = vector_of(bias), t = indices_of(targets);
  with_workspace(x, [&](void* workspace, int64_t* bytes) {
    return fh_linear_cross_entropy(xr.const_data_ptr(), stride_of(xr), w.const_data_ptr(), stride_of(w), data_of(b),
                                   dtype_code(b.defined() ? b.scalar_type() : x.scalar_type()),
                                   t.const_data_ptr<int64_t>(), ignore, static_cast<int>(reduction),
                                   loss.mutable_data_ptr<float>(), lse.mutable_data_ptr<float>(), workspace, bytes,
                                   dtype_code(x.scalar_type()), rows, cols, vocab, current_stream());
  });
  return {loss, lse};
}

at::Tensor loss_hip(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, const OptTensor& bias,
                    int64_t ignore, int64_t reduction) {
  return std::get<0>(loss_forward_hip(x, weight, targets, bias, ignore, reduction));
}

// (dx, dweight, dbias), empty where not wanted.
std::tuple<at::Tensor, at::Tensor, at::Tensor> loss_backward_hip(const at::Tensor& grad, const at::Tensor& x,
                                                                 const at::Tensor& weight, const at::Tensor& targets,
                                                                 const OptTensor& bias, const at::Tensor& lse,
                                                                 int64_t ignore, int64_t reduction, bool want_x,
                                                                 bool want_weight, bool want_bias) {
  check_loss(x, weight, targets, bias, reduction);
  const int64_t cols = x.size(-1), vocab = weight.size(0), rows = x.numel() / cols;
  TORCH_CHECK(strided_on(grad, x) && grad.scalar_type() == at::kFloat &&
                  grad.sizes() == (reduction == FH_REDUCE_NONE ? targets.sizes() : at::IntArrayRef{}),
              "linear_cross_entropy: grad must match the result");
  TORCH_CHECK(strided_on(lse, x) && lse.scalar_type() == at::kFloat && lse.dim() == 2 && lse.size(0) == rows &&
                  lse.size(1) == 2 && lse.is_contiguous(),
              "linear_cross_entropy: expected the forward's sums");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const at::ScalarType bias_type = bias.has_value() ? bias->scalar_type() : x.scalar_type();
  const auto make = [&](bool want, at::IntArrayRef sizes, at::ScalarType type) {
    const auto options = x.options().dtype(type);
    return !want ? at::empty({0}, options) : rows == 0 ? at::zeros(sizes, options) : at::empty(sizes, options);
  };
  at::Tensor dx = make(want_x, x.sizes(), x.scalar_type());
  at::Tensor dw = make(want_weight, weight.sizes(), x.scalar_type());
  at::Tensor db = make(want_bias, {vocab}, bias_type);
  if (rows == 0) return {dx, dw, db};
  const at::Tensor xr = rows_of(x, cols), w = rows_of(weight, cols), b = vector_of(bias), t = indices_of(targets);
  const at::Tensor g = grad.resolve_neg().contiguous();
  with_workspace(x, [&](void* workspace, int64_t* bytes) {
    return fh_linear_cross_entropy_backward(
        xr.const_data_ptr(), stride_of(xr), w.const_data_ptr(), stride_of(w), data_of(b), dtype_code(bias_type),
        t.const_data_ptr<int64_t>(), ignore, static_cast<int>(reduction), lse.const_data_ptr<float>(),
        g.const_data_ptr<float>(), want_x ? dx.mutable_data_ptr() : nullptr,
        want_weight ? dw.mutable_data_ptr() : nullptr, want_bias ? db.mutable_data_ptr() : nullptr, workspace, bytes,
        dtype_code(x.scalar_type()), rows, cols, vocab, current_stream());
  });
  return {dx, dw, db};
}

// Whether a step forms the gradients with the loss, for the upstream gradient to scale: one product of
// four fewer, for FP32 sums of the weight's size, which are written and read once more.  Against forming the
// logits again, at 4096 x 32768, 1024 x 131072 (FP32: 10007) and 2048 x 10007: 0.99 to 1.04 times as long at 768
// rows of 16 bits, 0.95 to 0.98 at 1024, 0.88 to 0.90 at 2048; FP32 0.86 to 1.01 at 128, 0.86 to 0.89 at 256.
bool ahead_of(const at::Tensor& x, int64_t reduction) {
  return reduction != FH_REDUCE_NONE && x.sym_numel() >= x.sym_size(-1) * (x.scalar_type() == at::kFloat ? 128 : 1024);
}

// (loss, places, sums of dx, dweight and dbias), the last three empty where not wanted.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> loss_ahead_hip(
    const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, const OptTensor& bias, int64_t ignore,
    int64_t reduction, bool want_x, bool want_weight, bool want_bias) {
  check_loss(x, weight, targets, bias, reduction);
  const int64_t cols = x.size(-1), vocab = weight.size(0), rows = x.numel() / cols;
  TORCH_CHECK(reduction != FH_REDUCE_NONE && rows > 0, "linear_cross_entropy: expected a sum or mean over some rows");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const auto floats = x.options().dtype(at::kFloat);
  at::Tensor loss = at::empty({}, floats), places = at::empty({rows + 1}, x.options().dtype(at::kInt));
  at::Tensor dx = want_x ? at::empty({rows, cols}, floats) : at::empty({0}, floats);
  at::Tensor dw = want_weight ? at::empty({vocab, cols}, floats) : at::empty({0}, floats);
  at::Tensor db = want_bias ? at::empty({vocab}, floats) : at::empty({0}, floats);
  const at::Tensor xr = rows_of(x, cols), w = rows_of(weight, cols), b = vector_of(bias), t = indices_of(targets);
  with_workspace(x, [&](void* workspace, int64_t* bytes) {
    return fh_linear_cross_entropy_ahead(
        xr.const_data_ptr(), stride_of(xr), w.const_data_ptr(), stride_of(w), data_of(b),
        dtype_code(b.defined() ? b.scalar_type() : x.scalar_type()), t.const_data_ptr<int64_t>(), ignore,
        static_cast<int>(reduction), loss.mutable_data_ptr<float>(), places.mutable_data_ptr<int>(),
        want_x ? dx.mutable_data_ptr<float>() : nullptr, want_weight ? dw.mutable_data_ptr<float>() : nullptr,
        want_bias ? db.mutable_data_ptr<float>() : nullptr, workspace, bytes, dtype_code(x.scalar_type()), rows, cols,
        vocab, current_stream());
  });
  return {loss, places, dx, dw, db};
}

// (dx, dweight, dbias) from these, empty where their sums are.
std::tuple<at::Tensor, at::Tensor, at::Tensor> loss_scale_hip(const at::Tensor& grad, const at::Tensor& x,
                                                              const at::Tensor& weight, const at::Tensor& targets,
                                                              const OptTensor& bias, const at::Tensor& places,
                                                              const at::Tensor& dx_sums, const at::Tensor& dw_sums,
                                                              const at::Tensor& db_sums, int64_t ignore,
                                                              int64_t reduction) {
  check_loss(x, weight, targets, bias, reduction);
  const int64_t cols = x.size(-1), vocab = weight.size(0), rows = x.numel() / cols;
  TORCH_CHECK(strided_on(grad, x) && grad.scalar_type() == at::kFloat && grad.dim() == 0,
              "linear_cross_entropy: grad must match the result");
  const auto matches = [&](const at::Tensor& t, int64_t count, at::ScalarType type) {
    return strided_on(t, x) && t.scalar_type() == type && t.is_contiguous() && (t.numel() == 0 || t.numel() == count);
  };
  TORCH_CHECK(matches(places, rows + 1, at::kInt) && places.numel() > 0 && matches(dx_sums, rows * cols, at::kFloat) &&
                  matches(dw_sums, vocab * cols, at::kFloat) && matches(db_sums, vocab, at::kFloat),
              "linear_cross_entropy: expected the forward's sums");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const at::ScalarType bias_type = bias.has_value() ? bias->scalar_type() : x.scalar_type();
  const auto make = [&](const at::Tensor& sums, at::IntArrayRef sizes, at::ScalarType type) {
    return at::empty(sums.numel() > 0 ? sizes : at::IntArrayRef{0}, x.options().dtype(type));
  };
  at::Tensor dx = make(dx_sums, x.sizes(), x.scalar_type()), dw = make(dw_sums, weight.sizes(), x.scalar_type()),
             db = make(db_sums, {vocab}, bias_type);
  const auto floats = [](const at::Tensor& t) { return t.numel() > 0 ? t.const_data_ptr<float>() : nullptr; };
  const auto out = [](at::Tensor& t) { return t.numel() > 0 ? t.mutable_data_ptr() : nullptr; };
  const at::Tensor t = indices_of(targets), g = grad.resolve_neg();
  check_status(fh_linear_cross_entropy_scale(
      g.const_data_ptr<float>(), t.const_data_ptr<int64_t>(), ignore, static_cast<int>(reduction),
      places.const_data_ptr<int>(), floats(dx_sums), floats(dw_sums), floats(db_sums), out(dx), out(dw), out(db),
      dtype_code(bias_type), dtype_code(x.scalar_type()), rows, cols, vocab, current_stream()));
  return {dx, dw, db};
}

// ---- autograd -----------------------------------------------------------------------

class EmbeddingFunction : public torch::autograd::Function<EmbeddingFunction> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& tokens, const at::Tensor& weight, double scale,
                            int64_t streams, int64_t padding) {
    static const auto op = find_op<at::Tensor(const at::Tensor&, const at::Tensor&, double, int64_t, int64_t)>(
        "flash_hypercons::_embedding");
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.sym_size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["streams"] = streams;
    ctx->saved_data["padding"] = padding;
    return op.call(tokens, weight, scale, streams, padding);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}};
    const at::Tensor tokens = ctx->get_saved_variables()[0], &grad = grads[0];
    const c10::SymInt vocab = ctx->saved_data["vocab"].toSymInt();
    const int64_t streams = ctx->saved_data["streams"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    if (at::GradMode::is_enabled()) {
      // From differentiable pieces, for a backward that builds a graph.
      const int64_t rows = vocab.expect_int(), cols = grad.size(-1);
      at::Tensor g = grad.to(at::kFloat);
      if (streams > 0) g = g.sum(-2);
      const at::Tensor t = tokens.reshape({-1}).to(at::kLong);
      const at::Tensor valid = (t >= 0).logical_and(t < rows).logical_and(t != padding);
      g = at::where(valid.unsqueeze(1), g.reshape({-1, cols}) * scale, at::zeros({}, g.options()));
      const at::Tensor dw = at::zeros({rows, cols}, g.options()).index_add(0, at::where(valid, t, at::zeros_like(t)), g);
      return {{}, dw.to(grad.scalar_type()), {}, {}, {}};
    }
    static const auto op =
        find_op<at::Tensor(const at::Tensor&, const at::Tensor&, c10::SymInt, double, int64_t, int64_t)>(
            "flash_hypercons::_embedding_backward");
    at::AutoDispatchBelowADInplaceOrView below;  // nothing is recorded: straight to the kernels
    return {{}, op.call(grad, tokens, vocab, scale, streams, padding), {}, {}, {}};
  }
};

at::Tensor embedding_autograd(const at::Tensor& tokens, const at::Tensor& weight, double scale, int64_t streams,
                              int64_t padding) {
  if (at::GradMode::is_enabled() && wants_grad(weight))
    return EmbeddingFunction::apply(tokens, weight, scale, streams, padding);
  static const auto op = find_op<at::Tensor(const at::Tensor&, const at::Tensor&, double, int64_t, int64_t)>(
      "flash_hypercons::_embedding");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(tokens, weight, scale, streams, padding);
}

// The gradients from differentiable pieces, for a backward that builds a graph.
variable_list loss_gradients(const at::Tensor& grad, const at::Tensor& x, const at::Tensor& weight,
                             const at::Tensor& targets, const at::Tensor& bias, int64_t ignore, int64_t reduction) {
  const int64_t cols = x.size(-1), vocab = weight.size(0);
  const at::Tensor t = targets.reshape({-1}).to(at::kLong), here = t != ignore;
  const at::Tensor valid = (t >= 0).logical_and(t < vocab);
  const at::Tensor xf = x.to(at::kFloat).reshape({-1, cols}), wf = weight.to(at::kFloat);
  at::Tensor z = at::where(here.unsqueeze(1), xf, at::zeros({}, xf.options())).mm(wf.t());
  if (bias.defined()) z = z + bias.to(at::kFloat);
  at::Tensor f = reduction == FH_REDUCE_NONE ? grad.reshape({-1}) : grad.expand({t.size(0)});
  if (reduction == FH_REDUCE_MEAN) f = f / here.sum();
  f = at::where(valid, f, at::full({}, NAN, f.options()));
  f = at::where(here, f, at::zeros({}, f.options())).unsqueeze(1);
  const at::Tensor hot = at::zeros_like(z).scatter(1, at::where(valid, t, at::zeros_like(t)).unsqueeze(1), 1.0);
  const at::Tensor dz = at::where(here.unsqueeze(1), (z.softmax(1) - hot) * f, at::zeros({}, z.options()));
  return {dz.mm(wf).reshape(x.sizes()).to(x.scalar_type()),
          dz.t().mm(at::where(here.unsqueeze(1), xf, at::zeros({}, xf.options()))).to(x.scalar_type()),
          bias.defined() ? dz.sum(0).to(bias.scalar_type()) : at::Tensor()};
}

class LossFunction : public torch::autograd::Function<LossFunction> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const at::Tensor& targets, const OptTensor& bias, int64_t ignore, int64_t reduction) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    const int64_t want = wanted(x, weight, targets, bias);
    ctx->saved_data["wanted"] = want;
    if (ahead_of(x, reduction)) {
      static const auto op = find_op<std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>(
          const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&, int64_t, int64_t, bool, bool, bool)>(
          "flash_hypercons::_linear_cross_entropy_ahead");
      auto [loss, places, dx, dw, db] =
          op.call(x, weight, targets, bias, ignore, reduction, want & 1, want & 2, want & 8);
      ctx->save_for_backward({x, weight, targets, bias.value_or(at::Tensor()), places, dx, dw, db});
      return loss;
    }
    static const auto op =
        find_op<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                   const OptTensor&, int64_t, int64_t)>(
            "flash_hypercons::_linear_cross_entropy_forward");
    auto [loss, lse] = op.call(x, weight, targets, bias, ignore, reduction);
    ctx->save_for_backward({x, weight, targets, bias.value_or(at::Tensor()), lse});
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}, {}};
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &targets = saved[2], &bias = saved[3];
    const int64_t ignore = ctx->saved_data["ignore"].toInt(), reduction = ctx->saved_data["reduction"].toInt();
    const int64_t want = ctx->saved_data["wanted"].toInt();
    const bool want_x = want & 1, want_weight = want & 2, want_bias = want & 8;
    at::Tensor dx, dw, db;
    if (at::GradMode::is_enabled()) {
      const variable_list g = loss_gradients(grads[0], x, weight, targets, bias, ignore, reduction);
      std::tie(dx, dw, db) = std::make_tuple(g[0], g[1], g[2]);
      return {want_x ? dx : at::Tensor(), want_weight ? dw : at::Tensor(), {}, want_bias ? db : at::Tensor(), {}, {}};
    }
    at::AutoDispatchBelowADInplaceOrView below;  // nothing is recorded: straight to the kernels
    if (saved.size() > 5) {
      static const auto op = find_op<std::tuple<at::Tensor, at::Tensor, at::Tensor>(
          const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&,
          const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, int64_t)>(
          "flash_hypercons::_linear_cross_entropy_scale");
      std::tie(dx, dw, db) = op.call(grads[0], x, weight, targets, optional_of(bias), saved[4], saved[5], saved[6],
                                     saved[7], ignore, reduction);
    } else {
      static const auto op = find_op<std::tuple<at::Tensor, at::Tensor, at::Tensor>(
          const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&,
          const at::Tensor&, int64_t, int64_t, bool, bool, bool)>("flash_hypercons::_linear_cross_entropy_backward");
      std::tie(dx, dw, db) = op.call(grads[0], x, weight, targets, optional_of(bias), saved[4], ignore, reduction,
                                     want_x, want_weight, want_bias);
    }
    return {want_x ? dx : at::Tensor(), want_weight ? dw : at::Tensor(), {}, want_bias ? db : at::Tensor(), {}, {}};
  }
};

at::Tensor loss_autograd(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                         const OptTensor& bias, int64_t ignore, int64_t reduction) {
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LossFunction::apply(x, weight, targets, bias, ignore, reduction);
  static const auto op = find_op<at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&,
                                            int64_t, int64_t)>("flash_hypercons::_linear_cross_entropy");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, targets, bias, ignore, reduction);
}

}  // namespace
}  // namespace flash_hypercons

TORCH_LIBRARY_FRAGMENT(flash_hypercons, m) {
  m.def("_embedding(Tensor tokens, Tensor weight, float scale, int streams, int padding) -> Tensor");
  m.def("_embedding_backward(Tensor grad, Tensor tokens, SymInt vocab, float scale, int streams, int padding) -> Tensor");
  m.def("_linear_cross_entropy(Tensor x, Tensor weight, Tensor targets, Tensor? bias, int ignore, int reduction) -> "
        "Tensor");
  m.def("_linear_cross_entropy_forward(Tensor x, Tensor weight, Tensor targets, Tensor? bias, int ignore, "
        "int reduction) -> (Tensor, Tensor)");
  m.def("_linear_cross_entropy_backward(Tensor grad, Tensor x, Tensor weight, Tensor targets, Tensor? bias, Tensor lse, "
        "int ignore, int reduction, bool want_x, bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)");
  m.def("_linear_cross_entropy_ahead(Tensor x, Tensor weight, Tensor targets, Tensor? bias, int ignore, int reduction, "
        "bool want_x, bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("_linear_cross_entropy_scale(Tensor grad, Tensor x, Tensor weight, Tensor targets, Tensor? bias, Tensor places, "
        "Tensor dx_sums, Tensor dw_sums, Tensor db_sums, int ignore, int reduction) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(flash_hypercons, CUDA, m) {
  m.impl("_linear_cross_entropy_ahead", &flash_hypercons::loss_ahead_hip);
  m.impl("_linear_cross_entropy_scale", &flash_hypercons::loss_scale_hip);
  m.impl("_embedding", &flash_hypercons::embedding_hip);
  m.impl("_embedding_backward", &flash_hypercons::embedding_backward_hip);
  m.impl("_linear_cross_entropy", &flash_hypercons::loss_hip);
  m.impl("_linear_cross_entropy_forward", &flash_hypercons::loss_forward_hip);
  m.impl("_linear_cross_entropy_backward", &flash_hypercons::loss_backward_hip);
}

TORCH_LIBRARY_IMPL(flash_hypercons, Autograd, m) {
  m.impl("_embedding", &flash_hypercons::embedding_autograd);
  m.impl("_linear_cross_entropy", &flash_hypercons::loss_autograd);
}
