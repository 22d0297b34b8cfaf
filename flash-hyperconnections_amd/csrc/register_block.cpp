// PyTorch-ROCm operators of the block between two stream mixings: layer norm, the
// linear layer with its epilogue, and the clipping of gradients (the reference has
// none of them).
//
// As in register.cpp, the implementations sit on the CUDA dispatch key, check their
// inputs, allocate results and workspaces with torch's allocator and call the C ABI
// on the current HIP stream; the differentiable operators have their autograd kernel
// here too, so that an eager step enters Python once a call.
#include <algorithm>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "register_parts.h"

namespace flash_hypercons {
namespace {

// ---- layer norm -------------------------------------------------------------------

void check_norm(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias) {
  TORCH_CHECK(x.is_cuda() && x.layout() == at::kStrided && x.dim() >= 1 && x.size(-1) >= 1 &&
                  element_type(x.scalar_type()),
              "layer_norm: expected a strided CUDA [..., C] tensor, C >= 1, in float32, float16, or bfloat16");
  for (const OptTensor* p : {&weight, &bias})
    if (p->has_value())
      TORCH_CHECK((*p)->dim() == 1 && (*p)->size(0) == x.size(-1) && strided_on(**p, x) &&
                      ((*p)->scalar_type() == x.scalar_type() || (*p)->scalar_type() == at::kFloat),
                  "layer_norm: expected weight and bias [C] on x's device, of its type or float32");
  TORCH_CHECK(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(),
              "layer_norm: expected weight and bias of one type");
}

at::ScalarType norm_params(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias) {
  return weight.has_value() ? weight->scalar_type() : bias.has_value() ? bias->scalar_type() : x.scalar_type();
}

std::tuple<at::Tensor, at::Tensor> norm_run(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                            double eps, bool want_stats) {
  check_norm(x, weight, bias);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t cols = x.size(-1);
  at::Tensor y = at::empty(x.sizes(), x.options());
  const int64_t rows = x.numel() / cols;
  at::Tensor stats = want_stats ? at::empty({rows, 2}, x.options().dtype(at::kFloat)) : at::Tensor();
  if (rows > 0) {
    const at::Tensor xr = rows_of(x, cols), w = vector_of(weight), b = vector_of(bias);
    check_status(fh_layer_norm(xr.const_data_ptr(), stride_of(xr), data_of(w), data_of(b),
                               dtype_code(norm_params(x, weight, bias)), eps, y.mutable_data_ptr(),
                               want_stats ? stats.mutable_data_ptr<float>() : nullptr, dtype_code(x.scalar_type()),
                               rows, cols, current_stream()));
  }
  return {y, stats};
}

at::Tensor layer_norm_hip(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  return std::get<0>(norm_run(x, weight, bias, eps, false));
}

std::tuple<at::Tensor, at::Tensor> layer_norm_forward_hip(const at::Tensor& x, const OptTensor& weight,
                                                          const OptTensor& bias, double eps) {
  return norm_run(x, weight, bias, eps, true);
}

// (dx, dweight, dbias); the last two in the parameters' type, empty where not wanted.
std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward_hip(const at::Tensor& grad, const at::Tensor& x,
                                                                       const OptTensor& weight, const OptTensor& bias,
                                                                       const at::Tensor& stats, bool want_weight,
                                                                       bool want_bias) {
  check_norm(x, weight, bias);
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  TORCH_CHECK(grad.sizes() == x.sizes() && strided_on(grad, x) && grad.scalar_type() == x.scalar_type(),
              "layer_norm: grad must match x");
  TORCH_CHECK(strided_on(stats, x) && stats.scalar_type() == at::kFloat && stats.dim() == 2 &&
                  stats.size(0) == rows && stats.size(1) == 2 && stats.is_contiguous(),
              "layer_norm: expected the forward's statistics");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  at::Tensor dx = at::empty(x.sizes(), x.options());
  const auto params = x.options().dtype(norm_params(x, weight, bias));
  if (rows == 0) {
    return {dx, at::zeros({want_weight ? cols : 0}, params), at::zeros({want_bias ? cols : 0}, params)};
  }
  at::Tensor dw = at::empty({want_weight ? cols : 0}, params), db = at::empty({want_bias ? cols : 0}, params);
  const at::Tensor xr = rows_of(x, cols), gr = rows_of(grad, cols), w = vector_of(weight);
  with_workspace(x, [&](void* workspace, int64_t* bytes) {
    return fh_layer_norm_backward(xr.const_data_ptr(), stride_of(xr), gr.const_data_ptr(), stride_of(gr), data_of(w),
                                  dtype_code(params.dtype().toScalarType()), stats.const_data_ptr<float>(),
                                  dx.mutable_data_ptr(), want_weight ? dw.mutable_data_ptr() : nullptr,
                                  want_bias ? db.mutable_data_ptr() : nullptr, workspace, bytes,
                                  dtype_code(x.scalar_type()), rows, cols, current_stream());
  });
  return {dx, dw, db};
}

// ---- linear ------------------------------------------------------------------------

void check_linear(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                  int64_t act) {
  TORCH_CHECK(x.is_cuda() && x.layout() == at::kStrided && x.dim() >= 1 && x.size(-1) >= 1 &&
                  element_type(x.scalar_type()),
              "linear: expected a strided CUDA [..., K] tensor, K >= 1, in float32, float16, or bfloat16");
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.size(0) >= 1 && strided_on(weight, x) &&
                  weight.scalar_type() == x.scalar_type(),
              "linear: expected weight [N, K], N >= 1, of x's type and device");
  TORCH_CHECK(!bias.has_value() ||
                  (bias->dim() == 1 && bias->size(0) == weight.size(0) && strided_on(*bias, x) &&
                   (bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat)),
              "linear: expected bias [N] on x's device, of its type or float32");
  if (residual.has_value()) {
    auto want = x.sizes().vec();
    want.back() = weight.size(0);
    TORCH_CHECK(residual->sizes() == at::IntArrayRef(want) && strided_on(*residual, x) &&
                    residual->scalar_type() == x.scalar_type(),
                "linear: expected residual [..., N] of x's type and device");
  }
  TORCH_CHECK(act >= FH_ACT_NONE && act <= FH_ACT_SILU, "linear: unknown activation");
}

std::tuple<at::Tensor, at::Tensor> linear_run(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                                              const OptTensor& residual, int64_t act, bool save) {
  check_linear(x, weight, bias, residual, act);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t cols = x.size(-1), outs = weight.size(0), rows = x.numel() / cols;
  auto shape = x.sizes().vec();
  shape.back() = outs;
  at::Tensor y = at::empty(shape, x.options());
  // The sum before the activation: FP32, or FP16 for either 16-bit type.
  save = save && act != FH_ACT_NONE;
  at::Tensor saved = at::empty({save ? rows : 0, outs},
                               x.options().dtype(x.scalar_type() == at::kFloat ? at::kFloat : at::kHalf));
  if (rows > 0) {
    const at::Tensor xr = rows_of(x, cols), w = rows_of(weight, cols), b = vector_of(bias);
    const at::Tensor r = residual.has_value() ? rows_of(*residual, outs) : at::Tensor();
    with_workspace(x, [&](void* workspace, int64_t* bytes) {
      return fh_linear(xr.const_data_ptr(), stride_of(xr), w.const_data_ptr(), stride_of(w), data_of(b),
                       dtype_code(b.defined() ? b.scalar_type() : x.scalar_type()), data_of(r),
                       r.defined() ? stride_of(r) : 0, static_cast<int>(act), y.mutable_data_ptr(),
                       save ? saved.mutable_data_ptr() : nullptr, workspace, bytes, dtype_code(x.scalar_type()), rows,
                       cols, outs, current_stream());
    });
  }
  return {y, saved};
}

at::Tensor linear_hip(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                      int64_t act) {
  return std::get<0>(linear_run(x, weight, bias, residual, act, false));
}

std::tuple<at::Tensor, at::Tensor> linear_forward_hip(const at::Tensor& x, const at::Tensor& weight,
                                                      const OptTensor& bias, const OptTensor& residual, int64_t act) {
  return linear_run(x, weight, bias, residual, act, true);
}

// (dx, dweight, dbias), empty where not wanted.
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_backward_hip(const at::Tensor& grad, const at::Tensor& x,
                                                                   const at::Tensor& weight, const OptTensor& bias,
                                                                   const at::Tensor& saved, int64_t act, bool want_x,
                                                                   bool want_weight, bool want_bias) {
  check_linear(x, weight, bias, std::nullopt, act);
  const int64_t cols = x.size(-1), outs = weight.size(0), rows = x.numel() / cols;
  auto shape = x.sizes().vec();
  shape.back() = outs;
  TORCH_CHECK(grad.sizes() == at::IntArrayRef(shape) && strided_on(grad, x) && grad.scalar_type() == x.scalar_type(),
              "linear: grad must match the result");
  const at::ScalarType saved_type = x.scalar_type() == at::kFloat ? at::kFloat : at::kHalf;
  TORCH_CHECK(act == FH_ACT_NONE || (strided_on(saved, x) && saved.scalar_type() == saved_type && saved.dim() == 2 &&
                                     saved.size(0) == rows && saved.size(1) == outs && saved.is_contiguous()),
              "linear: expected the forward's saved sums");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const at::ScalarType bias_type = bias.has_value() ? bias->scalar_type() : x.scalar_type();
  const auto make = [&](bool want, at::IntArrayRef sizes, at::ScalarType type) {
    const auto options = x.options().dtype(type);
    return !want ? at::empty({0}, options) : rows == 0 ? at::zeros(sizes, options) : at::empty(sizes, options);
  };
  at::Tensor dx = make(want_x, x.sizes(), x.scalar_type());
  at::Tensor dw = make(want_weight, weight.sizes(), x.scalar_type());
  at::Tensor db = make(want_bias, {outs}, bias_type);
  if (rows == 0) return {dx, dw, db};
  const at::Tensor xr = rows_of(x, cols), w = rows_of(weight, cols), g = rows_of(grad, outs);
  with_workspace(x, [&](void* workspace, int64_t* bytes) {
    return fh_linear_backward(xr.const_data_ptr(), stride_of(xr), w.const_data_ptr(), stride_of(w),
                              g.const_data_ptr(), stride_of(g), act == FH_ACT_NONE ? nullptr : saved.const_data_ptr(),
                              static_cast<int>(act), want_x ? dx.mutable_data_ptr() : nullptr,
                              want_weight ? dw.mutable_data_ptr() : nullptr,
                              want_bias ? db.mutable_data_ptr() : nullptr, dtype_code(bias_type), workspace, bytes,
                              dtype_code(x.scalar_type()), rows, cols, outs, current_stream());
  });
  return {dx, dw, db};
}

// ---- global norm and clipping -------------------------------------------------------

// Arrays that the kernels take as flat memory: every tensor without gaps or overlaps
// whatever its dimensions' order; the others through a contiguous copy.
struct Arrays {
  std::vector<const void*> data;
  std::vector<int64_t> sizes;
  std::vector<int> dtypes;
  std::vector<at::Tensor> copies;               // keep the copies alive
  std::vector<std::pair<at::Tensor, at::Tensor>> back;  // (copy, original) of gapped tensors

  Arrays(at::TensorList tensors, const char* op, bool inplace) {
    const size_t n = tensors.size();
    data.reserve(n);
    sizes.reserve(n);
    dtypes.reserve(n);
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (const at::Tensor& t : tensors) {
      TORCH_CHECK(t.is_cuda() && t.layout() == at::kStrided && element_type(t.scalar_type()) &&
                      t.device() == tensors[0].device(),
                  op, ": expected strided CUDA tensors of one device in float32, float16, or bfloat16");
      at::Tensor flat = t;
      if (t.is_neg() || !t.is_non_overlapping_and_dense()) {
        flat = t.resolve_neg().contiguous();
        copies.push_back(flat);
        if (inplace) back.emplace_back(flat, t);
      }
      // What is written in place has storage of its own from here on, where a lazy clone shared it.
      data.push_back(inplace ? flat.mutable_data_ptr() : flat.const_data_ptr());
      if (inplace && t.numel() > 0) {
        const auto at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) {
          TORCH_CHECK(t.stride(d) != 0 || t.size(d) == 1, op, ": a tensor's elements share memory");
          last += (t.size(d) - 1) * t.stride(d);
        }
        // Gapped tensors may interleave; they are copied, and not looked at here.
        if (t.is_non_overlapping_and_dense()) spans.emplace_back(at, at + (last + 1) * t.element_size());
      }
      sizes.push_back(flat.numel());
      dtypes.push_back(dtype_code(t.scalar_type()));
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      TORCH_CHECK(spans[i].first >= spans[i - 1].second, op, ": two tensors share memory");
  }
  int count() const { return static_cast<int>(data.size()); }
};

at::Tensor grad_norm_hip(at::TensorList tensors, double norm_type) {
  TORCH_CHECK(!tensors.empty(), "grad_norm: no tensors");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(tensors[0].device());
  const Arrays a(tensors, "grad_norm", false);
  at::Tensor norm = at::empty({}, tensors[0].options().dtype(at::kFloat));
  with_workspace(norm, [&](void* workspace, int64_t* bytes) {
    return fh_grad_norm(a.count(), a.data.data(), a.sizes.data(), a.dtypes.data(), norm_type,
                        norm.mutable_data_ptr<float>(), workspace, bytes, current_stream());
  });
  return norm;
}

at::Tensor clip_into(const at::TensorList tensors, Arrays& a, void* const* out, double max_norm, double norm_type) {
  at::Tensor norm = at::empty({}, tensors[0].options().dtype(at::kFloat));
  with_workspace(norm, [&](void* workspace, int64_t* bytes) {
    return fh_clip_gradients(a.count(), a.data.data(), out, a.sizes.data(), a.dtypes.data(), norm_type, max_norm,
                             norm.mutable_data_ptr<float>(), workspace, bytes, current_stream());
  });
  return norm;
}

std::tuple<std::vector<at::Tensor>, at::Tensor> clip_grads_hip(at::TensorList tensors, double max_norm,
                                                               double norm_type) {
  TORCH_CHECK(!tensors.empty(), "clip_grad_norm: no tensors");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(tensors[0].device());
  Arrays a(tensors, "clip_grad_norm", false);
  std::vector<at::Tensor> clipped;
  std::vector<void*> out;
  clipped.reserve(tensors.size());
  out.reserve(tensors.size());
  for (const at::Tensor& t : tensors) {
    // Dense tensors keep their strides, whose memory order the kernels copy; others are contiguous.
    const bool dense = !t.is_neg() && t.is_non_overlapping_and_dense();
    clipped.push_back(dense ? at::empty_strided(t.sizes(), t.strides(), t.options()) : at::empty(t.sizes(), t.options()));
    out.push_back(clipped.back().mutable_data_ptr());
  }
  at::Tensor norm = clip_into(tensors, a, out.data(), max_norm, norm_type);
  return {std::move(clipped), std::move(norm)};
}

at::Tensor clip_grads_inplace_hip(at::TensorList tensors, double max_norm, double norm_type) {
  TORCH_CHECK(!tensors.empty(), "clip_grad_norm_: no tensors");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(tensors[0].device());
  Arrays a(tensors, "clip_grad_norm_", true);
  at::Tensor norm = clip_into(tensors, a, nullptr, max_norm, norm_type);
  for (auto& [copy, original] : a.back) original.copy_(copy);
  for (const at::Tensor& t : tensors)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

// ---- autograd -----------------------------------------------------------------------

// The gradients from differentiable pieces, for a backward that builds a graph.
variable_list norm_gradients(const at::Tensor& grad, const at::Tensor& x, const at::Tensor& weight,
                             const at::Tensor& bias, double eps) {
  const at::Tensor xf = x.to(at::kFloat), g = grad.to(at::kFloat);
  const at::Tensor d = xf - xf.mean(-1, true);
  const at::Tensor r = (d.square().mean(-1, true) + eps).rsqrt(), n = d * r;
  const at::Tensor q = weight.defined() ? g * weight.to(at::kFloat) : g;
  const at::Tensor dx = r * (q - q.mean(-1, true) - n * (q * n).mean(-1, true));
  const int64_t cols = x.size(-1);
  const auto sum = [&](const at::Tensor& v, const at::Tensor& like) {
    return like.defined() ? v.reshape({-1, cols}).sum(0).to(like.scalar_type()) : at::Tensor();
  };
  return {dx.to(x.scalar_type()), sum(g * n, weight), sum(g, bias)};
}

class LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& weight, const OptTensor& bias,
                            double eps) {
    static const auto op = find_op<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const OptTensor&,
                                                                      const OptTensor&, double)>(
        "flash_hypercons::_layer_norm_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, stats] = op.call(x, weight, bias, eps);
    ctx->save_for_backward({x, weight.value_or(at::Tensor()), bias.value_or(at::Tensor()), stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["wanted"] = wanted(x, weight, bias);
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    if (!grads[0].defined()) return {{}, {}, {}, {}};
    if (at::GradMode::is_enabled()) {
      variable_list g = norm_gradients(grads[0], x, weight, bias, ctx->saved_data["eps"].toDouble());
      return {g[0], g[1], g[2], {}};
    }
    static const auto op =
        find_op<std::tuple<at::Tensor, at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const OptTensor&,
                                                               const OptTensor&, const at::Tensor&, bool, bool)>(
            "flash_hypercons::_layer_norm_backward");
    const int64_t want = ctx->saved_data["wanted"].toInt();
    const bool want_weight = want & 2, want_bias = want & 4;
    auto [dx, dw, db] = op.call(grads[0], x, optional_of(weight), optional_of(bias), stats, want_weight, want_bias);
    return {dx, want_weight ? dw : at::Tensor(), want_bias ? db : at::Tensor(), {}};
  }
};

at::Tensor layer_norm_autograd(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LayerNormFunction::apply(x, weight, bias, eps);
  static const auto op =
      find_op<at::Tensor(const at::Tensor&, const OptTensor&, const OptTensor&, double)>("flash_hypercons::_layer_norm");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, bias, eps);
}

// dz of a graph-building backward, from differentiable pieces.
at::Tensor activation_gradient(const at::Tensor& g, const at::Tensor& z, int64_t act) {
  switch (act) {
    case FH_ACT_RELU: return g * (z > 0).to(g.scalar_type());
    case FH_ACT_GELU: return at::gelu_backward(g, z, "none");
    case FH_ACT_GELU_TANH: return at::gelu_backward(g, z, "tanh");
    case FH_ACT_SILU: {
      const at::Tensor q = z.sigmoid();
      return g * q * (1 + z * (1 - q));
    }
    default: return g;
  }
}

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                            const OptTensor& residual, int64_t act) {
    static const auto op =
        find_op<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, const OptTensor&,
                                                   const OptTensor&, int64_t)>("flash_hypercons::_linear_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, sums] = op.call(x, weight, bias, residual, act);
    ctx->save_for_backward({x, weight, bias.value_or(at::Tensor()), sums});
    ctx->saved_data["act"] = act;
    ctx->saved_data["wanted"] = wanted(x, weight, bias, residual);
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &sums = saved[3], &grad = grads[0];
    const int64_t act = ctx->saved_data["act"].toInt();
    if (!grad.defined()) return {{}, {}, {}, {}, {}};
    const int64_t want = ctx->saved_data["wanted"].toInt();
    const bool want_x = want & 1, want_weight = want & 2, want_bias = want & 4;
    at::Tensor dx, dw, db;
    if (at::GradMode::is_enabled()) {
      const at::Tensor xf = x.to(at::kFloat).reshape({-1, x.size(-1)}), wf = weight.to(at::kFloat);
      at::Tensor z = xf.mm(wf.t());
      if (bias.defined()) z = z + bias.to(at::kFloat);
      const at::Tensor dz = activation_gradient(grad.to(at::kFloat).reshape({-1, weight.size(0)}), z, act);
      if (want_x) dx = dz.mm(wf).reshape(x.sizes()).to(x.scalar_type());
      if (want_weight) dw = dz.t().mm(xf).to(x.scalar_type());
      if (want_bias) db = dz.sum(0).to(bias.scalar_type());
    } else if (want_x || want_weight || want_bias) {
      static const auto op = find_op<std::tuple<at::Tensor, at::Tensor, at::Tensor>(
          const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&, const at::Tensor&, int64_t, bool,
          bool, bool)>("flash_hypercons::_linear_backward");
      auto got = op.call(grad, x, weight, optional_of(bias), sums, act, want_x, want_weight, want_bias);
      if (want_x) dx = std::get<0>(got);
      if (want_weight) dw = std::get<1>(got);
      if (want_bias) db = std::get<2>(got);
    }
    return {dx, dw, db, want & 8 ? grad : at::Tensor(), {}};
  }
};

at::Tensor linear_autograd(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                           const OptTensor& residual, int64_t act) {
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual)))
    return LinearFunction::apply(x, weight, bias, residual, act);
  static const auto op = find_op<at::Tensor(const at::Tensor&, const at::Tensor&, const OptTensor&, const OptTensor&,
                                            int64_t)>("flash_hypercons::_linear");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, bias, residual, act);
}

}  // namespace
}  // namespace flash_hypercons

TORCH_LIBRARY_FRAGMENT(flash_hypercons, m) {
  m.def("_layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("_layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  m.def("_layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, bool want_weight, "
        "bool want_bias) -> (Tensor, Tensor, Tensor)");
  m.def("_linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act) -> Tensor");
  m.def("_linear_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act) -> (Tensor, Tensor)");
  m.def("_linear_backward(Tensor grad, Tensor x, Tensor weight, Tensor? bias, Tensor saved, int act, bool want_x, "
        "bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)");
  m.def("_grad_norm(Tensor[] tensors, float norm_type) -> Tensor");
  m.def("_clip_grads(Tensor[] tensors, float max_norm, float norm_type) -> (Tensor[], Tensor)");
  m.def("_clip_grads_(Tensor(a!)[] tensors, float max_norm, float norm_type) -> Tensor");
}

TORCH_LIBRARY_IMPL(flash_hypercons, CUDA, m) {
  m.impl("_layer_norm", &flash_hypercons::layer_norm_hip);
  m.impl("_layer_norm_forward", &flash_hypercons::layer_norm_forward_hip);
  m.impl("_layer_norm_backward", &flash_hypercons::layer_norm_backward_hip);
  m.impl("_linear", &flash_hypercons::linear_hip);
  m.impl("_linear_forward", &flash_hypercons::linear_forward_hip);
  m.impl("_linear_backward", &flash_hypercons::linear_backward_hip);
  m.impl("_grad_norm", &flash_hypercons::grad_norm_hip);
  m.impl("_clip_grads", &flash_hypercons::clip_grads_hip);
  m.impl("_clip_grads_", &flash_hypercons::clip_grads_inplace_hip);
}

TORCH_LIBRARY_IMPL(flash_hypercons, Autograd, m) {
  m.impl("_layer_norm", &flash_hypercons::layer_norm_autograd);
  m.impl("_linear", &flash_hypercons::linear_autograd);
}
