// What the operators around the stream mixing share: checks of tensors, rows, workspaces and
// calls through the dispatcher.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <algorithm>
#include <optional>

#include "flash_hypercons.h"

namespace flash_hypercons {
namespace {

using OptTensor = std::optional<at::Tensor>;

bool element_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? FH_DTYPE_F32 : t == at::kBFloat16 ? FH_DTYPE_BF16 : FH_DTYPE_F16;
}

hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

void check_status(int rc) { TORCH_CHECK(rc == FH_OK, "flash_hypercons: ", fh_last_error()); }

bool strided_on(const at::Tensor& t, const at::Tensor& like) {
  return t.layout() == at::kStrided && t.device() == like.device();
}

// [..., cols] as rows of contiguous columns: in place where one stride leads from row
// to row, otherwise a copy.
at::Tensor rows_of(const at::Tensor& t, int64_t cols) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
  if (r.is_neg()) r = r.resolve_neg();
  if (cols > 1 && r.stride(1) != 1) r = r.contiguous();
  return r;
}

// A row's distance from the next; of a single row, whose stride may be anything, its length.
int64_t stride_of(const at::Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

at::Tensor vector_of(const OptTensor& t) {
  return t.has_value() && t->defined() ? t->resolve_neg().contiguous() : at::Tensor();
}

const void* data_of(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Runs call(workspace, bytes), the first time for the workspace's size alone.
template <typename Call>
void with_workspace(const at::Tensor& like, Call call) {
  int64_t bytes = 0;
  check_status(call(nullptr, &bytes));
  if (bytes == 0) {
    alignas(16) char none[16];  // any address will do
    check_status(call(none, &bytes));
    return;
  }
  const at::Tensor workspace = at::empty({bytes}, like.options().dtype(at::kByte));
  check_status(call(workspace.mutable_data_ptr(), &bytes));
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <typename Signature>
c10::TypedOperatorHandle<Signature> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

OptTensor optional_of(const at::Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && wants_grad(*t); }

// Which inputs need a gradient, as bits in the inputs' order.  (The node's own
// needs_input_grad leaves out optional inputs that were not given.)
template <typename... Inputs>
int64_t wanted(const Inputs&... inputs) {
  int64_t bits = 0, bit = 1;
  ((bits |= wants_grad(inputs) ? bit : 0, bit <<= 1), ...);
  return bits;
}

}  // namespace
}  // namespace flash_hypercons
