// What the torch ops share: checks of arguments, streams, pointers, and the two guards of their autograd functions.
// Everything has internal linkage.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include "fsctep.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc, const char* name) { TORCH_CHECK(rc == 0, name, " failed (", rc, "): ", fsc_last_error()); }

const Tensor& some(const optional<Tensor>& t) {
  static const Tensor none;
  return t.has_value() ? *t : none;
}

void require_gpu(std::initializer_list<std::reference_wrapper<const Tensor>> ts, const char* name) {
  const Tensor& first = ts.begin()->get();
  for (const Tensor& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK(t.is_cuda(), name, ": fsctep ops run on the GPU only (HIP kernels); got a ", t.device(), " tensor");
    TORCH_CHECK(t.device() == first.device(), name, ": tensors on ", first.device(), " and ", t.device());
  }
}

int32_t code_of(at::ScalarType t, const char* name) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16, name, " must be float32 or bfloat16, got ", t);
  return t == at::kFloat ? FSC_F32 : FSC_BF16;
}

// (rows, width) with a contiguous last dimension; rows may lie at any non-negative stride.
Tensor rows2d(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be (rows, width), got ", t.dim(), " dimensions");
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= 0) ? t : t.contiguous();
}
int64_t stride_of(const Tensor& t) { return t.size(0) <= 1 ? 0 : t.stride(0); }
// the row stride of a single row is of no meaning: 0 keeps it aligned
const void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.const_data_ptr() : nullptr; }
void* mptr(Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

template <typename Sig>
auto op_handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

// Whether a call goes through its autograd function: a gradient is wanted, or an input carries a forward-mode tangent,
// which the function refuses (below autograd it would be lost).
bool differentiates(std::initializer_list<std::reference_wrapper<const Tensor>> ts) {
  for (const Tensor& t : ts)
    if (t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined())) return true;
  return false;
}

// A backward op's call: below autograd unless a gradient of the gradient may be asked for, which then raises.
struct BackwardGuard {
  optional<at::AutoDispatchBelowADInplaceOrView> below;
  BackwardGuard() {
    if (!at::GradMode::is_enabled()) below.emplace();
  }
};

template <const char* const& NAME>
void refuse(const c10::OperatorHandle& op, torch::jit::Stack*) {
  TORCH_CHECK(false, op.schema().name(), ": ", NAME);
}
const char* const kGpuOnly = "fsctep ops run on the GPU only (HIP kernels)";

}  // namespace
