// What the bindings of the operators on token rows share: checks, rows as the kernels take them, whether a call is a plain one.
#pragma once
#include <ATen/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>

#include "../../include/gnb200.h"
#include "gn_torch.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check_status(int rc) { TORCH_CHECK(rc == GNB200_OK, gnb200_last_error(), " (status ", rc, ")"); }

int dtype_code(at::ScalarType t) { return t == at::kFloat ? GNB200_F32 : t == at::kHalf ? GNB200_F16 : t == at::kBFloat16 ? GNB200_BF16 : -1; }
int code_of(const Tensor& t) { return t.defined() ? dtype_code(t.scalar_type()) : GNB200_F32; }
const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

Tensor empty_like_sizes(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor none_of(const Tensor& like) { return empty_like_sizes({0}, like.scalar_type(), like); }

// Rows of contiguous channels at one distance: true and that distance, or false where the tensor has to be copied first.
bool uniform_rows(const Tensor& t, int64_t* stride) {
  const auto sizes = t.sizes(), strides = t.strides();
  const int64_t last = t.dim() - 1;
  if (last < 0 || (sizes[last] != 1 && strides[last] != 1)) return false;
  int64_t rows = 1, step = 0;
  for (int64_t d = last - 1; d >= 0; --d) {
    if (sizes[d] == 1) continue;
    if (rows == 1)
      step = strides[d];
    else if (strides[d] != step * rows)
      return false;
    rows *= sizes[d];
  }
  *stride = rows == 1 ? sizes[last] : step;
  return true;
}
// The rows as the vector kernels take them: in place where they lie on vector boundaries, or are contiguous from one on (as results are:
// the same frame); copied first otherwise.  x_type: of the call's x, whose vectors the others' follow.
Tensor as_rows(const Tensor& t, at::ScalarType x_type, int64_t* stride) {
  if (!t.defined() || t.numel() == 0) return t;
  const int64_t width = x_type == at::kFloat ? 4 : 8, C = t.size(-1), frame = width * (int64_t)t.element_size();
  const auto at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  if (uniform_rows(t, stride)) {
    if (C % width == 0 && *stride % width == 0 && at % 16 == 0) return t;
    if ((*stride == C || t.numel() == C) && at % frame == 0) return t;
  }
  Tensor c = empty_like_sizes(t.sizes(), t.scalar_type(), t);
  c.copy_(t);
  *stride = C;
  return c;
}

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// What the kernels ask for; nullptr where it is there, else the reason of the refusal.
const char* refusal_of_rows(const Tensor& x, const Tensor& weight, const Tensor& residual) {
  if (!x.device().is_cuda()) return "x must be a CUDA tensor; this package has no CPU path";
  if (x.dim() < 1 || x.size(-1) < 1) return "x must have shape (*, channels)";
  const auto st = x.scalar_type();
  if (dtype_code(st) < 0) return "x must be float32, float16 or bfloat16";
  if (residual.defined()) {
    if (residual.device() != x.device() || residual.sizes() != x.sizes()) return "residual must match x in sizes and device";
    if (residual.scalar_type() != st && residual.scalar_type() != at::kFloat) return "residual must have the dtype of x or float32";
  }
  if (weight.defined()) {
    if (weight.device() != x.device() || weight.dim() != 1 || weight.size(0) != x.size(-1) || !weight.is_contiguous())
      return "weight must be a contiguous vector of one element per channel on the device of x";
    if (weight.scalar_type() != st && weight.scalar_type() != at::kFloat) return "weight must have the dtype of x or float32";
  }
  return nullptr;
}

bool wants_graph(std::initializer_list<const Tensor*> tensors) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// The gradients' own gradients: an error, where an op without a formula would leave its term out.
void refuse_second(const char* name) { TORCH_CHECK(false, "gnb200: ", name, " is differentiable once; a gradient of its gradient was asked for"); }

// Tangents of forward mode: an error too, where the kernels would leave them out.
void refuse_tangents(const char* name, std::initializer_list<Tensor> tensors) {
  for (const Tensor& t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "gnb200: ", name, " has no derivative in forward mode");
}

bool plain(std::initializer_list<const Tensor*> tensors) {
  if (!gnb200_ops::only_cuda_sees(tensors)) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined()) return false;  // dual tensors
  return true;
}

}  // namespace
