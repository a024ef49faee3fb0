// torch binding of dropout with the residual's addition:
//   dropout_add(x, residual?, p, seed_at?, seed, layer) -> s     seed_at: the seed as a tensor of one int64, read by the kernel
//   dropout_mask(t, p, seed_at?, seed, layer, dtype) -> t where kept, over 1 - p, in `dtype`: the gradient of x, and its own gradient
// and the plain call with its autograd node.
#include "gn_torch_rows.h"

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

namespace {

const char* refusal_of_dropout(const Tensor& x, const Tensor& residual, double p, const Tensor& seed_at) {
  if (!x.device().is_cuda()) return "x must be a CUDA tensor; this package has no CPU path";
  if (dtype_code(x.scalar_type()) < 0) return "x must be float32, float16 or bfloat16";
  if (residual.defined()) {
    if (residual.device() != x.device() || residual.sizes() != x.sizes()) return "residual must match x in sizes and device";
    if (residual.scalar_type() != x.scalar_type() && residual.scalar_type() != at::kFloat) return "residual must have the dtype of x or float32";
  }
  if (!(p >= 0.0 && p * 4294967296.0 < 4294967295.5)) return "p must be at least 0 and less than 1";
  if (seed_at.defined() && (seed_at.device() != x.device() || seed_at.scalar_type() != at::kLong || seed_at.numel() != 1))
    return "a seed that is a tensor must have one element, int64, on the device of x";
  return nullptr;
}

Tensor dropout(const Tensor& x_in, const Tensor& residual_in, double p, const Tensor& seed_at, int64_t seed, int64_t layer, at::ScalarType type) {
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = x_in.contiguous(), residual = residual_in.defined() ? residual_in.contiguous() : residual_in;
  Tensor out = empty_like_sizes(x.sizes(), type, x);
  check_status(gnb200_dropout_add(data(x), data(residual), x.numel(), p, seed_at.defined() ? seed_at.const_data_ptr<int64_t>() : nullptr, (uint64_t)seed,
                                  (uint64_t)layer, code_of(x), dtype_code(type), out.mutable_data_ptr(), c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

Tensor dropout_add_op(const Tensor& x, const OptTensor& residual, double p, const OptTensor& seed_at, int64_t seed, int64_t layer) {
  if (const char* why = refusal_of_dropout(x, value(residual), p, value(seed_at))) TORCH_CHECK(false, "gnb200: ", why);
  refuse_tangents("dropout_add", {x, value(residual)});
  return dropout(x, value(residual), p, value(seed_at), seed, layer, residual.has_value() ? residual->scalar_type() : x.scalar_type());
}
Tensor dropout_mask_op(const Tensor& t, double p, const OptTensor& seed_at, int64_t seed, int64_t layer, at::ScalarType dtype) {
  if (const char* why = refusal_of_dropout(t, Tensor(), p, value(seed_at))) TORCH_CHECK(false, "gnb200: ", why);
  refuse_tangents("dropout_add", {t});
  TORCH_CHECK(dtype == t.scalar_type() || dtype == at::kFloat || (t.scalar_type() == at::kFloat && dtype_code(dtype) >= 0),
              "gnb200: dtype must be that of t, or one of them float32");
  return dropout(t, Tensor(), p, value(seed_at), seed, layer, dtype);
}
const auto& dropout_mask_handle() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnb200::dropout_mask", "").typed<decltype(dropout_mask_op)>();
  return op;
}

// The backward as a node of its own: what it keeps are a few numbers, and the seed where that is a tensor.  (As a torch::autograd::Function, whose context
// keeps values by name, a training step took 4 us more of the host's time.)
struct DropoutBackward : torch::autograd::Node {
  torch::autograd::SavedVariable seed_at;
  double p;
  int64_t seed, layer;
  at::ScalarType x_type;
  bool has_seed, residual;  // residual: it is the second input

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(residual ? 2 : 1);
    const Tensor& ds = grads[0];
    if (!ds.defined()) return out;
    const Tensor seed_tensor = has_seed ? seed_at.unpack(shared_from_this()) : Tensor();
    if (task_should_compute_output(0)) {
      // Through the dispatcher where a graph of the backward is asked for, as it has the mask's own gradient, and where somebody else looks at the
      // gradient: a batch of them, a dispatch mode.
      if (c10::GradMode::is_enabled() || !plain({&ds, &seed_tensor})) {
        out[0] = dropout_mask_handle().call(ds, p, opt(seed_tensor), seed, layer, x_type);
      } else {
        at::AutoDispatchBelowADInplaceOrView guard;
        out[0] = dropout(ds, Tensor(), p, seed_tensor, seed, layer, x_type);
      }
    }
    if (residual) out[1] = ds;
    return out;
  }
  std::string name() const override { return "DropoutAddBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    seed_at.reset_data();
  }
};

}  // namespace

Tensor gnb200_ops::dropout_add_direct(const Tensor& x, const Tensor& residual, double p, const Tensor& seed_at, int64_t seed, int64_t layer, bool* ok) {
  *ok = plain({&x, &residual, &seed_at}) && refusal_of_dropout(x, residual, p, seed_at) == nullptr;
  if (!*ok) return {};
  std::shared_ptr<DropoutBackward> node;
  if (wants_graph({&x, &residual})) {
    node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
    node->set_next_edges(residual.defined() ? torch::autograd::collect_next_edges(x, residual) : torch::autograd::collect_next_edges(x));
    node->p = p, node->seed = seed, node->layer = layer, node->x_type = x.scalar_type();
    node->has_seed = seed_at.defined(), node->residual = residual.defined();
    if (node->has_seed) node->seed_at = torch::autograd::SavedVariable(seed_at, false);
  }
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    out = dropout(x, residual, p, seed_at, seed, layer, residual.defined() ? residual.scalar_type() : x.scalar_type());
  }
  if (node) torch::autograd::set_history(out, node);
  return out;
}

TORCH_LIBRARY_FRAGMENT(gnb200, m) {
  m.def("dropout_add(Tensor x, Tensor? residual, float p, Tensor? seed_at, int seed, int layer) -> Tensor");
  m.def("dropout_mask(Tensor t, float p, Tensor? seed_at, int seed, int layer, ScalarType dtype) -> Tensor");
}
TORCH_LIBRARY_IMPL(gnb200, CUDA, m) {
  m.impl("dropout_add", &dropout_add_op);
  m.impl("dropout_mask", &dropout_mask_op);
}
// (registered to refuse with a message of this library)
TORCH_LIBRARY_IMPL(gnb200, CPU, m) {
  m.impl("dropout_add", &dropout_add_op);
  m.impl("dropout_mask", &dropout_mask_op);
}
