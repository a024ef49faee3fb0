// What gnb200_torch.so offers besides its ops.
#pragma once
#include <ATen/Tensor.h>

#include <initializer_list>
#include <tuple>

namespace gnb200_ops {

// Whether nothing but autograd and CUDA kernels would see an op on these tensors (gn_torch.cpp)
bool only_cuda_sees(std::initializer_list<const at::Tensor*> tensors);

// The module's call, if it is a plain one (see gn_torch.cpp); an undefined tensor otherwise.
__attribute__((visibility("default"))) at::Tensor group_norm_act_direct(const at::Tensor& X, const at::Tensor& weight,
                                                                        const at::Tensor& bias, int64_t G, double eps, int64_t act);

// Token rows (gn_torch_tokens.cpp): the public functions' calls where they are plain ones, autograd node included; `ok` false where
// Python has to look at the call.  Undefined tensors stand for absent arguments.  (y, sum), the latter undefined without a residual.
__attribute__((visibility("default"))) std::tuple<at::Tensor, at::Tensor> rms_norm_direct(const at::Tensor& x, const at::Tensor& weight,
                                                                                          const at::Tensor& residual, double eps,
                                                                                          double offset, bool* ok);
// (codes, scales, sum)
__attribute__((visibility("default"))) std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_quant_direct(
    const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, double eps, double offset, int64_t block, int64_t format,
    bool* ok);
__attribute__((visibility("default"))) std::tuple<at::Tensor, at::Tensor> rotary_direct(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions, const at::Tensor& inv_freq, at::IntArrayRef sections,
    const at::Tensor& q_weight, const at::Tensor& k_weight, double eps, double offset, bool interleaved, bool* ok);

}  // namespace gnb200_ops
