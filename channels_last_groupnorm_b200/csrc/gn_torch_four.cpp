// torch binding of rows in four bits (codes and scales: gn_four.cuh):
//   quantize_4bit(x, block, scale?) -> (codes, scales)
//   dequantize_4bit(codes, scales, channels, scale?, dtype) -> rows
//   rms_quant_4bit(x, residual?, weight?, eps, offset, block, scale?) -> (codes, scales, sum)      sum is empty without a residual
//   linear_4bit(codes, scales, weight_codes, weight_scales, scale?, weight_scale?, bias?, dtype) -> y
// codes: float4_e2m1fn_x2; scales: float8_e4m3fn in blocks of 16, float8_e8m0fnu in blocks of 32.  No gradients; and the plain calls.
#include "gn_torch_rows.h"

namespace {

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
at::ScalarType scales_type(int64_t block) { return block == 16 ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu; }
int64_t rows_of(const Tensor& t) {
  int64_t n = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
  return n;
}

const char* refusal_of_scale(const Tensor& scale, int64_t block, const Tensor& like) {
  if (!scale.defined()) return nullptr;
  if (block == 32) return "blocks of 32 have no scale of the whole tensor";
  if (scale.device() != like.device() || scale.scalar_type() != at::kFloat || scale.numel() != 1) return "scale must be one float32 on the device of the rows";
  return nullptr;
}
const char* refusal_of_quant(const Tensor& x, const Tensor& weight, const Tensor& residual, int64_t block, const Tensor& scale) {
  if (const char* why = refusal_of_rows(x, weight, residual)) return why;
  if (block != 16 && block != 32) return "block must be 16 or 32 channels";
  return refusal_of_scale(scale, block, x);
}
// codes of some rows and their scales; *block: what the scales' type says
const char* refusal_of_four(const Tensor& codes, const Tensor& scales, int64_t* block) {
  if (!codes.device().is_cuda()) return "codes must be a CUDA tensor; this package has no CPU path";
  if (codes.scalar_type() != at::kFloat4_e2m1fn_x2 || codes.dim() < 1 || codes.size(-1) < 16 || codes.size(-1) % 16 != 0)
    return "codes must be float4_e2m1fn_x2 of shape (*, channels / 2), whole blocks of 32 channels";
  *block = scales.scalar_type() == at::kFloat8_e4m3fn ? 16 : scales.scalar_type() == at::kFloat8_e8m0fnu ? 32 : 0;
  if (*block == 0) return "scales must be float8_e4m3fn (blocks of 16) or float8_e8m0fnu (blocks of 32)";
  if (scales.device() != codes.device() || scales.dim() != 2 || scales.size(0) != up(rows_of(codes), 128) ||
      scales.size(1) != up(codes.size(-1) * 2 / *block, 4) || !scales.is_contiguous())
    return "scales must be those of all rows of codes, contiguous, in tiles of 128 rows and 4 blocks";
  return nullptr;
}

// bytes of codes as the kernels take them
Tensor as_codes(const Tensor& codes) {
  if (codes.is_contiguous() && reinterpret_cast<uintptr_t>(codes.const_data_ptr()) % 16 == 0) return codes;
  return codes.view(at::kByte).clone(at::MemoryFormat::Contiguous);
}
const float* scale_at(const Tensor& scale) { return scale.defined() ? scale.const_data_ptr<float>() : nullptr; }

struct Four {
  Tensor codes, scales, sum;
};
// norm: with the root-mean-square norm in front
Four quantize(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, double offset, int64_t block, const Tensor& scale, bool norm) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t C = x.size(-1), rows = x.numel() / C, wide = up(C, 32);
  int64_t x_stride = C, r_stride = C;
  const auto st = x.scalar_type();
  const Tensor xr = as_rows(x, st, &x_stride), rr = as_rows(residual, st, &r_stride);
  Four out;
  at::DimVector sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = wide / 2;
  out.codes = empty_like_sizes(sizes, at::kFloat4_e2m1fn_x2, x);
  out.scales = empty_like_sizes({up(rows, 128), up(wide / block, 4)}, scales_type(block), x);
  if (residual.defined()) out.sum = empty_like_sizes(x.sizes(), residual.scalar_type(), x);
  if (rows == 0) return out;
  const auto stream = c10::cuda::getCurrentCUDAStream().stream();
  if (norm)
    check_status(gnb200_rms_fwd_4bit(data(xr), x_stride, data(rr), r_stride, data(weight), rows, C, eps, offset, code_of(x), code_of(residual), code_of(weight),
                                     (int)block, scale_at(scale), out.codes.mutable_data_ptr(), out.scales.mutable_data_ptr(),
                                     residual.defined() ? out.sum.mutable_data_ptr() : nullptr, stream));
  else
    check_status(gnb200_quantize_4bit(data(xr), x_stride, rows, C, code_of(x), (int)block, scale_at(scale), out.codes.mutable_data_ptr(),
                                      out.scales.mutable_data_ptr(), stream));
  return out;
}

const char* refusal_of_dequantize(const Tensor& codes, const Tensor& scales, int64_t channels, const Tensor& scale, at::ScalarType dtype) {
  int64_t block = 0;
  if (const char* why = refusal_of_four(codes, scales, &block)) return why;
  if (channels < 1 || up(channels, 32) != codes.size(-1) * 2) return "channels must be those that the codes were made of";
  if (dtype_code(dtype) < 0) return "dtype must be float32, float16 or bfloat16";
  return refusal_of_scale(scale, block, codes);
}
Tensor dequantize(const Tensor& codes, const Tensor& scales, int64_t channels, const Tensor& scale, at::ScalarType dtype) {
  c10::cuda::CUDAGuard guard(codes.device());
  at::DimVector sizes(codes.sizes().begin(), codes.sizes().end());
  sizes.back() = channels;
  Tensor out = empty_like_sizes(sizes, dtype, codes);
  const int64_t rows = rows_of(codes);
  if (rows == 0) return out;
  const Tensor c = as_codes(codes);
  check_status(gnb200_dequantize_4bit(data(c), data(scales), rows, channels, scales.scalar_type() == at::kFloat8_e4m3fn ? 16 : 32, scale_at(scale),
                                      dtype_code(dtype), out.mutable_data_ptr(), c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

const char* refusal_of_linear(const Tensor& codes, const Tensor& scales, const Tensor& w_codes, const Tensor& w_scales, const Tensor& scale,
                              const Tensor& w_scale, const Tensor& bias, at::ScalarType dtype) {
  int64_t block = 0, w_block = 0;
  if (const char* why = refusal_of_four(codes, scales, &block)) return why;
  if (w_codes.device() != codes.device() || w_codes.dim() != 2) return "weight_codes must have shape (features, channels / 2), on the device of codes";
  if (const char* why = refusal_of_four(w_codes, w_scales, &w_block)) return why;
  if (block != w_block || codes.size(-1) != w_codes.size(-1)) return "codes and weight_codes must have the same channels and blocks";
  if (const char* why = refusal_of_scale(scale, block, codes)) return why;
  if (const char* why = refusal_of_scale(w_scale, block, codes)) return why;
  if (bias.defined() && (bias.device() != codes.device() || bias.dim() != 1 || bias.size(0) != w_codes.size(0) || dtype_code(bias.scalar_type()) < 0 ||
                         !bias.is_contiguous()))
    return "bias must be a contiguous vector of one element per feature in float32, float16 or bfloat16";
  if (dtype_code(dtype) < 0) return "dtype must be float32, float16 or bfloat16";
  return nullptr;
}
Tensor linear(const Tensor& codes, const Tensor& scales, const Tensor& w_codes, const Tensor& w_scales, const Tensor& scale, const Tensor& w_scale,
              const Tensor& bias, at::ScalarType dtype) {
  c10::cuda::CUDAGuard guard(codes.device());
  at::DimVector sizes(codes.sizes().begin(), codes.sizes().end());
  sizes.back() = w_codes.size(0);
  Tensor out = empty_like_sizes(sizes, dtype, codes);
  const int64_t rows = rows_of(codes);
  if (out.numel() == 0) return out;
  const Tensor c = as_codes(codes), w = as_codes(w_codes);
  check_status(gnb200_linear_4bit(data(c), data(scales), scale_at(scale), data(w), data(w_scales), scale_at(w_scale), data(bias), rows, w_codes.size(0),
                                  codes.size(-1) * 2, scales.scalar_type() == at::kFloat8_e4m3fn ? 16 : 32, code_of(bias), dtype_code(dtype),
                                  out.mutable_data_ptr(), c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

std::tuple<Tensor, Tensor> quantize_op(const Tensor& x, int64_t block, const OptTensor& scale) {
  if (const char* why = refusal_of_quant(x, Tensor(), Tensor(), block, value(scale))) TORCH_CHECK(false, "gnb200: ", why);
  refuse_tangents("quantize_4bit", {x, value(scale)});
  Four f = quantize(x, Tensor(), Tensor(), 0.0, 0.0, block, value(scale), false);
  return {f.codes, f.scales};
}
std::tuple<Tensor, Tensor, Tensor> rms_quant_4bit_op(const Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps, double offset, int64_t block,
                                                     const OptTensor& scale) {
  if (const char* why = refusal_of_quant(x, value(weight), value(residual), block, value(scale))) TORCH_CHECK(false, "gnb200: ", why);
  refuse_tangents("rms_norm_quant_4bit", {x, value(weight), value(residual), value(scale)});
  Four f = quantize(x, value(weight), value(residual), eps, offset, block, value(scale), true);
  return {f.codes, f.scales, f.sum.defined() ? f.sum : none_of(x)};
}
Tensor dequantize_op(const Tensor& codes, const Tensor& scales, int64_t channels, const OptTensor& scale, at::ScalarType dtype) {
  if (const char* why = refusal_of_dequantize(codes, scales, channels, value(scale), dtype)) TORCH_CHECK(false, "gnb200: ", why);
  refuse_tangents("dequantize_4bit", {value(scale)});
  return dequantize(codes, scales, channels, value(scale), dtype);
}
Tensor linear_op(const Tensor& codes, const Tensor& scales, const Tensor& w_codes, const Tensor& w_scales, const OptTensor& scale, const OptTensor& w_scale,
                 const OptTensor& bias, at::ScalarType dtype) {
  if (const char* why = refusal_of_linear(codes, scales, w_codes, w_scales, value(scale), value(w_scale), value(bias), dtype)) TORCH_CHECK(false, "gnb200: ", why);
  refuse_tangents("linear_4bit", {value(scale), value(w_scale), value(bias)});
  return linear(codes, scales, w_codes, w_scales, value(scale), value(w_scale), value(bias), dtype);
}

}  // namespace

std::tuple<Tensor, Tensor> gnb200_ops::quantize_4bit_direct(const Tensor& x, int64_t block, const Tensor& scale, bool* ok) {
  *ok = plain({&x, &scale}) && !wants_graph({&x, &scale}) && refusal_of_quant(x, Tensor(), Tensor(), block, scale) == nullptr;
  if (!*ok) return {};
  at::AutoDispatchBelowADInplaceOrView guard;
  Four f = quantize(x, Tensor(), Tensor(), 0.0, 0.0, block, scale, false);
  return {f.codes, f.scales};
}
std::tuple<Tensor, Tensor, Tensor> gnb200_ops::rms_quant_4bit_direct(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, double offset,
                                                                     int64_t block, const Tensor& scale, bool* ok) {
  *ok = plain({&x, &weight, &residual, &scale}) && !wants_graph({&x, &weight, &residual, &scale}) &&
        refusal_of_quant(x, weight, residual, block, scale) == nullptr;
  if (!*ok) return {};
  at::AutoDispatchBelowADInplaceOrView guard;
  Four f = quantize(x, weight, residual, eps, offset, block, scale, true);
  return {f.codes, f.scales, f.sum};
}
Tensor gnb200_ops::dequantize_4bit_direct(const Tensor& codes, const Tensor& scales, int64_t channels, const Tensor& scale, at::ScalarType dtype, bool* ok) {
  *ok = plain({&codes, &scales, &scale}) && !wants_graph({&scale}) && refusal_of_dequantize(codes, scales, channels, scale, dtype) == nullptr;
  if (!*ok) return {};
  at::AutoDispatchBelowADInplaceOrView guard;
  return dequantize(codes, scales, channels, scale, dtype);
}
Tensor gnb200_ops::linear_4bit_direct(const Tensor& codes, const Tensor& scales, const Tensor& w_codes, const Tensor& w_scales, const Tensor& scale,
                                      const Tensor& w_scale, const Tensor& bias, at::ScalarType dtype, bool* ok) {
  *ok = plain({&codes, &scales, &w_codes, &w_scales, &scale, &w_scale, &bias}) && !wants_graph({&scale, &w_scale, &bias}) &&
        refusal_of_linear(codes, scales, w_codes, w_scales, scale, w_scale, bias, dtype) == nullptr;
  if (!*ok) return {};
  at::AutoDispatchBelowADInplaceOrView guard;
  return linear(codes, scales, w_codes, w_scales, scale, w_scale, bias, dtype);
}

TORCH_LIBRARY_FRAGMENT(gnb200, m) {
  m.def("quantize_4bit(Tensor x, int block, Tensor? scale) -> (Tensor, Tensor)");
  m.def("dequantize_4bit(Tensor codes, Tensor scales, int channels, Tensor? scale, ScalarType dtype) -> Tensor");
  m.def("rms_quant_4bit(Tensor x, Tensor? residual, Tensor? weight, float eps, float offset, int block, Tensor? scale) -> (Tensor, Tensor, Tensor)");
  m.def("linear_4bit(Tensor codes, Tensor scales, Tensor weight_codes, Tensor weight_scales, Tensor? scale, Tensor? weight_scale, Tensor? bias, "
        "ScalarType dtype) -> Tensor");
}
TORCH_LIBRARY_IMPL(gnb200, CUDA, m) {
  m.impl("quantize_4bit", &quantize_op);
  m.impl("dequantize_4bit", &dequantize_op);
  m.impl("rms_quant_4bit", &rms_quant_4bit_op);
  m.impl("linear_4bit", &linear_op);
}
// (registered to refuse with a message of this library)
TORCH_LIBRARY_IMPL(gnb200, CPU, m) {
  m.impl("quantize_4bit", &quantize_op);
  m.impl("dequantize_4bit", &dequantize_op);
  m.impl("rms_quant_4bit", &rms_quant_4bit_op);
  m.impl("linear_4bit", &linear_op);
}
