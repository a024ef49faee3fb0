// torch binding of the operators on token rows: torch.ops.gnb200.{rms_fwd, rms_bwd, rms_quant, rotary, rotary_bwd} over the C ABI,
// and the plain calls with their autograd nodes.
//   rms_fwd(x, residual?, weight?, eps, offset) -> (y, sum, rstd)       sum is empty without a residual
//   rms_bwd(dy, dsum?, sum, addend?, weight?, rstd, offset) -> (dx, dsum_out, dweight)    s = sum + addend; dsum_out, dweight empty where
//                                                                                      there are none
//   rms_quant(x, residual?, weight?, eps, offset, block, format) -> (codes, scales, sum)
//   rotary(q, k?, positions, inv_freq, sections, q_weight?, k_weight?, eps, offset, interleaved) -> (q, k)
//   rotary_bwd(dq, dk?, q, k?, positions, ...) -> (dq, dk, dq_weight, dk_weight)
// The functional ops serve tracing (torch.compile) and libtorch programs; eager calls of the package take the plain calls,
// which run the same code without the dispatcher and with a native autograd node.
#include "gn_torch_rows.h"

namespace {

// ------------------------------------------------------------------------------------------------
// Root-mean-square norm
// ------------------------------------------------------------------------------------------------
struct RmsOut {
  Tensor y, sum, rstd, scale;
};
// format < 0: y in x's type; else codes
RmsOut rms_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, double offset, bool want_rstd, int64_t block,
                   int format, bool checked = false) {
  if (!checked)
    if (const char* why = refusal_of_rows(x, weight, residual)) TORCH_CHECK(false, "gnb200: ", why);
  TORCH_CHECK(format < 0 || block == 0 || block == 32 || block == 64 || block == 128,
              "gnb200: block is 0 (one scale per row), 32, 64 or 128 channels, got ", block);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t C = x.size(-1), rows = x.numel() / C;
  int64_t x_stride = C, r_stride = C;
  const auto st = x.scalar_type();
  const Tensor xr = as_rows(x, st, &x_stride), rr = as_rows(residual, st, &r_stride);
  RmsOut out;
  if (residual.defined()) out.sum = empty_like_sizes(x.sizes(), residual.scalar_type(), x);
  const auto stream = c10::cuda::getCurrentCUDAStream().stream();
  if (format < 0) {
    out.y = empty_like_sizes(x.sizes(), x.scalar_type(), x);
    if (want_rstd) out.rstd = empty_like_sizes(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
    if (rows)
      check_status(gnb200_rms_fwd(data(xr), x_stride, data(rr), r_stride, data(weight), rows, C, eps, offset, code_of(x), code_of(residual),
                                  code_of(weight), out.y.mutable_data_ptr(), residual.defined() ? out.sum.mutable_data_ptr() : nullptr,
                                  want_rstd ? out.rstd.mutable_data_ptr<float>() : nullptr, stream));
    return out;
  }
  out.y = empty_like_sizes(x.sizes(), format == GNB200_E4M3 ? at::kFloat8_e4m3fn : at::kChar, x);
  at::DimVector scales(x.sizes().begin(), x.sizes().end());
  scales.back() = block ? (C + block - 1) / block : 1;
  out.scale = empty_like_sizes(scales, at::kFloat, x);
  if (rows)
    check_status(gnb200_rms_fwd_8bit(data(xr), x_stride, data(rr), r_stride, data(weight), rows, C, eps, offset, code_of(x),
                                     code_of(residual), code_of(weight), (int)block, format, out.y.mutable_data_ptr(),
                                     out.scale.mutable_data_ptr<float>(), residual.defined() ? out.sum.mutable_data_ptr() : nullptr, stream));
  return out;
}

struct RmsGrads {
  Tensor dx, dsum, dweight;  // dsum undefined where it would be dx
};
RmsGrads rms_backward(const Tensor& dy, const Tensor& dsum, const Tensor& sum, const Tensor& addend, const Tensor& weight, const Tensor& rstd,
                      double offset, bool want_dsum, bool want_dweight) {
  TORCH_CHECK(dy.device().is_cuda(), "gnb200: dy must be a CUDA tensor; this package has no CPU path");
  TORCH_CHECK(dtype_code(dy.scalar_type()) >= 0 && dy.dim() >= 1 && dy.size(-1) >= 1, "gnb200: dy must be (*, channels) in float32, float16 or bfloat16");
  TORCH_CHECK(sum.sizes() == dy.sizes() && sum.device() == dy.device() &&
                  (sum.scalar_type() == dy.scalar_type() || sum.scalar_type() == at::kFloat),
              "gnb200: sum must match dy in sizes and device and have its dtype or float32");
  TORCH_CHECK(!dsum.defined() || (dsum.sizes() == sum.sizes() && dsum.device() == sum.device() && dsum.scalar_type() == sum.scalar_type()),
              "gnb200: dsum must match sum in sizes, dtype and device");
  TORCH_CHECK(!addend.defined() || (addend.sizes() == dy.sizes() && addend.device() == dy.device() && addend.scalar_type() == dy.scalar_type()),
              "gnb200: addend must match dy in sizes, dtype and device");
  const int64_t C = dy.size(-1), rows = dy.numel() / C;
  TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == rows && rstd.device() == dy.device(),
              "gnb200: rstd must be the tensor returned by gnb200::rms_fwd for this input");
  TORCH_CHECK(!weight.defined() || (weight.dim() == 1 && weight.size(0) == C && weight.is_contiguous() && weight.device() == dy.device() &&
                                    (weight.scalar_type() == dy.scalar_type() || weight.scalar_type() == at::kFloat)),
              "gnb200: weight must be a contiguous vector of one element per channel in the dtype of dy or float32");
  c10::cuda::CUDAGuard guard(dy.device());
  int64_t dy_stride = C, ds_stride = C, s_stride = C, a_stride = C;
  const auto st = dy.scalar_type();
  const Tensor dyr = as_rows(dy, st, &dy_stride), dsr = as_rows(dsum, st, &ds_stride), sr = as_rows(sum, st, &s_stride),
               ar = as_rows(addend, st, &a_stride);
  const int dtype = code_of(dy), sum_dtype = code_of(sum);
  RmsGrads out;
  out.dx = empty_like_sizes(dy.sizes(), dy.scalar_type(), dy);
  if (want_dsum && sum_dtype != dtype) out.dsum = empty_like_sizes(dy.sizes(), sum.scalar_type(), dy);
  want_dweight = want_dweight && weight.defined();
  Tensor ws;
  size_t ws_bytes = 0;
  if (want_dweight) {
    out.dweight = empty_like_sizes({C}, weight.scalar_type(), dy);
    ws_bytes = gnb200_rms_bwd_workspace_bytes(rows, C, dtype, sum_dtype);
    if (ws_bytes) ws = empty_like_sizes({(int64_t)ws_bytes}, at::kByte, dy);
  }
  check_status(gnb200_rms_bwd(data(dyr), dy_stride, data(dsr), ds_stride, data(sr), s_stride, data(ar), a_stride, data(weight),
                              rstd.const_data_ptr<float>(), rows, C, offset, dtype, sum_dtype, code_of(weight), out.dx.mutable_data_ptr(),
                              out.dsum.defined() ? out.dsum.mutable_data_ptr() : nullptr,
                              want_dweight ? out.dweight.mutable_data_ptr() : nullptr, ws_bytes ? ws.mutable_data_ptr() : nullptr, ws_bytes,
                              c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

std::tuple<Tensor, Tensor, Tensor> rms_fwd_op(const Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps, double offset) {
  refuse_tangents("rms_norm", {x, value(weight), value(residual)});
  RmsOut o = rms_forward(x, value(weight), value(residual), eps, offset, true, 0, -1);
  return {o.y, o.sum.defined() ? o.sum : none_of(x), o.rstd};
}
std::tuple<Tensor, Tensor, Tensor> rms_bwd_op(const Tensor& dy, const OptTensor& dsum, const Tensor& sum, const OptTensor& addend,
                                              const OptTensor& weight, const Tensor& rstd, double offset) {
  refuse_tangents("rms_norm", {dy, value(dsum), sum, value(addend), value(weight), rstd});
  RmsGrads g = rms_backward(dy, value(dsum), sum, value(addend), value(weight), rstd, offset, true, true);
  return {g.dx, g.dsum.defined() ? g.dsum : none_of(sum), g.dweight.defined() ? g.dweight : none_of(sum)};
}
std::tuple<Tensor, Tensor, Tensor> rms_quant_op(const Tensor& x, const OptTensor& residual, const OptTensor& weight, double eps, double offset,
                                                int64_t block, int64_t format) {
  TORCH_CHECK(format == GNB200_E4M3 || format == GNB200_INT8, "gnb200: unknown format code ", format, " (0 e4m3, 1 int8)");
  refuse_tangents("rms_norm_quant", {x, value(weight), value(residual)});
  RmsOut o = rms_forward(x, value(weight), value(residual), eps, offset, false, block, (int)format);
  return {o.y, o.scale, o.sum.defined() ? o.sum : none_of(x)};
}

const auto& rms_bwd_handle() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnb200::rms_bwd", "").typed<decltype(rms_bwd_op)>();
  return op;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// (an absent argument is an empty optional: the node has no edge for it, and edges are counted over the present ones)
struct RmsFunction : torch::autograd::Function<RmsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual_arg, const OptTensor& weight_arg, double eps,
                               double offset) {
    const Tensor residual = value(residual_arg), weight = value(weight_arg);
    RmsOut o = rms_forward(x, weight, residual, eps, offset, true, 0, -1, true);
    ctx->set_materialize_grads(false);
    // The stored sum of a 16-bit stream is rounded: good enough for the gradient of x, whose terms are rounded alike, but it would cost
    // the weight's gradient, a sum in fp32 over all rows, what its 16 bits lack.  There the backward adds x and the residual again.
    const bool again = residual.defined() && residual.scalar_type() != at::kFloat && weight.defined() && weight.requires_grad();
    ctx->save_for_backward({again ? residual : residual.defined() ? o.sum : x, again ? x : Tensor(), weight, o.rstd});
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["x_type"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = residual.defined();
    if (residual.defined()) return {o.y, o.sum};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &dy = grads[0], dsum = grads.size() > 1 ? grads[1] : Tensor();
    const Tensor &sum = saved[0], &addend = saved[1], &weight = saved[2], &rstd = saved[3];
    const auto x_type = (at::ScalarType)ctx->saved_data["x_type"].toInt();
    const double offset = ctx->saved_data["offset"].toDouble();
    const bool residual = ctx->saved_data["residual"].toBool();
    const bool want_dsum = residual && ctx->needs_input_grad(1);
    const bool want_dweight = weight.defined() && ctx->needs_input_grad(residual ? 2 : 1);
    variable_list out(5);
    if (!dy.defined()) {  // the norm's output was not used: the sum's gradient passes
      if (dsum.defined()) {
        out[0] = dsum.scalar_type() == x_type ? dsum : dsum.to(x_type);
        out[1] = dsum;
      }
      return out;
    }
    // through the dispatcher, whose formula refuses a second derivative, where a graph of the backward is asked for or somebody else looks at the gradients
    if (c10::GradMode::is_enabled() || !plain({&dy, &dsum, &sum, &addend, &weight, &rstd})) {
      auto [dx, ds, dw] = rms_bwd_handle().call(dy, opt(dsum), sum, opt(addend), opt(weight), rstd, offset);
      out[0] = dx;
      if (want_dsum) out[1] = sum.scalar_type() == x_type ? dx : ds;
      if (want_dweight) out[2] = dw;
      return out;
    }
    RmsGrads g = rms_backward(dy, dsum, sum, addend, weight, rstd, offset, want_dsum, want_dweight);
    out[0] = g.dx;
    if (want_dsum) out[1] = g.dsum.defined() ? g.dsum : g.dx;
    out[2] = g.dweight;
    return out;
  }
};

struct RmsBackwardOnce : torch::autograd::Function<RmsBackwardOnce> {
  static variable_list forward(AutogradContext*, const Tensor& dy, const OptTensor& dsum, const Tensor& sum, const OptTensor& addend,
                               const OptTensor& weight, const Tensor& rstd, double offset) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [dx, ds, dw] = rms_bwd_handle().call(dy, dsum, sum, addend, weight, rstd, offset);
    return {dx, ds, dw};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    refuse_second("rms_norm");
    return {};
  }
};
std::tuple<Tensor, Tensor, Tensor> rms_bwd_autograd(const Tensor& dy, const OptTensor& dsum, const Tensor& sum, const OptTensor& addend,
                                                    const OptTensor& weight, const Tensor& rstd, double offset) {
  const Tensor ds = value(dsum), a = value(addend), w = value(weight);
  if (wants_graph({&dy, &ds, &sum, &a, &w, &rstd})) {
    variable_list out = RmsBackwardOnce::apply(dy, dsum, sum, addend, weight, rstd, offset);
    return {out[0], out[1], out[2]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return rms_bwd_handle().call(dy, dsum, sum, addend, weight, rstd, offset);
}

// ------------------------------------------------------------------------------------------------
// Rotary positions
// ------------------------------------------------------------------------------------------------
int64_t pairs_of(at::IntArrayRef sections) {
  int64_t n = 0;
  for (int64_t s : sections) n += s;
  return n;
}
bool channels_contiguous(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1; }

const char* refusal_of_heads(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections,
                             const Tensor& q_weight, const Tensor& k_weight) {
  if (!q.device().is_cuda()) return "q must be a CUDA tensor; this package has no CPU path";
  if (q.dim() != 3 && q.dim() != 4) return "q must have shape (tokens, heads, head_dim) or (batch, tokens, heads, head_dim)";
  const auto st = q.scalar_type();
  if (dtype_code(st) < 0) return "q must be float32, float16 or bfloat16";
  const int64_t nd = q.dim(), D = q.size(-1);
  if (D < 2 || D > 512) return "heads must have 2 to 512 channels";
  if (k.defined()) {
    if (k.device() != q.device() || k.scalar_type() != st || k.dim() != nd || k.size(-1) != D) return "k must match q in dtype, device, rank and head_dim";
    if (k.sizes().slice(0, nd - 2) != q.sizes().slice(0, nd - 2)) return "k must have the tokens of q";
  }
  if (sections.empty() || sections.size() > 8) return "sections must name the pairs of 1 to 8 axes";
  for (int64_t s : sections)
    if (s < 0 || s > 256) return "sections must not be negative, nor hold more pairs than a head";
  const int64_t pairs = pairs_of(sections);
  if (pairs < 1 || 2 * pairs > D) return "the sections' pairs must fit the head";
  if (positions.device() != q.device() || positions.dim() != nd - 1 || positions.size(-1) != (int64_t)sections.size() ||
      positions.sizes().slice(0, nd - 2) != q.sizes().slice(0, nd - 2))
    return "positions must have the tokens of q and one column per axis, on its device";
  const auto pt = positions.scalar_type();
  if (pt != at::kInt && pt != at::kLong && pt != at::kFloat) return "positions must be int32, int64 or float32";
  if (inv_freq.device() != q.device() || inv_freq.scalar_type() != at::kFloat || inv_freq.dim() != 1 || inv_freq.size(0) != pairs ||
      !inv_freq.is_contiguous())
    return "inv_freq must be a contiguous float32 vector of one frequency per pair on the device of q";
  for (const Tensor* w : {&q_weight, &k_weight})
    if (w->defined() && (w->device() != q.device() || w->dim() != 1 || w->size(0) != D || !w->is_contiguous() ||
                         (w->scalar_type() != st && w->scalar_type() != at::kFloat)))
      return "norm weights must be contiguous vectors of head_dim elements in the dtype of q or float32 on its device";
  if (k_weight.defined() && !k.defined()) return "a norm weight for keys without keys";
  return nullptr;
}

// strides of batch, token and head
void strides_of(const Tensor& t, int64_t (&out)[3]) {
  const bool batched = t.dim() == 4;
  out[0] = batched ? t.stride(0) : 0;
  out[1] = t.stride(batched ? 1 : 0);
  out[2] = t.stride(batched ? 2 : 1);
}
Tensor with_contiguous_channels(const Tensor& t) { return !t.defined() || channels_contiguous(t) ? t : t.contiguous(); }

gnb200_rotary_args args_of(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections,
                           const Tensor& q_weight, const Tensor& k_weight, double eps, double offset, bool interleaved) {
  const Tensor& any = q.defined() ? q : k;
  const bool batched = any.dim() == 4;
  gnb200_rotary_args a = {};
  a.batch = batched ? any.size(0) : 1;
  a.tokens = any.size(batched ? 1 : 0);
  a.q_heads = q.defined() ? q.size(-2) : 0;
  a.k_heads = k.defined() ? k.size(-2) : 0;
  a.head_dim = any.size(-1);
  a.positions = positions.const_data_ptr();
  a.pos_stride[0] = batched ? positions.stride(0) : 0;
  a.pos_stride[1] = positions.stride(batched ? 1 : 0);
  a.pos_stride[2] = positions.stride(-1);
  const auto pt = positions.scalar_type();
  a.pos_type = pt == at::kInt ? GNB200_POS_I32 : pt == at::kLong ? GNB200_POS_I64 : GNB200_POS_F32;
  a.axes = (int)sections.size();
  for (int i = 0; i < a.axes; ++i) a.sections[i] = (int)sections[i];
  a.inv_freq = inv_freq.const_data_ptr<float>();
  a.q_weight = q.defined() ? data(q_weight) : nullptr;
  a.k_weight = k.defined() ? data(k_weight) : nullptr;
  a.q_weight_dtype = code_of(q_weight);
  a.k_weight_dtype = code_of(k_weight);
  a.eps = eps;
  a.offset = offset;
  a.interleaved = interleaved;
  a.dtype = code_of(any);
  return a;
}
bool nothing(const gnb200_rotary_args& a) { return a.batch * a.tokens * (a.q_heads + a.k_heads) == 0; }

std::tuple<Tensor, Tensor> rotary_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& positions, const Tensor& inv_freq,
                                          at::IntArrayRef sections, const Tensor& q_weight, const Tensor& k_weight, double eps, double offset,
                                          bool interleaved) {
  if (const char* why = refusal_of_heads(q_in, k_in, positions, inv_freq, sections, q_weight, k_weight)) TORCH_CHECK(false, "gnb200: ", why);
  c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = with_contiguous_channels(q_in), k = with_contiguous_channels(k_in);
  const gnb200_rotary_args a = args_of(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved);
  Tensor qo = empty_like_sizes(q.sizes(), q.scalar_type(), q), ko;
  int64_t qs[3], ks[3] = {0, 0, 0};
  strides_of(q, qs);
  if (k.defined()) {
    ko = empty_like_sizes(k.sizes(), k.scalar_type(), k);
    strides_of(k, ks);
  }
  if (!nothing(a))
    check_status(gnb200_rotary_fwd(&a, data(q), qs, data(k), ks, qo.mutable_data_ptr(), k.defined() ? ko.mutable_data_ptr() : nullptr,
                                   c10::cuda::getCurrentCUDAStream().stream()));
  return {qo, ko};
}

struct RotaryGrads {
  Tensor dq, dk, dq_weight, dk_weight;
};
// dq or dk undefined: left out; q, k: what the forward got, needed where there is a weight
RotaryGrads rotary_backward(const Tensor& dq_in, const Tensor& dk_in, const Tensor& q_in, const Tensor& k_in, const Tensor& positions,
                            const Tensor& inv_freq, at::IntArrayRef sections, const Tensor& q_weight, const Tensor& k_weight, double eps,
                            double offset, bool interleaved) {
  const Tensor dq = with_contiguous_channels(dq_in), dk = with_contiguous_channels(dk_in);
  const Tensor& any = dq.defined() ? dq : dk;
  c10::cuda::CUDAGuard guard(any.device());
  const gnb200_rotary_args a = args_of(dq, dk, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved);
  RotaryGrads out;
  int64_t dqs[3] = {0, 0, 0}, dks[3] = {0, 0, 0}, qs[3] = {0, 0, 0}, ks[3] = {0, 0, 0};
  Tensor q, k;
  if (dq.defined()) {
    strides_of(dq, dqs);
    out.dq = empty_like_sizes(dq.sizes(), dq.scalar_type(), dq);
    if (q_weight.defined()) {
      TORCH_CHECK(q_in.defined() && q_in.sizes() == dq.sizes() && q_in.scalar_type() == dq.scalar_type() && q_in.device() == dq.device(),
                  "gnb200: q must match dq in sizes, dtype and device");
      q = with_contiguous_channels(q_in);
      strides_of(q, qs);
      out.dq_weight = empty_like_sizes(q_weight.sizes(), q_weight.scalar_type(), dq);
      if (dq.numel() == 0) out.dq_weight.zero_();
    }
  }
  if (dk.defined()) {
    strides_of(dk, dks);
    out.dk = empty_like_sizes(dk.sizes(), dk.scalar_type(), dk);
    if (k_weight.defined()) {
      TORCH_CHECK(k_in.defined() && k_in.sizes() == dk.sizes() && k_in.scalar_type() == dk.scalar_type() && k_in.device() == dk.device(),
                  "gnb200: k must match dk in sizes, dtype and device");
      k = with_contiguous_channels(k_in);
      strides_of(k, ks);
      out.dk_weight = empty_like_sizes(k_weight.sizes(), k_weight.scalar_type(), dk);
      if (dk.numel() == 0) out.dk_weight.zero_();
    }
  }
  if (nothing(a)) return out;
  const size_t ws_bytes = gnb200_rotary_bwd_workspace_bytes(&a);
  Tensor ws;
  if (ws_bytes) ws = empty_like_sizes({(int64_t)ws_bytes}, at::kByte, any);
  const auto ptr = [](const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
  check_status(gnb200_rotary_bwd(&a, data(dq), dqs, data(dk), dks, data(q), qs, data(k), ks, ptr(out.dq), ptr(out.dk), ptr(out.dq_weight),
                                 ptr(out.dk_weight), ptr(ws), ws_bytes, c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

std::tuple<Tensor, Tensor> rotary_op(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& inv_freq,
                                     at::IntArrayRef sections, const OptTensor& q_weight, const OptTensor& k_weight, double eps, double offset,
                                     bool interleaved) {
  refuse_tangents("rotary", {q, value(k), positions, inv_freq, value(q_weight), value(k_weight)});
  auto [qo, ko] = rotary_forward(q, value(k), positions, inv_freq, sections, value(q_weight), value(k_weight), eps, offset, interleaved);
  return {qo, ko.defined() ? ko : none_of(q)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> rotary_bwd_op(const Tensor& dq, const OptTensor& dk, const Tensor& q, const OptTensor& k,
                                                         const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections,
                                                         const OptTensor& q_weight, const OptTensor& k_weight, double eps, double offset,
                                                         bool interleaved) {
  if (const char* why = refusal_of_heads(dq, value(dk), positions, inv_freq, sections, value(q_weight), value(k_weight)))
    TORCH_CHECK(false, "gnb200: (gradients) ", why);
  refuse_tangents("rotary", {dq, value(dk), q, value(k), positions, inv_freq, value(q_weight), value(k_weight)});
  RotaryGrads g = rotary_backward(dq, value(dk), q, value(k), positions, inv_freq, sections, value(q_weight), value(k_weight), eps, offset,
                                  interleaved);
  const auto filled = [&](const Tensor& t) { return t.defined() ? t : none_of(dq); };
  return {filled(g.dq), filled(g.dk), filled(g.dq_weight), filled(g.dk_weight)};
}

const auto& rotary_bwd_handle() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gnb200::rotary_bwd", "").typed<decltype(rotary_bwd_op)>();
  return op;
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_arg, const OptTensor& q_weight_arg,
                               const OptTensor& k_weight_arg, const Tensor& positions, const Tensor& inv_freq,
                               const std::vector<int64_t>& sections, double eps, double offset, bool interleaved) {
    const Tensor k = value(k_arg), q_weight = value(q_weight_arg), k_weight = value(k_weight_arg);
    auto [qo, ko] = rotary_forward(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved);
    ctx->set_materialize_grads(false);
    // (a rotation alone needs nothing of its input)
    ctx->save_for_backward({q_weight.defined() ? q : Tensor(), k_weight.defined() ? k : Tensor(), q_weight, k_weight, positions, inv_freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["interleaved"] = interleaved;
    if (k.defined()) return {qo, ko};
    return {qo};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    const Tensor &dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(10);
    if (!dq.defined() && !dk.defined()) return out;
    const double eps = ctx->saved_data["eps"].toDouble(), offset = ctx->saved_data["offset"].toDouble();
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    // (as in RmsFunction)
    if (c10::GradMode::is_enabled() || !plain({&dq, &dk, &saved[0], &saved[1], &saved[2], &saved[3], &saved[4], &saved[5]})) {
      const auto& op = rotary_bwd_handle();
      if (!dq.defined()) {  // (the keys alone, in the queries' place)
        auto [gk, none, gkw, no_weight] = op.call(dk, OptTensor(), saved[1].defined() ? saved[1] : dk, OptTensor(), saved[4], saved[5], sections,
                                                  opt(saved[3]), OptTensor(), eps, offset, interleaved);
        out[1] = gk;
        if (saved[3].defined()) out[3] = gkw;
        return out;
      }
      auto [gq, gk, gqw, gkw] = op.call(dq, opt(dk), saved[0].defined() ? saved[0] : dq, opt(saved[1]), saved[4], saved[5], sections,
                                        opt(saved[2]), dk.defined() ? opt(saved[3]) : OptTensor(), eps, offset, interleaved);
      out[0] = gq;
      if (dk.defined()) out[1] = gk;
      if (saved[2].defined()) out[2] = gqw;
      if (saved[3].defined() && dk.defined()) out[3] = gkw;
      return out;
    }
    RotaryGrads g = rotary_backward(dq, dk, saved[0], saved[1], saved[4], saved[5], sections, saved[2], saved[3], eps, offset, interleaved);
    out[0] = g.dq;
    out[1] = g.dk;
    out[2] = g.dq_weight;
    out[3] = g.dk_weight;
    return out;
  }
};

struct RotaryBackwardOnce : torch::autograd::Function<RotaryBackwardOnce> {
  static variable_list forward(AutogradContext*, const Tensor& dq, const OptTensor& dk, const Tensor& q, const OptTensor& k,
                               const OptTensor& q_weight, const OptTensor& k_weight, const Tensor& positions, const Tensor& inv_freq,
                               const std::vector<int64_t>& sections, double eps, double offset, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [gq, gk, gqw, gkw] = rotary_bwd_handle().call(dq, dk, q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved);
    return {gq, gk, gqw, gkw};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    refuse_second("rotary");
    return {};
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor> rotary_bwd_autograd(const Tensor& dq, const OptTensor& dk, const Tensor& q, const OptTensor& k,
                                                               const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections,
                                                               const OptTensor& q_weight, const OptTensor& k_weight, double eps, double offset,
                                                               bool interleaved) {
  const Tensor dk_ = value(dk), k_ = value(k), qw = value(q_weight), kw = value(k_weight);
  if (wants_graph({&dq, &dk_, &q, &k_, &qw, &kw})) {
    variable_list out =
        RotaryBackwardOnce::apply(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, sections.vec(), eps, offset, interleaved);
    return {out[0], out[1], out[2], out[3]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return rotary_bwd_handle().call(dq, dk, q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved);
}

}  // namespace

std::tuple<Tensor, Tensor> gnb200_ops::rms_norm_direct(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps,
                                                       double offset, bool* ok) {
  *ok = plain({&x, &weight, &residual}) && refusal_of_rows(x, weight, residual) == nullptr;
  if (!*ok) return {};
  if (wants_graph({&x, &weight, &residual})) {
    variable_list out = RmsFunction::apply(x, opt(residual), opt(weight), eps, offset);
    return {out[0], out.size() > 1 ? out[1] : Tensor()};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  RmsOut o = rms_forward(x, weight, residual, eps, offset, false, 0, -1, true);
  return {o.y, o.sum};
}

std::tuple<Tensor, Tensor, Tensor> gnb200_ops::rms_quant_direct(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps,
                                                                double offset, int64_t block, int64_t format, bool* ok) {
  *ok = plain({&x, &weight, &residual}) && !wants_graph({&x, &weight, &residual}) && refusal_of_rows(x, weight, residual) == nullptr &&
        (block == 0 || block == 32 || block == 64 || block == 128) && (format == GNB200_E4M3 || format == GNB200_INT8);
  if (!*ok) return {};
  at::AutoDispatchBelowADInplaceOrView guard;
  RmsOut o = rms_forward(x, weight, residual, eps, offset, false, block, (int)format, true);
  return {o.y, o.scale, o.sum};
}

std::tuple<Tensor, Tensor> gnb200_ops::rotary_direct(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& inv_freq,
                                                     at::IntArrayRef sections, const Tensor& q_weight, const Tensor& k_weight, double eps,
                                                     double offset, bool interleaved, bool* ok) {
  *ok = plain({&q, &k, &positions, &inv_freq, &q_weight, &k_weight}) &&
        refusal_of_heads(q, k, positions, inv_freq, sections, q_weight, k_weight) == nullptr;
  if (!*ok) return {};
  if (wants_graph({&q, &k, &q_weight, &k_weight})) {
    variable_list out = RotaryFunction::apply(q, opt(k), opt(q_weight), opt(k_weight), positions, inv_freq, sections.vec(), eps, offset, interleaved);
    return {out[0], out.size() > 1 ? out[1] : Tensor()};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return rotary_forward(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved);
}

TORCH_LIBRARY_FRAGMENT(gnb200, m) {
  m.def("rms_fwd(Tensor x, Tensor? residual, Tensor? weight, float eps, float offset) -> (Tensor, Tensor, Tensor)");
  m.def("rms_bwd(Tensor dy, Tensor? dsum, Tensor sum, Tensor? addend, Tensor? weight, Tensor rstd, float offset) -> (Tensor, Tensor, Tensor)");
  m.def("rms_quant(Tensor x, Tensor? residual, Tensor? weight, float eps, float offset, int block, int format) -> (Tensor, Tensor, Tensor)");
  m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, int[] sections, Tensor? q_weight, Tensor? k_weight, float eps, "
        "float offset, bool interleaved) -> (Tensor, Tensor)");
  m.def("rotary_bwd(Tensor dq, Tensor? dk, Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, int[] sections, Tensor? q_weight, "
        "Tensor? k_weight, float eps, float offset, bool interleaved) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(gnb200, CUDA, m) {
  m.impl("rms_fwd", &rms_fwd_op);
  m.impl("rms_bwd", &rms_bwd_op);
  m.impl("rms_quant", &rms_quant_op);
  m.impl("rotary", &rotary_op);
  m.impl("rotary_bwd", &rotary_bwd_op);
}

TORCH_LIBRARY_IMPL(gnb200, Autograd, m) {
  m.impl("rms_bwd", &rms_bwd_autograd);
  m.impl("rotary_bwd", &rotary_bwd_autograd);
}

// (registered to refuse with a message of this library)
TORCH_LIBRARY_IMPL(gnb200, CPU, m) {
  m.impl("rms_fwd", &rms_fwd_op);
  m.impl("rms_bwd", &rms_bwd_op);
  m.impl("rms_quant", &rms_quant_op);
  m.impl("rotary", &rotary_op);
  m.impl("rotary_bwd", &rotary_bwd_op);
}
