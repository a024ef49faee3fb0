"""Fake-tensor kernels and the autograd formula of torch.ops.gnb200.*.

The reference registers its two ops without a Meta kernel or an autograd formula and disables
dynamo on the module (src/gnnhwc/custom_gn.py:63, its README lists torch.compile support as to
do).  With the registrations below the ops can be traced: `torch.compile` sees the output shapes
and strides without running a kernel, and `torch.ops.gnb200.fwd` is differentiable on its own
(its backward is `torch.ops.gnb200.bwd`).
"""
import torch


def _like(X):
    """Same sizes and storage order as X (channels-last or channels-first)."""
    n, c, r = X.shape
    if X.stride(1) == 1 or c == 1:
        return X.new_empty((n, r, c)).permute(0, 2, 1)
    return X.new_empty((n, c, r))


def _stats_dtype(X):
    return torch.float64 if X.dtype == torch.float64 else torch.float32


@torch.library.register_fake("gnb200::fwd")
def _fwd_fake(X, weight, bias, G, eps, act):
    n = X.shape[0]
    stats = X.new_empty((n, G), dtype=_stats_dtype(X))
    return _like(X), stats, torch.empty_like(stats)


@torch.library.register_fake("gnb200::bwd")
def _bwd_fake(dy, X, weight, bias, means, rstds, G, act):
    return _like(X), torch.empty_like(weight), torch.empty_like(bias)


@torch.library.register_fake("gnb200::bwd_f32")
def _bwd_f32_fake(dy, X, weight, bias, means, rstds, G, act):
    return _like(X), X.new_empty((2, X.shape[1]), dtype=_stats_dtype(X))


@torch.library.register_fake("gnb200::bwd_f32_peer")
def _bwd_f32_peer_fake(dy, X, weight, bias, means, rstds, G, act, peer_ptrs, rank):
    return _like(X), X.new_empty((2, X.shape[1]), dtype=_stats_dtype(X))


def _fwd_setup_context(ctx, inputs, output):
    X, weight, bias, G, eps, act = inputs
    _, means, rstds = output
    ctx.save_for_backward(X, weight, bias, means, rstds)
    ctx.G = G
    ctx.act = act


def _fwd_backward(ctx, dY, dmeans, drstds):
    X, weight, bias, means, rstds = ctx.saved_tensors
    # the kernels want dy in the storage order of X
    if X.stride(1) == 1 or X.shape[1] == 1:
        dy = dY.permute(0, 2, 1).contiguous().permute(0, 2, 1)
    else:
        dy = dY.contiguous()
    dx, dgamma, dbeta = torch.ops.gnb200.bwd(dy, X, weight, bias, means, rstds, ctx.G, ctx.act)
    return dx, dgamma, dbeta, None, None, None


torch.library.register_autograd("gnb200::fwd", _fwd_backward, setup_context=_fwd_setup_context)


# ---------------------------------------------------------------------------------------------- token rows


def _none_of(t):
    return t.new_empty((0,))


@torch.library.register_fake("gnb200::rms_fwd")
def _rms_fwd_fake(x, residual, weight, eps, offset):
    s = _none_of(x) if residual is None else torch.empty_like(residual, memory_format=torch.contiguous_format)
    return torch.empty_like(x, memory_format=torch.contiguous_format), s, x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.register_fake("gnb200::rms_bwd")
def _rms_bwd_fake(dy, dsum, sum, addend, weight, rstd, offset):
    ds = _none_of(sum) if sum.dtype == dy.dtype else torch.empty_like(sum, memory_format=torch.contiguous_format)
    return torch.empty_like(dy, memory_format=torch.contiguous_format), ds, _none_of(sum) if weight is None else torch.empty_like(weight)


@torch.library.register_fake("gnb200::rms_quant")
def _rms_quant_fake(x, residual, weight, eps, offset, block, format):
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn if format == 0 else torch.int8)
    scales = (x.shape[-1] + block - 1) // block if block else 1
    s = _none_of(x) if residual is None else torch.empty_like(residual, memory_format=torch.contiguous_format)
    return q, x.new_empty(x.shape[:-1] + (scales,), dtype=torch.float32), s


@torch.library.register_fake("gnb200::rotary")
def _rotary_fake(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved):
    contiguous = torch.contiguous_format
    return torch.empty_like(q, memory_format=contiguous), _none_of(q) if k is None else torch.empty_like(k, memory_format=contiguous)


@torch.library.register_fake("gnb200::rotary_bwd")
def _rotary_bwd_fake(dq, dk, q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved):
    contiguous = torch.contiguous_format
    return (torch.empty_like(dq, memory_format=contiguous), _none_of(dq) if dk is None else torch.empty_like(dk, memory_format=contiguous),
            _none_of(dq) if q_weight is None else torch.empty_like(q_weight), _none_of(dq) if k_weight is None else torch.empty_like(k_weight))


def _rms_setup_context(ctx, inputs, output):
    x, residual, weight, _, offset = inputs
    _, s, rstd = output
    ctx.has_residual = residual is not None
    ctx.offset = offset
    # (as the native node: x and the residual again where the stored sum is rounded and the weight's gradient wanted)
    again = ctx.has_residual and residual.dtype != torch.float32 and weight is not None and weight.requires_grad
    ctx.save_for_backward(residual if again else s if ctx.has_residual else x, x if again else None, weight, rstd)
    ctx.mark_non_differentiable(rstd) if ctx.has_residual else ctx.mark_non_differentiable(rstd, s)


def _rms_backward(ctx, dy, ds, drstd):
    s, addend, weight, rstd = ctx.saved_tensors
    dx, dres, dw = torch.ops.gnb200.rms_bwd(dy, ds if ctx.has_residual else None, s, addend, weight, rstd, ctx.offset)
    if not ctx.has_residual:
        dres = None
    elif s.dtype == dx.dtype:
        dres = dx
    return dx, dres, None if weight is None else dw, None, None


torch.library.register_autograd("gnb200::rms_fwd", _rms_backward, setup_context=_rms_setup_context)


def _rotary_setup_context(ctx, inputs, output):
    q, k, positions, inv_freq, ctx.sections, q_weight, k_weight, ctx.eps, ctx.offset, ctx.interleaved = inputs
    ctx.has_k = k is not None
    # (as the native node: a rotation alone needs nothing of its input)
    ctx.save_for_backward(None if q_weight is None else q, None if k_weight is None else k, positions, inv_freq, q_weight, k_weight)
    if not ctx.has_k:
        ctx.mark_non_differentiable(output[1])


def _rotary_backward(ctx, dq, dk):
    q, k, positions, inv_freq, q_weight, k_weight = ctx.saved_tensors
    gq, gk, gqw, gkw = torch.ops.gnb200.rotary_bwd(dq, dk if ctx.has_k else None, dq if q is None else q, k, positions, inv_freq, ctx.sections,
                                                   q_weight, k_weight, ctx.eps, ctx.offset, ctx.interleaved)
    return (gq, gk if ctx.has_k else None, None, None, None, None if q_weight is None else gqw, None if k_weight is None else gkw,
            None, None, None)


torch.library.register_autograd("gnb200::rotary", _rotary_backward, setup_context=_rotary_setup_context)


# ---------------------------------------------------------------------------------------------- rows in four bits, dropout


def _up(n, to):
    return (n + to - 1) // to * to


def _four_like(x, block):
    c = x.shape[-1]
    wide, rows = _up(c, 32), x.numel() // c
    return (x.new_empty(x.shape[:-1] + (wide // 2,), dtype=torch.float4_e2m1fn_x2),
            x.new_empty((_up(rows, 128), _up(wide // block, 4)), dtype=torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu))


@torch.library.register_fake("gnb200::quantize_4bit")
def _quantize_4bit_fake(x, block, scale):
    return _four_like(x, block)


@torch.library.register_fake("gnb200::rms_quant_4bit")
def _rms_quant_4bit_fake(x, residual, weight, eps, offset, block, scale):
    s = _none_of(x) if residual is None else torch.empty_like(residual, memory_format=torch.contiguous_format)
    return _four_like(x, block) + (s,)


@torch.library.register_fake("gnb200::dequantize_4bit")
def _dequantize_4bit_fake(codes, scales, channels, scale, dtype):
    return codes.new_empty(codes.shape[:-1] + (channels,), dtype=dtype)


@torch.library.register_fake("gnb200::linear_4bit")
def _linear_4bit_fake(codes, scales, weight_codes, weight_scales, scale, weight_scale, bias, dtype):
    return codes.new_empty(codes.shape[:-1] + (weight_codes.shape[0],), dtype=dtype)


@torch.library.register_fake("gnb200::dropout_add")
def _dropout_add_fake(x, residual, p, seed_at, seed, layer):
    return torch.empty_like(x, memory_format=torch.contiguous_format, dtype=x.dtype if residual is None else residual.dtype)


@torch.library.register_fake("gnb200::dropout_mask")
def _dropout_mask_fake(t, p, seed_at, seed, layer, dtype):
    return torch.empty_like(t, memory_format=torch.contiguous_format, dtype=dtype)


def _dropout_setup_context(ctx, inputs, output):
    x, residual, ctx.p, seed_at, ctx.seed, ctx.layer = inputs
    ctx.x_type, ctx.has_residual = x.dtype, residual is not None
    ctx.save_for_backward(seed_at)


def _dropout_backward(ctx, ds):
    dx = torch.ops.gnb200.dropout_mask(ds, ctx.p, ctx.saved_tensors[0], ctx.seed, ctx.layer, ctx.x_type) if ctx.needs_input_grad[0] else None
    return dx, ds if ctx.has_residual else None, None, None, None, None


torch.library.register_autograd("gnb200::dropout_add", _dropout_backward, setup_context=_dropout_setup_context)


def _mask_setup_context(ctx, inputs, output):
    t, ctx.p, seed_at, ctx.seed, ctx.layer, _ = inputs
    ctx.t_type = t.dtype
    ctx.save_for_backward(seed_at)


def _mask_backward(ctx, d):
    return torch.ops.gnb200.dropout_mask(d, ctx.p, ctx.saved_tensors[0], ctx.seed, ctx.layer, ctx.t_type), None, None, None, None, None


torch.library.register_autograd("gnb200::dropout_mask", _mask_backward, setup_context=_mask_setup_context)
