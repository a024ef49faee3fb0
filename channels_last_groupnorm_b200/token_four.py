"""Rows in four bits with block scales, and the product of two such matrices.

What a block's projections take in serving, one step below `rms_norm_quant`: `quantize_4bit` of any rows (activations, or a weight once),
`rms_norm_quant_4bit` of the norm's output, `linear_4bit` for the product on the 4-bit tensor cores (csrc/gn_four.cu,
csrc/gn_linear4.cu).  The reference has no counterpart.

Codes are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), dtype float4_e2m1fn_x2: two a byte, the first channel in the low half, in rows of
whole blocks of 32, zeros behind the channels.  A block of 16 channels has a scale in float8_e4m3fn beside a scale of the whole tensor in
float32; a block of 32 has a power of two in float8_e8m0fnu.  The tensor of scales has ceil(rows / 128) * 128 rows of ceil(blocks / 4) * 4; its
bytes lie in tiles of 128 rows and 4 blocks, in which row r, block b is byte (r % 32) * 16 + r % 128 // 32 * 4 + b % 4.
"""
import torch
import torch.nn as nn

from . import _native
from .token_rows import TYPES, check_rows, refuse_tangents

_quantize = _native.python_module.quantize_4bit
_dequantize = _native.python_module.dequantize_4bit
_rms_quant = _native.python_module.rms_quant_4bit
_linear = _native.python_module.linear_4bit

#: blocks and the dtypes of their scales
SCALE_TYPES = {16: torch.float8_e4m3fn, 32: torch.float8_e8m0fnu}


def _check_block(name, block, scale, device):
    if block not in SCALE_TYPES:
        raise ValueError("%s: block must be 16 or 32 channels, got %s" % (name, block))
    if scale is not None:
        if block == 32:
            raise ValueError("%s: blocks of 32 have no scale of the whole tensor" % name)
        if scale.numel() != 1 or scale.dtype != torch.float32 or scale.device != device:
            raise ValueError("%s: scale must be one float32 on the device of the rows, got %s %s on %s" % (name, tuple(scale.shape), scale.dtype, scale.device))


def _refuse_grad(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("%s has no gradient: call it under torch.no_grad()" % name)
    refuse_tangents(name, *tensors)


def _up(n, to):
    return (n + to - 1) // to * to


def _check_four(name, codes, scales):
    """The block that the scales' dtype says."""
    if not codes.is_cuda:
        raise ValueError("%s: codes must be a CUDA tensor; this package has no CPU path" % name)
    if codes.dtype != torch.float4_e2m1fn_x2 or codes.ndim < 1 or codes.shape[-1] < 16 or codes.shape[-1] % 16:
        raise ValueError("%s: codes must be float4_e2m1fn_x2 of shape (*, channels / 2), whole blocks of 32 channels, got %s %s"
                         % (name, tuple(codes.shape), codes.dtype))
    block = next((b for b, t in SCALE_TYPES.items() if t == scales.dtype), None)
    if block is None:
        raise ValueError("%s: scales must be float8_e4m3fn (blocks of 16) or float8_e8m0fnu (blocks of 32), got %s" % (name, scales.dtype))
    rows = 1
    for n in codes.shape[:-1]:
        rows *= n
    want = (_up(rows, 128), _up(codes.shape[-1] * 2 // block, 4))
    if scales.shape != want or scales.device != codes.device or not scales.is_contiguous():
        raise ValueError("%s: scales must be those of all rows of codes, contiguous %s on its device, got %s on %s"
                         % (name, want, tuple(scales.shape), scales.device))
    return block


def quantize_4bit(x, block=16, scale=None):
    """Rows as 4-bit codes and block scales: (codes, scales).

    x: (*, channels) in float32, float16 or bfloat16, read in place as by `rms_norm`.  block 16: the scale of a block is its largest magnitude over 6 *
    scale, rounded to e4m3, 2^-9 to 448; `scale`, one float32 on the device (None: 1) from 2^-100 to 2^117, belongs to the whole tensor.  block 32: the scale
    is 2^(floor(log2(largest magnitude)) - 2), and there is no `scale`.  A code is that of x over its scales, the nearest one, ties to the even
    code, saturating.  A NaN or an infinity makes the scale of its block NaN.  No gradient: it refuses to run where one would be recorded.
    """
    if not torch.compiler.is_compiling():
        out = _quantize(x, block, scale)
        if out is not None:
            return out
    check_rows("quantize_4bit", x, None, None)
    _check_block("quantize_4bit", block, scale, x.device)
    _refuse_grad("quantize_4bit", x, scale)
    return torch.ops.gnb200.quantize_4bit(x, int(block), scale)


def dequantize_4bit(codes, scales, channels=None, scale=None, dtype=torch.bfloat16):
    """What codes and scales stand for: code * block scale * scale, (*, channels) in `dtype`.  channels: what the codes were made of (None: all that
    their rows hold)."""
    channels = codes.shape[-1] * 2 if channels is None else channels
    if not torch.compiler.is_compiling():
        out = _dequantize(codes, scales, channels, scale, dtype)
        if out is not None:
            return out
    block = _check_four("dequantize_4bit", codes, scales)
    _check_block("dequantize_4bit", block, scale, codes.device)
    if channels < 1 or _up(channels, 32) != codes.shape[-1] * 2:
        raise ValueError("dequantize_4bit: channels must be those that the codes were made of, got %s for rows of %d" % (channels, codes.shape[-1] * 2))
    if dtype not in TYPES:
        raise ValueError("dequantize_4bit: dtype must be float32, float16 or bfloat16, got %s" % dtype)
    _refuse_grad("dequantize_4bit", scale)
    return torch.ops.gnb200.dequantize_4bit(codes, scales, int(channels), scale, dtype)


def rms_norm_quant_4bit(x, weight=None, residual=None, eps=1e-6, offset=0.0, block=16, scale=None):
    """`rms_norm` with its output as 4-bit codes and block scales: (codes, scales), or (codes, scales, s) with a residual.

    The norm's output is not rounded before it becomes codes; block and scale are those of `quantize_4bit`.  Inference only: it refuses to run
    where a gradient would be recorded.
    """
    if not torch.compiler.is_compiling():
        out = _rms_quant(x, weight, residual, eps, offset, block, scale)
        if out is not None:
            return out
    check_rows("rms_norm_quant_4bit", x, weight, residual)
    _check_block("rms_norm_quant_4bit", block, scale, x.device)
    _refuse_grad("rms_norm_quant_4bit", x, weight, residual, scale)
    if weight is not None:
        weight = weight.contiguous()
    codes, scales, s = torch.ops.gnb200.rms_quant_4bit(x, residual, weight, float(eps), float(offset), int(block), scale)
    return (codes, scales) if residual is None else (codes, scales, s)


def linear_4bit(codes, scales, weight_codes, weight_scales, scale=None, weight_scale=None, bias=None, dtype=torch.bfloat16):
    """The product of rows (*, channels) with a weight (features, channels), both in four bits: (*, features) in `dtype`.

    codes, scales and weight_codes, weight_scales: from `quantize_4bit` (or `rms_norm_quant_4bit`) with the same block, scale and weight_scale what they were
    made with.  bias: (features,) in float32, float16 or bfloat16.  Summed in 32 bits, rounded once.  No gradient.
    """
    if not torch.compiler.is_compiling():
        out = _linear(codes, scales, weight_codes, weight_scales, scale, weight_scale, bias, dtype)
        if out is not None:
            return out
    block = _check_four("linear_4bit", codes, scales)
    if weight_codes.ndim != 2 or weight_codes.device != codes.device:
        raise ValueError("linear_4bit: weight_codes must have shape (features, channels / 2) on the device of codes, got %s on %s"
                         % (tuple(weight_codes.shape), weight_codes.device))
    if _check_four("linear_4bit", weight_codes, weight_scales) != block or weight_codes.shape[-1] != codes.shape[-1]:
        raise ValueError("linear_4bit: codes and weight_codes must have the same channels and blocks, got rows of %d %s and %d %s"
                         % (codes.shape[-1] * 2, scales.dtype, weight_codes.shape[-1] * 2, weight_scales.dtype))
    _check_block("linear_4bit", block, scale, codes.device)
    _check_block("linear_4bit", block, weight_scale, codes.device)
    if bias is not None and (bias.shape != weight_codes.shape[:1] or bias.dtype not in TYPES or bias.device != codes.device):
        raise ValueError("linear_4bit: bias must be a vector of %d elements in float32, float16 or bfloat16 on the device of codes, got %s %s on %s"
                         % (weight_codes.shape[0], tuple(bias.shape), bias.dtype, bias.device))
    if dtype not in TYPES:
        raise ValueError("linear_4bit: dtype must be float32, float16 or bfloat16, got %s" % dtype)
    _refuse_grad("linear_4bit", scale, weight_scale, bias)
    if bias is not None:
        bias = bias.contiguous()
    return torch.ops.gnb200.linear_4bit(codes, scales, weight_codes, weight_scales, scale, weight_scale, bias, dtype)


class Linear4bit(nn.Module):
    """Linear4bit(weight, bias=None, block=16): a trained `nn.Linear`'s weight in four bits, for serving.

    `forward(x, scale=None)` quantises x and multiplies; `forward((codes, scales), scale)` takes what `RMSNorm.quantize_4bit` made with the same
    block and scale.  In blocks of 16 the weight's own scale is its largest finite magnitude over 6 * 448, so that the largest block scale is
    the largest e4m3.  `dtype`: that of the result for codes (x's own for x); the weight's by default.
    """

    def __init__(self, weight, bias=None, block=16, dtype=None):
        super().__init__()
        self.features, self.channels = weight.shape
        self.block = int(block)
        self.dtype = weight.dtype if dtype is None else dtype
        with torch.no_grad():
            scale = None
            if self.block == 16:
                # (of the finite ones: a NaN or an infinity makes its own feature NaN, not all of them)
                most = weight.abs().nan_to_num_(nan=0.0, posinf=0.0).amax() if weight.numel() else weight.new_zeros(())
                scale = (most.float() / (6 * 448)).clamp_min(2.0 ** -100).reshape(1)
            codes, scales = quantize_4bit(weight.detach(), self.block, scale)
        self.register_buffer("weight_codes", codes.view(torch.uint8))  # (the packed type has neither copies nor checkpoints)
        self.register_buffer("weight_scales", scales.view(torch.uint8))
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_linear(cls, linear, block=16):
        return cls(linear.weight, linear.bias, block)

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale  # stays in 32 bits where the module goes to 16
        super()._apply(fn, recurse)
        if scale is not None and self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, x, scale=None):
        if isinstance(x, torch.Tensor):
            dtype = x.dtype
            if x.ndim < 1 or x.shape[-1] != self.channels:
                raise ValueError("Linear4bit: expected input of shape (*, %d), got %s" % (self.channels, tuple(x.shape)))
            x = quantize_4bit(x, self.block, scale)
        else:
            dtype = self.dtype
        return linear_4bit(x[0], x[1], self.weight_codes.view(torch.float4_e2m1fn_x2), self.weight_scales.view(SCALE_TYPES[self.block]), scale,
                           self.weight_scale, self.bias, dtype)

    def extra_repr(self):
        return "{channels}, {features}, block={block}".format(channels=self.channels, features=self.features, block=self.block)
