"""Root-mean-square norm of token rows with the residual's addition, and the same with an 8-bit output and scales.

What the blocks around attention and feed-forward layers start with: `rms_norm` in training and inference, `rms_norm_quant`
in front of 8-bit products in inference.  Both run as one kernel that reads and writes every element once, but for rows of more than
some 16384 channels, which it reads two or three times (csrc/gn_rms.cu).  The reference has no counterpart.
"""
import torch
import torch.nn as nn

from . import _native

_rms_norm = _native.python_module.rms_norm
_rms_quant = _native.python_module.rms_quant

#: 8-bit types of `rms_norm_quant` and their codes in the C ABI
QUANT_FORMATS = {torch.float8_e4m3fn: 0, torch.int8: 1}
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _check(name, x, weight, residual):
    if not x.is_cuda:
        raise ValueError("%s: x must be a CUDA tensor; this package has no CPU path" % name)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("%s: x must have shape (*, channels), got %s" % (name, tuple(x.shape)))
    if x.dtype not in _TYPES:
        raise ValueError("%s: x must be float32, float16 or bfloat16, got %s" % (name, x.dtype))
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError("%s: residual must match x in sizes and device, got %s on %s for %s on %s"
                             % (name, tuple(residual.shape), residual.device, tuple(x.shape), x.device))
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError("%s: residual must have the dtype of x or float32, got %s for %s" % (name, residual.dtype, x.dtype))
    if weight is not None:
        if weight.shape != x.shape[-1:] or weight.device != x.device:
            raise ValueError("%s: weight must be a vector of %d elements on the device of x, got %s on %s"
                             % (name, x.shape[-1], tuple(weight.shape), weight.device))
        if weight.dtype not in (x.dtype, torch.float32):
            raise ValueError("%s: weight must have the dtype of x or float32, got %s for %s" % (name, weight.dtype, x.dtype))


def rms_norm(x, weight=None, residual=None, eps=1e-6, offset=0.0):
    """y = s * rsqrt(mean(s^2) + eps) * (offset + weight) over the last dimension, with s = x + residual.

    Returns y without a residual, else (y, s): s, rounded once to the residual's dtype, is the residual stream that the next block
    adds to; the norm itself takes the sum before that rounding.  x: (*, channels) in float32, float16 or bfloat16; contiguous rows
    and slices of a wider tensor whose channels, start and distance are whole 16-byte vectors are read in place, other layouts are copied first.  residual: x's sizes, x's dtype
    or float32.  weight: (channels,) in x's dtype or float32, or None for no weight; offset=1 is for weights stored as
    differences from one.  Differentiable once in x, weight and residual (a gradient of the gradients is an error); the weight's
    gradient is summed in a fixed order.
    """
    if not torch.compiler.is_compiling():
        out = _rms_norm(x, weight, residual, eps, offset)
        if out is not None:
            return out
    _check("rms_norm", x, weight, residual)
    if weight is not None:
        weight = weight.contiguous()
    y, s, _ = torch.ops.gnb200.rms_fwd(x, residual, weight, float(eps), float(offset))
    return y if residual is None else (y, s)


def rms_norm_quant(x, weight=None, residual=None, eps=1e-6, offset=0.0, block=0, dtype=torch.float8_e4m3fn):
    """`rms_norm` with its output as 8-bit codes: (codes, scales), or (codes, scales, s) with a residual; y = codes * scales.

    dtype: torch.float8_e4m3fn or torch.int8.  block: 0 for one scale per row (scales of shape (*, 1)), or 32, 64 or 128 channels
    that share one (shape (*, ceil(channels / block))).  A scale is the largest magnitude of its channels over the largest code (448
    or 127), at least 2^-126; a NaN among them makes it NaN.  A code is that of y / scale, rounded as a division rounds it, with y in 32
    bits.  Inference only: it refuses to run where
    a gradient would be recorded.
    """
    if dtype not in QUANT_FORMATS:
        raise ValueError("rms_norm_quant: dtype must be torch.float8_e4m3fn or torch.int8, got %s" % (dtype,))
    if not torch.compiler.is_compiling():
        out = _rms_quant(x, weight, residual, eps, offset, block, QUANT_FORMATS[dtype])
        if out is not None:
            return out
    _check("rms_norm_quant", x, weight, residual)
    if block not in (0, 32, 64, 128):
        raise ValueError("rms_norm_quant: block must be 0 (one scale per row), 32, 64 or 128, got %s" % (block,))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rms_norm_quant has no gradient: call it under torch.no_grad(), or use rms_norm")
    if weight is not None:
        weight = weight.contiguous()
    q, scale, s = torch.ops.gnb200.rms_quant(x, residual, weight, float(eps), float(offset), int(block), QUANT_FORMATS[dtype])
    return (q, scale) if residual is None else (q, scale, s)


class RMSNorm(nn.Module):
    """RMSNorm(num_channels, eps=1e-6, offset=0.0, affine=True, device=None, dtype=None)

    `forward(x, residual=None)` is `rms_norm`, `quantize(x, residual=None, block=0, dtype=torch.float8_e4m3fn)` is
    `rms_norm_quant`.  The weight starts so that offset + weight is one.
    """

    def __init__(self, num_channels: int, eps=1e-6, offset=0.0, affine=True, device=None, dtype=None):
        super().__init__()
        self.num_channels = num_channels
        self.eps = float(eps)
        self.offset = float(offset)
        self.affine = affine
        if affine:
            self.weight = nn.Parameter(torch.empty((num_channels,), device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.affine:
            nn.init.constant_(self.weight, 1.0 - self.offset)

    def _expect(self, x):
        if x.ndim < 1 or x.shape[-1] != self.num_channels:
            raise ValueError("RMSNorm: expected input of shape (*, %d), got %s" % (self.num_channels, tuple(x.shape)))

    def forward(self, x, residual=None):
        self._expect(x)
        return rms_norm(x, self.weight, residual, self.eps, self.offset)

    def quantize(self, x, residual=None, block=0, dtype=torch.float8_e4m3fn):
        self._expect(x)
        return rms_norm_quant(x, self.weight, residual, self.eps, self.offset, block, dtype)

    def extra_repr(self):
        return "{num_channels}, eps={eps}, offset={offset}, affine={affine}".format(**self.__dict__)
