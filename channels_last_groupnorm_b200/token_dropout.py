"""Dropout of a branch with the residual's addition, its mask made from a counter wherever it is needed and never stored.

What stands in front of the norms of a transformer block in training: `dropout_add` is one kernel that reads the branch's output and the
residual stream once, its backward another that reads the gradient (csrc/gn_dropout.cu).  The reference has no counterpart.
"""
import torch
import torch.nn as nn

from . import _native
from .token_rows import check_rows, refuse_tangents

_dropout_add = _native.python_module.dropout_add


def _signed(name, n):
    """A number of 64 bits, with or without a sign, as the ops take it."""
    n = int(n)
    if not -2 ** 63 <= n < 2 ** 64:
        raise ValueError("dropout_add: %s must fit 64 bits, got %d" % (name, n))
    return n - 2 ** 64 if n >= 2 ** 63 else n


def dropout_add(x, residual=None, p=0.1, seed=None, layer=0):
    """residual + dropout(x): an element of x is dropped with probability p, or divided by 1 - p; without a residual the dropout alone.

    x: (*) in float32, float16 or bfloat16.  residual: x's sizes, x's dtype or float32; the result has the residual's dtype, is summed in
    32 bits and rounded once.  Element i of x, counted in order, is kept where word i % 4 of Philox 4x32 with ten rounds, counter (i // 4,
    layer), key `seed`, is at least p * 2^32: the same seed and layer give the same mask whatever the layout, and different ones independent
    masks.  So each place in the model that drops has a layer of its own, and each step a seed, with one of its own for each rank that has a slice of the
    batch and each micro-batch: elements are counted from the first of this call's x.  seed: a number, or a tensor of one int64 on the device of x, which
    the kernels read, so that a captured graph follows it (it must keep its value until the backward has run); None only where nothing can be
    dropped.  0 <= p < 1.  A dropped
    element gives zero whatever it was.  Differentiable in x and residual.
    """
    at = seed if isinstance(seed, torch.Tensor) else None
    if not torch.compiler.is_compiling():
        out = _dropout_add(x, residual, p, seed, layer)
        if out is not None:
            return out
    check_rows("dropout_add", x.reshape(1) if x.ndim == 0 else x, None, residual)
    p = float(p)
    if not (p >= 0 and p * 2.0 ** 32 < 2.0 ** 32 - 0.5):
        raise ValueError("dropout_add: p must be at least 0 and less than 1, got %s" % p)
    if at is not None and (at.numel() != 1 or at.dtype != torch.int64 or at.device != x.device):
        raise ValueError("dropout_add: a seed that is a tensor must have one element, int64, on the device of x, got %s %s on %s"
                         % (tuple(at.shape), at.dtype, at.device))
    layer = _signed("layer", layer)
    if seed is None:
        if p > 0 and x.numel() > 0:
            raise ValueError("dropout_add: a seed is needed, another one for each step, rank and micro-batch: the same seed drops the same elements")
        seed = 0
    refuse_tangents("dropout_add", x, residual)
    return torch.ops.gnb200.dropout_add(x, residual, p, at, 0 if at is not None else _signed("seed", seed), layer)


class DropoutAdd(nn.Module):
    """DropoutAdd(p=0.1, layer=0)

    `forward(x, residual, seed)` is `dropout_add` in training, where the step's seed is needed; in evaluation it is the addition alone.  layer: another
    number for each of a model's modules, which drop the same elements otherwise.
    """

    def __init__(self, p=0.1, layer=0):
        super().__init__()
        self.p = float(p)
        self.layer = int(layer)
        if not 0 <= self.p < 1:
            raise ValueError("DropoutAdd: p must be at least 0 and less than 1, got %s" % p)

    def forward(self, x, residual=None, seed=None):
        if not self.training:
            return dropout_add(x, residual, 0.0, 0, self.layer)
        return dropout_add(x, residual, self.p, seed, self.layer)

    def extra_repr(self):
        return "p={p}, layer={layer}".format(**self.__dict__)
