"""Rotary positions with several axes on queries and keys, with or without the norm of each head in front.

Tokens of text have one position, those of images and videos a place in time, height and width: every axis turns its own
section of a head's pairs of channels.  `rotary` does queries and keys in one kernel that reads and writes them once, the
root-mean-square norm of each head included where weights are given (csrc/gn_rotary.cu).  The reference has no counterpart.
"""
import torch
import torch.nn as nn

from . import _native
from .token_rows import refuse_tangents

_rotary = _native.python_module.rotary
_TYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_HEAD_DIM = 512
MAX_AXES = 8


def _check(q, k, positions, inv_freq, sections, q_weight, k_weight):
    if not q.is_cuda:
        raise ValueError("rotary: q must be a CUDA tensor; this package has no CPU path")
    if q.ndim not in (3, 4):
        raise ValueError("rotary: q must have shape (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), got %s" % (tuple(q.shape),))
    if q.dtype not in _TYPES:
        raise ValueError("rotary: q must be float32, float16 or bfloat16, got %s" % q.dtype)
    d = q.shape[-1]
    if not 2 <= d <= MAX_HEAD_DIM:
        raise ValueError("rotary: heads must have 2 to %d channels, got %d" % (MAX_HEAD_DIM, d))
    if k is not None and (k.ndim != q.ndim or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != d or k.dtype != q.dtype or k.device != q.device):
        raise ValueError("rotary: k must match q in tokens, head_dim, dtype and device, got %s %s for %s %s"
                         % (tuple(k.shape), k.dtype, tuple(q.shape), q.dtype))
    if not 1 <= len(sections) <= MAX_AXES or any(s < 0 for s in sections):
        raise ValueError("rotary: sections must name the pairs of 1 to %d axes, got %s" % (MAX_AXES, tuple(sections)))
    pairs = sum(sections)
    if pairs < 1 or 2 * pairs > d:
        raise ValueError("rotary: %d pairs do not fit heads of %d channels" % (pairs, d))
    if positions.shape != q.shape[:-2] + (len(sections),) or positions.device != q.device:
        raise ValueError("rotary: positions must have shape %s on the device of q, got %s on %s"
                         % (tuple(q.shape[:-2]) + (len(sections),), tuple(positions.shape), positions.device))
    if positions.dtype not in (torch.int32, torch.int64, torch.float32):
        raise ValueError("rotary: positions must be int32, int64 or float32, got %s" % positions.dtype)
    if inv_freq.shape != (pairs,) or inv_freq.dtype != torch.float32 or inv_freq.device != q.device:
        raise ValueError("rotary: inv_freq must be a float32 vector of %d frequencies on the device of q, got %s %s on %s"
                         % (pairs, tuple(inv_freq.shape), inv_freq.dtype, inv_freq.device))
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or w.dtype not in (q.dtype, torch.float32) or w.device != q.device):
            raise ValueError("rotary: %s must be a vector of %d elements in the dtype of q or float32 on its device, got %s %s on %s"
                             % (name, d, tuple(w.shape), w.dtype, w.device))
    if k_weight is not None and k is None:
        raise ValueError("rotary: a norm weight for keys without keys")
    if torch.is_grad_enabled() and (inv_freq.requires_grad or positions.requires_grad):
        raise ValueError("rotary: has no gradient in positions or inv_freq")


def rotary(q, k, positions, inv_freq, sections, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, offset=0.0):
    """Turns the pairs of channels of every head of q and k by position * inv_freq; returns (q, k), new contiguous tensors.

    q, k: (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), each with heads of its own number; any strides with
    contiguous channels are read in place (slices of one projection's output, (batch, heads, tokens, head_dim) transposed).  k
    may be None.  positions: (*tokens, axes), int32, int64 or float32.  sections: pairs of each axis; inv_freq: float32, one
    frequency per pair, the first sections[0] of axis 0 and so on.  Pair i is channels (i, i + pairs), or (2 i, 2 i + 1) with
    interleaved=True; channels beyond the 2 * sum(sections) first ones pass.  q_weight, k_weight: weights of a root-mean-square
    norm of each head in front of the rotation, (offset + weight); None for no norm.  Differentiable once in q, k and the weights (a gradient of
    the gradients is an error).
    """
    if not torch.compiler.is_compiling() and not inv_freq.requires_grad and not positions.requires_grad:
        out = _rotary(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved)
        if out is not None:
            return out
    sections = [int(s) for s in sections]
    _check(q, k, positions, inv_freq, sections, q_weight, k_weight)
    refuse_tangents("rotary", q, k, positions, inv_freq, q_weight, k_weight)
    q_weight, k_weight = (w if w is None else w.contiguous() for w in (q_weight, k_weight))
    out = torch.ops.gnb200.rotary(q, k, positions, inv_freq.contiguous(), sections, q_weight, k_weight, float(eps), float(offset), bool(interleaved))
    return out[0], (None if k is None else out[1])


class AxialRotary(nn.Module):
    """AxialRotary(head_dim, sections, base=10000.0, shared=False, interleaved=False, qk_norm=False, eps=1e-6, device=None, dtype=None)

    `forward(q, k, positions)` is `rotary` with frequencies of base^(-j / n): with shared=False every axis has the whole range (n its
    own pairs), with shared=True the axes divide one range among them (n = all pairs), in the order of `sections`.  qk_norm
    adds the heads' norms with learned weights `q_weight` and `k_weight`.  The frequencies are no part of a checkpoint: a module that was
    built on the meta device has them again as soon as it leaves it (`to_empty`, then `load_state_dict` or `reset_parameters`).
    """

    def __init__(self, head_dim: int, sections, base=10000.0, shared=False, interleaved=False, qk_norm=False, eps=1e-6, device=None, dtype=None):
        super().__init__()
        self.head_dim = head_dim
        self.sections = tuple(int(s) for s in sections)
        self.interleaved = bool(interleaved)
        self.eps = float(eps)
        if not 1 <= len(self.sections) <= MAX_AXES or min(self.sections) < 0 or not 2 <= 2 * sum(self.sections) <= head_dim <= MAX_HEAD_DIM:
            raise ValueError("AxialRotary: %s pairs do not fit heads of %d channels" % (self.sections, head_dim))
        self.base = float(base)
        self.shared = bool(shared)
        self.register_buffer("inv_freq", self._frequencies(device), persistent=False)
        for name in ("q_weight", "k_weight"):
            self.register_parameter(name, nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype)) if qk_norm else None)

    def _frequencies(self, device):
        n = sum(self.sections)
        exponents = [i / n for i in range(n)] if self.shared else [i / s for s in self.sections for i in range(s)]
        return torch.tensor([self.base ** -e for e in exponents], dtype=torch.float32, device=device)

    def reset_parameters(self):
        """Weights of one and the frequencies of the module's base, as the constructor makes them."""
        self.inv_freq = self._frequencies(self.inv_freq.device)
        with torch.no_grad():
            for w in (self.q_weight, self.k_weight):
                if w is not None:
                    w.fill_(1.0)

    def _apply(self, fn, recurse=True):
        # Moved, but neither rounded nor emptied: frequencies stay in 32 bits where the module goes to 16, an angle of many turns needs
        # them, and to_empty() leaves them as they are, since no checkpoint brings them back.
        kept = self.inv_freq
        super()._apply(fn, recurse)
        device = self.inv_freq.device
        self.inv_freq = self._frequencies(device) if kept.is_meta and device.type != "meta" else kept.to(device)
        return self

    def forward(self, q, k, positions):
        return rotary(q, k, positions, self.inv_freq, self.sections, self.q_weight, self.k_weight, self.eps, self.interleaved)

    def extra_repr(self):
        return "{head_dim}, {sections}, interleaved={interleaved}, eps={eps}".format(**self.__dict__)
