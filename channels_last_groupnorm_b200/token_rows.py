"""What the operators on token rows ask of their arguments."""
import torch
from torch.autograd import forward_ad

TYPES = (torch.float32, torch.float16, torch.bfloat16)


def check_rows(name, x, weight, residual):
    if not x.is_cuda:
        raise ValueError("%s: x must be a CUDA tensor; this package has no CPU path" % name)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("%s: x must have shape (*, channels), got %s" % (name, tuple(x.shape)))
    if x.dtype not in TYPES:
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


def refuse_tangents(name, *tensors):
    """Forward mode, torch.func.jvp too, whose wrapped tensors the ops do not see: an error where its tangents would be left out."""
    if not torch.compiler.is_compiling() and forward_ad._current_level >= 0:
        if any(t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise NotImplementedError("%s has no derivative in forward mode" % name)
