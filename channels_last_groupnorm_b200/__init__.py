"""B200-native channels-last GroupNorm with fused activation (drop-in for `gnnhwc`), and operators on token rows."""
from .gn_nhwc import ACTIVATION_CODES, GN_NHWC, GN_NHWC_Func
from .token_norm import QUANT_FORMATS, RMSNorm, rms_norm, rms_norm_quant
from .token_rotary import AxialRotary, rotary
from . import _compile  # noqa: F401  (fake-tensor kernels and autograd formula of torch.ops.gnb200.*)

__all__ = ["GN_NHWC", "GN_NHWC_Func", "ACTIVATION_CODES", "RMSNorm", "rms_norm", "rms_norm_quant", "QUANT_FORMATS", "AxialRotary", "rotary"]
