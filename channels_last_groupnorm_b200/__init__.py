"""B200-native channels-last GroupNorm with fused activation (drop-in for `gnnhwc`), and operators on token rows."""
from .gn_nhwc import ACTIVATION_CODES, GN_NHWC, GN_NHWC_Func
from .token_norm import QUANT_FORMATS, RMSNorm, rms_norm, rms_norm_quant
from .token_rotary import AxialRotary, rotary
from .token_dropout import DropoutAdd, dropout_add
from .token_four import Linear4bit, dequantize_4bit, linear_4bit, quantize_4bit, rms_norm_quant_4bit
from . import _compile  # noqa: F401  (fake-tensor kernels and autograd formula of torch.ops.gnb200.*)

__all__ = ["GN_NHWC", "GN_NHWC_Func", "ACTIVATION_CODES", "RMSNorm", "rms_norm", "rms_norm_quant", "QUANT_FORMATS", "AxialRotary", "rotary", "DropoutAdd",
           "dropout_add", "Linear4bit", "linear_4bit", "quantize_4bit", "dequantize_4bit", "rms_norm_quant_4bit"]
