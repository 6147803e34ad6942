from .checkpoint import restore_fp8, save_fp8
from .fp8 import E4M3_MAX, calc_diff, dequantize_fp8_blockwise, quantize_fp8_blockwise
from .norm import KeptRows, check_readout, layer_norm, layer_norm_backward, layer_norm_forward
from .pack import route_pack, route_pack_reference
from .projection import fp8_weight_grad, linear, norm_linear

__all__ = [
    "E4M3_MAX",
    "KeptRows",
    "calc_diff",
    "check_readout",
    "dequantize_fp8_blockwise",
    "fp8_weight_grad",
    "layer_norm",
    "layer_norm_backward",
    "layer_norm_forward",
    "linear",
    "norm_linear",
    "quantize_fp8_blockwise",
    "restore_fp8",
    "route_pack",
    "route_pack_reference",
    "save_fp8",
]
