"""8-bit activation checkpoints: what a training step keeps between its forward and backward pass, in e4m3.

``save_fp8`` stores ``x [rows, width]`` as e4m3 codes and one fp32 scale per row and 128 columns, the layout of
``quantize_fp8_blockwise(x, power_of_two=True)`` (so ``dequantize_fp8_blockwise`` reads it too), by one sm_100a
kernel.  A scale is the least power of two that brings its block's largest finite value within 448: dividing by it
is exact, so a value is off by its one rounding, at most 2^-4 of itself down to 2^-6 of the scale, and the restored
value is exact in bf16.  Infinities and NaN come back as NaN and leave their block's other values alone.
Code rows start on 16-byte boundaries (``codes.stride(0)`` is the width rounded up to 16).

``restore_fp8`` gives the values back; :func:`~.norm.layer_norm_backward` and :func:`~.projection.fp8_weight_grad`
read a checkpoint directly, which is cheaper.  Autograd sees neither call (tangents of forward mode and traces are
refused); :func:`~.projection.linear` and :func:`~.projection.norm_linear` are the differentiable forms that keep such
a checkpoint.
"""

from __future__ import annotations

import torch

from .. import _native


def save_fp8(x: torch.Tensor):
    """``x [rows, width]`` (bf16, fp16 or fp32 on a GPU) as ``(codes [rows, width] e4m3, scales [rows, ceil(width / 128)])``."""
    return _native.load().save_fp8(x)


def restore_fp8(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``save_fp8``'s ``(codes, scales)`` as ``dtype``.

    A finite value beyond the type's range (a largest value that was rounded up) becomes the type's largest.
    """
    return _native.load().restore_fp8(codes, scales, dtype)
