"""Projections whose backward pass reads an 8-bit checkpoint of their input.

``fp8_weight_grad`` computes a projection's weight gradient from the gradient of its output and the checkpoint,
without a dequantised copy (autograd does not see the call, and a trace is refused).  ``linear`` and ``norm_linear``
are the differentiable forms: the forward product and the input's gradient are plain matrix products; what is kept in
between is the 8-bit checkpoint alone.
``norm_linear`` runs a layer norm in front, and one checkpoint (the normalised rows) serves both backward passes:
with ``n = h w + b``, ``dW = dz^T n = (dz^T h) w + (sum dz) b^T``.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .norm import KeptRows, _adjacent, _forward, _no_code_gradient, _recorded, layer_norm_backward, layer_norm_forward


def fp8_weight_grad(dy, codes, scales, norm_weight=None, norm_bias=None, *, dtype=None, bias_grad: bool = True):
    """``(dweight [out, width], dbias [out])`` of ``y = X W^T + c`` for ``dy [rows, out]`` (bf16, fp16 or fp32).

    ``X [rows, width]`` is the checkpoint ``(codes, scales)`` of :func:`~.checkpoint.save_fp8` or of a norm kept as
    ``"fp8"``; with ``norm_weight`` (and ``norm_bias``), ``[width]`` of dy's type or fp32, the projection's input was
    ``X * norm_weight + norm_bias``.  Both results have dy's type, or ``dtype`` fp32; ``dbias`` is None without
    ``bias_grad``.  Products are exact (dy enters as bf16 terms that hold all of its bits down to 2^-133, the
    checkpoint's values are exact in bf16; scales that are no powers of two round them to bf16) and summed in fp32 on
    the tensor cores, which cut what they add.  So no more than 2048 rows of an fp32 ``dy`` go into one sum, 4096 of a
    16-bit one into an fp32 result, 8192 into a 16-bit result, and those sums are joined by rounded additions: fp32
    results are 7e-7 and 2e-6 of their norm off, whatever the number of rows, 16-bit ones 4e-6 beside their rounding.
    """
    return _native.load().fp8_weight_grad(dy, codes, scales, norm_weight, norm_bias, dtype, bias_grad)


def _backward_as_written(backward):
    """A projection's backward pass: its products in the parameters' type, also where it runs under autocast."""

    @functools.wraps(backward)
    def run(ctx, dz):
        with torch.autocast(dz.device.type, enabled=False):
            return backward(ctx, dz)

    return once_differentiable(run)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.wants = ctx.needs_input_grad
        kept = _native.load().save_fp8(x, True) if ctx.wants[1] else (None, None)
        ctx.save_for_backward(*kept, weight)
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @_backward_as_written
    def backward(ctx, dz):
        codes, scales, weight = ctx.saved_tensors
        dz = _adjacent(dz).to(weight.dtype)  # autocast may have changed the product's type
        dx = dz @ weight if ctx.wants[0] else None
        dweight = dbias = None
        if ctx.wants[1]:
            dweight, dbias = fp8_weight_grad(dz, codes, scales, bias_grad=ctx.wants[2])
        elif ctx.wants[2]:
            dbias = dz.sum(0)
        return dx, dweight, dbias


def linear(x, weight, bias=None):
    """Differentiable ``x [rows, width] @ weight [features, width]^T + bias`` that keeps ``x`` in 8 bits."""
    _check_projection(x.dtype, x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _Linear.apply(x, weight, bias)
    return torch.nn.functional.linear(x, weight, bias)


class _NormLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, norm_bias, weight, bias, eps, scales, hidden, block, dtype):
        normed, kept = _forward(x, norm_weight, norm_bias, eps, scales, hidden, block, dtype, "fp8", True)
        ctx.save_for_backward(kept.rows, kept.scales, kept.rstd, norm_weight, norm_bias, weight)
        return torch.nn.functional.linear(normed, weight, bias)

    @staticmethod
    @_backward_as_written
    def backward(ctx, dz):
        codes, scales, rstd, norm_weight, norm_bias, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        dz = _adjacent(dz).to(weight.dtype)  # autocast may have changed the product's type
        dx = dnw = dnb = dweight = dbias = None
        if need[0] or need[1] or need[2]:
            dx, dnw, dnb = layer_norm_backward(dz @ weight, KeptRows(codes, scales, None, rstd), norm_weight,
                                               want_dx=need[0], want_params=need[1] or need[2])
        if need[3]:
            dweight, dbias = fp8_weight_grad(dz, codes, scales, norm_weight, norm_bias, bias_grad=need[4])
        elif need[4]:
            dbias = dz.sum(0)
        return (dx, dnw if need[1] else None, dnb if need[2] else None, dweight, dbias, None, None, None, None, None)


def norm_linear(x, norm_weight, norm_bias, weight, bias=None, eps: float = 1e-5, *, scales=None, hidden=None,
                block: int = 128, dtype=None):
    """Differentiable ``layer_norm(x) @ weight^T + bias`` that keeps only the normalised rows, in 8 bits.

    ``x``, ``scales``, ``hidden``, ``block`` and ``dtype`` are :func:`~.norm.layer_norm_forward`'s; ``weight
    [features, width]`` and ``bias [features]`` have the type of the normalised rows.  There is no forward-mode
    derivative (a tangent raises).
    """
    _no_code_gradient(x)
    out = (dtype or torch.bfloat16) if x.dtype == torch.float8_e4m3fn else x.dtype
    _check_projection(out, x, weight, bias)
    if _recorded(x, norm_weight, norm_bias, weight, bias):
        return _NormLinear.apply(x, norm_weight, norm_bias, weight, bias, eps, scales, hidden, block, dtype)
    normed, _ = layer_norm_forward(x, norm_weight, norm_bias, eps, scales=scales, hidden=hidden, block=block,
                                   dtype=dtype)
    return torch.nn.functional.linear(normed, weight, bias)


def _check_projection(dtype, x, weight, bias):
    if x.dim() != 2 or weight.dim() != 2 or weight.shape[1] != x.shape[1]:
        raise ValueError("expected rows [rows, width] and a weight [features, width]")
    if weight.dtype != dtype or (bias is not None and (bias.dtype != dtype or tuple(bias.shape) != (weight.shape[0],))):
        raise ValueError("weight and bias [features] must have the rows' type")
