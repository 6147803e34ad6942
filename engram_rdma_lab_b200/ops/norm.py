"""Layer norm over looked-up rows, forward and backward (sm_100a kernels).

The rows are what a lookup returns: ``[tokens, width]`` bf16 (fp16 and fp32 work too), or e4m3 codes with their
scales, which the kernel multiplies in as it reads (no dequantised copy).  The backward pass reads what the forward
pass kept: the rows themselves with three fp32 numbers per row (``keep="exact"``), or the normalised rows in 8 bits
with one (``keep="fp8"``; the format of :mod:`.checkpoint`), half of bf16's bytes.  Normalised values are what suits
8 bits: a row's common offset and size are gone before the rounding, so e4m3's relative precision is spent on what
the gradient needs, and the same checkpoint serves the projection behind the norm
(:func:`~.projection.fp8_weight_grad`).

Sums over rows and columns are held in fp32 (a row whose deviations are past 1.8e19 has an infinite or unknown variance:
its ``y`` is the bias, or NaN) and joined in a fixed order: equal inputs give equal bits on equal GPUs,
and a row's ``y`` does not depend on the rows beside it.  Everything runs on the current stream and can be captured
into CUDA graphs (capture the functional pair, not autograd's backward pass).  A kernel whose bounded wait for its
own copies ran out reports that: the read-out calls that follow raise, and :func:`check_readout` asks.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _native

_KEEP = {None: 0, "exact": 1, "fp8": 2}


class _KeptRows(NamedTuple):
    rows: torch.Tensor
    scales: Optional[torch.Tensor]
    mean: Optional[torch.Tensor]
    rstd: torch.Tensor


class KeptRows(_KeptRows):
    """What ``layer_norm_forward`` keeps: ``(x, None, mean, rstd)`` or ``(codes, scales, None, rstd)``.

    Beside the four, ``shift`` is what the rounding of ``mean`` left (None: zeros): a row's mean is ``mean + shift``,
    which counts where its offset is many times its deviation.
    """

    shift: Optional[torch.Tensor] = None

    def __new__(cls, rows, scales, mean, rstd, shift=None):
        self = tuple.__new__(cls, (rows, scales, mean, rstd))
        if shift is not None:
            self.shift = shift
        return self


def _keep_mode(keep) -> int:
    try:
        return _KEEP[keep]
    except (KeyError, TypeError):
        raise ValueError('keep must be None, "exact" or "fp8"') from None


def _forward(x, weight, bias, eps, scales, hidden, block, dtype, keep, recorded):
    mode = _keep_mode(keep)
    y, codes, code_scales, mean, rstd, shift = _native.load().norm_forward(
        x, weight, bias, eps, scales, hidden, block, dtype, mode, recorded)
    if mode == 0:
        return y, None
    if mode == 2:
        return y, KeptRows(codes, code_scales, None, rstd)
    return y, KeptRows(x, None, mean, rstd, shift)


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, *, scales=None, hidden=None, block: int = 128,
                       dtype=None, keep=None):
    """``(y, kept)`` with ``y = (x - mean) / sqrt(var + eps) * weight + bias`` for each row of ``x [tokens, width]``.

    ``x`` is bf16, fp16 or fp32 (``y`` has its type), or e4m3 codes with ``scales`` as ``fetch`` returns both:
    ``scales [tokens, width // hidden * ceil(hidden / block)]`` fp32 of either layout, one per ``block`` columns of
    each looked-up row of ``hidden`` columns (default: the width); ``y`` is then ``dtype`` (default bf16).
    ``weight`` and ``bias [width]`` have y's type or are fp32.  ``keep`` says what the backward pass will read:
    nothing (``kept`` is None), ``"exact"`` (``x`` itself, which must stay unchanged) or ``"fp8"``.  Codes of a lookup
    are kept as ``"fp8"`` only: the next fetch reuses their memory.  Autograd does not see this call (tangents of
    forward mode are refused), nor does a trace, which is refused (:func:`layer_norm` is their form).
    """
    return _forward(x, weight, bias, eps, scales, hidden, block, dtype, keep, False)


def layer_norm_backward(dy, kept: KeptRows, weight=None, *, want_dx: bool = True, want_params: bool = True):
    """``(dx, dweight, dbias)`` for the gradient ``dy [tokens, width]`` of ``layer_norm_forward``'s ``y``.

    ``dx`` has dy's type (for looked-up codes it is the gradient of the dequantised rows), ``dweight`` and ``dbias``
    the weight's type; both are None without a ``weight``.  What is not wanted is None and not computed.
    """
    return _native.load().norm_backward(dy, kept.rows, kept.scales, kept.mean, kept.rstd, weight, want_dx, want_params,
                                        getattr(kept, "shift", None))


def check_readout(device=None) -> None:
    """Wait for the device (default: the current one) and raise if a read-out kernel gave up waiting on it.

    Every read-out call raises then too, but it looks when it is made: replays of captured calls report nothing, nor do
    the last calls before their results are used.  Results computed before this returns are good.
    """
    device = torch.device("cuda" if device is None else f"cuda:{device}" if isinstance(device, int) else device)
    if device.type != "cuda":
        raise ValueError("read-out kernels run on GPUs")
    index = torch.cuda.current_device() if device.index is None else device.index
    torch.cuda.synchronize(index)
    _native.load().check_readout(index)


def _adjacent(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _no_code_gradient(x: torch.Tensor):
    if x.dtype == torch.float8_e4m3fn and x.requires_grad:
        raise ValueError("float8_e4m3fn rows get no gradient; layer_norm_backward gives their dequantised rows'")


def _recorded(*tensors) -> bool:
    """Whether autograd has to see a call: a gradient is wanted, a trace records, or forward-mode differentiation
    carries a tangent.

    The kernels' results carry no tangent, which counts as zero (the autograd functions raise instead), and a trace
    takes them as constants (it records an autograd function as one operation).
    """
    given = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given) or torch.jit.is_tracing():
        return True
    # Without an open level there are no tangents (and asking each tensor takes as long as the call).
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in given)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, scales, hidden, block, dtype, keep):
        y, kept = _forward(x, weight, bias, eps, scales, hidden, block, dtype, keep, True)
        ctx.save_for_backward(*kept, kept.shift, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        *kept, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dweight, dbias = layer_norm_backward(_adjacent(dy), KeptRows(*kept), weight,
                                                 want_dx=need[0], want_params=need[1] or need[2])
        return dx, dweight if need[1] else None, dbias if need[2] else None, None, None, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, *, scales=None, hidden=None, block: int = 128, dtype=None,
               keep: str = "fp8"):
    """Differentiable layer norm of ``x [tokens, width]``; the arguments are :func:`layer_norm_forward`'s.

    ``keep`` (``"fp8"``, also for fp32 rows, or ``"exact"``) chooses what is kept for the backward pass; nothing is
    kept where no gradient is wanted.  ``"exact"`` keeps ``x`` itself: rows that ``EngramBuffer.fetch`` returned last
    until the next fetch, after which the backward pass raises (not after the replay of a captured fetch, which nothing
    counts), so take ``"fp8"`` or a copy where fetches run ahead of backward passes.  There is no forward-mode
    derivative (a tangent raises).  Looked-up e4m3 codes get no gradient themselves (:func:`layer_norm_backward` gives
    their rows').
    """
    if _keep_mode(keep) == 0:
        raise ValueError('keep must be "exact" or "fp8"')
    _no_code_gradient(x)
    if _recorded(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, scales, hidden, block, dtype, keep)
    return layer_norm_forward(x, weight, bias, eps, scales=scales, hidden=hidden, block=block, dtype=dtype)[0]
