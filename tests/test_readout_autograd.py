"""The differentiable read-out forms under forward-mode differentiation, tracing and autocast.

A stand-in computes what the kernels do from elementary operations on the CPU.  Like the extension's, its results are
new tensors that autograd knows nothing of: no history, no tangent, and a trace sees them as constants.
"""

import functools
import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.utils.checkpoint

from engram_rdma_lab_b200 import _native, ops
from engram_rdma_lab_b200.models import EngramReadout

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def unseen(function):
    """Run in a thread of its own, where no trace, autocast or gradient mode of the caller reaches."""

    @functools.wraps(function)
    def call(self, *args, **kwargs):
        plain = [a.detach() if isinstance(a, torch.Tensor) else a for a in args]
        result = []

        def work():
            with torch.no_grad():
                result.append(function(self, *plain, **kwargs))

        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        return result[0]

    return call


class StandIn:
    @unseen
    def norm_forward(self, x, weight, bias, eps, scales, hidden, block, dtype, keep, recorded=False):
        mean = x.double().mean(1, keepdim=True)
        rstd = 1 / torch.sqrt(((x.double() - mean) ** 2).mean(1, keepdim=True) + eps)
        h = (x.double() - mean) * rstd
        y = h if weight is None else h * weight.double()
        y = (y if bias is None else y + bias.double()).to(x.dtype)
        codes, code_scales = ops.quantize_fp8_blockwise(h.float(), power_of_two=True) if keep == 2 else (None, None)
        exact = keep == 1
        return (y, codes, code_scales, mean[:, 0].float() if exact else None, rstd[:, 0].float() if keep else None,
                torch.zeros(len(x)) if exact else None)

    @unseen
    def norm_backward(self, dy, rows, scales, mean, rstd, weight, want_dx, want_params, shift):
        if weight is not None and weight.dtype not in (dy.dtype, FP32):
            raise ValueError("weight must have the rows' type or float32")
        r = rstd.double()[:, None]
        h = (rows.double() - mean.double()[:, None]) * r if scales is None else self.rows(rows, scales)
        g = dy.double() if weight is None else dy.double() * weight.double()
        dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        parameters = want_params and weight is not None
        return (dx.to(dy.dtype) if want_dx else None, (dy.double() * h).sum(0).to(weight.dtype) if parameters else None,
                dy.double().sum(0).to(weight.dtype) if parameters else None)

    @staticmethod
    def rows(codes, scales):
        return codes.double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]

    @unseen
    def save_fp8(self, x, recorded=False):
        return ops.quantize_fp8_blockwise(x.float(), power_of_two=True)

    @unseen
    def fp8_weight_grad(self, dy, codes, scales, norm_weight, norm_bias, dtype, want_bias):
        x = self.rows(codes, scales)
        if norm_weight is not None:
            x = x * norm_weight.double()
        if norm_bias is not None:
            x = x + norm_bias.double()
        out = dtype or dy.dtype
        return (dy.double().t() @ x).to(out), dy.double().sum(0).to(out) if want_bias else None


@pytest.fixture(autouse=True)
def stand_in(monkeypatch):
    native = StandIn()
    monkeypatch.setattr(_native, "load", lambda: native)


def randn(seed, *shape, dtype=FP32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def leaves(dtype=FP32, out=24, width=256, norm=None):
    """x, norm weight and bias, projection weight and bias."""
    norm = norm or dtype
    return (randn(1, 10, width, dtype=dtype), 1 + randn(2, width, dtype=norm) / 4, randn(3, width, dtype=norm),
            randn(4, out, width, dtype=dtype) / 8, randn(5, out, dtype=dtype))


FORMS = {
    "layer_norm": (lambda x, nw, nb, w, b: ops.layer_norm(x, nw, nb), (0, 1, 2)),
    "layer_norm exact": (lambda x, nw, nb, w, b: ops.layer_norm(x, nw, nb, keep="exact"), (0, 1, 2)),
    "norm_linear": (ops.norm_linear, (0, 1, 2, 3, 4)),
}


# ---------------------------------------------------------------- forward mode
@pytest.mark.parametrize("grad", ["no grad", "grad", "required"])
@pytest.mark.parametrize("form", FORMS)
def test_a_tangent_is_refused_and_not_dropped(form, grad):
    call, arguments = FORMS[form]
    for k in arguments:
        values = list(leaves())
        with forward_ad.dual_level(), torch.set_grad_enabled(grad != "no grad"):
            values[k] = forward_ad.make_dual(values[k], torch.ones_like(values[k]))
            if grad == "required":
                values = [v if j == k else v.requires_grad_() for j, v in enumerate(values)]
            with pytest.raises(NotImplementedError, match="jvp"):
                call(*values)


@pytest.mark.parametrize("form", FORMS)
def test_calls_without_a_tangent_run_while_a_level_is_open(form):
    call, _ = FORMS[form]
    want = call(*leaves())
    with forward_ad.dual_level():
        assert torch.equal(call(*leaves()), want)


def test_linear_carries_tangents():
    """Nothing is kept where no gradient is wanted: a plain product, which forward mode differentiates."""
    x, _, _, w, b = leaves()
    tangent = randn(7, *x.shape)
    with forward_ad.dual_level():
        y = ops.linear(forward_ad.make_dual(x, tangent), w, b)
        torch.testing.assert_close(forward_ad.unpack_dual(y).tangent, tangent @ w.t())


# ---------------------------------------------------------------- tracing
@pytest.mark.filterwarnings("ignore::DeprecationWarning", "ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_a_trace_computes_with_its_own_inputs(form, grad):
    call, _ = FORMS[form]
    first = [t.requires_grad_(grad) for t in leaves()]
    if grad and form != "norm_linear":  # torch traces no function whose result is new to it and requires grad
        with pytest.raises(RuntimeError, match="constant"):
            torch.jit.trace(call, first, check_trace=False)
        return
    traced = torch.jit.trace(call, first, check_trace=False)
    other = [2 + t.detach() * 3 for t in leaves()]
    assert torch.equal(traced(*other), call(*other))


# ---------------------------------------------------------------- autocast
@pytest.mark.parametrize("dtype,other", [(FP32, BF16), (BF16, FP16), (FP16, BF16)])
@pytest.mark.parametrize("form", ["linear", "norm_linear"])
def test_gradients_do_not_depend_on_where_backward_runs(form, dtype, other):
    """A backward pass inside the region computes what it does outside: products in the parameters' type."""
    def gradients(inside):
        x, nw, nb, w, b = (t.requires_grad_() for t in leaves(dtype))
        used = (x, w, b) if form == "linear" else (x, nw, nb, w, b)
        with torch.autocast("cpu", other):
            z = ops.linear(x, w, b) if form == "linear" else ops.norm_linear(x, nw, nb, w, b)
            assert z.dtype == other
            if inside:
                return torch.autograd.grad(z, used, randn(9, *z.shape, dtype=other))
        return torch.autograd.grad(z, used, randn(9, *z.shape, dtype=other))

    for a, c in zip(gradients(True), gradients(False)):
        assert a.dtype == c.dtype == dtype and torch.equal(a, c)


@pytest.mark.parametrize("form", [*FORMS, "linear"])
def test_recomputed_under_activation_checkpointing(form):
    call = FORMS[form][0] if form in FORMS else lambda x, nw, nb, w, b: ops.linear(x, w, b)
    results = []
    for recompute in (False, True):
        values = [t.requires_grad_() for t in leaves()]
        z = torch.utils.checkpoint.checkpoint(call, *values, use_reentrant=False) if recompute else call(*values)
        z.backward(randn(9, *z.shape))
        results.append([t.grad for t in values])
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(*results))


# ---------------------------------------------------------------- the module
@pytest.mark.parametrize("rows", [BF16, FP16, FP32])
def test_a_readout_with_fp32_parameters_takes_16_bit_rows(rows):
    """The rows' values are exact in fp32: parameters and result have the module's type."""
    torch.manual_seed(1)
    readout = EngramReadout(64, 4, 24, bias=True, dtype=FP32)
    x = randn(1, 10, 256, dtype=rows).requires_grad_()
    z = readout(x)
    parameters = list(readout.parameters())
    want = ops.norm_linear(x.detach().float(), *parameters[:4])
    assert z.dtype == FP32 and torch.equal(z, want)
    dz = randn(2, *z.shape)
    got = torch.autograd.grad(z, [x, *parameters], dz)
    assert got[0].dtype == rows and all(torch.equal(a, c) for a, c in zip(got[1:], torch.autograd.grad(want, parameters, dz)))
    with torch.autocast("cpu", BF16):
        assert readout(x).dtype == BF16


def test_a_readout_refuses_rows_that_its_type_cannot_hold():
    with pytest.raises(ValueError, match="rows' type"):
        EngramReadout(64, 4, 24, dtype=FP16)(randn(1, 10, 256, dtype=BF16))
    with pytest.raises(ValueError, match="rows' type"):
        EngramReadout(64, 4, 24, dtype=BF16)(randn(1, 10, 256))
    with pytest.raises(ValueError):
        EngramReadout(64, 4, 24, dtype=FP32)(randn(1, 10, 256).to(torch.float8_e4m3fn))
