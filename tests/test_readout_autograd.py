"""The differentiable read-out forms under forward-mode differentiation, tracing and autocast.

A stand-in computes what the kernels do from elementary operations on the CPU.  Like the extension's, its results are
new tensors that autograd knows nothing of: no history, no tangent, and a trace sees them as constants.
"""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from engram_rdma_lab_b200 import _native, ops

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


class StandIn:
    @staticmethod
    def _new(t):
        return None if t is None else torch.frombuffer(bytearray(t.detach().contiguous().view(torch.uint8).numpy().tobytes()),
                                                       dtype=t.dtype).view(t.shape)

    def norm_forward(self, x, weight, bias, eps, scales, hidden, block, dtype, keep):
        with torch.no_grad():
            x = x.detach()
            mean = x.double().mean(1, keepdim=True)
            rstd = 1 / torch.sqrt(((x.double() - mean) ** 2).mean(1, keepdim=True) + eps)
            h = (x.double() - mean) * rstd
            y = h if weight is None else h * weight.detach().double()
            y = (y if bias is None else y + bias.detach().double()).to(x.dtype)
            codes, code_scales = self.save_fp8(h) if keep == 2 else (None, None)
            exact = keep == 1
            return (self._new(y), codes, code_scales, self._new(mean[:, 0].float()) if exact else None,
                    self._new(rstd[:, 0].float()) if keep else None, torch.zeros(len(x)) if exact else None)

    def norm_backward(self, dy, rows, scales, mean, rstd, weight, want_dx, want_params, shift):
        assert weight is None or weight.dtype in (dy.dtype, FP32)
        with torch.no_grad():
            n = dy.shape[1]
            r = rstd.double()[:, None]
            h = (rows.double() - mean.double()[:, None]) * r if scales is None else self._rows(rows, scales)
            g = dy.double() if weight is None else dy.double() * weight.detach().double()
            dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).sum(1, keepdim=True) / n)
            parameters = want_params and weight is not None
            return (self._new(dx.to(dy.dtype)) if want_dx else None,
                    self._new((dy.double() * h).sum(0).to(weight.dtype)) if parameters else None,
                    self._new(dy.double().sum(0).to(weight.dtype)) if parameters else None)

    @staticmethod
    def _rows(codes, scales):
        return codes.double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]

    def save_fp8(self, x):
        codes, scales = ops.quantize_fp8_blockwise(x.detach().float(), power_of_two=True)
        return codes, self._new(scales)

    def fp8_weight_grad(self, dy, codes, scales, norm_weight, norm_bias, dtype, want_bias):
        with torch.no_grad():
            x = self._rows(codes, scales)
            if norm_weight is not None:
                x = x * norm_weight.detach().double()
            if norm_bias is not None:
                x = x + norm_bias.detach().double()
            dy64 = dy.detach().double()
            out = dtype or dy.dtype
            return self._new((dy64.t() @ x).to(out)), self._new(dy64.sum(0).to(out)) if want_bias else None


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
