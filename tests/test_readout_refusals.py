"""Arguments that the read-out operators refuse (before any device is touched, so this needs no GPU)."""

import pytest
import torch

from engram_rdma_lab_b200 import _native
from engram_rdma_lab_b200.models import EngramReadout
from engram_rdma_lab_b200.ops import (
    KeptRows,
    fp8_weight_grad,
    layer_norm,
    layer_norm_backward,
    layer_norm_forward,
    linear,
    norm_linear,
    restore_fp8,
    save_fp8,
)

pytestmark = pytest.mark.skipif(not _native.available(), reason="extension not built")

F8 = torch.float8_e4m3fn


def rows(m=4, n=256, dtype=torch.bfloat16):
    return torch.zeros(m, n).to(dtype)


def codes(m=4, n=256):
    return torch.zeros(m, n).to(F8)


def scales(m=4, n=2):
    return torch.ones(m, n)


@pytest.mark.parametrize("call,message", [
    (lambda: layer_norm_forward(torch.zeros(4)), "rows must be"),
    (lambda: layer_norm_forward(torch.zeros(4, 0)), "rows must be"),
    (lambda: layer_norm_forward(rows().t()), "adjacent columns"),
    (lambda: layer_norm_forward(rows(dtype=torch.float64)), "bfloat16, float16, float32"),
    (lambda: layer_norm_forward(rows(dtype=torch.int32)), "bfloat16, float16, float32"),
    (lambda: layer_norm_forward(rows(), dtype=torch.float32), "dtype can be chosen"),
    (lambda: layer_norm_forward(rows(), hidden=64), "hidden describes"),
    (lambda: layer_norm_forward(rows(), scales=scales()), "need scales"),
    (lambda: layer_norm_forward(codes()), "need scales"),
    (lambda: layer_norm_forward(codes(), scales=scales(), hidden=96), "hidden must divide"),
    (lambda: layer_norm_forward(codes(), scales=scales(), hidden=0), "hidden must divide"),
    (lambda: layer_norm_forward(codes(), scales=scales(4, 3)), "scales must be float32"),
    (lambda: layer_norm_forward(codes(), scales=scales(3, 2)), "scales must be float32"),
    (lambda: layer_norm_forward(codes(), scales=scales().double()), "scales must be float32"),
    (lambda: layer_norm_forward(codes(), scales=scales(), block=0), "block must be positive"),
    (lambda: layer_norm_forward(codes(), scales=scales(), dtype=F8), "dtype must be"),
    (lambda: layer_norm_forward(codes(), scales=scales(), keep="exact"), "kept as"),
    (lambda: layer_norm_forward(rows(), keep="all"), "keep must be"),
    (lambda: layer_norm_forward(rows(), keep=["fp8"]), "keep must be"),
    (lambda: layer_norm_forward(rows(), eps=-1e-5), "eps must not be negative"),
    (lambda: layer_norm_forward(rows(), eps=float("nan")), "eps must not be negative"),
    (lambda: layer_norm_forward(rows(), None, torch.zeros(256)), "a bias needs a weight"),
    (lambda: layer_norm_forward(rows(), torch.zeros(255)), "weight must be contiguous"),
    (lambda: layer_norm_forward(rows(), torch.zeros(1).expand(256)), "weight must be contiguous"),
    (lambda: layer_norm_forward(rows(), torch.zeros(256).half()), "weight must have"),
    (lambda: layer_norm_forward(rows(), torch.zeros(256), torch.zeros(256).bfloat16()), "bias must be"),
    (lambda: layer_norm_forward(rows()), "on a GPU"),
    (lambda: layer_norm(rows(), keep=None), "keep must be"),
    (lambda: layer_norm(codes().requires_grad_(), scales=scales()), "get no gradient"),
    (lambda: norm_linear(codes().requires_grad_(), None, None, rows(8), scales=scales()), "get no gradient"),
    (lambda: layer_norm_backward(rows(), KeptRows(rows(3), None, torch.zeros(3), torch.zeros(3))), "shape of the kept rows"),
    (lambda: layer_norm_backward(rows(dtype=torch.float16), KeptRows(rows(), None, torch.zeros(4), torch.zeros(4))), "rows' type"),
    (lambda: layer_norm_backward(rows(), KeptRows(rows(), None, None, torch.zeros(4))), "mean must be"),
    (lambda: layer_norm_backward(rows(), KeptRows(rows(), None, torch.zeros(4), torch.zeros(3))), "rstd must be"),
    (lambda: layer_norm_backward(rows(), KeptRows(codes(), scales(4, 1), None, torch.zeros(4))), "scales must be"),
    (lambda: layer_norm_backward(rows(), KeptRows(rows(), scales(), None, torch.zeros(4))), "codes must be float8"),
    (lambda: layer_norm_backward(codes(), KeptRows(codes(), scales(), None, torch.zeros(4))), "dy must be"),
    (lambda: layer_norm_backward(rows(1).t(), KeptRows(codes(256, 1), scales(256, 1), None, torch.zeros(256))), "on a GPU"),
    (lambda: layer_norm_backward(torch.zeros(4, 1).expand(4, 256), KeptRows(codes(), scales(), None, torch.zeros(4))), "adjacent"),
    (lambda: save_fp8(torch.zeros(4)), "activations must be"),
    (lambda: save_fp8(rows(dtype=torch.int8)), "activations must be"),
    (lambda: save_fp8(rows().t()), "adjacent columns"),
    (lambda: save_fp8(rows()), "on a GPU"),
    (lambda: restore_fp8(rows(), scales()), "codes must be float8"),
    (lambda: restore_fp8(codes(), scales(4, 3)), "scales must be"),
    (lambda: restore_fp8(codes(), scales(), torch.float64), "dtype must be"),
    (lambda: restore_fp8(codes(), scales()), "on a GPU"),
    (lambda: fp8_weight_grad(rows(3, 8), codes(), scales()), "same rows"),
    (lambda: fp8_weight_grad(codes(4, 8), codes(), scales()), "dy must be"),
    (lambda: fp8_weight_grad(rows(4, 8), codes(), scales(), dtype=torch.float16), "dtype must be"),
    (lambda: fp8_weight_grad(rows(4, 8), codes(), scales(), None, torch.zeros(256)), "a bias needs"),
    (lambda: fp8_weight_grad(rows(4, 8), codes(), scales(), torch.zeros(8)), "weight must be contiguous"),
    (lambda: fp8_weight_grad(rows(4, 8), codes(), scales()), "on a GPU"),
    (lambda: linear(rows(), rows(8, 128)), "expected rows"),
    (lambda: linear(rows(), rows(8, dtype=torch.float32)), "must have the rows' type"),
    (lambda: norm_linear(rows(), None, None, rows(8), torch.zeros(7).bfloat16()), "must have the rows' type"),
    (lambda: EngramReadout(64, 0, 8), "must be positive"),
])
def test_refusals(call, message):
    with pytest.raises(ValueError, match=message):
        call()


def test_readout_module_parameters():
    readout = EngramReadout(64, 4, 24, bias=True)
    shapes = {name: tuple(p.shape) for name, p in readout.named_parameters()}
    assert shapes == {"norm_weight": (256,), "norm_bias": (256,), "weight": (24, 256), "bias": (24,)}
    with pytest.raises(ValueError, match="expected rows"):
        readout(rows(4, 128))
