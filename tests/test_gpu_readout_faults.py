"""How a read-out kernel's given-up wait is reported.  No wait runs out here: the word that a kernel would set is set
from the host."""

import pytest
import torch

from engram_rdma_lab_b200 import _native
from engram_rdma_lab_b200.ops import (
    check_readout,
    fp8_weight_grad,
    layer_norm_backward,
    layer_norm_forward,
    restore_fp8,
    save_fp8,
)

from .test_gpu_readout import BF16, _gpu, randn  # noqa: F401

pytestmark = pytest.mark.gpu


def test_every_call_and_the_check_report_it():
    C = _native.load()
    x = randn(1, 4, 256, dtype=BF16)
    codes, scales = save_fp8(x)
    _, kept = layer_norm_forward(x, keep="exact")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = layer_norm_forward(x)
    check_readout()
    calls = [lambda: layer_norm_forward(x), lambda: layer_norm_backward(x, kept), lambda: save_fp8(x),
             lambda: restore_fp8(codes, scales), lambda: fp8_weight_grad(x, codes, scales)]
    assert C.debug_readout_fault(0, 5) == 0
    try:
        for call in (*calls, check_readout, lambda: check_readout(0), lambda: check_readout("cuda:0")):
            with pytest.raises(RuntimeError, match="gave up waiting"):
                call()
        graph.replay()  # a replay runs no host code that could look
        with pytest.raises(RuntimeError, match="gave up waiting"):
            check_readout(torch.device("cuda", 0))
    finally:
        assert C.debug_readout_fault(0, 0) == 5
    check_readout()
    for call in calls:
        call()
