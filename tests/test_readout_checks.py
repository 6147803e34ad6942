"""Argument checks of the read-out operators beyond test_readout_refusals.py (no GPU is touched)."""

import copy
import pickle

import pytest
import torch

from engram_rdma_lab_b200 import _native
from engram_rdma_lab_b200.ops import KeptRows, check_readout, fp8_weight_grad, layer_norm_backward, layer_norm_forward, restore_fp8, save_fp8

pytestmark = pytest.mark.skipif(not _native.available(), reason="extension not built")


@pytest.mark.parametrize("shift", [torch.zeros(3), torch.zeros(4, 1), torch.zeros(4).double(), torch.zeros(8)[::2]])
def test_the_second_part_of_a_mean_is_checked(shift):
    x = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="shift must be"):
        layer_norm_backward(x, KeptRows(x, None, torch.zeros(4), torch.ones(4), shift))


@pytest.mark.filterwarnings("ignore::DeprecationWarning", "ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("call", [
    lambda x: layer_norm_forward(x)[0],
    lambda x: layer_norm_backward(x, KeptRows(x, None, x[:, 0].contiguous(), x[:, 0].contiguous()))[0],
    lambda x: save_fp8(x)[1],
    lambda x: restore_fp8(x.to(torch.float8_e4m3fn), torch.ones(4, 2)),
    lambda x: fp8_weight_grad(x, x.to(torch.float8_e4m3fn), torch.ones(4, 2))[0],
])
def test_a_trace_is_refused(call):
    """A trace would not see the call and keep its result as a constant."""
    with pytest.raises(RuntimeError, match="constant"):
        torch.jit.trace(call, (torch.zeros(4, 256),), check_trace=False)


def test_a_check_of_another_kind_of_device():
    with pytest.raises(ValueError, match="on GPUs"):
        check_readout("cpu")


def test_kept_rows_are_four_and_carry_the_rest_of_the_mean():
    """They unpack as (rows, scales, mean, rstd); copies have what is beside the four, a tuple of the four has none."""
    kept = KeptRows(torch.ones(4, 8), None, torch.zeros(4), torch.ones(4), torch.full((4,), 2.0))
    rows, scales, mean, rstd = kept
    assert rows is kept.rows and scales is None and mean is kept.mean and rstd is kept.rstd
    for same in (copy.copy(kept), copy.deepcopy(kept), pickle.loads(pickle.dumps(kept))):
        assert torch.equal(same.shift, kept.shift) and torch.equal(same.rows, rows) and len(same) == 4
    assert KeptRows(*kept).shift is None and kept._replace(rstd=mean).shift is None
