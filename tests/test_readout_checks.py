"""Argument checks of the read-out operators beyond test_readout_refusals.py (no GPU is touched)."""

import pytest
import torch

from engram_rdma_lab_b200 import _native
from engram_rdma_lab_b200.ops import KeptRows, layer_norm_backward

pytestmark = pytest.mark.skipif(not _native.available(), reason="extension not built")


@pytest.mark.parametrize("shift", [torch.zeros(3), torch.zeros(4, 1), torch.zeros(4).double(), torch.zeros(8)[::2]])
def test_the_second_part_of_a_mean_is_checked(shift):
    x = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="shift must be"):
        layer_norm_backward(x, KeptRows(x, None, torch.zeros(4), torch.ones(4), shift))
