"""Read-out operators at the ends of fp32."""

import pytest
import torch

from engram_rdma_lab_b200.ops import layer_norm_forward, restore_fp8

from .test_gpu_readout import FP32, _gpu, randn  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- infinities
# Whole chunks in a warp and in a block, single elements in a warp and in a block, rows read more than once.
@pytest.mark.parametrize("n", [256, 1024, 16384, 100, 1001, 16400, 20001])
@pytest.mark.parametrize("eps", [0.0, 1e-60])
def test_infinite_normalised_values_are_kept_as_nan(n, eps):
    """A row whose squares underflow has variance 0 and, without eps, infinite normalised values.  The format keeps
    what is not finite as NaN and leaves a block without finite values at scale 1."""
    x = randn(n, 3, n)
    x[1] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 1e-30, -1e-30)
    y, kept = layer_norm_forward(x, None, None, eps, keep="fp8")
    assert torch.isinf(kept.rstd[1]) and not torch.isfinite(y[1]).any()
    assert restore_fp8(kept.rows, kept.scales, FP32)[1].isnan().all()
    assert torch.equal(kept.scales[1], torch.ones_like(kept.scales[1]))
    for r in (0, 2):
        assert torch.isfinite(y[r]).all() and torch.isfinite(restore_fp8(kept.rows, kept.scales, FP32)[r]).all()
