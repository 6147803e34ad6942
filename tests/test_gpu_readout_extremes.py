"""Read-out operators at the ends of fp32."""

import pytest
import torch

from engram_rdma_lab_b200.ops import layer_norm_forward, restore_fp8

from .test_gpu_readout import BF16, F8, FP16, FP32, _gpu, params, randn  # noqa: F401

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


@pytest.mark.parametrize("n", [256, 1024, 100, 1001, 20001])
def test_rows_whose_variance_is_beyond_fp32_give_no_finite_garbage(n):
    """Squares past 3.4e38: the variance is infinite (rstd 0, y the bias) or, where its correction overflows as well,
    unknown, and then the row is NaN; it is never computed with rstd = 1 / sqrt(eps)."""
    x = torch.stack([randn(n, n) * 1e20, 1e30 * (1 + randn(n + 1, n).abs() / 16), randn(n + 2, n)])
    w, b = params(n, FP32)
    y, kept = layer_norm_forward(x, w, b, keep="exact")
    for r in (0, 1):
        assert y[r].isnan().all() or torch.equal(y[r], b)
        assert kept.rstd[r].isnan() or kept.rstd[r] == 0
    assert torch.isfinite(y[2]).all()


@pytest.mark.parametrize("n", [256, 1000])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_restore_keeps_infinite_values_infinite(n, dtype):
    """Scales of another origin may be infinite: their values are infinities (NaN for codes of zero), while finite
    values past the type's range become its largest."""
    codes = torch.ones(3, n, device="cuda").to(F8)
    codes[:, 1], codes[:, 2] = torch.tensor(-2.0).to(F8), torch.tensor(0.0).to(F8)
    scales = torch.ones(3, -(-n // 128), device="cuda")
    scales[1, 0], scales[2] = float("inf"), 2.0 ** 127
    x = restore_fp8(codes, scales, dtype)
    assert torch.isposinf(x[1, 0]) and torch.isneginf(x[1, 1]) and x[1, 2].isnan() and torch.isinf(x[1, 3:128]).all()
    assert torch.isfinite(x[0]).all() and torch.isfinite(x[1, 128:]).all() and torch.isfinite(x[2]).all()
    assert x[2, 1] == (-torch.finfo(dtype).max)
