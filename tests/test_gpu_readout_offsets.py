"""Layer norm of fp32 rows whose offset is thousands of times their deviation, against 64 bits.

The rows are 4096 + N(0, 1).  ``x - m`` is exact for a first mean ``m`` (two fp32 values within a factor of two), and
what ``m`` is off by comes back as the mean of ``x - m``, a sum of values of the deviation's size.  So a normalised
value is off by a few U of a deviation.  Rounding the corrected mean to one fp32 number instead costs up to 2^-12,
half a step at 4096, in every value of a row.
"""

import pytest

from engram_rdma_lab_b200.ops import layer_norm_forward

from .test_gpu_readout import DEPTH, EPS, FP32, U, _gpu, close, norm_exact, params, randn, rounded  # noqa: F401

pytestmark = pytest.mark.gpu

# A warp, a block and single elements per row, and rows that are read more than once.
WIDTHS = [256, 6144, 4097, 12290, 20001]


def rows_far_from_zero(m, n):
    return 4096 + randn(n, m, n)


def h_tolerance(x, h, rstd):
    """The correction is a sum of x - m (|x - m| is at most the deviation and m's own error, DEPTH U 4100 < .03), one
    more rounding takes it off, and rstd is half of what its sum of squares is off by, and a few U."""
    d = (x.double() - x.double().mean(1, keepdim=True)).abs()
    return rstd[:, None] * (DEPTH * U * (d.mean(1, keepdim=True) + 0.03) + 4 * U * d) + (DEPTH / 2 + 8) * U * h.abs()


@pytest.mark.parametrize("n", WIDTHS)
def test_forward_of_rows_far_from_zero(n):
    x = rows_far_from_zero(16, n)
    w, b = params(n, FP32)
    want, h, _, rstd = norm_exact(x, w, b)
    y, _ = layer_norm_forward(x, w, b, EPS)
    t = h_tolerance(x, h, rstd) * w.double().abs() + 2 * U * ((h * w.double()).abs() + b.double().abs())
    close(y, want, t + rounded(want, FP32), "y")
