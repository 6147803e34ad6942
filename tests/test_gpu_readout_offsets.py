"""Layer norm of fp32 rows whose offset is thousands of times their deviation, against 64 bits.

The rows are 4096 + N(0, 1).  ``x - m`` is exact for a first mean ``m`` (two fp32 values within a factor of two), and
what ``m`` is off by comes back as the mean of ``x - m``, a sum of values of the deviation's size.  So a normalised
value is off by a few U of a deviation.  Rounding the corrected mean to one fp32 number instead costs up to 2^-12,
half a step at 4096, in every value of a row.
"""

import pytest
import torch

from engram_rdma_lab_b200.ops import KeptRows, layer_norm, layer_norm_backward, layer_norm_forward

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


@pytest.mark.parametrize("n", WIDTHS)
def test_backward_of_exact_rows_far_from_zero(n):
    m = 64
    x, dy = rows_far_from_zero(m, n), randn(n + 1, m, n)
    w, b = params(n, FP32)
    _, h, _, rstd = norm_exact(x, w, b)
    th = h_tolerance(x, h, rstd)
    _, kept = layer_norm_forward(x, w, b, EPS, keep="exact")
    dx, dw, db = layer_norm_backward(dy, kept, w)
    g = dy.double() * w.double()
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    t1 = DEPTH * U * g.abs().mean(1, keepdim=True)
    t2 = DEPTH * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * th).mean(1, keepdim=True)
    want = rstd[:, None] * (g - c1 - h * c2)
    t = rstd[:, None] * (t1 + t2 * h.abs() + th * c2.abs() + 6 * U * (g.abs() + c1.abs() + (h * c2).abs()))
    close(dx, want, t + (DEPTH / 2 + 8) * U * want.abs() + rounded(want, FP32), "dx")
    # A column's sum: no term goes through more additions than there are rows.
    dy64, want = dy.double(), (dy.double() * h).sum(0)
    t = (dy64.abs() * (th + 2 * U * h.abs())).sum(0) + m * U * (dy64 * h).abs().sum(0)
    close(dw, want, t + rounded(want, FP32), "dweight")
    close(db, dy64.sum(0), m * U * dy64.abs().sum(0) + rounded(dy64.sum(0), FP32), "dbias")


def test_autograd_reads_what_the_forward_pass_kept():
    x, dy = rows_far_from_zero(20, 1000), randn(3, 20, 1000)
    w, b = params(1000, FP32)
    _, kept = layer_norm_forward(x, w, b, EPS, keep="exact")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(layer_norm(*leaves, EPS, keep="exact"), leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(got, layer_norm_backward(dy, kept, w)))


def test_a_single_mean_per_row_still_serves():
    """Statistics of another origin: rows, one fp32 mean and one rstd per row."""
    x, dy = randn(1, 30, 768), randn(2, 30, 768)
    w, _ = params(768, FP32)
    _, h, mean, rstd = norm_exact(x)
    kept = KeptRows(x, None, mean.float(), rstd.float())
    dx, dw, _ = layer_norm_backward(dy, kept, w)
    # x - mean: the mean's rounding and the difference's, 2 U of 8 (no value is larger), rstd's rounding and the product's.
    dh = 16 * U * rstd[:, None] + 4 * U * h.abs()
    dy64 = dy.double()
    t = (dy64.abs() * dh).sum(0) + 30 * U * (dy64 * h).abs().sum(0)
    close(dw, (dy64 * h).sum(0), t + rounded((dy64 * h).sum(0), FP32), "dweight")
    assert torch.isfinite(dx).all()
