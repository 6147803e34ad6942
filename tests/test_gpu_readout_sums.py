"""Sums of the weight gradient: every bit of a gradient counts, over one row and over very many."""

import pytest
import torch

from engram_rdma_lab_b200.ops import fp8_weight_grad, save_fp8

from .test_gpu_readout import BF16, FP16, FP32, U, _gpu, checkpoint, close, params, randn, rounded, weight_grad_exact  # noqa: F401

pytestmark = pytest.mark.gpu


def exact_rows(codes, scales):
    return codes.double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_weight_grad_of_one_row_is_the_products(dtype):
    """One row times powers of two: every bit of dy has to arrive, for a result with room for it."""
    n, out = 256, 264
    x = torch.exp2(torch.randint(-6, 9, (1, n), device="cuda").float())
    codes, scales = save_fp8(x)
    bits = torch.randint(0, 1 << 23, (1, out), device="cuda", dtype=torch.int32)
    dy = ((127 << 23) + bits | 1).view(FP32).to(dtype)  # fp32: all 24 bits, the last one set
    want = dy.double().t() @ exact_rows(codes, scales)
    got, sums = fp8_weight_grad(dy, codes, scales, dtype=FP32)
    assert torch.equal(got.double(), want) and torch.equal(sums.double(), dy.double()[0])


@pytest.mark.parametrize("dtype", [FP16, FP32])
@pytest.mark.parametrize("m", [256, 512])
def test_weight_grad_holds_all_terms_of_a_gradient(m, dtype):
    """The last terms go through m / 16 additions into an accumulator that grows as a square root (2/3 of its last
    size on average); a cut takes U of it on average.  The smaller terms before them add 2^-7 of that.  A dropped
    third term of fp32 would cost ~5e-6, the largest term first 2.5e-6, a dropped second term of fp16 1e-3."""
    codes, scales = save_fp8(randn(m, m, 1000))
    dy = randn(m + 1, m, 700, dtype=dtype)
    want = dy.double().t() @ exact_rows(codes, scales)
    got, _ = fp8_weight_grad(dy, codes, scales, dtype=FP32)
    assert (got.double() - want).norm() <= 1.02 * (m / 16) * U * 2 / 3 * want.norm()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("signs", ["one", "both"])
@pytest.mark.parametrize("m,n,out", [(8192, 256, 136), (262_144, 256, 264)])
def test_weight_grad_of_very_many_rows(m, n, out, signs, dtype):
    """An accumulator of an fp32 result takes 2048 rows of fp32 or 4096 of bf16, 16 at a time (those of smaller terms of
    dy before add 2^-7 of it), before it is rounded into the sum of its like.  A cut is U of the accumulator on average, which grows linearly
    (1/2 of its last size on average) where all terms have one sign, as a square root (2/3) otherwise; joining p
    parts rounds p times, half a U each."""
    x, dy = randn(m, m, n), randn(m + 1, m, out)
    if signs == "one":
        x, dy = x.abs(), dy.abs()
    codes, scales = save_fp8(x)
    dy = dy.to(dtype)
    rows, want = exact_rows(codes, scales), 0
    for at in range(0, m, 65536):
        want = want + dy[at:at + 65536].double().t() @ rows[at:at + 65536]
    got, sums = fp8_weight_grad(dy, codes, scales, dtype=FP32)
    most = 2048 if dtype == FP32 else 4096
    bound = 1.02 * (most / 16) * U * (1 / 2 if signs == "one" else 2 / 3) + m / most / 2 * U
    assert (got.double() - want).norm() <= bound * want.norm()
    # Column sums of dy: 32 parts of m / 32 rows by eight warps, then 8 + 32 additions.
    total = dy.double().sum(0)
    close(sums, total, (m / 256 + 40) * U * dy.double().abs().sum(0) + rounded(total, FP32), "dbias")


@pytest.mark.parametrize("n", [12288, 12290])  # rows of the result on 16-byte boundaries, and not
def test_weight_grad_of_many_rows_into_a_wide_result(n):
    """Parts of the rows whose results would fill gigabytes side by side are joined a few at a time, with the norm
    folded in once."""
    m, out = 33_000, 2048
    codes, scales = save_fp8(randn(1, m, n))
    dy = randn(2, m, out, dtype=FP32)
    w, b = params(n, FP32)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got, _ = fp8_weight_grad(dy, codes, scales, w, b)
    torch.cuda.synchronize()
    planes, results = 3 * m * out * 2, out * n * 4
    assert torch.cuda.max_memory_allocated() - before <= planes + results + (512 << 20) + (16 << 20)
    rows = exact_rows(codes, scales).mul_(w.double()).add_(b.double())
    want = dy.double().t() @ rows
    bound = 1.02 * 128 * U * 2 / 3 + (m / 2048 + 4) * U
    assert (got.double() - want).norm() <= bound * want.norm()
    assert torch.equal(got, fp8_weight_grad(dy, codes, scales, w, b)[0])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m", [8191, 8193, 20_000])  # one accumulator, and several
def test_weight_grad_of_many_rows_in_16_bits(m, dtype):
    codes, scales = checkpoint(m, m, 1040)
    dy = randn(m + 1, m, 520, dtype=dtype)
    w, b = params(1040, dtype)
    (want, t), (sums, tb) = weight_grad_exact(dy, codes, scales, w, b)
    dw, db = fp8_weight_grad(dy, codes, scales, w, b)
    close(dw, want, t + rounded(want, dtype), "dweight")
    close(db, sums, tb + rounded(sums, dtype), "dbias")
    assert torch.equal(dw, fp8_weight_grad(dy, codes, scales, w, b)[0])
