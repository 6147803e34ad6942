"""Read-out operators on the GPU against plain implementations in 64 bits.

Tolerances count roundings.  U = 2^-24 is half a step of fp32.  An output is rounded once to its type (half a step,
``eps / 2``), and fp32 intermediates add a few U of the largest term that enters them.  A sum of terms t_i that is
split over lanes and joined as a tree is off by at most DEPTH * U * sum|t_i|, DEPTH the additions a term goes through.
"""

import pytest
import torch

from engram_rdma_lab_b200.models import EngramReadout
from engram_rdma_lab_b200.ops import (
    KeptRows,
    dequantize_fp8_blockwise,
    fp8_weight_grad,
    layer_norm,
    layer_norm_backward,
    layer_norm_forward,
    linear,
    norm_linear,
    quantize_fp8_blockwise,
    restore_fp8,
    save_fp8,
)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    torch.cuda.set_device(0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape, dtype=FP32):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tolerance, what):
    """Every element within its own tolerance (and the same non-finite ones)."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), f"{what}: non-finite values differ"
    worst = ((got - want).abs() - tolerance)[fine]
    assert worst.numel() == 0 or worst.max() <= 0, f"{what}: off by {worst.max():.3g} more than allowed"


def rounded(want, dtype):
    """What one rounding to `dtype` may change: half a step, or half the smallest subnormal."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return want.abs() * half_step(dtype) + tiny


# ---------------------------------------------------------------- 8-bit format
def e4m3_exact(v):
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp_min(-6).double() - 3)
    return torch.round(v / step) * step


def format_exact(x):
    """The 8-bit form of float64 `x`: (values, scales), from the definition."""
    m, n = x.shape
    out, scales = torch.empty_like(x), torch.empty(m, -(-n // 128), dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        part = x[:, b * 128:(b + 1) * 128]
        finite = torch.isfinite(part)
        top = torch.where(finite, part.abs(), 0).amax(1)
        k = torch.full_like(top, -126)
        for e in range(-126, 121):
            k = torch.where(448 * 2.0 ** (e - 1) < top, float(e), k)
        s = torch.where(top > 0, torch.exp2(k), 1)
        scales[:, b] = s
        codes = e4m3_exact(torch.where(finite, part, 0) / s[:, None])
        out[:, b * 128:(b + 1) * 128] = torch.where(finite, codes * s[:, None], torch.nan)
    return out, scales


SIZES = [(1, 1), (1, 128), (3, 129), (5, 127), (2, 16), (33, 1000), (17, 4097), (64, 6144), (9, 12288)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n", SIZES)
def test_save_is_the_format_and_restore_gives_its_values(m, n, dtype):
    x = (randn(m * n, m, n) * torch.exp2(4 * randn(n, m, 1))).to(dtype)
    codes, scales = save_fp8(x)
    want, want_scales = format_exact(x.double())
    assert codes.shape == (m, n) and codes.dtype == F8 and codes.stride(0) % 16 == 0
    assert torch.equal(scales.double(), want_scales)
    values = codes.double() * want_scales.repeat_interleave(128, 1)[:, :n]
    assert torch.equal(values, want)
    for out in (BF16, FP16, FP32):
        assert torch.equal(restore_fp8(codes, scales, out), want.clamp(-torch.finfo(out).max, torch.finfo(out).max).to(out))


def test_save_agrees_with_the_blockwise_quantiser_of_tables():
    x = randn(5, 40, 512, dtype=BF16)
    codes, scales = save_fp8(x)
    want, want_scales = quantize_fp8_blockwise(x, power_of_two=True)
    assert torch.equal(scales, want_scales) and torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(dequantize_fp8_blockwise(codes, scales), restore_fp8(codes, scales))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_save_of_borders_and_non_finite_values(dtype):
    largest, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.zeros(12, 300, device="cuda", dtype=dtype)
    x[1, :200] = largest
    x[2] = least
    x[3] = least * torch.finfo(dtype).eps  # the smallest subnormal
    x[4, 5], x[4, 140] = float("inf"), float("-inf")
    x[4, 6] = 3.0
    x[5, 299] = float("nan")
    x[5, 298] = -7.0
    x[6] = 448.0  # the largest value of scale 1
    x[7] = 449.0 if dtype != BF16 else 450.0
    x[8, :64], x[8, 64:] = 1.0, 2.0 ** -9  # codes that are subnormal
    x[9] = torch.linspace(-464, 464, 300, device="cuda").to(dtype)
    x[10] = float("nan")
    x[11] = -0.0
    codes, scales = save_fp8(x)
    want, want_scales = format_exact(x.double())
    assert torch.equal(scales.double(), want_scales)
    got = restore_fp8(codes, scales, FP32).double()
    want = want.clamp(-torch.finfo(FP32).max, torch.finfo(FP32).max)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    back = restore_fp8(codes, scales, dtype)
    assert torch.isfinite(back[1]).all()  # a largest value that was rounded up comes back as the type's largest


def test_save_reads_strided_rows_and_restore_strided_codes():
    wide = randn(3, 20, 700, dtype=BF16)
    for view in (wide[:, 100:612], wide[::2, 3:260], wide[3:4, :1].expand(6, 1), wide[5].expand(4, 700)):
        codes, scales = save_fp8(view)
        again, again_scales = save_fp8(view.contiguous())
        assert torch.equal(codes.view(torch.uint8), again.view(torch.uint8)) and torch.equal(scales, again_scales)
    packed = again.contiguous()[:, 1:]  # code rows on odd addresses
    col_major = torch.empty(again_scales.shape[1], 4, device="cuda").t().copy_(again_scales)
    want = restore_fp8(again[:, 1:].clone(), again_scales)
    assert torch.equal(restore_fp8(packed, col_major), want)


def test_save_and_restore_of_no_rows():
    codes, scales = save_fp8(torch.empty(0, 200, device="cuda", dtype=BF16))
    assert codes.shape == (0, 200) and scales.shape == (0, 2)
    assert restore_fp8(codes, scales).shape == (0, 200)


def test_offsets_beyond_32_bits():
    m, n = 178_000, 12_288  # 2.19e9 elements
    x = torch.empty(m, n, device="cuda", dtype=BF16)
    x[-3:] = randn(1, 3, n, dtype=BF16)
    codes, scales = save_fp8(x)
    tail, tail_scales = save_fp8(x[-3:].clone())
    assert torch.equal(codes[-3:].view(torch.uint8), tail.view(torch.uint8)) and torch.equal(scales[-3:], tail_scales)
    del codes
    y, kept = layer_norm_forward(x, keep="fp8")
    y_tail, kept_tail = layer_norm_forward(x[-3:].clone(), keep="fp8")
    assert torch.equal(y[-3:], y_tail) and torch.equal(kept.rows[-3:].view(torch.uint8), kept_tail.rows.view(torch.uint8))
    dx, _, _ = layer_norm_backward(x, kept, want_params=False)
    dx_tail, _, _ = layer_norm_backward(x[-3:].clone(), kept_tail, want_params=False)
    assert torch.equal(dx[-3:], dx_tail)


# ---------------------------------------------------------------- layer norm
def norm_exact(x, weight=None, bias=None, eps=EPS):
    """(y, h, mean, rstd) in 64 bits."""
    x = x.double()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / torch.sqrt((d * d).mean(1) + eps)
    h = d * rstd[:, None]
    y = h if weight is None else h * weight.double()
    return (y if bias is None else y + bias.double()), h, mean, rstd


def h_tolerance(x, h, rstd):
    """fp32 error of a normalised value: x - mean is off by a few U of the row's largest |x| (its rounding and the
    mean's; the mean's own sum is corrected by the second pass to within 2 U of it), rstd by 16 U of itself (the
    sum of squares goes through at most ~48 additions of same-signed terms, each half a U on average towards rstd's
    square root, plus the division)."""
    top = x.double().abs().amax(1, keepdim=True)
    return 4 * U * top * rstd[:, None] + 32 * U * h.abs()


def y_tolerance(x, weight, bias, dtype, eps=EPS):
    y, h, _, rstd = norm_exact(x, weight, bias, eps)
    t = h_tolerance(x, h, rstd)
    if weight is not None:
        t = t * weight.double().abs() + 2 * U * (h * weight.double()).abs()
    if bias is not None:
        t = t + 2 * U * bias.double().abs()
    return t + rounded(y, dtype)


def params(n, dtype, seed=7):
    return (1 + 0.3 * randn(seed, n)).to(dtype), (0.3 * randn(seed + 1, n)).to(dtype)


@pytest.mark.parametrize("affine", ["none", "weight", "both", "both fp32"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n", SIZES)
def test_norm_forward(m, n, dtype, affine):
    x = (randn(m + n, m, n) * 3 + randn(n, 1, n)).to(dtype)
    w, b = params(n, FP32 if "fp32" in affine else dtype)
    w, b = (None if affine == "none" else w), (b if "both" in affine else None)
    want, h, mean, rstd = norm_exact(x, w, b)
    tolerance = y_tolerance(x, w, b, dtype)
    y, kept = layer_norm_forward(x, w, b, EPS)
    assert kept is None and y.dtype == dtype
    close(y, want, tolerance, "y")
    y2, kept = layer_norm_forward(x, w, b, EPS, keep="exact")
    assert torch.equal(y, y2) and kept.rows is x
    top = x.double().abs().amax(1)
    close(kept.mean, mean, 4 * U * top, "mean")
    close(kept.rstd, rstd, 32 * U * rstd + 4 * U * top * rstd * rstd * (x.double() - mean[:, None]).abs().amax(1) * rstd, "rstd")
    y3, kept = layer_norm_forward(x, w, b, EPS, keep="fp8")
    assert torch.equal(y, y3)
    check_kept(kept, x, h, rstd)


def check_kept(kept, x, h, rstd):
    """A kept value is the normalised one, off by fp32's error, then by one e4m3 rounding: 2^-4 of itself, or half
    the smallest subnormal step (2^-10) of its scale; the scale is the format's, or its neighbour where the
    block's largest value is within fp32's error of the border."""
    t = h_tolerance(x, h, rstd)
    n = h.shape[1]
    values = restore_fp8(kept.rows, kept.scales, FP32).double()
    scale = kept.scales.double().repeat_interleave(128, 1)[:, :n]
    close(values, h, t + (h.abs() + t) * 2.0 ** -4 + scale * 2.0 ** -10, "kept rows")
    _, want = format_exact(h)
    _, low = format_exact(h.abs() - t)
    _, high = format_exact(h.abs() + t)
    got = kept.scales.double()
    assert ((got == want) | (got == low) | (got == high)).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_norm_forward_of_rows_with_a_large_offset(dtype):
    # fp32 sums of squares would lose all digits of a deviation that is 2^-12 of the offset.
    x = (4096 + randn(3, 6, 6144)).to(dtype)
    want, h, _, rstd = norm_exact(x)
    y, _ = layer_norm_forward(x, None, None, EPS)
    close(y, want, y_tolerance(x, None, None, dtype), "y")


@pytest.mark.parametrize("n", [1, 2, 100, 256, 6144])
def test_norm_of_constant_rows_and_of_one_column(n):
    x = torch.stack([torch.zeros(n), torch.full((n,), 5.0), torch.full((n,), -1e4)]).cuda().to(BF16)
    w, b = params(n, BF16)
    y, kept = layer_norm_forward(x, w, b, EPS, keep="fp8")
    # x equals its mean: at most the mean's rounding, U |x|, times rstd = 1 / sqrt(eps), remains of h.
    tolerance = 2 * U * x.double().abs() * EPS ** -0.5 * w.double().abs() + rounded(b.double().expand(3, n), BF16)
    close(y, b.double().expand(3, n), tolerance, "y")
    assert torch.equal(kept.scales[0], torch.ones_like(kept.scales[0])) and not kept.rows[0].float().any()


def test_non_finite_values_stay_in_their_rows():
    x = randn(4, 5, 6144, dtype=BF16)
    w, b = params(6144, BF16)
    clean, kept_clean = layer_norm_forward(x, w, b, keep="fp8")
    bad = x.clone()
    bad[1, 17], bad[3, 6000] = float("nan"), float("inf")
    y, kept = layer_norm_forward(bad, w, b, keep="fp8")
    for r in (0, 2, 4):
        assert torch.equal(y[r], clean[r]) and torch.equal(kept.rows[r].view(torch.uint8), kept_clean.rows[r].view(torch.uint8))
    assert y[1].isnan().all() and y[3].isnan().all()
    dx, dw, _ = layer_norm_backward(x, kept, w)
    assert torch.isfinite(dx[[0, 2, 4]]).all() and dx[[1, 3]].isnan().all() and dw.isnan().all()


def test_norm_reads_strided_rows():
    wide = randn(9, 12, 2000, dtype=BF16)
    for view in (wide[:, 8:1032], wide[::3, 5:517], wide[4].expand(3, 2000), wide[:, 7:8]):
        w, b = params(view.shape[1], BF16)
        for keep in ("exact", "fp8"):
            y, kept = layer_norm_forward(view, w, b, keep=keep)
            y2, kept2 = layer_norm_forward(view.contiguous(), w, b, keep=keep)
            close(y, norm_exact(view, w, b)[0], y_tolerance(view, w, b, BF16), "y")
            close(y2, norm_exact(view, w, b)[0], y_tolerance(view, w, b, BF16), "y")
            dy = randn(2, *view.shape, dtype=BF16)
            for a, c in zip(layer_norm_backward(dy, kept, w), backward_exact(dy, kept, w)):
                assert a.shape == c[0].shape
                close(a, *c, "gradients")


def lookup(seed, tokens, entries, hidden, block, layout="columns"):
    """e4m3 codes and scales as a fetch returns them, and the rows they stand for (float64)."""
    packs = -(-hidden // block)
    there = torch.rand(tokens, entries, 1, generator=gen(seed + 1), device="cuda") > 0.2
    codes = (randn(seed, tokens, entries, hidden) * there).reshape(tokens, -1).to(F8)
    values = torch.exp2(-torch.randint(0, 9, (tokens, entries, packs), generator=gen(seed + 2), device="cuda").float()) * there
    values = values.reshape(tokens, -1)
    if layout == "columns":
        padded = (tokens + 3) // 4 * 4
        scales = torch.zeros(entries * packs * padded, device="cuda").as_strided(values.shape, (1, padded)).copy_(values)
    else:
        scales = values.contiguous()
    wide = values.view(tokens, entries, packs).repeat_interleave(block, 2)[:, :, :hidden].reshape(tokens, -1)
    return codes, scales, codes.double() * wide.double()


@pytest.mark.parametrize("layout", ["columns", "rows"])
@pytest.mark.parametrize("out", [BF16, FP16, FP32])
@pytest.mark.parametrize("tokens,entries,hidden,block", [
    (1, 24, 256, 128), (7, 24, 256, 128), (5, 4, 64, 128), (3, 3, 144, 128), (2, 5, 80, 16), (6, 24, 512, 128), (4, 1, 16, 128),
    (9, 2, 256, 256), (3, 7, 48, 20), (2, 1, 1001, 128),
])
def test_norm_of_looked_up_codes(tokens, entries, hidden, block, out, layout):
    codes, scales, x = lookup(tokens * hidden, tokens, entries, hidden, block, layout)
    w, b = params(entries * hidden, out)
    want, h, _, rstd = norm_exact(x, w, b)
    y, kept = layer_norm_forward(codes, w, b, EPS, scales=scales, hidden=hidden, block=block, dtype=out, keep="fp8")
    assert y.dtype == out
    close(y, want, y_tolerance(x, w, b, out), "y")
    check_kept(kept, x, h, rstd)


# ---------------------------------------------------------------- backward
DEPTH = 64 + 32  # additions of a row's sum: a thread's own terms of up to 12288 columns, then lanes and warps


def backward_exact(dy, kept, weight):
    """((dx, tolerance), (dweight, tolerance), (dbias, tolerance)) from what was kept, in 64 bits."""
    dy64 = dy.double()
    m, n = dy.shape
    if kept.scales is None:
        mean, rstd = kept.mean.double(), kept.rstd.double()[:, None]
        h = (kept.rows.double() - mean[:, None]) * rstd
        dh = 3 * U * (kept.rows.double().abs() + mean.abs()[:, None]) * rstd + 2 * U * h.abs()
    else:
        rstd = kept.rstd.double()[:, None]
        h = kept.rows.double() * kept.scales.double().repeat_interleave(128, 1)[:, :n]
        dh = torch.zeros_like(h)
    w = torch.ones(n, device="cuda", dtype=torch.float64) if weight is None else weight.double()
    g = dy64 * w
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    t1 = DEPTH * U * g.abs().mean(1, keepdim=True)
    t2 = DEPTH * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * dh).mean(1, keepdim=True)
    dx = rstd * (g - c1 - h * c2)
    t = rstd * (t1 + t2 * h.abs() + dh * c2.abs() + 6 * U * (g.abs() + c1.abs() + (h * c2).abs()))
    out = [(dx, t + rounded(dx, dy.dtype))]
    if weight is not None:
        # A column's sum: at most ~m / 8 + 300 additions in the worst split of the rows.
        depth = m / 8 + 300
        dw, db = (dy64 * h).sum(0), dy64.sum(0)
        tw = (dy64.abs() * (dh + 2 * U * h.abs())).sum(0) + depth * U * (dy64 * h).abs().sum(0)
        out += [(dw, tw + rounded(dw, weight.dtype)), (db, depth * U * dy64.abs().sum(0) + rounded(db, weight.dtype))]
    return out


@pytest.mark.parametrize("params_type", ["none", "same", "fp32"])
@pytest.mark.parametrize("keep", ["exact", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n", SIZES + [(700, 64), (2500, 256), (300, 777), (1500, 6144), (160, 12288)])
def test_norm_backward(m, n, dtype, keep, params_type):
    x = (randn(m + n, m, n) * 2 + randn(n, 1, n)).to(dtype)
    dy = randn(m * 3 + n, m, n, dtype=dtype)
    w, b = params(n, FP32 if params_type == "fp32" else dtype)
    if params_type == "none":
        w = b = None
    _, kept = layer_norm_forward(x, w, b, EPS, keep=keep)
    got = layer_norm_backward(dy, kept, w)
    for name, a, c in zip(("dx", "dweight", "dbias"), got, backward_exact(dy, kept, w)):
        close(a, *c, name)
    if w is None:
        assert got[1] is None and got[2] is None
    else:
        assert got[1].dtype == w.dtype and got[2].dtype == w.dtype
        dx, none1, none2 = layer_norm_backward(dy, kept, w, want_params=False)
        assert torch.equal(dx, got[0]) and none1 is None and none2 is None
        none, dw, db = layer_norm_backward(dy, kept, w, want_dx=False)
        assert none is None
        for name, a, c in zip(("dweight", "dbias"), (dw, db), backward_exact(dy, kept, w)[1:]):
            close(a, *c, name)
    assert all(a is None or torch.equal(a, c) for a, c in zip(got, layer_norm_backward(dy, kept, w)))


def test_norm_backward_of_no_rows():
    x = torch.empty(0, 300, device="cuda", dtype=BF16)
    w, b = params(300, BF16)
    for keep in ("exact", "fp8"):
        y, kept = layer_norm_forward(x, w, b, keep=keep)
        dx, dw, db = layer_norm_backward(x, kept, w)
        assert y.shape == dx.shape == (0, 300) and not dw.any() and not db.any()


def test_norm_backward_reads_strided_gradients():
    x = randn(1, 30, 1024, dtype=BF16)
    w, b = params(1024, BF16)
    _, kept = layer_norm_forward(x, w, b, keep="exact")
    wide = randn(2, 30, 3000, dtype=BF16)
    for dy in (wide[:, 8:1032], wide[:, 3:1027], wide[4, :1024].expand(30, 1024)):
        for a, c in zip(layer_norm_backward(dy, kept, w), backward_exact(dy, kept, w)):
            close(a, *c, "gradients")


def test_norm_gradient_against_differences():
    """<dx, v> + <dw, vw> + <db, vb> against a central difference of L = sum dy * norm(x, w, b) in 64 bits: the
    difference is off by its third-order term, ~step^2, and its rounding, ~2^-53 / step."""
    m, n, step = 6, 500, 1e-5
    x, dy = randn(1, m, n), randn(2, m, n)
    w, b = params(n, FP32)
    v, vw, vb = randn(3, m, n).double(), randn(4, n).double(), randn(5, n).double()
    _, kept = layer_norm_forward(x, w, b, EPS, keep="exact")
    dx, dw, db = layer_norm_backward(dy, kept, w)

    def loss(t):
        return (dy.double() * norm_exact(x.double() + t * v, w.double() + t * vw, b.double() + t * vb)[0]).sum()

    difference = (loss(step) - loss(-step)) / (2 * step)
    terms = [(dx.double() * v), (dw.double() * vw), (db.double() * vb)]
    got = sum(t.sum() for t in terms)
    size = sum(t.abs().sum() for t in terms)
    assert (got - difference).abs() <= 200 * U * size + 1e-7 * size


@pytest.mark.parametrize("keep", ["exact", "fp8"])
def test_layer_norm_autograd(keep):
    m, n = 50, 768
    x = randn(1, m, n, dtype=BF16).requires_grad_()
    w, b = (p.requires_grad_() for p in params(n, BF16))
    dy = randn(3, m, n, dtype=BF16)
    y = layer_norm(x, w, b, EPS, keep=keep)
    assert torch.equal(y, layer_norm_forward(x.detach(), w.detach(), b.detach(), EPS)[0])
    got = torch.autograd.grad(y, (x, w, b), dy)
    _, kept = layer_norm_forward(x.detach(), w.detach(), b.detach(), EPS, keep=keep)
    for a, c in zip(got, layer_norm_backward(dy, kept, w.detach())):
        assert torch.equal(a, c)
    # A broadcast gradient, and leaves that want none.
    (dx,) = torch.autograd.grad(layer_norm(x, w.detach(), None, EPS, keep=keep).sum(), (x,))
    assert torch.equal(dx, layer_norm_backward(torch.ones_like(dy), kept, w.detach(), want_params=False)[0])
    (db,) = torch.autograd.grad(layer_norm(x.detach(), w.detach(), b, EPS, keep=keep), (b,), dy)
    assert torch.equal(db, got[2])
    with torch.no_grad():
        assert not layer_norm(x, w, b, EPS, keep=keep).requires_grad


def test_layer_norm_keeps_exact_rows_from_being_changed():
    x = randn(1, 8, 128)
    w, b = (p.requires_grad_() for p in params(128, FP32))
    y = layer_norm(x, w, b, keep="exact")
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# Widths at which another kernel, or another of its variants, takes the call: whole chunks in a warp (256, 512), in a
# block (1024 and up), at the most (16384), past it; single elements in a warp (300), in a block (513, 8193), past it.
@pytest.mark.parametrize("keep", ["exact", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("m,n", [(1200, 8), (700, 264), (700, 512), (300, 520), (500, 1024), (5, 1032), (300, 4096), (3, 12304),
                                 (160, 16384), (4, 16400), (900, 300), (900, 511), (500, 513), (160, 8191), (160, 8193), (5, 12289),
                                 (3, 16385), (2, 20001)])
def test_norm_at_the_borders_of_its_variants(m, n, dtype, keep):
    x = (randn(m + n, m, n) * 2 + randn(n, 1, n)).to(dtype)
    dy = randn(m * 3 + n, m, n, dtype=dtype)
    w, b = params(n, dtype)
    want, h, _, rstd = norm_exact(x, w, b)
    y, kept = layer_norm_forward(x, w, b, EPS, keep=keep)
    close(y, want, y_tolerance(x, w, b, dtype), "y")
    if keep == "fp8":
        check_kept(kept, x, h, rstd)
    for name, a, c in zip(("dx", "dweight", "dbias"), layer_norm_backward(dy, kept, w), backward_exact(dy, kept, w)):
        close(a, *c, name)
    # A row's bits do not depend on the rows beside it.
    one, _ = layer_norm_forward(x[m - 1:], w, b, EPS)
    assert torch.equal(one, y[m - 1:])


def test_norm_of_many_looked_up_tokens():
    codes, scales, x = lookup(3, 3000, 6, 256, 128)
    w, b = params(1536, BF16)
    y, kept = layer_norm_forward(codes, w, b, EPS, scales=scales, hidden=256, keep="fp8")
    want, h, _, rstd = norm_exact(x, w, b)
    close(y, want, y_tolerance(x, w, b, BF16), "y")
    check_kept(kept, x, h, rstd)


# ---------------------------------------------------------------- weight gradient
def checkpoint(seed, m, n):
    return save_fp8(randn(seed, m, n) * torch.exp2(randn(seed + 1, 1, n)))


def weight_grad_exact(dy, codes, scales, w=None, b=None):
    """((dweight, tolerance), (dbias, tolerance)) before the rounding to the result's type."""
    n, m = codes.shape[1], codes.shape[0]
    x = codes.double() * scales.double().repeat_interleave(128, 1)[:, :n]
    dy = dy.double()
    sums, sums_abs = dy.sum(0), dy.abs().sum(0)
    grad, size = dy.t() @ x, dy.abs().t() @ x.abs()
    # Products are exact; a tensor core adds 16 at a time and may cut instead of round (2 U, and as much
    # again for the alignment of the 16), a split of the rows adds at most 300 more.
    depth = m / 16 + 300
    t, tb = 4 * U * depth * size, (m / 8 + 300) * U * sums_abs
    if w is not None:
        t = t * w.double().abs() + 4 * U * (grad * w.double()).abs()
        grad = grad * w.double()
    if b is not None:
        grad = grad + sums[:, None] * b.double()
        t = t + (tb[:, None] + 4 * U * sums_abs[:, None]) * b.double().abs()
    return (grad, t), (sums, tb)


@pytest.mark.parametrize("fold", ["none", "weight", "both"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n,out", [(1, 1, 1), (1, 256, 8), (3, 130, 5), (16, 128, 128), (63, 64, 200), (65, 1001, 129), (100, 256, 72),
                                     (129, 4097, 33), (500, 640, 264), (1000, 6144, 256), (2100, 384, 1024), (5000, 128, 16)])
def test_weight_grad(m, n, out, dtype, fold):
    codes, scales = checkpoint(m + n, m, n)
    dy = randn(out + m, m, out, dtype=dtype)
    w, b = params(n, dtype)
    w, b = (None if fold == "none" else w), (b if fold == "both" else None)
    (want, t), (sums, tb) = weight_grad_exact(dy, codes, scales, w, b)
    dw, db = fp8_weight_grad(dy, codes, scales, w, b)
    assert dw.shape == (out, n) and dw.dtype == dtype and db.shape == (out,) and db.dtype == dtype
    close(dw, want, t + rounded(want, dtype), "dweight")
    close(db, sums, tb + rounded(sums, dtype), "dbias")
    dw32, none = fp8_weight_grad(dy, codes, scales, w, b, dtype=FP32, bias_grad=False)
    assert dw32.dtype == FP32 and none is None
    close(dw32, want, t + rounded(want, FP32), "dweight fp32")
    assert torch.equal(dw32, fp8_weight_grad(dy, codes, scales, w, b, dtype=FP32)[0])


def test_weight_grad_of_no_rows():
    codes, scales = save_fp8(torch.empty(0, 200, device="cuda", dtype=BF16))
    w, b = params(200, BF16)
    dw, db = fp8_weight_grad(torch.empty(0, 24, device="cuda", dtype=BF16), codes, scales, w, b)
    assert dw.shape == (24, 200) and not dw.any() and not db.any()


def test_weight_grad_of_strided_operands():
    m, n, out = 150, 384, 96
    codes, scales = checkpoint(5, m, n + 40)
    wide = randn(6, m, 400, dtype=BF16)
    col_major = torch.empty(4, 152, device="cuda").t()[:m].copy_(scales)
    for dy in (wide[:, 8:104], wide[:, 3:99], wide[7, :96].expand(m, 96), wide[:, :96].clone()):
        for c, s in ((codes, scales), (codes, col_major)):
            (want, t), _ = weight_grad_exact(dy, c, s)
            close(fp8_weight_grad(dy, c, s)[0], want, t + rounded(want, BF16), "dweight")
    packed = codes.contiguous()[:, 1:257]  # code rows on odd addresses
    dy, s = wide[:, :96], scales[:, :2]
    (want, t), _ = weight_grad_exact(dy, packed, s)
    close(fp8_weight_grad(dy, packed, s)[0], want, t + rounded(want, BF16), "dweight")


def test_weight_grad_rounds_values_whose_scales_are_no_powers_of_two():
    """amax / 448 scales: a decoded value is rounded to bf16 once, half a step of it."""
    m, n, out = 200, 300, 64
    codes, scales = quantize_fp8_blockwise(randn(1, m, n))
    dy = randn(2, m, out, dtype=BF16)
    (want, t), (sums, tb) = weight_grad_exact(dy, codes, scales)
    x = codes.double().abs() * scales.double().repeat_interleave(128, 1)[:, :n]
    dw, db = fp8_weight_grad(dy, codes, scales, dtype=FP32)
    close(dw, want, t + half_step(BF16) * (dy.double().abs().t() @ x) + rounded(want, FP32), "dweight")
    close(db, sums, tb + rounded(sums, FP32), "dbias")


def test_weight_grad_scales_far_from_one_and_non_finite_codes():
    m, n, out = 70, 256, 40
    x = randn(1, m, n) * torch.exp2(torch.randint(-60, 60, (m, 1), generator=gen(2), device="cuda").float())
    x[:, 128:] *= 2.0 ** 20
    codes, scales = save_fp8(x)
    dy = (randn(3, m, out) * torch.exp2(-torch.log2(x.abs().amax(1, keepdim=True)))).to(BF16)
    (want, t), _ = weight_grad_exact(dy, codes, scales)
    close(fp8_weight_grad(dy, codes, scales, dtype=FP32)[0], want, t + rounded(want, FP32), "dweight")
    bad = x.clone()
    bad[11, 5] = float("nan")
    codes, scales = save_fp8(bad)
    dw, db = fp8_weight_grad(dy, codes, scales, dtype=FP32)
    assert dw[:, 5].isnan().all() and torch.isfinite(dw[:, :5]).all() and torch.isfinite(dw[:, 6:]).all() and torch.isfinite(db).all()
    dy[3, 7] = float("inf")
    codes, scales = save_fp8(x)
    dw, db = fp8_weight_grad(dy, codes, scales, dtype=FP32)
    assert not torch.isfinite(dw[7]).any() and torch.isinf(db[7]) and torch.isfinite(dw[:7]).all() and torch.isfinite(dw[8:]).all()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_keeps_its_input_in_8_bits(dtype):
    x = randn(1, 90, 320, dtype=dtype).requires_grad_()
    w, c = randn(2, 64, 320, dtype=dtype).requires_grad_(), randn(3, 64, dtype=dtype).requires_grad_()
    z = linear(x, w, c)
    assert torch.equal(z, torch.nn.functional.linear(x, w, c))
    dz = randn(4, 90, 64, dtype=dtype)
    dx, dw, dc = torch.autograd.grad(z, (x, w, c), dz)
    want = fp8_weight_grad(dz, *save_fp8(x.detach()))
    assert torch.equal(dx, dz @ w.detach()) and torch.equal(dw, want[0]) and torch.equal(dc, want[1])


def test_projections_under_autocast():
    x = randn(1, 40, 256, dtype=BF16).requires_grad_()
    w = randn(2, 32, 256, dtype=BF16).requires_grad_()
    nw, nb = (p.requires_grad_() for p in params(256, BF16))
    with torch.autocast("cuda", FP16):
        z = linear(x, w) + norm_linear(x, nw, nb, w)
    z.float().sum().backward()
    assert all(t.grad.dtype == BF16 and torch.isfinite(t.grad).all() for t in (x, w, nw, nb))


def test_norm_linear_is_its_parts():
    x = randn(1, 200, 768, dtype=BF16).requires_grad_()
    nw, nb = (p.requires_grad_() for p in params(768, BF16))
    w, c = randn(2, 128, 768, dtype=BF16).requires_grad_(), randn(3, 128, dtype=BF16).requires_grad_()
    z = norm_linear(x, nw, nb, w, c)
    dz = randn(4, 200, 128, dtype=BF16)
    got = torch.autograd.grad(z, (x, nw, nb, w, c), dz)
    with torch.no_grad():
        y, kept = layer_norm_forward(x, nw, nb, keep="fp8")
        assert torch.equal(z, torch.nn.functional.linear(y, w, c))
        want = (*layer_norm_backward(dz @ w, kept, nw), *fp8_weight_grad(dz, kept.rows, kept.scales, nw, nb))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # The formula, in 64 bits, from the rows before their rounding: e4m3 is off by at most 2^-4 of each value.
    leaves = [t.detach().double().requires_grad_() for t in (x, nw, nb, w, c)]
    z64 = norm_exact(leaves[0], leaves[1], leaves[2])[0]
    h = norm_exact(leaves[0])[1].detach()
    z64 = z64 @ leaves[3].t() + leaves[4]
    g64 = torch.autograd.grad(z64, leaves, dz.double())
    off = (got[3].double() - g64[3]).abs()
    # (2^-4 of each kept value, and of each block's smallest) + bf16's rounding, over the sum's terms
    kept_off = h.abs() * 2.0 ** -4 + 2.0 ** -10 * kept.scales.double().repeat_interleave(128, 1)
    bound = dz.double().abs().t() @ (kept_off * nw.detach().double().abs())
    assert (off <= bound * 1.01 + rounded(g64[3], BF16) * 1.1).all()


@pytest.mark.parametrize("tokens", [1, 77])
def test_readout_of_a_fetch_trains_while_the_buffer_is_reused(port, monkeypatch, tokens):
    """fetch -> readout -> another fetch into the same memory -> backward."""
    import torch.distributed as dist

    from engram_rdma_lab_b200 import EngramBuffer
    from engram_rdma_lab_b200.models import make_indices, quantized_fp8_shard

    monkeypatch.setenv("ENGRAM_EGM_ENABLE", "1")
    own_group = not dist.is_initialized()
    if own_group:
        dist.init_process_group("gloo", rank=0, world_size=1, init_method=f"tcp://127.0.0.1:{port}")
    group = dist.group.WORLD
    entries, hidden, most, ept, packs = (512, 515), 256, 128, 6, 2
    sizes = EngramBuffer.get_storage_size_hint(group, entries, hidden, most, ept, F8, packs)
    buffer = EngramBuffer(group, *sizes, True, *EngramBuffer.get_theoretical_config(group, 2, most, ept), explicitly_destroy=True)
    buffer.set_config(entries, hidden, most, ept, F8, packs)
    storages, table_scales = quantized_fp8_shard(0, 1, entries, hidden, packs, "cuda")
    buffer.write(storages, table_scales)
    torch.manual_seed(3)
    readouts = [EngramReadout(hidden, ept, 48, bias=True, device="cuda") for _ in entries]
    indices = make_indices(0, 1, entries, tokens, ept, epoch=1, padding=0.1, device="cuda")
    outputs = buffer.fetch_all(indices)
    rows = [(d.clone(), s.clone()) for d, s in outputs]
    results = [readout(d, s) for readout, (d, s) in zip(readouts, outputs)]
    buffer.fetch_all(make_indices(0, 1, entries, tokens, ept, epoch=2, padding=0.1, device="cuda"))
    dz = randn(8, tokens, 48, dtype=BF16)
    torch.autograd.backward(results, [dz, dz])
    for readout, result, (data, scales) in zip(readouts, results, rows):
        wide = scales.repeat_interleave(128, 1)
        x = data.double() * wide.double()
        y, _ = layer_norm_forward(data, readout.norm_weight.detach(), readout.norm_bias.detach(), scales=scales, hidden=hidden)
        close(y, norm_exact(x, readout.norm_weight.detach(), readout.norm_bias.detach())[0],
              y_tolerance(x, readout.norm_weight.detach(), readout.norm_bias.detach(), BF16), "normalised rows")
        assert torch.equal(result, torch.nn.functional.linear(y, readout.weight, readout.bias))
        _, kept = layer_norm_forward(data, readout.norm_weight.detach(), readout.norm_bias.detach(), scales=scales, hidden=hidden, keep="fp8")
        dw, db = fp8_weight_grad(dz, kept.rows, kept.scales, readout.norm_weight.detach(), readout.norm_bias.detach())
        _, dnw, dnb = layer_norm_backward(dz @ readout.weight.detach(), kept, readout.norm_weight.detach())
        for got, want in zip((readout.weight, readout.bias, readout.norm_weight, readout.norm_bias), (dw, db, dnw, dnb)):
            assert torch.equal(got.grad, want)
    buffer.destroy()
    if own_group:
        dist.destroy_process_group()


def step(x, dy, dz, w, b):
    y, kept = layer_norm_forward(x, w, b, keep="fp8")
    return (y, *layer_norm_backward(dy, kept, w), *fp8_weight_grad(dz, kept.rows, kept.scales, w, b), restore_fp8(*save_fp8(dy)))


def test_captured_steps_replay_with_new_inputs_and_share_nothing():
    m, n, out = 300, 1024, 136
    w, b = params(n, BF16)
    inputs = [[randn(s, m, n, dtype=BF16), randn(s + 1, m, n, dtype=BF16), randn(s + 2, m, out, dtype=BF16)] for s in (1, 5)]
    graphs, results = [], []
    step(*inputs[0], w, b)
    torch.cuda.synchronize()
    for values in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(*values, w, b))
        graphs.append(graph)
    for seed in (20, 30):
        for k, values in enumerate(inputs):
            for j, v in enumerate(values):
                v.copy_(randn(seed + 7 * k + j, *v.shape, dtype=BF16))
        want = [[t.clone() for t in step(*values, w, b)] for values in inputs]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):  # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(results, want):
            assert all(torch.equal(a, c) for a, c in zip(got, expected))


def test_calls_run_on_the_current_stream():
    m, n, out = 2048, 2048, 256
    w, b = params(n, BF16)
    x, dy, dz = randn(1, m, n, dtype=BF16), randn(2, m, n, dtype=BF16), randn(3, m, out, dtype=BF16)
    want = step(x, dy, dz, w, b)
    stream = torch.cuda.Stream()
    late = [torch.zeros_like(t) for t in (x, dy, dz)]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)  # the inputs come late on this stream
        for t, v in zip(late, (x, dy, dz)):
            t.copy_(v)
        got = step(*late, w, b)
    stream.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_wait_that_ran_out_refuses_what_follows():
    """The word that a kernel sets when it gives up, set here by hand."""
    from engram_rdma_lab_b200 import _native

    C = _native.load()
    x = randn(1, 4, 256, dtype=BF16)
    codes, scales = save_fp8(x)
    assert C.debug_readout_fault(0, 5) == 0
    try:
        with pytest.raises(RuntimeError, match="gave up waiting"):
            layer_norm_forward(x)
        with pytest.raises(RuntimeError, match="gave up waiting"):
            fp8_weight_grad(x, codes, scales)
    finally:
        assert C.debug_readout_fault(0, 0) == 5
    layer_norm_forward(x)


def test_calls_from_several_threads():
    """Two threads on streams of their own: nothing is shared between calls."""
    import threading

    m, n, out = 400, 1536, 200
    w, b = params(n, BF16)
    inputs = [[randn(s, m, n, dtype=BF16), randn(s + 1, m, n, dtype=BF16), randn(s + 2, m, out, dtype=BF16)] for s in (1, 5)]
    want = [step(*values, w, b) for values in inputs]
    torch.cuda.synchronize()
    failures = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = step(*inputs[k], w, b)
        stream.synchronize()
        if not all(torch.equal(a, c) for a, c in zip(got, want[k])):
            failures.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_other_tensors_are_left_alone():
    """Results are new tensors: the memory around inputs, and rows behind a view's last, do not change."""
    big = randn(1, 40, 1024, dtype=BF16)
    before = big.clone()
    w, b = params(512, BF16)
    x = big[:30, 256:768]
    _, kept = layer_norm_forward(x, w, b, keep="exact")
    layer_norm_backward(big[5:35, :512], kept, w)
    codes, scales = save_fp8(x)
    fp8_weight_grad(big[:30, 8:100], codes, scales)
    assert torch.equal(big, before)
    assert isinstance(kept, KeptRows)
