"""Argument checks of the read-out operators beyond test_readout_refusals.py (no GPU is touched)."""

import copy
import pickle
import types

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.masked
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from engram_rdma_lab_b200 import _native
from engram_rdma_lab_b200.ops import (
    KeptRows,
    check_readout,
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


# ---------------------------------------------------------------- tensors without memory
def masked(t):
    return torch.masked.masked_tensor(t, torch.ones_like(t, dtype=torch.bool))


def freed(t):
    t = t.clone()
    t.untyped_storage().resize_(0)
    return t


def shortened(t):
    t = t.clone()
    t.untyped_storage().resize_(t.untyped_storage().nbytes() - 1)
    return t


def misaligned(t):
    return torch.frombuffer(bytearray(t.numel() * t.element_size() + 1), dtype=t.dtype, offset=1).view(t.shape)


def fake(t):
    with FakeTensorMode():
        return torch.empty(t.shape, dtype=t.dtype)


def functional(t):
    return torch._to_functional_tensor(t)


KINDS = {
    "fake": fake,
    "functional": functional,
    "zeros": lambda t: torch._efficientzerotensor(t.shape, dtype=t.dtype),
    "negated": torch._neg_view,
    "masked": masked,
    "freed": freed,
    "shortened": shortened,
    "misaligned": misaligned,
    "sparse": lambda t: t.to_sparse(),
}
F8 = torch.float8_e4m3fn


def arguments():
    return dict(x=torch.ones(4, 256), dy=torch.ones(4, 256), scales=torch.ones(4, 2), codes=torch.ones(4, 256).to(F8),
                weight=torch.ones(256), bias=torch.ones(256), mean=torch.zeros(4), rstd=torch.ones(4), shift=torch.zeros(4))


CALLS = {
    "forward": (lambda a: layer_norm_forward(a["x"], a["weight"], a["bias"]), ["x", "weight", "bias"]),
    "forward of codes": (lambda a: layer_norm_forward(a["codes"], a["weight"], scales=a["scales"], dtype=torch.float32),
                         ["codes", "scales", "weight"]),
    "backward": (lambda a: layer_norm_backward(a["dy"], KeptRows(a["x"], None, a["mean"], a["rstd"], a["shift"]), a["weight"]),
                 ["dy", "x", "mean", "rstd", "shift", "weight"]),
    "backward of codes": (lambda a: layer_norm_backward(a["dy"], KeptRows(a["codes"], a["scales"], None, a["rstd"]), a["weight"]),
                          ["dy", "codes", "scales", "rstd", "weight"]),
    "save": (lambda a: save_fp8(a["x"]), ["x"]),
    "restore": (lambda a: restore_fp8(a["codes"], a["scales"]), ["codes", "scales"]),
    "weight gradient": (lambda a: fp8_weight_grad(a["dy"], a["codes"], a["scales"], a["weight"], a["bias"]),
                        ["dy", "codes", "scales", "weight", "bias"]),
}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("call", CALLS)
def test_tensors_without_plain_memory_are_refused(call, kind):
    """Their pointers are null or past their end, or their values are not what lies there."""
    run, names = CALLS[call]
    with pytest.raises(ValueError, match="on a GPU"):  # nothing else is wrong
        run(arguments())
    for name in names:
        given = arguments()
        if given[name].dtype == F8 and kind in ("negated", "masked", "sparse", "functional", "misaligned"):
            continue  # there is no such tensor of codes
        given[name] = KINDS[kind](given[name])
        with pytest.raises((ValueError, RuntimeError)) as refusal:
            run(given)
        assert "on a GPU" not in str(refusal.value), name


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("call", [*CALLS, "layer_norm", "linear", "norm_linear"])
def test_a_graph_of_the_dispatcher_is_refused(call):
    """make_fx on real tensors would not see the calls, in autograd functions neither, and keep constants."""
    a = arguments()
    forms = {
        "layer_norm": lambda x: layer_norm(x, a["weight"].requires_grad_(), a["bias"]),
        "linear": lambda x: linear(x, torch.ones(8, 256, requires_grad=True)),
        "norm_linear": lambda x: norm_linear(x, a["weight"].requires_grad_(), a["bias"], torch.ones(8, 256)),
    }
    run = forms.get(call) or (lambda x: CALLS[call][0](a)[0])
    with pytest.raises(RuntimeError, match="constant"):
        make_fx(run)(a["x"])


def test_kept_rows_of_another_kind_serve():
    """Anything with the four fields does; the second part of the mean is then zeros."""
    kept = types.SimpleNamespace(rows=torch.ones(4, 8), scales=None, mean=torch.zeros(4), rstd=torch.ones(4))
    with pytest.raises(ValueError, match="on a GPU"):
        layer_norm_backward(torch.ones(4, 8), kept)


@pytest.mark.parametrize("call", CALLS)
def test_a_tangent_is_refused(call):
    """The results of direct calls carry none, which would count as zero."""
    run, names = CALLS[call]
    for name in names:
        with forward_ad.dual_level():
            given = arguments()
            if given[name].dtype == F8:
                continue
            given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
            with pytest.raises(ValueError, match="tangent"):
                run(given)
            with pytest.raises(ValueError, match="on a GPU"):  # an open level alone is none
                run(arguments())
