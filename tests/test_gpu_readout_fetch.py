"""Training on fetched bf16 rows: the next fetch overwrites them, and autograd has to know."""

import pytest
import torch
import torch.distributed as dist

from engram_rdma_lab_b200 import EngramBuffer
from engram_rdma_lab_b200.models import EngramReadout, make_indices, normal_bf16_shard
from engram_rdma_lab_b200.ops import layer_norm, layer_norm_backward, layer_norm_forward

from .test_gpu_readout import BF16, _gpu, params, randn  # noqa: F401

pytestmark = pytest.mark.gpu

ENTRIES, HIDDEN, MOST, EPT = (512, 515), 128, 64, 3


@pytest.fixture
def buffer(port, monkeypatch):
    monkeypatch.setenv("ENGRAM_EGM_ENABLE", "1")
    own_group = not dist.is_initialized()
    if own_group:
        dist.init_process_group("gloo", rank=0, world_size=1, init_method=f"tcp://127.0.0.1:{port}")
    group = dist.group.WORLD
    sizes = EngramBuffer.get_storage_size_hint(group, ENTRIES, HIDDEN, MOST, EPT, BF16, 0)
    buffer = EngramBuffer(group, *sizes, True, *EngramBuffer.get_theoretical_config(group, 2, MOST, EPT), explicitly_destroy=True)
    buffer.set_config(ENTRIES, HIDDEN, MOST, EPT, BF16, 0)
    buffer.write(normal_bf16_shard(0, 1, ENTRIES, HIDDEN, "cuda"))
    yield buffer
    buffer.destroy()
    if own_group:
        dist.destroy_process_group()


def indices(epoch, tokens=40):
    return make_indices(0, 1, ENTRIES, tokens, EPT, epoch=epoch, padding=0.1, device="cuda")


@pytest.mark.parametrize("tokens", [40, 7, 64])
@pytest.mark.parametrize("which", ["fetch", "fetch_all"])
def test_rows_kept_exact_are_refused_after_the_next_fetch(buffer, which, tokens):
    w, b = (p.requires_grad_() for p in params(HIDDEN * EPT, BF16))
    data = buffer.fetch_all(indices(1))[0]
    dy = randn(2, *data.shape, dtype=BF16)
    results = [layer_norm(x, w, b, keep="exact") for x in (data, data.detach(), data[3:, :])]
    # (also where the number of tokens, and with it the tensors that a fetch returns, changed)
    after = getattr(buffer, which)(indices(2, tokens))
    if which == "fetch":
        for hook in after:
            hook()
    for y in results:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.backward(y, dy[:len(y)])


def test_rows_kept_exact_serve_until_the_next_fetch(buffer):
    w, b = params(HIDDEN * EPT, BF16)
    leaves = [w.clone().requires_grad_(), b.clone().requires_grad_()]
    for epoch in (1, 2, 3):  # the same number of tokens: the fetch returns the same tensors
        data = buffer.fetch_all(indices(epoch))[1]
        dy = randn(epoch, *data.shape, dtype=BF16)
        x = data.detach().requires_grad_()
        got = torch.autograd.grad(layer_norm(x, *leaves, keep="exact"), (x, *leaves), dy)
        _, kept = layer_norm_forward(data.clone(), w, b, keep="exact")
        assert all(torch.equal(a, c) for a, c in zip(got, layer_norm_backward(dy, kept, w)))


def test_a_readout_keeps_nothing_of_the_buffer(buffer):
    torch.manual_seed(3)
    readout = EngramReadout(HIDDEN, EPT, 16, device="cuda")
    data = buffer.fetch_all(indices(1))[0]
    dz = randn(4, len(data), 16, dtype=BF16)
    want = torch.autograd.grad(readout(data.clone()), list(readout.parameters()), dz)
    z = readout(data)
    buffer.fetch_all(indices(2))
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(z, list(readout.parameters()), dz), want))


def test_fetches_in_inference_mode(buffer):
    with torch.inference_mode():
        first = buffer.fetch_all(indices(1))[0]
        y = layer_norm(first)
        again = buffer.fetch_all(indices(1))[0]
        assert torch.equal(layer_norm(again), y)
    data = buffer.fetch_all(indices(1, 9))[0]
    assert not data.is_inference() and layer_norm(data).shape == (9, HIDDEN * EPT)
