"""Gradients under activation checkpointing and saved-tensor hooks: the packed
scan and window attention give the same bits as without."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


def _inputs(dev, dtype):
    g = torch.Generator(device=dev).manual_seed(31)
    T, H, Hkv, Dh = 333, 4, 2, 64
    fused = torch.randn(T, (H + 2 * Hkv) * Dh, device=dev, generator=g).to(dtype)
    gy = torch.randn(T, H, Dh, device=dev, generator=g).to(dtype)
    return fused, gy, torch.tensor([0, 100, 100, 290, T], device=dev)  # int64: the forward makes an int32 copy


def _attend(mr, fused, cu):
    q, k, v = (t.unflatten(1, (-1, 64)) for t in fused.split([256, 128, 128], 1))
    return mr.window_attention_packed(q, k, v, cu, 70, sinks=3)


def _scan(mr, fused, cu):
    a, x = torch.sigmoid(fused[:, :256]), fused[:, 256:]
    y, final = mr.rglru_scan_packed_with_state(a, x, cu)
    return y + final.sum()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("run", [_attend, _scan])
def test_checkpointed_call(mr, cuda_dev, run, dtype):
    fused, gy, cu = _inputs(cuda_dev, dtype)
    gy = gy if run is _attend else gy.flatten(1).float()
    grads = []
    for wrap in (False, True):
        leaf = fused.clone().requires_grad_()
        y = checkpoint(run, mr, leaf, cu, use_reentrant=False) if wrap else run(mr, leaf, cu)
        junk = [torch.full((n,), 0x7f7f7f7f, dtype=torch.int32, device=cuda_dev) for n in (5, 512, 4096)]
        grads.append(torch.autograd.grad(y, leaf, gy)[0])
        del junk
    assert torch.equal(*grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("run", [_attend, _scan])
def test_saved_on_the_host(mr, cuda_dev, run, dtype):
    """What the backward gets back is dense where the forward read slices of a fused projection."""
    fused, gy, cu = _inputs(cuda_dev, dtype)
    gy = gy if run is _attend else gy.flatten(1).float()
    leaf = fused.clone().requires_grad_()
    want, = torch.autograd.grad(run(mr, leaf, cu), leaf, gy)
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        y = run(mr, leaf, cu)
    assert torch.equal(torch.autograd.grad(y, leaf, gy)[0], want)
