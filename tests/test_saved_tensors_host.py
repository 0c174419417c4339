"""The attention's backward works on what autograd hands back, which under
checkpointing and saved-tensor hooks is not the forward's memory: the entry
point's arguments are recorded here in place of a launch."""

import importlib
import types

import pytest
import torch

W = importlib.import_module("mlx-recurrence_b200.window")


class _Record:
    def __init__(self):
        self.calls = {}

    def __call__(self, dev, name, *args):
        self.calls[name] = args


@pytest.fixture
def record(monkeypatch):
    r = _Record()
    # the real size function, everything else recorded
    sizes = types.SimpleNamespace(mr_window_attn_bwd_workspace_bytes=lambda *a: 64)
    fake = types.SimpleNamespace(require_cuda=lambda *t: t[0].device, call_on=r, addr=W._lib.addr, load=lambda: sizes,
                                 DTYPE_CODE=W._lib.DTYPE_CODE)
    monkeypatch.setattr(W, "_lib", fake)
    return r


def _backward_under_hooks(record, pack, unpack, int64):
    T, Hq, Hkv, Dh = 24, 4, 2, 32
    fused = torch.randn(T, (Hq + 2 * Hkv) * Dh).requires_grad_()
    q, k, v = (t.unflatten(1, (-1, Dh)) for t in fused.split([Hq * Dh, Hkv * Dh, Hkv * Dh], 1))
    cu = torch.tensor([0, 10, T], dtype=torch.int64 if int64 else torch.int32)
    handed = []

    def give(t):
        handed.append(unpack(t))
        return handed[-1]

    with torch.autograd.graph.saved_tensors_hooks(pack, give):
        y = W.window_attention_packed(q, k, v, cu, 4)
    y.backward(torch.ones_like(y))
    gy, y_, low, lse, q_, k_, v_, qt, qh, kt, kh, vt, vh, cu_ = record.calls["mr_window_attn_bwd"][:14]
    return handed, (q_, k_, v_, cu_, lse), (qt, qh, kt, kh, vt, vh), (Hq, Hkv, Dh)


@pytest.mark.parametrize("int64", [True, False])
def test_backward_reads_the_tensors_it_is_handed(record, int64):
    """Hooks that give back contiguous copies: their addresses and strides, not those of the forward's slices."""
    handed, ptrs, strides, (Hq, Hkv, Dh) = _backward_under_hooks(record, lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format), int64)
    alive = {t.data_ptr() for t in handed}
    assert all(p in alive for p in ptrs)
    assert strides == (Hq * Dh, Dh, Hkv * Dh, Dh, Hkv * Dh, Dh)


def test_backward_takes_slices_in_place_without_hooks(record):
    _, _, strides, (Hq, Hkv, Dh) = _backward_under_hooks(record, lambda t: t, lambda t: t, True)
    row = (Hq + 2 * Hkv) * Dh
    assert strides == (row, Dh) * 3


def test_backward_copies_what_is_handed_back_misaligned(record):
    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype)[1:]
        return flat.copy_(t.flatten()).view(t.shape)

    _, ptrs, strides, (Hq, Hkv, Dh) = _backward_under_hooks(record, lambda t: t, shifted, True)
    assert all(p % 16 == 0 for p in ptrs[:3])
    assert strides == (Hq * Dh, Dh, Hkv * Dh, Dh, Hkv * Dh, Dh)
