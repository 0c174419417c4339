"""Refusals of the packed scan and of window attention: wrong shapes, types,
devices and values raise before any launch (Python), and the C entry points
return their status codes (the pointers here are never read)."""

import ctypes
import importlib

import pytest
import torch


def _lm():
    m = importlib.import_module("mlx-recurrence_b200._lib")
    return m, m.load()


def test_packed_scan_refuses_bad_shapes(mr):
    a, cu = torch.rand(10, 4), torch.tensor([0, 10])
    for args in ((a, a[:, :3], cu), (a[None], a[None], cu), (a[:, :0], a[:, :0], cu)):
        with pytest.raises(ValueError, match="a and x must both be"):
            mr.rglru_scan_packed(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        mr.rglru_scan_packed(a, a, cu)


def test_window_attention_refuses_bad_arguments(mr):
    q, k = torch.randn(2, 8, 4, 64), torch.randn(2, 8, 2, 64)
    bad = [
        (dict(q=q[0]), "must be"), (dict(v=k[:, :7]), "must be"), (dict(k=k[:, :7], v=k[:, :7]), "multiple of Hkv"),
        (dict(q=q[:, :, :3]), "multiple of Hkv"), (dict(k=k[..., :32], v=k[..., :32]), "must be"),
        (dict(q=q[..., :40], k=k[..., :40], v=k[..., :40]), "Dh=40"), (dict(window=0), "window"),
        (dict(sinks=-1), "sinks"), (dict(sinks=65), "sinks"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
        (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    ]
    for change, match in bad:
        args = dict(q=q, k=k, v=k, window=4) | change
        with pytest.raises(ValueError, match=match):
            mr.window_attention(**args)
    for bad in (dict(window=4.0), dict(sinks=1.5)):
        with pytest.raises(TypeError):
            mr.window_attention(**(dict(q=q, k=k, v=k, window=4) | bad))
    with pytest.raises(RuntimeError, match="CUDA"):
        mr.window_attention(q, k, k, 4)
    with pytest.raises(ValueError, match="must be"):
        mr.window_attention_packed(q, k, k, torch.tensor([0, 8]), 4)


def test_step_refuses_bad_shapes(mr):
    q, k = torch.randn(2, 4, 64), torch.randn(2, 2, 64)
    c = torch.zeros(2, 9, 2, 64)
    with pytest.raises(ValueError, match="multiple of Hkv"):
        mr.window_attention_step(q[:, :3], k, k, c, c.clone(), torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="CUDA"):
        mr.window_attention_step(q, k, k, c, c.clone(), torch.zeros(2, dtype=torch.long))


def test_references_on_the_cpu(mr):
    """The plain loops, against each other's special cases: a window as long as the sequence is causal attention, a
    window of one returns v, and the packed scan's loop equals the dense one per sequence."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 9, h, 32, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    full = mr.window_attention_reference(q, k, v, 9)
    assert torch.equal(full, mr.window_attention_reference(q, k, v, 2, sinks=9))
    one = mr.window_attention_reference(q, k, v, 1)
    assert torch.allclose(one, v.repeat_interleave(2, 2))
    a, x = torch.rand(10, 3, generator=g), torch.randn(10, 3, generator=g)
    y = mr.rglru_scan_packed_reference(a, x, torch.tensor([0, 4, 4, 9]))
    assert torch.equal(y[4:9], mr.rglru_scan_reference(a[None, 4:9], x[None, 4:9])[0]) and (y[9] == 0).all()


def test_c_abi_status_codes(mr):
    m, lib = _lm()
    p, n = ctypes.c_void_p(256), None
    assert lib.mr_rglru_packed_fwd(p, p, p, 1, 7, 8, 4, n, p, n, n, n, 0, n) == m.MR_E_DTYPE
    assert lib.mr_rglru_packed_fwd(p, p, p, 1, 1, 8, 0, n, p, n, n, n, 0, n) == m.MR_E_SHAPE
    assert lib.mr_rglru_packed_fwd(p, p, p, 1, 1, 1 << 31, 4, n, p, n, n, n, 0, n) == m.MR_E_SHAPE
    assert lib.mr_rglru_packed_fwd(p, p, p, 1, 1, 8, 1 << 31, n, p, n, n, n, 0, n) == m.MR_E_SHAPE
    assert lib.mr_rglru_packed_fwd(p, p, p, 1, 1, 300, 4, n, p, n, n, n, 0, n) == m.MR_E_WORKSPACE
    assert lib.mr_rglru_packed_fwd(n, p, p, 1, 1, 8, 4, n, p, n, n, n, 0, n) == m.MR_E_ALIGN
    assert lib.mr_rglru_packed_workspace_bytes(128, 64) == 0 < lib.mr_rglru_packed_workspace_bytes(129, 64)
    assert lib.mr_rglru_packed_bwd(p, n, p, p, p, p, -1, 1, 8, 4, n, p, p, n, n, 0, n) == m.MR_E_SHAPE

    def fwd(q=p, ts=64, cu=p, S=1, L=0, dtype=1, T=8, Hq=2, Hkv=1, Dh=64, window=4, sinks=0, scale=0.1, y=p):
        return lib.mr_window_attn_fwd(q, p, p, ts, 64, 64, 64, 64, 64, cu, S, L, dtype, T, Hq, Hkv, Dh, window, sinks,
                                      scale, y, n, n, n)

    for change, code in ((dict(dtype=5), m.MR_E_DTYPE), (dict(Hq=3, Hkv=2), m.MR_E_SHAPE), (dict(Dh=48), m.MR_E_SHAPE),
                         (dict(window=0), m.MR_E_SHAPE), (dict(sinks=65), m.MR_E_SHAPE), (dict(scale=0.0), m.MR_E_SHAPE),
                         (dict(ts=60), m.MR_E_ALIGN), (dict(q=ctypes.c_void_p(8)), m.MR_E_ALIGN), (dict(y=n), m.MR_E_ALIGN),
                         (dict(cu=n, S=2, L=3), m.MR_E_SHAPE), (dict(T=-1), m.MR_E_SHAPE)):
        assert fwd(**change) == code, change
    assert fwd(T=0) == m.MR_OK
    rc = lib.mr_window_attn_bwd(p, p, p, p, p, p, p, 64, 64, 64, 64, 64, 64, p, 1, 0, 1, 8, 2, 1, 64, 4, 0, 0.1, p, p, p, n,
                                0, n)
    assert rc == m.MR_E_WORKSPACE
    assert lib.mr_window_step(p, p, p, p, p, p, 1, 1, 2, 3, 2, 64, 9, 1, 0.1, p, n) == m.MR_E_SHAPE
    assert lib.mr_window_step(p, p, p, p, p, p, 1, 1, 2, 2, 2, 64, 4, 4, 0.1, p, n) == m.MR_E_SHAPE
    assert lib.mr_window_step(p, p, p, p, p, p, 1, 9, 2, 2, 2, 64, 5, 4, 0.1, p, n) == m.MR_E_DTYPE
    assert lib.mr_window_step(p, n, p, p, p, p, 1, 1, 2, 2, 2, 64, 5, 4, 0.1, p, n) == m.MR_E_ALIGN
    assert lib.mr_window_cache(p, p, 64, 64, 64, 64, n, 2, 3, 1, 8, 1, 64, 5, 1, p, p, n) == m.MR_E_SHAPE
    assert lib.mr_window_cache(p, p, 60, 64, 64, 64, p, 2, 0, 1, 8, 1, 64, 5, 1, p, p, n) == m.MR_E_ALIGN


@pytest.mark.gpu
def test_refusals_on_the_device(mr, cuda_dev):
    a, cu = torch.rand(10, 4, device=cuda_dev), torch.tensor([0, 10], device=cuda_dev)
    for bad, match in ((cu[None], "1-D"), (cu.float(), "int32 or int64"), (cu.cpu(), "must be on"), (cu[:0], "1-D"),
                       ([0, 10], "1-D")):
        with pytest.raises(ValueError, match=match):
            mr.rglru_scan_packed(a, a, bad)
    with pytest.raises(ValueError, match="h0 must have"):
        mr.rglru_scan_packed(a, a, cu, h0=torch.zeros(2, 4, device=cuda_dev))
    q, k = torch.randn(3, 4, 64, device=cuda_dev), torch.randn(3, 2, 64, device=cuda_dev)
    c, pos = [torch.zeros(3, 9, 2, 64, device=cuda_dev) for _ in range(2)], torch.zeros(3, dtype=torch.long, device=cuda_dev)

    def step(**change):
        args = dict(q=q, k=k, v=k, cache_k=c[0], cache_v=c[1], pos=pos, sinks=2) | change
        return mr.window_attention_step(**args)

    step()
    for change, match in ((dict(cache_k=c[0].half()), "contiguous"), (dict(cache_k=c[0].transpose(1, 2)), "caches"),
                          (dict(cache_v=c[0]), "overlap"), (dict(sinks=9), "caches"), (dict(pos=pos[:2]), "pos"),
                          (dict(pos=pos.float()), "pos"), (dict(pos=pos.cpu()), "pos"),
                          (dict(cache_k=c[0][:2], cache_v=c[1][:2]), "caches"),
                          (dict(cache_k=torch.zeros(3, 18, 2, 64, device=cuda_dev)[:, ::2]), "contiguous")):
        with pytest.raises(ValueError, match=match):
            step(**change)
    y = mr.rglru_scan_packed(a.requires_grad_(), a, cu)
    g, = torch.autograd.grad(y.sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), a)
