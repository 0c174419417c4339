"""The packed RG-LRU scan where what one chunk hands to the next matters: gates
near one (bits must not depend on how far the other blocks have come) and
gates whose products leave float32's range though the recurrence does not."""

import pytest
import torch

import _packed_oracle as O

pytestmark = pytest.mark.gpu


def _grads(mr, a, x, cu, h0, gy, gf):
    leaves = [t.detach().clone().requires_grad_() for t in (a, x, h0)]
    y, final = mr.rglru_scan_packed_with_state(leaves[0], leaves[1], cu, h0=leaves[2])
    return [y.detach(), final.detach(), *torch.autograd.grad((y, final), leaves, (gy, gf))]


def _check(mr, a, x, cu, h0, gy, gf):
    got = _grads(mr, a, x, cu, h0, gy, gf)
    y, _, final = O.scan_forward(a, x, cu, h0)
    ga, gx, gh = O.scan_backward(a, x, cu, gy, gf, h0)
    ty, tf, ta, tx, th = O.scan_bounds(a, x, cu, gy, gf, h0)
    for name, g, w, t in (("y", got[0], y, ty), ("final", got[1], final, tf), ("grad_a", got[2], ga, ta),
                          ("grad_x", got[3], gx, tx), ("grad_h0", got[4], gh, th)):
        O.check(name, g, w, t)
    return got


# ---- the same bits every time ------------------------------------------------------------------


@pytest.mark.parametrize("dtype,D,lens", [(torch.bfloat16, 128, [40000]), (torch.float32, 33, [9000, 3, 12000]),
                                          (torch.float16, 512, [30000, 20000])])
def test_results_do_not_vary(mr, cuda_dev, dtype, D, lens):
    """Gates of 0.985 to 1: a chunk's product is far from zero, so every chunk depends on those before it. Alone, and
    beside another stream's work, which delays some blocks."""
    g = torch.Generator(device=cuda_dev).manual_seed(41)
    r = dict(device=cuda_dev, generator=g)
    T, S, cu = sum(lens), len(lens), O.borders(lens).to(cuda_dev)
    a = (1 - 0.015 * torch.rand(T, D, **r)).to(dtype)
    x, gy = torch.randn(T, D, **r).to(dtype), torch.randn(T, D, **r)
    h0, gf = torch.randn(S, D, **r), torch.randn(S, D, **r)
    want = _grads(mr, a, x, cu, h0, gy, gf)
    side, busy = torch.cuda.Stream(cuda_dev), torch.randn(2048, 2048, device=cuda_dev)
    torch.cuda.synchronize()
    for n in range(12):
        if n >= 4:
            with torch.cuda.stream(side):
                for _ in range(n):
                    busy @ busy
        for name, p, q in zip(("y", "final", "grad_a", "grad_x", "grad_h0"), _grads(mr, a, x, cu, h0, gy, gf), want):
            assert torch.equal(p, q), (name, n, int((p != q).sum()))
    torch.cuda.synchronize()


def test_gates_near_one_against_float64(mr, cuda_dev):
    g = torch.Generator().manual_seed(42)
    lens, D = [1500, 0, 700], 36
    T = sum(lens)
    a = 1 - 0.01 * torch.rand(T, D, generator=g)
    x, gy, h0, gf = (torch.randn(n, D, generator=g) for n in (T, T, 3, 3))
    _check(mr, *(t.to(cuda_dev) for t in (a, x, O.borders(lens), h0, gy, gf)))
