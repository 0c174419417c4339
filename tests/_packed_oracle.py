"""Float64 statements of the packed RG-LRU scan and of sliding-window attention
with sinks, each with the elementwise error that the kernels' arithmetic can
reach at most (derived beside each bound)."""

import math

import torch

U32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def borders(lens, pad_front=0):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0).tolist()), dtype=torch.int64)


# ---- RG-LRU ------------------------------------------------------------------------------------


def scan_forward(a, x, cu, h0=None):
    """y [T, D], h_{t-1} [T, D], final [S, D] in float64."""
    a, x = a.double(), x.double()
    T, D = a.shape
    y, before = torch.zeros_like(a), torch.zeros_like(a)
    final = []
    for s, (lo, hi) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
        h = torch.zeros(D, dtype=torch.float64, device=a.device) if h0 is None else h0[s].double()
        for t in range(lo, hi):
            before[t] = h
            h = a[t] * h + x[t]
            y[t] = h
        final.append(h)
    return y, before, torch.stack(final) if final else torch.zeros(0, D, dtype=torch.float64, device=a.device)


def scan_backward(a, x, cu, gy, gf=None, h0=None):
    """grad_a, grad_x, grad_h0, the adjoint's step-by-step formulas."""
    _, before, _ = scan_forward(a, x, cu, h0)
    a, gy = a.double(), gy.double()
    gx = torch.zeros_like(a)
    gh0 = []
    for s, (lo, hi) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
        carry = torch.zeros(a.shape[1], dtype=torch.float64, device=a.device) if gf is None else gf[s].double()
        for t in range(hi - 1, lo - 1, -1):
            gx[t] = gy[t] + carry
            carry = a[t] * gx[t]
        gh0.append(carry)
    return gx * before, gx, torch.stack(gh0)


def scan_bounds(a, x, cu, gy, gf=None, h0=None):
    """Elementwise error bounds of (y, final, grad_a, grad_x, grad_h0) in float32.

    Every result is a sum of path products a_t .. a_{s+1} x_s. However the steps
    are grouped, a path of n = t - s + 1 steps goes through at most n products,
    n sums and 6 further joins (thread, warp, CTA, look-back), so its relative
    error is below (2 n + 6) u <= 8 n u. With M = scan(|a|, |x|), the sum of
    n |path| over all paths is E = scan(|a|, M), and the error is below 8 u E."""
    A, X, G = a.double().abs(), x.double().abs(), gy.double().abs()
    H = None if h0 is None else h0.double().abs()
    F = None if gf is None else gf.double().abs()
    M, Mb, Mf = scan_forward(A, X, cu, H)
    E, Eb, Ef = scan_forward(A, M, cu, H)
    _, P, Ph = scan_backward(A, X, cu, G, F, H)
    _, Q, Qh = scan_backward(A, X, cu, P, F, H)
    # grad_a = adj * h_{t-1}: the factors' errors, and one product
    return 8 * U32 * E, 8 * U32 * Ef, 8 * U32 * (Q * Mb + P * Eb) + U32 * P * Mb, 8 * U32 * Q, 8 * U32 * (Qh + Ph)


# ---- attention ---------------------------------------------------------------------------------


def visible(T, cu, window, sinks, device="cpu"):
    """[T, T] truth values from the definition, token by token of each sequence."""
    see = torch.zeros(T, T, dtype=torch.bool)
    for lo, hi in zip(cu[:-1].tolist(), cu[1:].tolist()):
        n = hi - lo
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        see[lo:hi, lo:hi] = (j <= i) & ((i - j < window) | (j < sinks))
    return see.to(device)


class Attention:
    """y, gradients and bounds for q [T, Hq, Dh], k, v [T, Hkv, Dh], gy.

    Rows and keys outside every sequence, and masked terms, are left out of
    every sum (not multiplied by zero)."""

    def __init__(self, q, k, v, cu, window, sinks, gy=None, scale=None):
        dev, dt = q.device, q.dtype
        T, Hq, Dh = q.shape
        G = Hq // k.shape[1]
        scale = Dh ** -0.5 if scale is None else scale
        see = visible(T, cu, window, sinks, dev)
        alive, keys = see.any(1), see.any(0)

        def clean(t, m):
            return torch.where(m[:, None, None], t.double(), 0.0).transpose(0, 1)

        q, k, v = clean(q, alive), clean(k, keys).repeat_interleave(G, 0), clean(v, keys).repeat_interleave(G, 0)
        s = (q @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
        p = torch.where(see, torch.softmax(s, -1), 0.0)  # a row that sees nothing: all NaN before the mask
        y = p @ v
        # what the kernels round: the operand type's half step r for P and dS where the tensor cores take them (float32
        # runs unrounded), the output type's half step, and float32 sums. Scores: Dh products and sums, the scale and
        # the exponent's own factor, (Dh + 4) u sum |q||k| scale absolute, which is relative in p, twice (row and sum)
        r = 0.0 if dt == torch.float32 else half_step(dt)
        out = half_step(dt)
        size = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~see, 0.0)
        relp = 2 * (Dh + 4) * U32 * size.amax(-1, keepdim=True) + 8 * U32
        n = see.sum(1)[:, None] * U32 + 4 * U32
        pv = p @ v.abs()
        self.y = y.transpose(0, 1)
        # P is at most 1 and the sum that divides it at least 1: `low`, half of its type's smallest step, per visible key
        low = self.tiny(dt)
        seen = see.double()
        ty = (r + relp + n) * pv * (1 + r) + low * (seen @ v.abs())
        ty = ty + out * (y.abs() + ty) + low
        self.tol_y = ty.transpose(0, 1)
        if gy is None:
            return
        gy = clean(gy, alive)
        delta = (gy * y).sum(-1, keepdim=True)
        dp = gy @ v.transpose(1, 2)
        ds = p * (dp - delta)
        self.gq = (ds @ k * scale).transpose(0, 1)

        def shared(t):
            return t.unflatten(0, (-1, G)).sum(1).transpose(0, 1)

        self.gk, self.gv = shared(ds.transpose(1, 2) @ q * scale), shared(p.transpose(1, 2) @ gy)
        # dS: its rounding r; the error of p; of dp (Dh sums); of delta, which comes from the rounded y
        edp = (Dh + 4) * U32 * (gy.abs() @ v.abs().transpose(1, 2))
        edelta = (gy.abs() * ty).sum(-1, keepdim=True) + (Dh + 4) * U32 * (gy * y).abs().sum(-1, keepdim=True)
        # (dS lies in its type at a power-of-two scale of at most max |gy|)
        eds = torch.where(see, (r + relp) * ds.abs() + (1 + r) * p * (edp + edelta) + low * gy.abs().max(), 0.0)
        nq = G * see.sum(0)[None, None] * U32 + 4 * U32
        tq = scale * (eds @ k.abs() + n * (ds.abs() @ k.abs()))
        tk = shared(scale * (eds.transpose(1, 2) @ q.abs() + nq.transpose(1, 2) * (ds.abs().transpose(1, 2) @ q.abs())))
        pe = p * (r + relp) + low * seen
        tv = shared(pe.transpose(1, 2) @ gy.abs() + nq.transpose(1, 2) * (p.transpose(1, 2) @ gy.abs()))
        self.tol_gq = tq.transpose(0, 1) * (1 + out) + out * self.gq.abs() + low
        self.tol_gk = tk * (1 + out) + out * self.gk.abs() + low
        self.tol_gv = tv * (1 + out) + out * self.gv.abs() + low

    @staticmethod
    def tiny(dt):
        """Half a step among the smallest numbers of the type, where relative steps end."""
        return {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38, torch.float64: 0.0}[dt]


def check(name, got, want, tol):
    got, want = got.detach().double(), want.detach()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    d = (got - want).abs() - tol
    at = int(d.argmax())
    assert float(d.detach().max()) <= 0, (f"{name}: off by {float((got - want).abs().flatten()[at]):.3g}, allowed "
                                 f"{float(tol.expand_as(want).flatten()[at]):.3g} (value {float(want.flatten()[at]):.3g}, "
                                 f"index {at})")
