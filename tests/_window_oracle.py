"""Float64 statement of sliding-window attention with bounds for what the
kernels round, kept apart from each other: the probabilities (`r`, the operand
type's half step, or its square where the rounding's remainder is carried
along), y's rounding, the remainder y_low that the backward gets beside y, and
dS at a scale of its own per row."""

import math

import torch

from _packed_oracle import Attention, U32, half_step, visible


class Window:
    """q [T, Hq, Dh], k, v [T, Hkv, Dh], gy like q. `y`, `tol_pre` (before y is rounded), `tol_y`, `tol_sum` (of y +
    y_low), and with gy `gq`, `gk`, `gv` and their bounds."""

    def __init__(self, q, k, v, cu, window, sinks, gy=None, scale=None, r=None):
        dev, dt = q.device, q.dtype
        T, Hq, Dh = q.shape
        G = Hq // k.shape[1]
        scale = Dh ** -0.5 if scale is None else scale
        see = visible(T, cu, window, sinks, dev)
        alive, keys = see.any(1), see.any(0)

        def clean(t, m):
            return torch.where(m[:, None, None], t.double(), 0.0).transpose(0, 1)

        q, k, v = clean(q, alive), clean(k, keys).repeat_interleave(G, 0), clean(v, keys).repeat_interleave(G, 0)
        p = torch.softmax((q @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf), -1)
        p = torch.where(see, p, 0.0)
        y = p @ v
        out, low = half_step(dt), Attention.tiny(dt)
        r = (0.0 if dt == torch.float32 else half_step(dt)) if r is None else r
        size = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~see, 0.0)
        # scores: Dh products and sums, the scale, the exponent's own factor; relative in p, twice (its row and the sum)
        relp = 2 * (Dh + 4) * U32 * size.amax(-1, keepdim=True) + 8 * U32
        n = see.sum(1)[:, None] * U32 + 4 * U32
        seen = see.double()
        pre = (r + relp + n) * (p @ v.abs()) * (1 + r) + low * (seen @ v.abs())
        ty = pre + out * (y.abs() + pre) + low
        # y_low rounds what y's rounding dropped, at most out (|y| + pre), to the same type
        tsum = pre + out * out * (y.abs() + pre) * (1 + out) + low + U32 * (y.abs() + pre)
        self.y, self.tol_pre, self.tol_y, self.tol_sum = (t.transpose(0, 1) for t in (y, pre, ty, tsum))
        if gy is None:
            return
        gy = clean(gy, alive)
        delta = (gy * y).sum(-1, keepdim=True)
        ds = p * (gy @ v.transpose(1, 2) - delta)
        self.gq = (ds @ k * scale).transpose(0, 1)

        def shared(t):
            return t.unflatten(0, (-1, G)).sum(1).transpose(0, 1)

        self.gk, self.gv = shared(ds.transpose(1, 2) @ q * scale), shared(p.transpose(1, 2) @ gy)
        edp = (Dh + 4) * U32 * (gy.abs() @ v.abs().transpose(1, 2))
        edelta = (gy.abs() * (ty if dt == torch.float32 else tsum)).sum(-1, keepdim=True)
        edelta = edelta + (Dh + 4) * U32 * (gy * y).abs().sum(-1, keepdim=True)
        # dS is rounded at a power-of-two scale that takes its row's bound B = |gy| |v| + |delta| (norms; the largest over
        # what the row sees) to 2^13 .. 2^14: half of the type's smallest step is then low / 2^13 of B, doubled here for
        # the norms' own rounding. grad_q: the query's B. grad_k: the largest of the queries that see the key.
        vmax = torch.where(see, v.norm(dim=-1)[:, None, :], 0.0).amax(-1, keepdim=True)
        B = 2 * gy.norm(dim=-1, keepdim=True) * vmax
        lowq = low * 2.0 ** -12 * B if dt == torch.float16 else torch.full_like(B, low)
        lowk = torch.where(see, lowq, 0.0).amax(1, keepdim=True)  # [H, 1, keys]
        lowk = lowk.unflatten(0, (-1, G)).amax(1).repeat_interleave(G, 0)
        err = torch.where(see, (r + relp) * ds.abs() + (1 + r) * p * (edp + edelta), 0.0)
        nq = G * see.sum(0)[None, None] * U32 + 4 * U32
        tq = scale * ((err + lowq * seen) @ k.abs() + n * (ds.abs() @ k.abs()))
        tk = shared(scale * ((err + lowk * seen).transpose(1, 2) @ q.abs()
                             + nq.transpose(1, 2) * (ds.abs().transpose(1, 2) @ q.abs())))
        pe = p * (r + relp) + low * seen
        tv = shared(pe.transpose(1, 2) @ gy.abs() + nq.transpose(1, 2) * (p.transpose(1, 2) @ gy.abs()))
        self.tol_gq = tq.transpose(0, 1) * (1 + out) + out * self.gq.abs() + low
        self.tol_gk = tk * (1 + out) + out * self.gk.abs() + low
        self.tol_gv = tv * (1 + out) + out * self.gv.abs() + low
