"""The sequence mixers over packed batches as workloads: the RG-LRU recurrence over sequences of different
lengths, sliding-window attention with sinks (training and prefill) and its one-token decode step.

Each case can run in a plain form (elementary torch operations in float32) or through this repository's
operators (`own`), and `exact` states the same results in float64 from the definitions.
"""

import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ---- cases -----------------------------------------------------------------------------------------------------


def listed():
    return [
        # one short fine-tuning example batch: launch latency of forward + backward
        dict(name="scan_tiny", op="scan", dtype="bf16", T=300, D=128, seqs=3, state=False),
        # a packed training batch of documents at the width and token count of the RG-LRU configuration
        dict(name="scan_train", op="scan", dtype="bf16", T=32768, D=2560, seqs=24, state=False),
        # one long document continued from a state (truncated back-propagation), few channels
        dict(name="scan_long", op="scan", dtype="fp16", T=131072, D=512, seqs=1, state=True),
        # float32, a width that no vector divides, many ragged sequences with states
        dict(name="scan_f32_odd", op="scan", dtype="f32", T=9973, D=1001, seqs=97, state=True),
        # a short packed batch: latency of attention forward + backward
        dict(name="attn_tiny", op="attn", dtype="bf16", T=333, Hq=4, Hkv=2, Dh=64, window=128, sinks=4, seqs=3),
        # a training step of local attention at the heads of the GLA configuration, dense batch of two rows
        dict(name="attn_train", op="attn", dtype="bf16", T=16384, Hq=32, Hkv=32, Dh=64, window=1024, sinks=0, seqs=0),
        # packed documents, grouped heads of 128, a long window and sinks: the largest
        dict(name="attn_train_gqa", op="attn", dtype="bf16", T=16001, Hq=16, Hkv=4, Dh=128, window=2048, sinks=4, seqs=7),
        # float32 training of a small model, ragged
        dict(name="attn_f32", op="attn", dtype="f32", T=3001, Hq=8, Hkv=4, Dh=32, window=300, sinks=2, seqs=5),
        # prefill of several prompts, leaving the caches that decoding starts from
        dict(name="prefill", op="prefill", dtype="fp16", T=12000, Hq=16, Hkv=8, Dh=128, window=1024, sinks=4, seqs=9),
        # one user decoding: latency
        dict(name="step_one", op="step", dtype="bf16", B=1, Hq=8, Hkv=2, Dh=64, window=512, sinks=4),
        # a serving batch at different positions, some slots free
        dict(name="step_batch", op="step", dtype="bf16", B=96, Hq=16, Hkv=4, Dh=128, window=2048, sinks=4),
        # one shared key/value head, odd window
        dict(name="step_mqa", op="step", dtype="fp16", B=33, Hq=10, Hkv=1, Dh=64, window=1023, sinks=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "attn", "attn", "prefill", "step", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "f32"])
    if op == "scan":
        D = _log(rng, 32, 4096)
        T = _log(rng, 64, min(131072, 83_000_000 // D))
        return dict(op=op, dtype=dtype, T=T, D=D, seqs=_log(rng, 1, max(2, T // 40)), state=rng.random() < 0.5)
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4])
    Dh = rng.choice([32, 64, 64, 96, 128, 128])
    sinks = rng.choice([0, 1, 4, 4, 13])
    window = _log(rng, 16, 2048)
    if op == "step":
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 96), Hq=Hq, Hkv=Hkv, Dh=Dh, window=window, sinks=sinks)
    top = 16000 if dtype != "f32" else 4000
    T = _log(rng, 64, top)
    return dict(op=op, dtype=dtype, T=T, Hq=min(Hq, 16), Hkv=Hkv, Dh=Dh, window=window, sinks=sinks,
                seqs=_log(rng, 1, max(2, min(64, T // 30))))


def _generator(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed))


def _lengths(T, seqs, seed=0):
    """Lengths that sum to T, ragged (exponential), the same for every seed of a case's inputs."""
    g = _generator(1000 * seqs + T, "cpu")
    w = torch.empty(seqs, dtype=torch.float64).exponential_(generator=g) + 0.02
    cuts = torch.floor(torch.cumsum(w, 0) / w.sum() * T).to(torch.int64)
    cuts[-1] = T
    return torch.diff(cuts, prepend=torch.zeros(1, dtype=torch.int64))


def _case_lengths(case):
    if not case["seqs"]:  # a dense batch of two rows
        return torch.tensor([case["T"] // 2] * 2)
    return _lengths(case["T"], case["seqs"])


def _positions(case):
    """Positions of the tokens that a decoding batch is at: some near the start, most past the window."""
    g = _generator(77 + case["B"], "cpu")
    pos = (torch.rand(case["B"], generator=g, dtype=torch.float64) * 3 * case["window"]).to(torch.int64)
    if case["B"] >= 8:
        pos[:: case["B"] // 2] = -1  # free slots of the batch
    else:
        pos += 2 * case["window"]
    return pos


def prepare(case, seed):
    dt, g = DTYPES[case["dtype"]], _generator(seed)
    f = dict(device="cuda", dtype=torch.float32, generator=g)
    st = dict(case)
    if case["op"] == "scan":
        T, D, S = case["T"], case["D"], case["seqs"]
        lam = torch.rand(D, **f) * (6.9 - 2.2) + 2.2
        r = torch.sigmoid(torch.randn(T, D, **f))
        a = torch.sigmoid(lam) ** (8.0 * r)
        st["a"] = a.to(dt)
        st["x"] = (torch.sqrt(1.0 - a * a) * torch.sigmoid(torch.randn(T, D, **f)) * torch.randn(T, D, **f)).to(dt)
        st["gy"] = torch.randn(T, D, **f)
        lens = _case_lengths(case)
        if case["state"]:
            st["h0"], st["gf"] = torch.randn(S, D, **f), torch.randn(S, D, **f)
    elif case["op"] == "step":
        B, slots = case["B"], case["window"] + case["sinks"]
        st["q"] = torch.randn(B, case["Hq"], case["Dh"], **f).to(dt)
        st["k"], st["v"] = (torch.randn(B, case["Hkv"], case["Dh"], **f).to(dt) for _ in range(2))
        st["cache_k"], st["cache_v"] = (torch.randn(B, slots, case["Hkv"], case["Dh"], **f).to(dt) for _ in range(2))
        st["pos"] = _positions(case).cuda()
        return st
    else:
        T = case["T"]
        st["q"] = torch.randn(T, case["Hq"], case["Dh"], **f).to(dt)
        st["k"], st["v"] = (torch.randn(T, case["Hkv"], case["Dh"], **f).to(dt) for _ in range(2))
        if case["op"] == "attn":
            st["gy"] = torch.randn(T, case["Hq"], case["Dh"], **f).to(dt)
        lens = _case_lengths(case)
    st["cu"] = torch.nn.functional.pad(torch.cumsum(lens, 0), (1, 0)).to(torch.int32).cuda()
    if case["op"] == "attn":
        for n in ("q", "k", "v"):
            st[n].requires_grad_()
    if case["op"] == "scan":
        for n in ("a", "x", "h0"):
            if n in st:
                st[n].requires_grad_()
    return st


# ---- one pass --------------------------------------------------------------------------------------------------


def run(st):
    return {"scan": _run_scan, "attn": _run_attn, "prefill": _run_prefill, "step": _run_step}[st["op"]](st)


def _run_scan(st):
    if own:
        mr = importlib.import_module("mlx-recurrence_b200")
        if st["state"]:
            y, final = mr.rglru_scan_packed_with_state(st["a"], st["x"], st["cu"], h0=st["h0"])
            grads = torch.autograd.grad((y, final), (st["a"], st["x"], st["h0"]), (st["gy"], st["gf"]))
            return {"y": y, "final": final, "grads": grads}
        y = mr.rglru_scan_packed(st["a"], st["x"], st["cu"])
        return {"y": y, "grads": torch.autograd.grad(y, (st["a"], st["x"]), st["gy"])}
    return _plain_scan(st)


def _run_attn(st):
    if own:
        mr = importlib.import_module("mlx-recurrence_b200")
        if st["seqs"]:
            y = mr.window_attention_packed(st["q"], st["k"], st["v"], st["cu"], st["window"], sinks=st["sinks"])
        else:
            q, k, v = (st[n].unflatten(0, (2, -1)) for n in ("q", "k", "v"))
            y = mr.window_attention(q, k, v, st["window"], sinks=st["sinks"]).flatten(0, 1)
        return {"y": y, "grads": torch.autograd.grad(y, (st["q"], st["k"], st["v"]), st["gy"])}
    with torch.enable_grad():
        q, k, v = (st[n].detach().float().requires_grad_() for n in ("q", "k", "v"))
        y = _plain_attn(q, k, v, st["cu"], st["window"], st["sinks"])
        grads = torch.autograd.grad(y, (q, k, v), st["gy"].float())
    dt = st["q"].dtype
    return {"y": y.detach().to(dt), "grads": tuple(t.to(dt) for t in grads)}


def _run_prefill(st):
    if own:
        mr = importlib.import_module("mlx-recurrence_b200")
        y, ck, cv = mr.window_attention_packed_with_state(st["q"], st["k"], st["v"], st["cu"], st["window"],
                                                          sinks=st["sinks"])
        return {"y": y, "cache_k": ck, "cache_v": cv}
    y = _plain_attn(st["q"].float(), st["k"].float(), st["v"].float(), st["cu"], st["window"], st["sinks"])
    # slot s < sinks holds token s; slot sinks + r holds the last token t >= sinks with (t - sinks) % window == r
    n = torch.diff(st["cu"].long())[:, None]
    slot = torch.arange(st["sinks"] + st["window"], device=n.device)[None]
    ring = slot - st["sinks"]
    last = torch.div(n - 1 - st["sinks"] - ring, st["window"], rounding_mode="floor") * st["window"] + slot
    tok = torch.where(ring < 0, slot, last)
    ok = (tok < n) & ((ring < 0) | (tok >= st["sinks"]))
    at = torch.where(ok, st["cu"].long()[:-1, None] + tok, 0)
    caches = [torch.where(ok[..., None, None], t[at], 0) for t in (st["k"], st["v"])]
    return {"y": y.to(st["q"].dtype), "cache_k": caches[0], "cache_v": caches[1]}


def _run_step(st):
    if own:
        mr = importlib.import_module("mlx-recurrence_b200")
        y = mr.window_attention_step(st["q"], st["k"], st["v"], st["cache_k"], st["cache_v"], st["pos"],
                                     sinks=st["sinks"])
        return {"y": y, "cache_k": st["cache_k"], "cache_v": st["cache_v"]}
    pos, sinks, window, ck, cv = st["pos"], st["sinks"], st["window"], st["cache_k"], st["cache_v"]
    B, Hq, Dh = st["q"].shape
    Hkv = ck.shape[2]
    active = pos >= 0
    slot = torch.where(pos < sinks, pos, sinks + (pos - sinks) % window).clamp(min=0)
    rows = torch.arange(B, device=pos.device)
    keep = active[:, None, None]
    ck[rows, slot] = torch.where(keep, st["k"], ck[rows, slot])
    cv[rows, slot] = torch.where(keep, st["v"], cv[rows, slot])
    seen = torch.arange(sinks + window, device=pos.device)[None] <= pos[:, None]
    q = st["q"].float().view(B, Hkv, Hq // Hkv, Dh) * Dh ** -0.5
    s = torch.matmul(q, ck.float().permute(0, 2, 3, 1))
    s = torch.where(seen[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    y = torch.matmul(p, cv.float().permute(0, 2, 1, 3)) / torch.where(z > 0, z, 1.0)
    return {"y": y.reshape(B, Hq, Dh).to(st["q"].dtype), "cache_k": ck, "cache_v": cv}


# ---- plain forms -----------------------------------------------------------------------------------------------


def _doubling_scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 0 by doubling: after step n, (a, x) compose the last 2^n steps."""
    n = 1
    while n < a.shape[0]:
        x = torch.cat((x[:n], torch.addcmul(x[n:], a[n:], x[:-n])))
        a = torch.cat((a[:n], a[n:] * a[:-n]))
        n *= 2
    return x


def _plain_scan(st):
    with torch.no_grad():
        a, x, cu = st["a"].float(), st["x"].float(), st["cu"].long()
        some = torch.diff(cu) > 0
        first, last = cu[:-1][some], cu[1:][some] - 1
        starts = torch.zeros(a.shape[0], 1, dtype=torch.bool, device=a.device)
        starts[first] = True
        h0 = torch.zeros(cu.numel() - 1, a.shape[1], device=a.device) if "h0" not in st else st["h0"].detach()
        inner = torch.where(starts, 0.0, a)
        x = x.index_add(0, first, a[first] * h0[some])
        y = _doubling_scan(inner, x)
        before = torch.cat((torch.zeros_like(y[:1]), y[:-1]))
        before[first] = h0[some]
        g = st["gy"]
        if st["state"]:
            g = g.index_add(0, last, st["gf"][some])
        nxt = torch.cat((inner[1:], torch.zeros_like(inner[:1])))
        adj = _doubling_scan(nxt.flip(0), g.flip(0)).flip(0)
        dt = st["a"].dtype
        ga, gx = (adj * before).to(dt), adj.to(dt)
        if not st["state"]:
            return {"y": y, "grads": (ga, gx)}
        final = h0.clone()
        final[some] = y[last]
        gh0 = st["gf"].clone()
        gh0[some] = a[first] * adj[first]
        return {"y": y, "final": final, "grads": (ga, gx, gh0)}


def _plain_attn(q, k, v, cu, window, sinks):
    """Blocks of 128 queries against the blocks of keys that their windows reach, and each row's sinks apart."""
    T, Hq, Dh = q.shape
    Hkv = k.shape[1]
    n, back = 128, -(-(window - 1) // 128)
    nb = -(-T // n)
    pad = nb * n - T
    pos = torch.arange(nb * n, device=q.device)
    seq = torch.searchsorted(cu[1:].contiguous(), pos.to(cu.dtype), right=True)
    start = torch.where(pos < T, cu.long()[seq.clamp(max=cu.numel() - 2)], pos)

    def blocks(t):  # [nb, Hkv, (back + 1) * n, Dh]
        t = torch.nn.functional.pad(t, (0, 0, 0, 0, back * n, pad)).view(nb + back, n, Hkv, Dh)
        return t.unfold(0, back + 1, 1).permute(0, 2, 4, 1, 3).flatten(2, 3)

    qb = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, pad)).view(nb, n, Hkv, Hq // Hkv, Dh).permute(0, 2, 3, 1, 4)
    qb = (qb * Dh ** -0.5).flatten(2, 3)  # [nb, Hkv, G * n, Dh]
    s = torch.matmul(qb, blocks(k).transpose(-1, -2)).unflatten(2, (-1, n))  # [nb, Hkv, G, n, keys]
    i = pos.view(nb, n, 1)
    j = (torch.arange(nb, device=q.device)[:, None] - back) * n + torch.arange((back + 1) * n, device=q.device)
    j = j[:, None, :]
    ok = (j <= i) & (i - j < window) & (j >= start.view(nb, n, 1))
    s = torch.where(ok[:, None, None], s, -math.inf)
    if sinks:
        at = start[:, None] + torch.arange(sinks, device=q.device)
        far = (at <= pos[:, None] - window).view(nb, n, sinks)  # the sinks that the window has left
        at = at.clamp(max=T - 1)
        ks = k[at].view(nb, n, sinks, Hkv, Dh).permute(0, 3, 1, 4, 2)  # [nb, Hkv, n, Dh, sinks]
        qs = qb.unflatten(2, (-1, n)).transpose(2, 3)  # [nb, Hkv, n, G, Dh]
        ss = torch.matmul(qs, ks).transpose(2, 3)
        s = torch.cat((s, torch.where(far[:, None, None], ss, -math.inf)), -1)
    p = torch.exp(s - s.detach().amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    keys = (back + 1) * n
    y = torch.matmul(p[..., :keys].flatten(2, 3), blocks(v)).unflatten(2, (-1, n))
    if sinks:
        vs = v[at].view(nb, n, sinks, Hkv, Dh).permute(0, 3, 1, 2, 4)
        y = y + torch.matmul(p[..., keys:].transpose(2, 3), vs).transpose(2, 3)
    return y.permute(0, 3, 1, 2, 4).reshape(nb * n, Hq, Dh)[:T]


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def _pairs(lens, window, sinks):
    """Visible (query, key) pairs of sequences of these lengths."""
    n = 0
    for L in lens.tolist():
        full = min(L, window)
        n += full * (full + 1) // 2 + (L - full) * window
        if sinks and L > window:  # query i >= window also sees min(sinks, i - window + 1) sinks
            far = L - window
            head = min(far, sinks)
            n += head * (head + 1) // 2 + (far - head) * sinks
    return n


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "scan":
        n = case["T"] * case["D"]
        s = case["seqs"] * case["D"] * 4 * 4 if case["state"] else 0
        return {"bytes": n * (2 * e + 4) + n * (2 * e + 4 + 2 * e) + s, "flops": 8 * n}
    qo, kv = case["Hq"] * case["Dh"] * e, 2 * case["Hkv"] * case["Dh"] * e
    if case["op"] == "step":
        seen = torch.clamp(_positions(case) + 1, max=case["window"] + case["sinks"]).clamp(min=0)
        n = int(seen.sum())
        return {"bytes": n * kv + case["B"] * (2 * qo + kv), "flops": 4 * n * case["Hq"] * case["Dh"]}
    pairs = _pairs(_case_lengths(case), case["window"], case["sinks"])
    f = 4 * pairs * case["Hq"] * case["Dh"]
    if case["op"] == "prefill":
        slots = case["seqs"] * (case["window"] + case["sinks"])
        return {"bytes": case["T"] * (2 * qo + kv) + slots * kv, "flops": f}
    # forward: q, k, v in, y out; backward: q, k, v, y, gy in, three gradients out
    return {"bytes": case["T"] * (5 * qo + 3 * kv), "flops": 3.5 * f}


# ---- the definitions in float64 --------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "scan":
            return _exact_scan(st)
        if case["op"] == "step":
            return _exact_step(st)
        y, grads = _exact_attn(st)
        if case["op"] == "attn":
            return {"y": y, "grads": grads}
        return {"y": y, "cache_k": None, "cache_v": None}


def _exact_scan(st):
    """Step by step over all sequences at once, each padded to the longest."""
    lens = torch.diff(st["cu"].long()).tolist()
    S, D, top = len(lens), st["a"].shape[1], max(lens)
    if top * S * D * 8 * 6 > 100e9:
        return None
    z = dict(dtype=torch.float64, device="cuda")
    a, x, g = torch.zeros(top, S, D, **z), torch.zeros(top, S, D, **z), torch.zeros(top, S, D, **z)
    at = 0
    for s, n in enumerate(lens):
        a[:n, s], x[:n, s], g[:n, s] = (st[m].detach()[at:at + n].double() for m in ("a", "x", "gy"))
        if st["state"] and n:
            g[n - 1, s] += st["gf"][s].double()
        at += n
    h0 = st["h0"].detach().double() if st["state"] else torch.zeros(S, D, **z)
    h, hs = h0, torch.empty(top, S, D, **z)
    for t in range(top):
        h = torch.addcmul(x[t], a[t], h, out=hs[t])
    adj = torch.zeros(S, D, **z)
    adjs = torch.empty(top, S, D, **z)
    for t in range(top - 1, -1, -1):
        adj = torch.add(g[t], adj, out=adjs[t])
        adj = adj * a[t]  # what reaches the step before
    y = torch.cat([hs[:n, s] for s, n in enumerate(lens)])
    gx = torch.cat([adjs[:n, s] for s, n in enumerate(lens)])
    before = torch.cat([torch.cat((h0[s:s + 1], hs[:n, s]))[:n] for s, n in enumerate(lens)])
    if not st["state"]:
        return {"y": y, "grads": (gx * before, gx)}
    final = torch.stack([hs[n - 1, s] if n else h0[s] for s, n in enumerate(lens)])
    gh0 = torch.stack([a[0, s] * adjs[0, s] if n else st["gf"][s].double() for s, n in enumerate(lens)])
    return {"y": y, "final": final, "grads": (gx * before, gx, gh0)}


def _exact_attn(st):
    """Sequence by sequence, some queries at a time against all keys before them, with the softmax's own formulas."""
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    gy = st["gy"].double() if "gy" in st else None
    G, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    y, gq, gk, gv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    cu = st["cu"].tolist()
    for lo, hi in zip(cu[:-1], cu[1:]):
        for b in range(lo, hi, 512):
            e = min(hi, b + 512)
            i = torch.arange(b, e, device=q.device)[:, None]
            j = torch.arange(lo, e, device=q.device)[None]
            see = (j <= i) & ((i - j < st["window"]) | (j - lo < st["sinks"]))
            cols = torch.nonzero(see.any(0))[:, 0]
            see, cols = see[:, cols], cols + lo
            kk, vv = (t[cols].repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))  # [Hq, keys, Dh]
            qq = q[b:e].transpose(0, 1)
            p = torch.softmax((qq @ kk.transpose(1, 2) * scale).masked_fill(~see, -math.inf), -1)
            o = p @ vv
            y[b:e] = o.transpose(0, 1)
            if gy is None:
                continue
            go = gy[b:e].transpose(0, 1)
            ds = p * (go @ vv.transpose(1, 2) - (go * o).sum(-1, keepdim=True)) * scale
            gq[b:e] = (ds @ kk).transpose(0, 1)
            gk[cols] += (ds.transpose(1, 2) @ qq).unflatten(0, (-1, G)).sum(1).transpose(0, 1)
            gv[cols] += (p.transpose(1, 2) @ go).unflatten(0, (-1, G)).sum(1).transpose(0, 1)
    return y, (gq, gk, gv)


def _exact_step(st):
    """Row by row: the visible tokens are the slots up to the position, the newest from the call's own k and v."""
    pos, sinks, window = st["pos"].tolist(), st["sinks"], st["window"]
    B, Hq, Dh = st["q"].shape
    Hkv = st["cache_k"].shape[2]
    y = torch.zeros(B, Hq, Dh, dtype=torch.float64, device="cuda")
    for b, p in enumerate(pos):
        if p < 0:
            continue
        slot = p if p < sinks else sinks + (p - sinks) % window
        kk, vv = (st[n][b, :p + 1].double() for n in ("cache_k", "cache_v"))
        kk[slot], vv[slot] = st["k"][b].double(), st["v"][b].double()
        for h in range(Hkv):
            hs = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            w = torch.softmax(st["q"][b, hs].double() @ kk[:, h].T / math.sqrt(Dh), -1)
            y[b, hs] = w @ vv[:, h]
    return {"y": y, "cache_k": None, "cache_v": None}
