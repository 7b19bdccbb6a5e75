"""What is measured of the state-space mixer's operators and of gradient clipping.

Cases of ``short_conv``, ``short_conv_step``, ``selective_scan``,
``selective_scan_step`` and ``clip_grad_norm_``: their inputs, one pass through
each, its plain form in elementary torch operations in 32 bits, and its exact
values in 64 bits.  Sizes follow the framework's mixer (1536 hidden, 2048 inner
channels, 4096-token windows, documents of 32 to 4096 tokens) and the ranges
around them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
TAPS = 4  # the framework's ShortConv


# --------------------------------------------------------------------------- cases


def listed():
    return [
        # A training step's ShortConv: one micro-batch of windows at the mixer's inner width.
        dict(name="conv_train", op="conv", train=True, batch=4, tokens=4096, width=2048, docs=0, dtype="bf16"),
        # The same layer over a short packed batch in fp32, an odd width: documents restart the convolution.
        dict(name="conv_packed_fp32", op="conv", train=True, batch=1, tokens=3001, width=1003, docs=7, dtype="fp32"),
        # One decoded token for each of 96 requests, states in a pool of slots: latency counts.
        dict(name="conv_step", op="conv_step", batch=96, slots=128, width=2048, dtype="bf16"),
        # A training step of the scan at the mixer's width over four windows, gated: the largest of the scans.
        dict(name="scan_train", op="scan", train=True, batch=4, tokens=4096, width=2048, state=16, groups=1, docs=0,
             gate=True, dtype="bf16"),
        # Packed pretraining windows: two windows of ragged documents, the state restarts at each.
        dict(name="scan_packed", op="scan", train=True, batch=1, tokens=8192, width=2048, state=16, groups=1, docs=24,
             gate=True, dtype="bf16"),
        # Fine-tuning in fp32 on a few odd-sized sequences, ungated, B and C in two groups of channels.
        dict(name="scan_train_fp32", op="scan", train=True, batch=3, tokens=777, width=1000, state=16, groups=2, docs=0,
             gate=False, dtype="fp32"),
        # One long prompt, read once, its state kept for decoding: few rows, a long axis.
        dict(name="scan_prompt", op="scan", train=False, batch=1, tokens=16384, width=2048, state=16, groups=1, docs=0,
             gate=True, dtype="bf16"),
        # A few short prompts at once with a narrower state, in fp16.
        dict(name="scan_prompt_short", op="scan", train=False, batch=6, tokens=130, width=1536, state=8, groups=1,
             docs=0, gate=True, dtype="fp16"),
        # One decoded token of one request: the smallest call there is.
        dict(name="scan_step_one", op="scan_step", batch=1, slots=1, width=2048, state=16, groups=1, dtype="bf16"),
        # One decoded token for each of 512 requests: the states' traffic counts.
        dict(name="scan_step_many", op="scan_step", batch=512, slots=640, width=2048, state=16, groups=1, dtype="bf16"),
        # Clipping between backward and optimizer: one mixer block's fp32 gradients, in their own type.
        dict(name="clip_block", op="clip", layers=1, hidden=1536, width=2048, dtype="fp32", out="fp32", ratio=0.3),
        # A 28-layer stack's bf16 gradients clipped into the optimizer's fp32 gradients: hundreds of tensors.
        dict(name="clip_stack", op="clip", layers=28, hidden=1536, width=2048, dtype="bf16", out="fp32", ratio=0.3),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan", "scan_step", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("conv", "scan"):
        packed = rng.random() < 0.4
        budget = 4 * 4096 * 2048
        width = _log(rng, 64, 2560)
        tokens = _log(rng, 1, 16384)
        batch = 1 if packed else _log(rng, 1, 64)
        while batch * tokens * width > budget // 2:
            if batch > 1:
                batch = (batch + 1) // 2
            else:
                tokens = (tokens + 1) // 2
        docs = _log(rng, 1, max(1, min(200, tokens // 8))) if packed else 0
        train = rng.random() < 0.6
        if op == "conv":
            return dict(op="conv", train=train, batch=batch, tokens=tokens, width=width, docs=docs, dtype=dtype)
        groups = rng.choice([1, 1, 2, 4])
        state = rng.choice([4, 8, 16, 16, 16, 24, 32])
        while batch * tokens * width * state > budget * 8 and tokens > 1:
            tokens = (tokens + 1) // 2
        docs = min(docs, max(1, tokens // 2)) if packed else 0
        return dict(op="scan", train=train, batch=batch, tokens=tokens, width=width // groups * groups, state=state,
                    groups=groups, docs=docs, gate=rng.random() < 0.7, dtype=dtype)
    if op == "conv_step":
        batch = _log(rng, 1, 1024)
        return dict(op="conv_step", batch=batch, slots=batch + rng.randint(0, batch), width=_log(rng, 64, 4096),
                    dtype=dtype)
    if op == "scan_step":
        batch, groups = _log(rng, 1, 512), rng.choice([1, 1, 2, 4])
        return dict(op="scan_step", batch=batch, slots=batch + rng.randint(0, batch),
                    width=_log(rng, 64, 2048) // groups * groups, state=rng.choice([4, 8, 16, 16, 32]), groups=groups,
                    dtype=dtype)
    return dict(op="clip", layers=_log(rng, 1, 28), hidden=_log(rng, 64, 1536), width=_log(rng, 64, 2048), dtype=dtype,
                out=rng.choice([dtype, "fp32"]), ratio=round(rng.uniform(0.05, 1.5), 3))


# --------------------------------------------------------------------------- inputs


def _doc_bounds(tokens, docs, rng):
    """Boundaries of `docs` documents over the tokens, their lengths spread over their logarithm."""
    parts = [math.exp(rng.uniform(math.log(32), math.log(4096))) for _ in range(docs)]
    total, at, cuts = sum(parts), 0.0, [0]
    for p in parts[:-1]:
        at += p
        cuts.append(min(tokens, int(at / total * tokens)))
    return cuts + [tokens]


def _block_shapes(hidden, width):
    """Parameters of one mixer block: projections, taps, norms and the small vectors beside them."""
    rank = max(1, hidden // 12)
    return [(hidden,), (4 * width, hidden), (rank, hidden), (width, rank), (16, hidden), (width, TAPS), (width, TAPS),
            (width, TAPS), (16,), (width,), (128,), (hidden, width)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    rng = random.Random(int(seed))
    c, dt = dict(case), DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0, dtype=dt, grad=False):
        t = (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)
        return t.requires_grad_() if grad else t

    s = {"case": c}
    op = c["op"]
    if op == "clip":
        shapes = [x for _ in range(c["layers"]) for x in _block_shapes(c["hidden"], c["width"])]
        s["grads"] = [randn(*x, scale=10.0 ** rng.uniform(-4, -2)) for x in shapes]
        # the optimizer's gradients: views of one flat buffer, end to end
        sizes = [math.prod(x) for x in shapes]
        s["flat"] = torch.empty(sum(sizes), device="cuda", dtype=DTYPES[c["out"]])
        s["out"] = [v.view(x) for v, x in zip(s["flat"].split(sizes), shapes)]
        # a clipping bound that the norm exceeds (ratio < 1) or not, as in a run's bad and good steps
        total = math.sqrt(sum(float(x.double().square().sum()) for x in s["grads"]))
        s["max_norm"] = total * c["ratio"]
        return s
    width = c["width"]
    if op in ("conv", "conv_step"):
        s["weight"] = randn(width, TAPS, scale=0.5, dtype=torch.float32, grad=op == "conv" and c["train"])
        s["bias"] = randn(width, scale=0.1, dtype=torch.float32, grad=op == "conv" and c["train"])
    else:
        n, groups = c["state"], c["groups"]
        a = -torch.arange(1, n + 1, device="cuda", dtype=torch.float32).repeat(width, 1)
        s["A"] = a * torch.exp(randn(width, n, scale=0.1, dtype=torch.float32))
        s["D"] = randn(width, scale=0.1, shift=1.0, dtype=torch.float32)
        step = torch.exp(torch.rand(width, device="cuda", generator=g) * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias): log-uniform in [1e-3, 1e-1]
        if op == "scan" and c["train"]:
            for k in ("A", "D", "dt_bias"):
                s[k].requires_grad_()
    if op in ("conv_step", "scan_step"):
        rows = c["batch"]
        s["slots"] = torch.randperm(c["slots"], device="cuda", generator=g)[:rows].to(torch.int32)
        # x and z leave one projection side by side, as do dt, B and C: rows of wider tensors
        xz = randn(rows, 2 * width)
        s["x"], s["z"] = xz[:, :width], xz[:, width:]
        if op == "conv_step":
            s["state"] = randn(c["slots"], width, TAPS - 1, dtype=torch.float32)
            return s
        s["dt"] = randn(rows, width, scale=0.5)
        bc = randn(rows, 2 * groups * n)
        s["B"], s["C"] = (t.reshape(rows, groups, n) for t in bc.split(groups * n, dim=1))
        s["state"] = randn(c["slots"], width, n, scale=0.1, dtype=torch.float32)
        return s
    b, t, grad = c["batch"], c["tokens"], c["train"]
    seqs = c["docs"] or b
    if c["docs"]:
        bounds = _doc_bounds(t, c["docs"], rng)
        s["bounds"] = bounds
        s["cu_seqlens"] = torch.tensor(bounds, device="cuda", dtype=torch.int32)
    xz = randn(b, t, 2 * width)
    leaf = (lambda v: v.detach().requires_grad_()) if grad else (lambda v: v)
    s["dy"] = randn(b, t, width)
    if op == "conv":
        s["x"] = leaf(xz[..., :width])
        s["h0"] = leaf(randn(seqs, width, TAPS - 1, dtype=torch.float32))
        s["dht"] = randn(seqs, width, TAPS - 1, dtype=torch.float32)
        return s
    s["x"] = leaf(torch.nn.functional.silu(xz[..., :width].float()).to(dt))
    s["z"] = leaf(xz[..., width:]) if c["gate"] else None
    s["dt"] = leaf(randn(b, t, width, scale=0.5))
    bc = randn(b, t, 2 * groups * n)
    s["B"], s["C"] = (leaf(v.reshape(b, t, groups, n)) for v in bc.split(groups * n, dim=2))
    s["h0"] = leaf(randn(seqs, width, n, scale=0.1, dtype=torch.float32))
    s["dht"] = randn(seqs, width, n, scale=0.1, dtype=torch.float32)
    return s


# --------------------------------------------------------------------------- one pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import sophia_b200

    c = s["case"]
    if c["op"] == "clip":
        norm = sophia_b200.clip_grad_norm_(s["grads"], s["max_norm"], out=s["out"])
        return {"norm": norm, "out": s["flat"]}
    if c["op"] == "conv_step":
        return {"y": sophia_b200.short_conv_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"]),
                "state": s["state"]}
    if c["op"] == "scan_step":
        y = sophia_b200.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], s["D"], s["z"],
                                            s["dt_bias"], slots=s["slots"])
        return {"y": y, "state": s["state"]}
    kw = dict(initial_state=s["h0"], output_final_state=True, cu_seqlens=s.get("cu_seqlens"))
    if c["op"] == "conv":
        y, ht = sophia_b200.short_conv(s["x"], s["weight"], s["bias"], **kw)
        names = ("x", "weight", "bias", "h0")
    else:
        y, ht = sophia_b200.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], **kw)
        names = tuple(k for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "h0") if s[k] is not None)
    out = {"y": y, "final_state": ht}
    if c["train"]:
        grads = torch.autograd.grad((y, ht), [s[k] for k in names], (s["dy"], s["dht"]))
        out |= {"d_" + k: v for k, v in zip(names, grads)}
    return out


def _run_plain(s):
    c = s["case"]
    with torch.no_grad():
        if c["op"] == "clip":
            return _plain_clip(s)
        if c["op"] == "conv_step":
            return _plain_conv_step(s)
        if c["op"] == "scan_step":
            return _plain_scan_step(s)
        return _plain_conv(s) if c["op"] == "conv" else _plain_scan(s)


def _silu(v):
    return v / (1 + torch.exp(-v))


def _silu_slope(v):
    p = 1 / (1 + torch.exp(-v))
    return p * (1 + v * (1 - p))


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _plain_clip(s):
    squares = torch.stack([g.float().square().sum() for g in s["grads"]])
    norm = squares.sum().sqrt()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * coef)
    return {"norm": norm, "out": s["flat"]}


def _plain_conv_step(s):
    at = s["slots"].long()
    x = s["x"].float()
    window = torch.cat([s["state"][at], x[:, :, None]], dim=2)
    y = _silu((window * s["weight"]).sum(-1) + s["bias"])
    s["state"][at] = window[:, :, 1:]
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _plain_scan_step(s):
    at, c = s["slots"].long(), s["case"]
    x = s["x"].float()
    d = _softplus(s["dt"].float() + s["dt_bias"])
    b, cc = (s[k].float().repeat_interleave(c["width"] // c["groups"], dim=1) for k in ("B", "C"))
    h = s["state"][at] * torch.exp(d[:, :, None] * s["A"]) + (d * x)[:, :, None] * b
    y = ((h * cc).sum(-1) + s["D"] * x) * _silu(s["z"].float())
    s["state"][at] = h
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _starts(s):
    """Per token and sequence: flat positions of the sequences' first and last tokens (empty ones left out)."""
    c = s["case"]
    cu = s.get("cu_seqlens")
    if cu is None:
        cu = torch.arange(c["batch"] + 1, device="cuda") * c["tokens"]
    cu = cu.long()
    full = (cu[1:] > cu[:-1]).nonzero()[:, 0]
    return cu[:-1][full], cu[1:][full] - 1, full


def _position(s):
    """[tokens, all sequences flat] each token's place in its sequence."""
    first, last, _ = _starts(s)
    n = s["case"]["batch"] * s["case"]["tokens"]
    mark = torch.zeros(n, device="cuda", dtype=torch.long)
    mark[first] = first
    return torch.arange(n, device="cuda") - torch.cummax(mark, 0).values


def _plain_conv(s):
    c = s["case"]
    n, width, hist = c["batch"] * c["tokens"], c["width"], TAPS - 1
    first, last, full = _starts(s)
    x, w, h0 = s["x"].float().reshape(n, width), s["weight"], s["h0"]
    pos = _position(s)
    seq = torch.zeros(n, device="cuda", dtype=torch.long)
    seq[first] = 1
    seq = full[torch.cumsum(seq, 0) - 1]

    def tap(back):  # the input `back` tokens before each one, the history where the sequence has none
        past = torch.cat([x.new_zeros(back, width), x])[:n]
        from_state = h0[seq, :, (hist - back + pos).clamp(0, hist - 1)]
        return torch.where((pos >= back)[:, None], past, from_state)

    taps = [tap(hist - k) if k < hist else x for k in range(TAPS)]
    pre = s["bias"] + sum(w[:, k] * taps[k] for k in range(TAPS))
    final = h0.clone()
    lengths = last - first + 1
    for k in range(hist):  # the last inputs of every sequence, older ones out of its initial state
        back = hist - 1 - k
        old = h0[full, :, (lengths + k).clamp(max=hist - 1)]
        final[full, :, k] = torch.where((lengths > back)[:, None], x[(last - back).clamp(min=0)], old)
    out = {"y": _silu(pre).to(s["x"].dtype).reshape(c["batch"], c["tokens"], width), "final_state": final}
    if not c["train"]:
        return out
    dpre = s["dy"].float().reshape(n, width) * _silu_slope(pre)
    dx, dh0 = torch.zeros_like(x), torch.zeros_like(h0)
    dht = s["dht"]
    for k in range(TAPS):
        back = hist - k
        part = dpre * w[:, k]
        inside = (pos >= back)[:, None]
        dx[: max(n - back, 0)] += torch.where(inside, part, 0.0)[back:]
        for p in range(back):  # the first tokens of each sequence read its initial state
            rows = (first + p)[lengths > p]
            dh0[full[lengths > p], :, hist - back + p] += part[rows]
    for k in range(hist):
        back = hist - 1 - k
        reach = lengths > back
        dx[(last - back)[reach]] += dht[full[reach], :, k]
        rest = full[~reach]
        dh0[rest, :, (lengths + k)[~reach]] += dht[rest, :, k]
    empty = torch.ones(h0.shape[0], device="cuda", dtype=torch.bool)
    empty[full] = False
    dh0[empty] += dht[empty]
    out["d_x"] = dx.to(s["x"].dtype).reshape(s["x"].shape)
    out["d_weight"] = torch.stack([(dpre * taps[k]).sum(0) for k in range(TAPS)], dim=1)
    out["d_bias"] = dpre.sum(0)
    out["d_h0"] = dh0
    return out


def _linear_scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the first axis, by doubling; both are overwritten."""
    step = 1
    while step < a.shape[0]:
        b[step:] = torch.addcmul(b[step:], a[step:], b[:-step])
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def _plain_scan(s):
    c = s["case"]
    b_, t_, width, n, groups = c["batch"], c["tokens"], c["width"], c["state"], c["groups"]
    rows = b_ * t_
    first, last, full = _starts(s)
    x, dtr = (s[k].float().reshape(rows, width) for k in ("x", "dt"))
    z = None if s["z"] is None else s["z"].float().reshape(rows, width)
    bb, cc = (s[k].float().reshape(rows, groups, 1, n) for k in ("B", "C"))
    raw = dtr + s["dt_bias"]
    d = _softplus(raw)
    shape = (rows, groups, width // groups, n)
    A, h0, dht = s["A"], s["h0"], s["dht"]
    decay = torch.exp(d[:, :, None] * A)
    feed = ((d * x).view(rows, groups, -1, 1) * bb).reshape(rows, width, n)
    feed[first] += decay[first] * h0[full]
    a = decay.clone()
    a[first] = 0
    h = _linear_scan(a, feed)
    final = h0.clone()
    final[full] = h[last]
    y = (h.view(shape) * cc).sum(-1).reshape(rows, width) + s["D"] * x
    gate = 1.0 if z is None else _silu(z)
    like = s["x"].dtype
    out = {"y": (y * gate).to(like).reshape(b_, t_, width), "final_state": final}
    if not c["train"]:
        return out
    dout = s["dy"].float().reshape(rows, width)
    dy = dout * gate
    a = decay.clone()
    a[first] = 0
    a = torch.cat([a[1:], torch.zeros_like(a[:1])]).flip(0)
    g = (dy.view(rows, groups, -1, 1) * cc).reshape(rows, width, n)
    g[last] += dht[full]
    g = _linear_scan(a, g.flip(0)).flip(0)
    del a
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = h0[full]
    back = decay * g
    dlog = back * before
    del before, decay
    dh0 = dht.clone()
    dh0[full] = back[first]
    gb = (g.view(shape) * bb).sum(-1).reshape(rows, width)
    dd = (dlog * A).sum(-1) + gb * x
    draw_ = dd * (1 / (1 + torch.exp(-raw)))
    out["d_x"] = (gb * d + dy * s["D"]).to(like).reshape(b_, t_, width)
    out["d_dt"] = draw_.to(like).reshape(b_, t_, width)
    out["d_A"] = (dlog * d[:, :, None]).sum(0)
    out["d_B"] = (g.view(shape) * (d * x).view(rows, groups, -1, 1)).sum(2).to(like).reshape(b_, t_, groups, n)
    out["d_C"] = (h.view(shape) * dy.view(rows, groups, -1, 1)).sum(2).to(like).reshape(b_, t_, groups, n)
    out["d_D"] = (dy * x).sum(0)
    if z is not None:
        out["d_z"] = (dout * y * _silu_slope(z)).to(like).reshape(b_, t_, width)
    out["d_dt_bias"] = draw_.sum(0)
    out["d_h0"] = dh0
    return out


# --------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = dict(case)
    size = SIZE[c["dtype"]]
    if c["op"] == "clip":
        n = c["layers"] * sum(math.prod(x) for x in _block_shapes(c["hidden"], c["width"]))
        return {"bytes": n * (size + SIZE[c["out"]]), "flops": 3 * n}
    width = c["width"]
    if c["op"] == "conv_step":
        per = c["batch"] * width
        return {"bytes": per * (2 * size + 2 * 4 * (TAPS - 1)) + width * 4 * (TAPS + 1), "flops": per * (2 * TAPS + 4)}
    if c["op"] == "scan_step":
        n, per = c["state"], c["batch"] * width
        rows = per * 4 * size + c["batch"] * 2 * c["groups"] * n * size
        return {"bytes": rows + per * 2 * 4 * n + width * 4 * (n + 2), "flops": per * (7 * n + 12)}
    seqs, per = c["docs"] or c["batch"], c["batch"] * c["tokens"] * width
    if c["op"] == "conv":
        state = seqs * width * (TAPS - 1) * 4
        if not c["train"]:
            return {"bytes": per * 2 * size + 2 * state, "flops": per * (2 * TAPS + 4)}
        return {"bytes": per * 4 * size + 4 * state, "flops": per * (6 * TAPS + 20)}
    n, gate = c["state"], 1 if c["gate"] else 0
    state, bc = seqs * width * n * 4, c["batch"] * c["tokens"] * 2 * c["groups"] * n * size
    if not c["train"]:
        return {"bytes": per * (3 + gate) * size + bc + 2 * state, "flops": per * (7 * n + 12)}
    # x, dt, z, dy and B, C once; y and the gradients once
    return {"bytes": per * (6 + 2 * gate) * size + 2 * bc + 4 * state, "flops": per * (24 * n + 40)}


# --------------------------------------------------------------------------- exact values


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits: token by token, document by document."""
    s = prepare(case, seed)
    c = s["case"]
    with torch.no_grad():
        if c["op"] == "clip":
            total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
            k = min(1.0, s["max_norm"] / (total + 1e-6))
            return {"norm": torch.tensor(total, dtype=torch.float64),
                    "out": torch.cat([g.reshape(-1).double() * k for g in s["grads"]])}
        v = {k: x.detach().double() if torch.is_tensor(x) and x.is_floating_point() else x for k, x in s.items()}
        if c["op"] == "conv_step":
            return _exact_conv_step(v)
        if c["op"] == "scan_step":
            return _exact_scan_step(v)
        spans = _exact_spans(v)
        return _exact_conv(v, spans) if c["op"] == "conv" else _exact_scan(v, spans)


def _exact_spans(v):
    """(sequence, batch row, first token, end) of every sequence."""
    c = v["case"]
    if c["docs"]:
        return [(i, 0, lo, hi) for i, (lo, hi) in enumerate(zip(v["bounds"], v["bounds"][1:]))]
    return [(i, i, 0, c["tokens"]) for i in range(c["batch"])]


def _exact_conv_step(v):
    state, at = v["state"], v["slots"].long()
    pre = v["bias"] + v["weight"][:, -1] * v["x"]
    for k in range(TAPS - 1):
        pre = pre + v["weight"][:, k] * state[at, :, k]
    new = state.clone()
    new[at] = torch.cat([state[at][..., 1:], v["x"].unsqueeze(-1)], -1)
    return {"y": pre * torch.sigmoid(pre), "state": new}


def _exact_scan_step(v):
    c, at, x = v["case"], v["slots"].long(), v["x"]
    d = torch.logaddexp(v["dt"] + v["dt_bias"], torch.zeros((), dtype=torch.float64, device=x.device))
    group = torch.arange(c["width"], device=x.device) // (c["width"] // c["groups"])
    new = v["state"].clone()
    y = v["D"] * x
    for n in range(c["state"]):
        h = new[at, :, n] * torch.exp(d * v["A"][:, n]) + d * x * v["B"][:, group, n]
        y = y + h * v["C"][:, group, n]
        new[at, :, n] = h
    return {"y": y * v["z"] * torch.sigmoid(v["z"]), "state": new}


def _exact_conv(v, spans):
    c, hist = v["case"], TAPS - 1
    x, w = v["x"], v["weight"]
    y, final = torch.empty_like(x), v["h0"].clone()
    dx, dw, db, dh0 = torch.empty_like(x), torch.zeros_like(w), torch.zeros_like(v["bias"]), torch.zeros_like(v["h0"])
    for i, row, lo, hi in spans:
        seq = torch.cat([v["h0"][i].T, x[row, lo:hi]])  # [hist + length, width]
        length = hi - lo
        pre = v["bias"] + sum(w[:, k] * seq[k:k + length] for k in range(TAPS))
        gate = torch.sigmoid(pre)
        y[row, lo:hi] = pre * gate
        final[i] = seq[length:].T
        if c["train"]:
            dpre = v["dy"][row, lo:hi] * (gate + pre * gate * (1 - gate))
            dseq = torch.zeros_like(seq)
            dseq[length:] += v["dht"][i].T
            for k in range(TAPS):
                dseq[k:k + length] += dpre * w[:, k]
                dw[:, k] += (dpre * seq[k:k + length]).sum(0)
            db += dpre.sum(0)
            dh0[i] = dseq[:hist].T
            dx[row, lo:hi] = dseq[hist:]
    out = {"y": y, "final_state": final}
    return out | {"d_x": dx, "d_weight": dw, "d_bias": db, "d_h0": dh0} if c["train"] else out


def _exact_scan(v, spans):
    c = v["case"]
    width, n, groups = c["width"], c["state"], c["groups"]
    if c["batch"] * c["tokens"] * width * n > 1 << 30:
        return None
    # sequences of one length run side by side, token after token
    lengths = sorted({hi - lo for _, _, lo, hi in spans})
    if sum(lengths) > 20000:
        return None
    x, dtr, z = v["x"], v["dt"], v["z"]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    raw = dtr + v["dt_bias"]
    d = torch.logaddexp(raw, zero)
    group = torch.arange(width, device=x.device) // (width // groups)
    A, D = v["A"], v["D"]
    y, final, dh0 = torch.empty_like(x), v["h0"].clone(), v["dht"].clone()
    grads = {k: torch.zeros_like(v[k]) for k in ("x", "dt", "A", "B", "C", "D", "dt_bias")}
    dz = None if z is None else torch.zeros_like(z)
    for length in lengths:
        if not length:
            continue
        at = [(i, row, lo) for i, row, lo, hi in spans if hi - lo == length]
        ids, rows, los = (torch.tensor(u, device=x.device) for u in zip(*at))
        h = v["h0"][ids]
        kept = []
        for t in range(length):
            p = (rows, los + t)
            e = torch.exp(d[p][..., None] * A)
            kept.append((h, e) if c["train"] else None)
            h = e * h + (d[p] * x[p])[..., None] * v["B"][p][:, group]
            out = (h * v["C"][p][:, group]).sum(-1) + D * x[p]
            y[p] = out if z is None else out * z[p] * torch.sigmoid(z[p])
            if c["train"] and z is not None:
                sg = torch.sigmoid(z[p])
                dz[p] = v["dy"][p] * out * (sg + z[p] * sg * (1 - sg))
        final[ids] = h
        if not c["train"]:
            continue
        carry = v["dht"][ids]
        for t in range(length - 1, -1, -1):
            p = (rows, los + t)
            prev, e = kept.pop()
            bg, cg = v["B"][p][:, group], v["C"][p][:, group]
            ds = v["dy"][p] if z is None else v["dy"][p] * z[p] * torch.sigmoid(z[p])
            u = (d[p] * x[p])[..., None]
            here = e * prev + u * bg
            carry = carry + ds[..., None] * cg
            split = (len(at), groups, width // groups, n)
            grads["C"][p] = (ds[..., None] * here).reshape(split).sum(2)
            grads["B"][p] = (carry * u).reshape(split).sum(2)
            feed = (carry * bg).sum(-1)
            slope = carry * e * prev
            grads["A"] += (slope * d[p][..., None]).sum(0)
            grads["x"][p] = feed * d[p] + ds * D
            grads["D"] += (ds * x[p]).sum(0)
            low = ((slope * A).sum(-1) + feed * x[p]) * torch.sigmoid(raw[p])
            grads["dt"][p] = low
            grads["dt_bias"] += low.sum(0)
            carry = carry * e
        dh0[ids] = carry
    out = {"y": y, "final_state": final}
    if c["train"]:
        out |= {"d_" + k: g for k, g in grads.items()}
        out["d_h0"] = dh0
        if dz is not None:
            out["d_z"] = dz
    return out
