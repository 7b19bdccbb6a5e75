"""What is measured of the gated linear recurrence, its single-token step, and the
residual norm with its dropout.

Cases of ``gated_recurrence``, ``gated_recurrence_step`` and ``residual_norm``: their
inputs, one pass through each, its plain form in elementary torch operations in
32 bits, and its exact values in 64 bits.  Sizes follow the framework's mixers
(1536 hidden, 2048 inner channels, 4096-token windows, documents of 32 to 4096
tokens) and the ranges around them.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


# --------------------------------------------------------------------------- cases


def listed():
    return [
        # A training step of the recurrence at the mixer's width over four windows, gated: the largest of its kind.
        dict(name="rec_train", op="rec", train=True, batch=4, tokens=4096, width=2048, docs=0, z=True, dtype="bf16"),
        # Packed pretraining windows: two windows of ragged documents, the state restarts at each.
        dict(name="rec_packed", op="rec", train=True, batch=1, tokens=8192, width=2048, docs=24, z=True, dtype="bf16"),
        # Fine-tuning in fp32 on a few odd-sized sequences of an odd width, without an output gate.
        dict(name="rec_train_fp32", op="rec", train=True, batch=3, tokens=777, width=1003, docs=0, z=False, dtype="fp32"),
        # One long prompt, read once, its state kept for decoding: one row, a long axis.
        dict(name="rec_prompt", op="rec", train=False, batch=1, tokens=32768, width=2048, docs=0, z=True, dtype="bf16"),
        # A few short prompts at once in fp16.
        dict(name="rec_prompt_short", op="rec", train=False, batch=6, tokens=130, width=1536, docs=0, z=True,
             dtype="fp16"),
        # One decoded token of one request: the smallest call there is.
        dict(name="rec_step_one", op="step", batch=1, slots=1, width=2048, z=True, dtype="bf16"),
        # One decoded token for each of 512 requests, states in a pool of slots.
        dict(name="rec_step_many", op="step", batch=512, slots=640, width=2048, z=True, dtype="bf16"),
        # Between two mixers of a training step under autocast: fp32 residual, bf16 branch, every part in use.
        dict(name="norm_train", op="norm", train=True, batch=4, tokens=4096, width=1536, post=True, gate=True, scale=True,
             p=0.1, dtype="bf16", stream="fp32"),
        # The same place in a wider bf16 stack without dropout or gate: norms and residual scale alone, the largest.
        dict(name="norm_train_wide", op="norm", train=True, batch=2, tokens=4096, width=4096, post=True, gate=False,
             scale=True, p=0.0, dtype="bf16", stream="bf16"),
        # Fine-tuning in fp32 at an odd width, dropout on.
        dict(name="norm_odd_fp32", op="norm", train=True, batch=3, tokens=777, width=1003, post=False, gate=True,
             scale=False, p=0.2, dtype="fp32", stream="fp32"),
        # A long prompt's residual stream: forward alone, in 16 bits.
        dict(name="norm_prompt", op="norm", train=False, batch=1, tokens=16384, width=1536, post=True, gate=True,
             scale=True, p=0.0, dtype="fp16", stream="fp16"),
        # One token of one request between two mixers: latency counts.
        dict(name="norm_step", op="norm", train=False, batch=1, tokens=1, width=1536, post=True, gate=True, scale=True,
             p=0.0, dtype="bf16", stream="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    """A width: mostly whole groups of eight channels, odd ones among them."""
    w = _log(rng, 64, hi)
    return w if rng.random() < 0.35 else w // 8 * 8


def draw(rng):
    op = rng.choice(["rec", "rec", "rec", "step", "norm", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "step":
        batch = _log(rng, 1, 1024)
        return dict(op=op, batch=batch, slots=batch + rng.randint(0, batch), width=_width(rng, 4096),
                    z=rng.random() < 0.7, dtype=dtype)
    budget = 4 * 4096 * 2048
    width = _width(rng, 2560 if op == "rec" else 4096)
    packed = op == "rec" and rng.random() < 0.4
    tokens = _log(rng, 1, 16384)
    batch = 1 if packed else _log(rng, 1, 64)
    while batch * tokens * width > (budget if dtype != "fp32" else budget // 2):
        if batch > 1:
            batch = (batch + 1) // 2
        else:
            tokens = (tokens + 1) // 2
    train = rng.random() < 0.6
    if op == "rec":
        docs = _log(rng, 1, max(1, min(200, tokens // 8))) if packed else 0
        return dict(op=op, train=train, batch=batch, tokens=tokens, width=width, docs=docs, z=rng.random() < 0.7,
                    dtype=dtype)
    return dict(op=op, train=train, batch=batch, tokens=tokens, width=width, post=rng.random() < 0.6,
                gate=rng.random() < 0.6, scale=rng.random() < 0.6,
                p=round(rng.uniform(0.02, 0.5), 3) if train and rng.random() < 0.6 else 0.0, dtype=dtype,
                stream=rng.choice([dtype, "fp32"]))


# --------------------------------------------------------------------------- inputs


def _doc_bounds(tokens, docs, rng):
    """Boundaries of `docs` documents over the tokens, their lengths spread over their logarithm."""
    parts = [math.exp(rng.uniform(math.log(32), math.log(4096))) for _ in range(docs)]
    total, at, cuts = sum(parts), 0.0, [0]
    for p in parts[:-1]:
        at += p
        cuts.append(min(tokens, int(at / total * tokens)))
    return cuts + [tokens]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 6389 + 29)
    rng = random.Random(int(seed))
    c, dt = dict(case), DTYPES[case["dtype"]]
    op, width = c["op"], c["width"]
    grad = bool(c.get("train"))

    def randn(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)

    def leaf(v):
        return v.detach().requires_grad_() if grad else v

    s = {"case": c}
    if op == "norm":
        lead, wide = (c["batch"], c["tokens"]), DTYPES[c["stream"]]
        s["residual"] = leaf(randn(*lead, width, scale=2.0, dtype=wide))
        s["branch"] = leaf(randn(*lead, width, scale=0.5))
        # the gate's logits leave a projection beside others: rows of a wider tensor
        s["gate"] = leaf(randn(*lead, 2 * width)[..., width:]) if c["gate"] else None
        s["weight"] = leaf(randn(width, scale=0.1, shift=1.0, dtype=torch.float32))
        s["branch_weight"] = leaf(randn(width, scale=0.1, shift=1.0, dtype=torch.float32)) if c["post"] else None
        s["scale"] = leaf(randn(width, scale=0.05, shift=0.3, dtype=torch.float32)) if c["scale"] else None
        # the dropout's key, on the device as a captured step keeps it, and the call's number
        s["key"] = torch.randint(0, 2 ** 62, (1,), device="cuda", generator=g)
        s["call"] = rng.randrange(2 ** 16)
        if grad:
            s["d_stream"], s["d_normed"] = randn(*lead, width, dtype=wide), randn(*lead, width)
        return s
    # rates: decays of exp(A) at a full gate from a few tokens' memory to a thousand's
    u = torch.rand(width, device="cuda", generator=g)
    s["A"] = leaf(-torch.exp(u * math.log(2000.0) + math.log(1e-3)))
    s["decay_bias"] = leaf(randn(width, scale=0.3, dtype=torch.float32))
    s["gate_bias"] = leaf(randn(width, scale=0.3, dtype=torch.float32))
    if op == "step":
        rows = c["batch"]
        s["slots"] = torch.randperm(c["slots"], device="cuda", generator=g)[:rows].to(torch.int32)
        lead, states = (rows,), c["slots"]
    else:
        lead, states = (c["batch"], c["tokens"]), c["docs"] or c["batch"]
        if c["docs"]:
            s["bounds"] = _doc_bounds(c["tokens"], c["docs"], rng)
            s["cu_seqlens"] = torch.tensor(s["bounds"], device="cuda", dtype=torch.int32)
    # x and z leave one projection side by side, the two gates another: rows of wider tensors
    xz, gates = randn(*lead, 2 * width), randn(*lead, 2 * width)
    s["x"], s["z"] = leaf(xz[..., :width]), leaf(xz[..., width:]) if c["z"] else None
    s["decay"], s["gate"] = leaf(gates[..., :width]), leaf(gates[..., width:])
    s["state"] = leaf(randn(states, width, scale=0.5, dtype=torch.float32))
    if grad:
        s["dy"], s["d_final"] = randn(*lead, width), randn(states, width, dtype=torch.float32)
    return s


# --------------------------------------------------------------------------- one pass


REC_LEAVES = ("x", "decay", "gate", "A", "z", "decay_bias", "gate_bias", "state")
NORM_LEAVES = ("residual", "branch", "weight", "branch_weight", "gate", "scale")


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import sophia_b200

    c = s["case"]
    if c["op"] == "step":
        y = sophia_b200.gated_recurrence_step(s["x"], s["decay"], s["gate"], s["A"], s["state"], s["z"], s["decay_bias"],
                                              s["gate_bias"], slots=s["slots"])
        return {"y": y, "state": s["state"]}
    if c["op"] == "rec":
        outs = sophia_b200.gated_recurrence(s["x"], s["decay"], s["gate"], s["A"], s["z"], s["decay_bias"], s["gate_bias"],
                                            initial_state=s["state"], output_final_state=True,
                                            cu_seqlens=s.get("cu_seqlens"))
        out = {"y": outs[0], "final_state": outs[1]}
        names, seeds = REC_LEAVES, ("dy", "d_final")
    else:
        outs = sophia_b200.residual_norm(s["residual"], s["branch"], s["weight"], branch_weight=s["branch_weight"],
                                         gate=s["gate"], scale=s["scale"], dropout_p=c["p"], seed=s["key"],
                                         offset=s["call"], eps=EPS)
        out = {"stream": outs[0], "normed": outs[1]}
        names, seeds = NORM_LEAVES, ("d_stream", "d_normed")
    if c["train"]:
        names = tuple(k for k in names if s[k] is not None)
        grads = torch.autograd.grad(outs, [s[k] for k in names], [s[k] for k in seeds])
        out |= {"d_" + k: v for k, v in zip(names, grads)}
    return out


def _run_plain(s):
    with torch.no_grad():
        return {"rec": _plain_rec, "step": _plain_step, "norm": _plain_norm}[s["case"]["op"]](s)


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _gates(s, dtype=torch.float32):
    """(sigmoid of the decay logits, decay, normaliser squared, input gate)."""
    r = _sigmoid(s["decay"].float() + s["decay_bias"])
    low = (s["A"] * r).to(dtype)
    return r, torch.exp(low), -torch.expm1(2 * low), _sigmoid(s["gate"].float() + s["gate_bias"])


def _plain_step(s):
    at = s["slots"].long()
    _, a, w, i = _gates(s)
    h = a * s["state"][at] + w.sqrt() * i * s["x"].float()
    s["state"][at] = h
    if s["z"] is not None:
        z = s["z"].float()
        h = h * z * _sigmoid(z)
    return {"y": h.to(s["x"].dtype), "state": s["state"]}


def _doubling(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the first axis, by doubling the span of tokens joined so far."""
    a, b = a.clone(), b.clone()
    n, step = a.shape[0], 1
    while step < n:
        b[step:] += a[step:] * b[:-step].clone()
        a[step:] *= a[:-step].clone()
        step *= 2
    return b


def _bounds(s):
    """Flat first and last tokens of the sequences that have any, and their numbers."""
    c = s["case"]
    cu = s["cu_seqlens"].long() if c["docs"] else torch.arange(c["batch"] + 1, device="cuda") * c["tokens"]
    full = (cu[1:] > cu[:-1]).nonzero()[:, 0]
    return cu[:-1][full], cu[1:][full] - 1, full


def _plain_rec(s):
    c = s["case"]
    width, shape, dt = c["width"], s["x"].shape, s["x"].dtype
    first, last, full = _bounds(s)

    def flat(v):
        return v.reshape(-1, width)

    # decays next to one and their products over thousands of tokens: 64 bits, 32 lose them
    r, a, w, i = (flat(v) for v in _gates(s, torch.float64))
    x, h0 = flat(s["x"].float()), s["state"]
    z = None if s["z"] is None else flat(s["z"].float())
    root = w.sqrt()
    fed = root * i * x
    fed[first] += a[first] * h0[full]
    joined = a.clone()
    joined[first] = 0
    h = _doubling(joined, fed)
    final = h0.clone()
    final[full] = h[last].float()
    p = None if z is None else _sigmoid(z)
    y = h if z is None else h * z * p
    out = {"y": y.to(dt).reshape(shape), "final_state": final}
    if not c["train"]:
        return out
    dy = flat(s["dy"].float())
    g = dy if z is None else dy * z * p
    g = g.double()
    g[last] += s["d_final"][full]
    after = torch.cat([a[1:], a.new_zeros(1, width)])
    after[last] = 0
    g = _doubling(after.flip(0), g.flip(0)).flip(0)
    prev = torch.cat([h.new_zeros(1, width), h[:-1]])
    prev[first] = h0[full].double()
    d_h0 = s["d_final"].clone()
    d_h0[full] = (a[first] * g[first]).float()
    # low = A r:  d h / d low = a h' - (a^2 / root) i x, with 0 where the normaliser is 0
    slope = torch.where(w > 0, a * a / root.clamp(min=1e-30), torch.zeros_like(w))
    d_low = g * (a * prev - slope * i * x)
    d_decay = d_low * s["A"] * r * (1 - r)
    d_gate = g * root * x * i * (1 - i)

    def shaped(v):
        return v.to(dt).reshape(shape)

    def total(v):
        return v.sum(0, dtype=torch.float64).float()

    out |= {"d_x": shaped(g * root * i), "d_decay": shaped(d_decay), "d_gate": shaped(d_gate), "d_A": total(d_low * r)}
    if z is not None:
        out["d_z"] = shaped(dy * h * p * (1 + z * (1 - p)))
    return out | {"d_decay_bias": total(d_decay), "d_gate_bias": total(d_gate), "d_state": d_h0}


M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85  # Philox4x32 (Salmon et al., 2011)


def _kept(s):
    """Which elements of [rows, width] the dropout keeps: four per counter (column / 4, row, 0, call)."""
    c = s["case"]
    rows, width, low = c["batch"] * c["tokens"], c["width"], 0xFFFFFFFF
    quads = (width + 3) // 4
    k0, k1 = s["key"] & low, (s["key"] >> 32) & low
    c0 = torch.arange(quads, device="cuda").expand(rows, quads)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, quads)
    c2, c3 = torch.zeros_like(c0), torch.full_like(c0, s["call"])
    for _ in range(10):
        p0, p1 = c0 * M0, c2 * M1  # 64-bit products, wrapped: their halves are right
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + W0) & low, (k1 + W1) & low
    words = torch.stack([c0, c1, c2, c3], dim=-1).reshape(rows, 4 * quads)[:, :width]
    return words >= round(c["p"] * 2 ** 32)


def _plain_norm(s):
    c, width = s["case"], s["case"]["width"]
    wide, dt, shape = s["residual"].dtype, s["branch"].dtype, s["branch"].shape

    def flat(v):
        return None if v is None else v.float().reshape(-1, width)

    x, o, gate = flat(s["residual"]), flat(s["branch"]), flat(s["gate"])
    scale = 1.0 if s["scale"] is None else s["scale"]
    keep = _kept(s).float() / (1 - c["p"]) if c["p"] else 1.0
    ro = torch.rsqrt(o.square().mean(1, keepdim=True) + EPS) if c["post"] else None
    u = o * ro * s["branch_weight"] if c["post"] else o
    p = 1.0 if gate is None else _sigmoid(gate)
    v = x + scale * keep * p * u
    rv = torch.rsqrt(v.square().mean(1, keepdim=True) + EPS)
    out = {"stream": v.to(wide).reshape(shape), "normed": (v * rv * s["weight"]).to(dt).reshape(shape)}
    if not c["train"]:
        return out
    dn = flat(s["d_normed"])
    t = dn * s["weight"]
    dv = flat(s["d_stream"]) + rv * (t - v * rv.square() * (t * v).mean(1, keepdim=True))

    def total(q):
        return q.sum(0, dtype=torch.float64).float()

    du = dv * scale * keep * p
    do = du
    out |= {"d_residual": dv.to(wide).reshape(shape), "d_weight": total(dn * v * rv)}
    if c["post"]:
        out["d_branch_weight"] = total(du * o * ro)
        t = du * s["branch_weight"]
        do = ro * (t - o * ro.square() * (t * o).mean(1, keepdim=True))
    out["d_branch"] = do.to(dt).reshape(shape)
    if gate is not None:
        out["d_gate"] = (du * u * (1 - p)).to(dt).reshape(shape)
    if s["scale"] is not None:
        out["d_scale"] = total(dv * keep * p * u)
    return out


# --------------------------------------------------------------------------- work


def work(case):
    c = dict(case)
    size, width = SIZE[c["dtype"]], c["width"]
    per = c["batch"] * c.get("tokens", 1) * width
    if c["op"] == "step":
        return {"bytes": per * ((4 + c["z"]) * size + 8) + 3 * 4 * width, "flops": per * 40}
    if c["op"] == "rec":
        state, z = (c["docs"] or c["batch"]) * width * 4, int(c["z"])
        if not c["train"]:
            return {"bytes": per * (4 + z) * size + 2 * state, "flops": per * 45}
        # x, the gates, z and dy once; y and the gradients once
        return {"bytes": per * (8 + 2 * z) * size + 4 * state, "flops": per * 130}
    wide, gate = SIZE[c["stream"]], int(c["gate"])
    if not c["train"]:
        return {"bytes": per * (2 * wide + (2 + gate) * size), "flops": per * (16 + 8 * gate)}
    # residual, branch, gate and both outputs' gradients once; outputs and gradients once
    return {"bytes": per * (4 * wide + (4 + 2 * gate) * size), "flops": per * (50 + 20 * gate + (15 if c["p"] else 0))}


# --------------------------------------------------------------------------- exact values


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits: token by token, differentiated by autograd."""
    c = dict(case)
    if c["op"] == "rec" and c["tokens"] > (16384 if c["train"] else 40000):
        return None
    s = prepare(case, seed)
    v = {k: x.detach().double().requires_grad_(x.requires_grad) if torch.is_tensor(x) and x.is_floating_point() else x
         for k, x in s.items()}
    if c["op"] == "step":
        return _exact_step(v)
    outs, names, seeds = _exact_rec(v) if c["op"] == "rec" else _exact_norm(v)
    out = {k: t.detach() for k, t in outs.items()}
    if c["train"]:
        names = [k for k in names if v[k] is not None]
        grads = torch.autograd.grad(list(outs.values()), [v[k] for k in names], [v[k] for k in seeds])
        out |= {"d_" + k: g for k, g in zip(names, grads)}
    return out


def _exact_parts(v):
    """Decay and what enters the state."""
    log_a = v["A"] * torch.sigmoid(v["decay"] + v["decay_bias"])
    return log_a.exp(), (-torch.expm1(2 * log_a)).sqrt() * torch.sigmoid(v["gate"] + v["gate_bias"]) * v["x"]


def _exact_step(v):
    a, b = _exact_parts(v)
    state, y = v["state"].clone(), []
    for row, slot in enumerate(v["slots"].tolist()):
        state[slot] = state[slot] * a[row] + b[row]
        y.append(state[slot])
    y = torch.stack(y)
    return {"y": y if v["z"] is None else y * torch.nn.functional.silu(v["z"]), "state": state}


def _exact_rec(v):
    c = v["case"]
    a, b = _exact_parts(v)
    a, b = a.unbind(1), b.unbind(1)
    bounds = v["bounds"] if c["docs"] else [0, c["tokens"]]
    outs, finals = [], []
    for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        h = v["state"][i:i + 1] if c["docs"] else v["state"]
        for t in range(lo, hi):
            h = a[t] * h + b[t]
            outs.append(h)
        finals.append(h)
    y = torch.stack(outs, 1)
    if v["z"] is not None:
        y = y * torch.nn.functional.silu(v["z"])
    return {"y": y, "final_state": torch.cat(finals)}, REC_LEAVES, ("dy", "d_final")


def _mask(key, call, rows, width, p):
    """The dropout's mask from the generator's definition, in numpy's unsigned integers."""
    u32, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    quads = (width + 3) // 4
    x = [np.tile(np.arange(quads, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), quads),
         np.zeros(rows * quads, np.uint64), np.full(rows * quads, call, np.uint64)]
    keys = [key & 0xFFFFFFFF, key >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        even, odd = x[0] * np.uint64(M0), x[2] * np.uint64(M1)
        x = [odd >> half ^ x[1] ^ np.uint64(keys[0]), odd & u32, even >> half ^ x[3] ^ np.uint64(keys[1]), even & u32]
        keys = [(k + w) & 0xFFFFFFFF for k, w in zip(keys, (W0, W1))]
    words = np.stack(x, axis=-1).reshape(rows, 4 * quads)[:, :width]
    return words >= np.uint64(round(p * 2 ** 32))


def _exact_norm(v):
    c, width = v["case"], v["case"]["width"]

    def rms(t):
        return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt()

    u = v["branch"]
    if c["post"]:
        u = rms(u) * v["branch_weight"]
    if c["gate"]:
        u = u * torch.sigmoid(v["gate"])
    if c["p"]:
        kept = torch.from_numpy(_mask(int(v["key"]), v["call"], c["batch"] * c["tokens"], width, c["p"])).to(u.device)
        u = torch.where(kept.reshape(u.shape), u / (1 - c["p"]), torch.zeros_like(u))
    if c["scale"]:
        u = u * v["scale"]
    stream = v["residual"] + u
    return {"stream": stream, "normed": rms(stream) * v["weight"]}, NORM_LEAVES, ("d_stream", "d_normed")
