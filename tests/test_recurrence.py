"""``gated_recurrence`` and ``gated_recurrence_step`` against a plain float64 statement of
the formulas (``recurrence_reference.py``) on the same inputs, gradients by
autograd of that statement and by differences.

Tolerances, derived beforehand.  Kernels compute in fp32 and round once.
* Outputs stored in 16 bits: one rounding, at most half a step, 2^-8 (bf16) or 2^-11 (fp16) of an element, plus the
  fp32 term.  In the Frobenius norm the same: |e_i| <= r |v_i| for every i gives |e| <= r |v|, and no less holds for
  certain (a norm that one element of mantissa 1 dominates may have all of r).
* fp32: a sigmoid has at most 5 roundings and two approximations of 2^-22, the decay and the
  normaliser follow within 8 roundings: 2^-20 = 1e-6 of each input of the recurrence.  A state that
  remembers up to n tokens adds n roundings of 2^-24, here n <= 1500: 9e-5 in the worst case, 2.3e-6 typically.
  Elements: 1e-4 of max(|ref|, rms(ref)); Frobenius: 1e-5.
* Sums over tokens (dA, biases): their terms carry the errors above with signs of their own; the sums themselves
  are compensated over tiles.  The terms may cancel, so the bound is taken relative to the largest of the sums, 1e-5.
"""

from __future__ import annotations

import pytest
import torch

import sophia_b200
import recurrence_reference as ref

ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
gpu = pytest.mark.gpu
NAMES = ("x", "decay", "gate", "A", "z", "decay_bias", "gate_bias", "h0")
SUMS = ("A", "decay_bias", "gate_bias")


def close(name, got, want, dtype, total=False):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, name
    if not want.numel():
        return
    assert torch.isfinite(got).all(), name
    if total:
        assert (got - want).abs().max() <= 1e-5 * want.abs().max() + 1e-30, name
        return
    rms = want.square().mean().sqrt()
    tol = ROUND[dtype] * want.abs() + 1e-4 * torch.maximum(want.abs(), rms)
    tol = tol + (2.0 ** -24 if dtype == torch.float16 else 0.0)  # fp16 subnormals
    assert ((got - want).abs() - tol).max() <= 0, f"{name}: {float((got - want).abs().max())} off, rms {float(rms)}"
    assert (got - want).norm() <= (1e-5 + ROUND[dtype]) * want.norm() + 1e-30, name


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, scale=1.0, dtype=torch.float32: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)


def cu_of(lengths):
    if lengths is None:
        return None
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], device="cuda", dtype=torch.int32)


def inputs(rn, dtype, B, T, E, N, z=True, biases=True, state=True, grad=True, pad=0):
    """Slices of wider tensors (`pad` elements beside them, so that rows may start anywhere)."""
    act = lambda: rn(B, T, E + pad, dtype=dtype)[..., pad:]  # noqa: E731
    ts = {"x": act(), "decay": act(), "gate": act(), "A": -torch.exp(rn(E, scale=2.0) - 2), "z": act() if z else None,
          "decay_bias": rn(E, scale=0.5) if biases else None, "gate_bias": rn(E, scale=0.5) if biases else None,
          "h0": rn(N, E) if state else None}
    return {k: None if v is None else v.detach().requires_grad_(grad) for k, v in ts.items()}


def call(ts, cu, final=True):
    return sophia_b200.gated_recurrence(*(ts[k] for k in NAMES[:-1]), initial_state=ts["h0"], output_final_state=final,
                                        cu_seqlens=cu)


def check(ts, cu, dy, dht):
    dtype = ts["x"].dtype
    y, ht = call(ts, cu)
    leaves = [k for k in NAMES if ts[k] is not None]
    got = torch.autograd.grad((y, ht), [ts[k] for k in leaves], (dy, dht))
    r = {k: None if v is None else v.detach().double().requires_grad_() for k, v in ts.items()}
    ry, rht = ref.recurrence(*(r[k] for k in NAMES), cu)
    want = torch.autograd.grad((ry, rht), [r[k] for k in leaves], (dy.double(), dht.double()), allow_unused=True)
    assert y.dtype == dtype and ht.dtype == torch.float32
    close("y", y, ry, dtype)
    close("final_state", ht, rht, torch.float32)
    for k, a, b in zip(leaves, got, want):
        close("d_" + k, a, torch.zeros_like(a) if b is None else b, ts[k].dtype, total=k in SUMS)
    assert sophia_b200._lib.device_error(reset=True) == 0


CASES = [  # dtype, B, T, E, z, biases, state, elements beside the rows, documents
    (torch.float32, 1, 1, 1, True, True, True, 0, None),
    (torch.float32, 2, 3, 5, True, True, True, 0, None),
    (torch.float32, 2, 31, 64, False, False, False, 0, None),
    (torch.float32, 2, 33, 68, True, True, True, 4, None),
    (torch.float32, 3, 300, 131, True, False, True, 1, None),
    (torch.bfloat16, 1, 1, 8, True, True, True, 0, None),
    (torch.bfloat16, 2, 63, 64, True, True, True, 0, None),
    (torch.bfloat16, 2, 64, 72, False, True, True, 8, None),
    (torch.bfloat16, 2, 65, 63, True, True, True, 1, None),
    (torch.bfloat16, 1, 1500, 200, True, True, True, 8, None),
    (torch.bfloat16, 1, 700, 129, True, True, False, 2, None),
    (torch.float16, 5, 129, 40, True, True, True, 0, None),
    (torch.float16, 2, 200, 77, False, False, True, 3, None),
    (torch.float16, 3, 1025, 96, True, True, True, 0, None),
    (torch.float32, 1, 40, 8, True, True, True, 0, (1, 2, 3, 0, 1, 17, 9, 7, 0)),
    (torch.float32, 1, 300, 70, True, True, False, 0, (0, 0, 32, 31, 1, 1, 64, 100, 71)),
    (torch.bfloat16, 1, 640, 64, True, True, True, 0, (0, 64, 1, 1, 1, 8, 75, 300, 126, 64, 0)),
    (torch.bfloat16, 1, 150, 33, False, True, True, 1, (150,)),
    (torch.float16, 1, 1000, 24, True, True, True, 0, (7,) * 142 + (6,)),
]


@gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "").replace(" ", "") for v in c)[:80])
def test_forward_and_gradients(case):
    dtype, B, T, E, z, biases, state, pad, docs = case
    rn, N = gen(7), len(docs) if docs else B
    ts = inputs(rn, dtype, B, T, E, N, z, biases, state, pad=pad)
    check(ts, cu_of(docs), rn(B, T, E, dtype=dtype), rn(N, E))


@gpu
def test_few_rows_share_their_tiles_over_ctas_and_many_do_not():
    """Rows from one (a cluster of eight CTAs a row) to 40 x 8 groups of channels (one CTA each)."""
    for dtype, B, T, E in ((torch.bfloat16, 1, 1153, 64), (torch.bfloat16, 40, 200, 512), (torch.float32, 20, 130, 512)):
        rn = gen(B)
        check(inputs(rn, dtype, B, T, E, B), None, rn(B, T, E, dtype=dtype), rn(B, E))


@gpu
def test_the_same_call_gives_the_same_bits():
    rn = gen(3)
    ts = inputs(rn, torch.bfloat16, 1, 3000, 192, 5)
    cu = cu_of((1000, 1, 999, 0, 1000))
    dy, dht = rn(1, 3000, 192, dtype=torch.bfloat16), rn(5, 192)
    runs = []
    for _ in range(3):
        y, ht = call(ts, cu)
        runs.append((y, ht, *torch.autograd.grad((y, ht), [ts[k] for k in NAMES], (dy, dht))))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@gpu
def test_prompt_in_pieces_and_single_tokens():
    """A prompt in two calls, then token by token in a pool of slots: the states and outputs of one call."""
    rn = gen(5)
    ts = inputs(rn, torch.bfloat16, 3, 220, 96, 3, grad=False)
    y, ht = call(ts, None)
    part = {k: v[:, :150] if k in ("x", "decay", "gate", "z") else v for k, v in ts.items()}
    y0, h = call(part, None)
    close("y", y0, y[:, :150].double(), torch.bfloat16)
    pool = torch.full((7, 96), float("nan"), device="cuda")
    slots = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
    pool[slots.long()] = h
    for t in range(150, 220):
        got = sophia_b200.gated_recurrence_step(ts["x"][:, t], ts["decay"][:, t], ts["gate"][:, t], ts["A"], pool, ts["z"][:, t],
                                                ts["decay_bias"], ts["gate_bias"], slots=slots)
        close("y", got, y[:, t].double(), torch.bfloat16)
    close("state", pool[slots.long()], ht.double(), torch.float32)
    assert pool[[1, 3, 5, 6]].isnan().all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,E,pad", [(1, 1, 0), (2, 7, 1), (5, 64, 0), (300, 130, 2), (3, 2050, 0)])
def test_step(dtype, rows, E, pad):
    rn = gen(rows + E)
    ts = {k: (v[0] if k in ("x", "decay", "gate", "z") else v) for k, v in
          inputs(rn, dtype, 1, rows, E, 1, grad=False, pad=pad).items()}
    pool = rn(rows + 4, E)
    slots = torch.randperm(rows + 4, device="cuda")[:rows].to(torch.int32)
    slots[rows // 2] = -3  # a padding row
    before = pool.clone()
    y = sophia_b200.gated_recurrence_step(ts["x"], ts["decay"], ts["gate"], ts["A"], pool, ts["z"], ts["decay_bias"],
                                          ts["gate_bias"], slots=slots)
    d = {k: v.double() for k, v in ts.items()}
    at = slots.long().clamp(min=0)
    ry, rh = ref.recurrence(d["x"][:, None], d["decay"][:, None], d["gate"][:, None], d["A"], d["z"][:, None],
                            d["decay_bias"], d["gate_bias"], before.double()[at], None)
    live = slots >= 0
    close("y", y[live], ry[:, 0][live], dtype)
    close("state", pool[at[live]], rh[live], torch.float32)
    assert not y[~live].any()
    rest = torch.ones(rows + 4, dtype=torch.bool, device="cuda")
    rest[at[live]] = False
    assert torch.equal(pool[rest], before[rest])
    assert sophia_b200._lib.device_error(reset=True) == 0


@gpu
def test_slot_past_the_pool_is_padding_and_reported():
    rn = gen(1)
    x = rn(2, 16)
    pool = rn(3, 16)
    before = pool.clone()
    slots = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    y = sophia_b200.gated_recurrence_step(x, x, x, -torch.ones(16, device="cuda"), pool, slots=slots)
    assert not y[0].any() and torch.equal(pool[[0, 2]], before[[0, 2]])
    assert sophia_b200._lib.device_error(reset=True) == 11


@gpu
def test_gates_at_their_ends():
    """Closed and open gates (padding's logits of -1e4, infinities) and rates from none to forgetting at once: the state
    passes through padded tokens, and every gradient stays finite.  A run of tokens starts from P h + c, the composed
    maps of the runs in front: for padded runs that is h bit by bit (P = 1, c = 0).  For the run and the tile that still
    hold real tokens, here 10, the composition has other roundings than the tokens one by one: at most one of 2^-24 of
    |P h| + |c| per token and composition, twice, so 2 (10 + 8) 2^-24 < 3e-6 of the largest state or input."""
    E = 64
    rn = gen(9)
    for dtype in (torch.float32, torch.bfloat16):
        ts = inputs(rn, dtype, 1, 80, E, 1, z=False, biases=False, grad=False)
        ts["A"] = -torch.logspace(-30, 3, E, device="cuda")
        for k in ("decay", "gate"):
            ts[k] = ts[k].contiguous()
        ts["decay"][:, 10:70] = -1e4
        ts["gate"][:, 20:30] = float("-inf")
        ts["decay"][:, 40:50] = float("-inf")
        ts["decay"][:, 70] = 1e4
        ts["gate"][:, 71] = float("inf")
        ts["decay"][:, 72] = float("inf")
        for k in ("x", "decay", "gate", "A", "h0"):
            ts[k].requires_grad_()
        y, ht = call(ts, None)
        assert torch.isfinite(y).all()
        assert (y[:, 16:32] == y[:, 16:17]).all()
        size = max(float(ts["x"].detach().abs().max()), float(ts["h0"].detach().abs().max()))
        assert ((y[:, 10:70] - y[:, 9:10]).abs().double() <= 3e-6 * size + ROUND[dtype] * y[:, 9:10].abs().double()).all()
        r = {k: None if v is None else v.detach().double() for k, v in ts.items()}
        ry, rht = ref.recurrence(*(r[k] for k in NAMES), None)
        close("y", y, ry, dtype)
        close("final_state", ht, rht, torch.float32)
        grads = torch.autograd.grad((y, ht), [ts[k] for k in ("x", "decay", "gate", "h0")], (torch.ones_like(y), ht.detach()))
        assert all(torch.isfinite(g).all() for g in grads)
        assert not grads[1][:, 10:70].any()


@gpu
def test_positive_rate_is_not_a_number_in_its_channel():
    rn = gen(14)
    ts = inputs(rn, torch.float32, 2, 40, 70, 2, grad=False)
    y, ht = call(ts, None)
    bad = dict(ts, A=ts["A"].clone())
    bad["A"][[3, 68]] = torch.tensor([0.5, float("nan")], device="cuda")
    by, bht = call(bad, None)
    hit = torch.zeros(70, dtype=torch.bool, device="cuda")
    hit[[3, 68]] = True
    assert by[..., hit].isnan().all() and torch.equal(by[..., ~hit], y[..., ~hit]) and torch.equal(bht[:, ~hit], ht[:, ~hit])
    pool = ts["h0"].clone()
    step = sophia_b200.gated_recurrence_step(*(bad[k][:, 0] for k in ("x", "decay", "gate")), bad["A"], pool)
    assert step[:, hit].isnan().all() and torch.isfinite(step[:, ~hit]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_expanded_transposed_and_far_rows(dtype):
    """Strides that the tile copies have no map for, and rows more than 2^31 elements apart: the same bits."""
    rn = gen(15)
    A = -torch.ones(64, device="cuda")
    run = lambda t: sophia_b200.gated_recurrence(t, t, t, A, t)[0]  # noqa: E731
    wide = torch.empty(2 ** 31 + 2 ** 20, device="cuda", dtype=dtype)
    far = torch.as_strided(wide, (2, 40, 64), (2 ** 31, 64, 1))
    far.copy_(rn(2, 40, 64))
    apart = torch.as_strided(wide, (1, 33, 64), (0, 2 ** 26, 1))
    for t in (rn(1, 40, 64, dtype=dtype).expand(3, 40, 64), rn(3, 1, 64, dtype=dtype).expand(3, 40, 64),
              rn(40, 3, 64, dtype=dtype).transpose(0, 1), rn(3, 64, 40, dtype=dtype).transpose(1, 2), far):
        close("y", run(t), run(t.contiguous()).double(), dtype)
    apart.copy_(rn(1, 33, 64))
    close("y", run(apart), run(apart.contiguous()).double(), dtype)


@gpu
def test_not_a_number_stays_in_its_document_and_channel():
    rn = gen(4)
    cu = cu_of((70, 3, 127))
    ts = inputs(rn, torch.bfloat16, 1, 200, 72, 3)
    clean, clean_ht = call(ts, cu)
    dy, dht = torch.ones_like(clean), torch.ones_like(clean_ht)
    base = torch.autograd.grad((clean, clean_ht), [ts["x"], ts["h0"]], (dy, dht))
    for bad in (float("nan"), float("inf")):
        dirty = dict(ts)
        with torch.no_grad():
            dirty["x"] = ts["x"].clone()
            dirty["x"][0, 71, 5] = bad
        dirty["x"].requires_grad_()
        y, ht = call(dirty, cu)
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[0, 71:73, 5] = True
        assert torch.equal(y[~hit], clean[~hit]) and not torch.isfinite(y[hit]).any()
        assert not torch.isfinite(ht[1, 5]) and torch.equal(ht[[0, 2]], clean_ht[[0, 2]])
        got = torch.autograd.grad((y, ht), [dirty["x"], dirty["h0"]], (dy, dht))
        other = torch.ones(200, dtype=torch.bool, device="cuda")
        other[70:73] = False
        assert torch.equal(got[0][:, other], base[0][:, other])
        assert torch.equal(got[1][[0, 2]], base[1][[0, 2]])


@gpu
def test_gradients_against_differences():
    """Directional derivatives of the kernel's own forward in fp32: central differences of step e have an error of
    e^2 f''' / 6 and 2^-24 |f| / e; with e = 1e-2 and values around one, 1e-3 of the directions' size."""
    rn = gen(13)
    ts = inputs(rn, torch.float32, 2, 50, 36, 2)
    dy, dht = rn(2, 50, 36), rn(2, 36)

    def f(t):
        y, ht = call(t, None)
        return (y.double() * dy).sum() + (ht.double() * dht).sum()

    grads = torch.autograd.grad(f(ts), [ts[k] for k in NAMES])
    for k, g in zip(NAMES, grads):
        v = rn(*ts[k].shape)
        if k == "A":
            v = v * ts[k].detach()  # keeps the rates negative
        e = 1e-2
        up, down = (dict(ts, **{k: ts[k].detach() + s * e * v}) for s in (1, -1))
        diff = (f(up) - f(down)).item() / (2 * e)
        assert abs(diff - (g * v).sum().item()) <= 2e-3 * (g.norm() * v.norm()).item(), k


@gpu
def test_no_tokens_no_rows_and_no_outputs_asked():
    rn = gen(2)
    A = -torch.ones(24, device="cuda")
    h0 = rn(2, 24).requires_grad_()
    empty = rn(2, 0, 24, dtype=torch.bfloat16)
    y, ht = sophia_b200.gated_recurrence(empty, empty, empty, A.requires_grad_(), initial_state=h0, output_final_state=True)
    assert y.shape == (2, 0, 24) and torch.equal(ht, h0)
    dA, dh0 = torch.autograd.grad(ht, [A, h0], torch.ones_like(ht))
    assert not dA.any() and (dh0 == 1).all()
    none = rn(0, 5, 24)
    y, ht = sophia_b200.gated_recurrence(none, none, none, A, output_final_state=True)
    assert y.shape == (0, 5, 24) and ht.shape == (0, 24)
    x = rn(1, 9, 24)
    y, ht = sophia_b200.gated_recurrence(x, x, x, A)
    assert ht is None
    assert sophia_b200.gated_recurrence_step(rn(0, 24), rn(0, 24), rn(0, 24), A.detach(), rn(3, 24)).shape == (0, 24)


@gpu
def test_refusals():
    rn = gen(0)
    x, A, f = rn(2, 5, 16), -torch.ones(16, device="cuda"), sophia_b200.gated_recurrence
    step = sophia_b200.gated_recurrence_step
    with pytest.raises(ValueError):
        f(x[0], x[0], x[0], A)
    with pytest.raises(ValueError):
        f(x, x[:, :4], x, A)
    with pytest.raises(ValueError):
        f(x, x, x, A[:8])
    with pytest.raises(ValueError):
        f(x, x, x, A, cu_seqlens=torch.tensor([0, 5], device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError):
        f(x, x, x, A, initial_state=rn(3, 16))
    with pytest.raises(AssertionError):
        f(x, x, x, A, initial_state=rn(2, 16, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError):
        f(x.double(), x, x, A)
    with pytest.raises(RuntimeError):
        f(x.cpu(), x, x, A)
    with pytest.raises(RuntimeError):
        f(x, x, x, A.cpu())
    with pytest.raises(ValueError):
        step(x[0], x[0], x[0], A, rn(4, 16))
    with pytest.raises(ValueError):
        step(x[0], x[0], x[0], A, rn(8, 16), slots=torch.zeros(5, device="cuda"))
    with pytest.raises(NotImplementedError):
        step(x[0], x[0], x[0], A.clone().requires_grad_(), rn(8, 16))
    y = f(x.requires_grad_(), x, x, A)[0]
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError):
        g.sum().backward()


@gpu
def test_malformed_table_is_reported():
    x = torch.randn(1, 40, 16, device="cuda")
    cu = torch.tensor([0, 30, 20, 40], device="cuda", dtype=torch.int32)
    sophia_b200.gated_recurrence(x, x, x, -torch.ones(16, device="cuda"), cu_seqlens=cu, output_final_state=True)
    assert sophia_b200._lib.device_error(reset=True) == 3


@gpu
def test_other_stream_captured_and_replayed():
    """The calls run on the caller's stream and in a graph; a replay reads what its inputs hold by then."""
    rn = gen(6)
    ts = inputs(rn, torch.bfloat16, 2, 300, 64, 2)
    dy, dht = rn(2, 300, 64, dtype=torch.bfloat16), rn(2, 64)
    leaves = [ts[k] for k in NAMES]

    def step():
        y, ht = call(ts, None)
        return (y, ht, *torch.autograd.grad((y, ht), leaves, (dy, dht)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        ts["x"].copy_(rn(2, 300, 64, dtype=torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


@gpu
def test_compiled_and_mixed_types():
    rn = gen(8)
    ts = inputs(rn, torch.float32, 2, 70, 48, 2)
    with torch.no_grad():
        ts["x"] = ts["x"].bfloat16()
    ts["x"].requires_grad_()
    y, ht = call(ts, None)
    assert y.dtype == torch.bfloat16
    fn = torch.compile(lambda t: call(t, None), fullgraph=True)
    cy, cht = fn(ts)
    assert torch.equal(cy, y) and torch.equal(cht, ht)
    dy, dht = torch.ones_like(y), torch.ones_like(ht)
    for a, b in zip(torch.autograd.grad((y, ht), [ts[k] for k in NAMES], (dy, dht)),
                    torch.autograd.grad((cy, cht), [ts[k] for k in NAMES], (dy, dht))):
        assert torch.equal(a, b)


@gpu
def test_no_grad_keeps_nothing():
    ts = inputs(gen(1), torch.bfloat16, 1, 512, 64, 1)
    with torch.no_grad():
        y, _ = call(ts, None)
    assert not y.requires_grad
    frozen = {k: v.detach() for k, v in ts.items()}
    y2, _ = call(frozen, None)
    assert torch.equal(y, y2) and y2.grad_fn is None


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinite_gradient_leaves_infinite_sums(dtype):
    """dA and the biases' gradients are sums over the tokens: one infinite term makes them infinite, as the plain sum,
    where it is the only one (a gradient that enters at a sequence's first token reaches no other); other channels
    keep their bits."""
    rn = gen(21)
    E, T = 70, 200
    ts = inputs(rn, dtype, 2, T, E, 2, z=False)
    leaves = [ts[k] for k in SUMS]
    dy = rn(2, T, E, dtype=dtype)
    base = torch.autograd.grad(call(ts, None, False)[0], leaves, dy)
    # the token's own factors from the formulas (autograd adds the two parts of d(A r), which may be inf - inf)
    x, decay, gate, A, db, gb, h0 = (ts[k].detach().double()[i][..., 5] for k, i in (
        ("x", (1, 0)), ("decay", (1, 0)), ("gate", (1, 0)), ("A", ...), ("decay_bias", ...), ("gate_bias", ...), ("h0", 1)))
    r, i = torch.sigmoid(decay + db), torch.sigmoid(gate + gb)
    a = torch.exp(A * r)
    n = torch.sqrt(1 - a * a)
    d_rate = a * h0 - a * a / n * i * x
    want = {"A": d_rate * r, "decay_bias": d_rate * A * r * (1 - r), "gate_bias": n * x * i * (1 - i)}
    rest = torch.arange(E, device="cuda") != 5
    for value in (float("inf"), -float("inf")):
        bad = dy.clone()
        bad[1, 0, 5] = value
        got = torch.autograd.grad(call(ts, None, False)[0], leaves, bad)
        for name, g, b in zip(SUMS, got, base):
            assert g[5] == value * torch.sign(want[name]), name
            assert torch.equal(g[rest], b[rest]), name


@gpu
@pytest.mark.parametrize("dtype,T", [(torch.float32, 75), (torch.bfloat16, 700)])
def test_states_that_forget_at_once(dtype, T):
    """Rates so steep that no state outlives a token, -inf the steepest: h = i x, whatever went before, and
    nothing of the gradients comes through a decay of 0 -- not even times a rate of 1e38.  A closed gate still lets the
    state through."""
    rn = gen(22)
    E = 66
    ts = inputs(rn, dtype, 2, T, E, 2, z=False, biases=False)
    leaves = [ts[k] for k in ("x", "decay", "gate", "A", "h0")]
    dy, dht = rn(2, T, E, dtype=dtype), rn(2, E)
    runs = []
    for rate in (-1e30, -1e34, -1e38, -3.4e38, float("-inf")):
        with torch.no_grad():
            ts["A"].fill_(rate)
        y, ht = call(ts, None)
        runs.append([t.detach() for t in (y, ht, *torch.autograd.grad((y, ht), leaves, (dy, dht)))])
        close("y", y, torch.sigmoid(ts["gate"].detach().double()) * ts["x"].detach().double(), dtype)
        pool = ts["h0"].detach().clone()
        step = sophia_b200.gated_recurrence_step(*(ts[k].detach()[:, 0] for k in ("x", "decay", "gate")), ts["A"].detach(),
                                                 pool)
        assert torch.equal(step, y.detach()[:, 0])
    for run in runs:
        assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))
    d_decay, d_A, d_h0 = runs[0][3], runs[0][5], runs[0][6]
    assert not d_decay.any() and not d_A.any() and not d_h0.any()
    with torch.no_grad():
        ts["decay"].fill_(float("-inf"))
        y, ht = call(ts, None)
    assert torch.equal(ht, ts["h0"].detach()) and torch.equal(y[:, 0], ts["h0"].detach().to(dtype))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_give_the_same_bits(dtype):
    """Expanded, transposed and odd rows against contiguous ones: the copies differ, a channel's arithmetic and the split
    over a cluster's CTAs (both by the sizes alone) do not, forward and backward."""
    rn = gen(16)
    A = -torch.exp(rn(64))

    def run(t):
        t = t.detach().requires_grad_()
        y, ht = sophia_b200.gated_recurrence(t, t, t, A, t, output_final_state=True)
        return y, ht, torch.autograd.grad((y, ht), t, (torch.ones_like(y), torch.ones_like(ht)))[0]

    for t in (rn(1, 300, 64, dtype=dtype).expand(3, 300, 64), rn(3, 1, 64, dtype=dtype).expand(3, 300, 64),
              rn(300, 3, 64, dtype=dtype).transpose(0, 1), rn(3, 64, 300, dtype=dtype).transpose(1, 2),
              rn(3, 300, 67, dtype=dtype)[..., 3:], rn(3, 300, 66, dtype=dtype)[..., 1:65]):
        assert all(torch.equal(a, b) for a, b in zip(run(t), run(t.contiguous())))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [-44.0, -60.0, -80.0])
def test_nearly_closed_input_gates(dtype, shift):
    """Gates of e^-44 to e^-80 let that share of the inputs in, on a state that starts from nothing: the bounds above,
    which are relative to the outputs' own size."""
    rn = gen(24)
    ts = inputs(rn, dtype, 2, 150, 72, 2, state=False)
    ts["gate_bias"] = (ts["gate_bias"].detach() + shift).requires_grad_()
    check(ts, None, rn(2, 150, 72, dtype=dtype), rn(2, 72))
    d = {k: None if v is None else v.detach() for k, v in ts.items()}
    pool = torch.zeros(2, 72, device="cuda")
    y = sophia_b200.gated_recurrence_step(*(d[k][:, 0] for k in ("x", "decay", "gate")), d["A"], pool, d["z"][:, 0],
                                          d["decay_bias"], d["gate_bias"])
    r = {k: None if v is None else v.double() for k, v in d.items()}
    close("step", y, ref.recurrence(*(r[k] for k in NAMES), None)[0][:, 0], dtype)


def test_kept_states_have_the_size_that_the_library_asks_for():
    """What the traced form allocates is what the library computes, at every size."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    lib, op = sophia_b200._lib.load(), torch.ops.sophia_b200.gated_recurrence_fwd.default
    with FakeTensorMode():
        for io, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16)):
            for B, T, E in ((1, 1, 1), (2, 31, 8), (3, 32, 5), (1, 64, 64), (2, 65, 7), (1, 129, 2048), (2, 0, 3)):
                x, A = torch.empty(B, T, E, dtype=dtype, device="cuda"), torch.empty(E, device="cuda")
                y, ht, saved = op(x, x, x, A, None, None, None, None, None, True, True)
                assert y.shape == x.shape and y.dtype == dtype and ht.shape == (B, E)
                assert saved.shape == (lib.kda_b200_recurrence_saved_bytes(B, T, E, io),)
