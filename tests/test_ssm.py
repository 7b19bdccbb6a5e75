"""State-space operators: ``short_conv``, ``selective_scan`` and their single-token
steps, against plain float64 statements of the formulas (``ssm_reference.py``) on
the same inputs, gradients by autograd of those statements and by differences.

Tolerances, derived beforehand.  Kernels compute in fp32 and round once.
* Outputs stored in 16 bits: one rounding, at most 2^-8 (bf16) or 2^-11 (fp16)
  of an element and half of that in the Frobenius norm, plus the fp32 term below.
* fp32: a recurrence adds one rounding (2^-24) per token to a state that remembers up to
  1 / (1 - a) tokens; with the steps used here (d >= 1e-3, A <= -0.5, up to 600
  tokens) that is at most 600 * 2^-24 = 4e-5 of the state's size in the worst case and
  sqrt(600) * 2^-24 = 1.5e-6 typically.  Elements: 1e-4 of max(|ref|, rms(ref)); Frobenius: 1e-5.
"""

from __future__ import annotations

import pytest
import torch

import sophia_b200
import ssm_reference as ref

ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
gpu = pytest.mark.gpu


def close_each(name, got, want, dtype):
    """Every value within its rounding and the arithmetic's error."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, name
    if not want.numel():
        return
    assert torch.isfinite(got).all(), name
    rms = want.square().mean().sqrt()
    tol = ROUND[dtype] * want.abs() + 1e-4 * torch.maximum(want.abs(), rms)
    tol = tol + (2.0 ** -24 if dtype == torch.float16 else 0.0)  # fp16 subnormals
    worst = ((got - want).abs() - tol).max()
    assert worst <= 0, f"{name}: {float((got - want).abs().max())} off, rms {float(rms)}"


def close(name, got, want, dtype):
    close_each(name, got, want, dtype)
    got, want = got.detach().double(), want.detach().double()
    assert (got - want).norm() <= (1e-5 + ROUND[dtype] / 2) * want.norm() + 1e-30, name


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, scale=1.0, dtype=torch.float32: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)


def doubles(ts):
    return {k: (v.detach().double().requires_grad_(v.requires_grad) if v is not None else None) for k, v in ts.items()}


def cu_of(lengths):
    if lengths is None:
        return None
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], device="cuda", dtype=torch.int32)


# --------------------------------------------------------------------------- convolution

CONV = [  # dtype, B, T, C, W, bias, state, silu, documents
    (torch.float32, 1, 1, 1, 4, True, True, True, None),
    (torch.float32, 2, 3, 5, 4, True, True, True, None),
    (torch.float32, 2, 37, 12, 4, False, False, False, None),
    (torch.float32, 3, 130, 9, 3, True, True, True, None),
    (torch.float32, 2, 20, 8, 2, True, True, True, None),
    (torch.float32, 2, 9, 8, 1, True, True, True, None),
    (torch.bfloat16, 2, 200, 64, 4, True, True, True, None),
    (torch.bfloat16, 1, 65, 24, 4, True, False, True, None),
    (torch.float16, 2, 33, 40, 4, True, True, True, None),
    (torch.float32, 1, 40, 8, 4, True, True, True, (1, 2, 3, 0, 1, 17, 9, 7, 0)),
    (torch.bfloat16, 1, 150, 16, 4, True, False, True, (0, 64, 1, 1, 1, 8, 75)),
    (torch.float32, 1, 12, 7, 3, True, True, False, (1, 1, 1, 1, 2, 2, 4)),
]


@gpu
@pytest.mark.parametrize("case", CONV, ids=lambda c: "-".join(str(v).replace("torch.", "").replace(" ", "") for v in c))
def test_conv_forward_and_gradients(case):
    dtype, B, T, C, W, with_bias, with_state, silu, docs = case
    rn, cu = gen(11), cu_of(docs)
    N = len(docs) if docs else B
    ts = {"x": rn(B, T, 2 * C, dtype=dtype)[..., :C].detach().requires_grad_(),  # a slice: strided rows
          "weight": rn(C, W, scale=0.5).requires_grad_(),
          "bias": rn(C, scale=0.2).requires_grad_() if with_bias else None,
          "h0": rn(N, C, W - 1).requires_grad_() if with_state else None}
    y, ht = sophia_b200.short_conv(ts["x"], ts["weight"], ts["bias"], activation="silu" if silu else None,
                                   initial_state=ts["h0"], output_final_state=True, cu_seqlens=cu)
    dy, dht = rn(B, T, C, dtype=dtype), rn(N, C, W - 1)
    leaves = [k for k, v in ts.items() if v is not None]
    got = torch.autograd.grad((y, ht), [ts[k] for k in leaves], (dy, dht))
    r = doubles(ts)
    ry, rht = ref.conv(r["x"], r["weight"], r["bias"], r["h0"], cu, silu)
    want = torch.autograd.grad((ry, rht), [r[k] for k in leaves], (dy.double(), dht.double()), allow_unused=True)
    assert y.dtype == dtype and ht.dtype == torch.float32
    close("y", y, ry, dtype)
    close("final_state", ht, rht, torch.float32)
    for k, a, b in zip(leaves, got, want):
        close("d_" + k, a, torch.zeros_like(a) if b is None else b, ts[k].dtype)
    assert sophia_b200._lib.device_error(reset=True) == 0


@gpu
def test_conv_steps_continue_a_prompt():
    rn = gen(5)
    x, w, b = rn(3, 20, 48, dtype=torch.bfloat16), rn(48, 4, scale=0.5), rn(48)
    whole, _ = sophia_b200.short_conv(x, w, b)
    y, state = sophia_b200.short_conv(x[:, :13], w, b, output_final_state=True)
    assert torch.equal(y, whole[:, :13])
    pool = torch.zeros(6, 48, 3, device="cuda")
    slots = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
    pool[slots.long()] = state
    for t in range(13, 20):
        assert torch.equal(sophia_b200.short_conv_step(x[:, t], pool, w, b, slots=slots), whole[:, t])
    _, final = sophia_b200.short_conv(x, w, b, output_final_state=True)
    assert torch.equal(pool[slots.long()], final)
    assert not pool[[1, 3, 5]].any()


# --------------------------------------------------------------------------- scan


def scan_tensors(dtype, B, T, E, N, G, gate, skip, bias, state, docs, seed=3):
    rn = gen(seed)
    nseq = len(docs) if docs else B
    wide = rn(B, T, 2 * E, dtype=dtype)
    bc = rn(B, T, 2 * G * N, dtype=dtype)
    leaf = lambda t: t.detach().requires_grad_()  # noqa: E731
    ts = {"x": leaf(wide[..., :E]), "dt": leaf(rn(B, T, E, scale=0.7, dtype=dtype)),
          "A": leaf(-torch.exp(rn(E, N, scale=0.7))),
          "B": leaf(bc[..., :G * N].reshape(B, T, G, N)), "C": leaf(bc[..., G * N:].reshape(B, T, G, N)),
          "D": leaf(rn(E)) if skip else None, "z": leaf(wide[..., E:]) if gate else None,
          "dt_bias": leaf(rn(E) - 2.0) if bias else None, "h0": leaf(rn(nseq, E, N)) if state else None}
    return ts, rn(B, T, E, dtype=dtype), rn(nseq, E, N)


SCAN = [  # dtype, B, T, E, N, G, gate, skip, bias, state, softplus, documents
    (torch.float32, 1, 1, 1, 1, 1, True, True, True, True, True, None),
    (torch.float32, 2, 7, 3, 16, 1, True, True, True, True, True, None),
    (torch.float32, 1, 9, 16, 16, 1, False, False, False, False, True, None),
    (torch.float32, 2, 255, 20, 16, 1, True, True, True, False, True, None),
    (torch.float32, 1, 256, 17, 8, 1, True, True, True, True, True, None),
    (torch.float32, 1, 257, 34, 5, 2, False, True, True, True, True, None),
    (torch.float32, 1, 600, 16, 16, 1, True, True, True, True, True, None),
    (torch.float32, 2, 64, 70, 24, 1, True, True, True, True, True, None),   # padded states: 24 of 32
    (torch.float32, 1, 65, 64, 64, 1, False, True, True, True, True, None),
    (torch.float32, 1, 130, 40, 33, 2, True, True, False, True, True, None),
    (torch.float32, 2, 70, 450, 3, 150, True, True, True, True, True, None),  # many groups: four states a lane
    (torch.float32, 2, 70, 448, 16, 64, True, True, True, True, True, None),
    (torch.float32, 2, 37, 480, 32, 60, False, True, True, True, True, None),
    (torch.float32, 1, 75, 320, 7, 80, True, True, True, True, True, (1, 2, 0, 7, 8, 9, 1, 47)),
    (torch.bfloat16, 2, 61, 640, 16, 80, True, True, True, True, True, None),
    (torch.bfloat16, 2, 130, 32, 16, 1, True, True, True, True, True, None),
    (torch.bfloat16, 1, 300, 48, 16, 2, True, True, True, False, True, None),
    (torch.bfloat16, 1, 100, 64, 32, 1, True, True, True, True, True, None),
    (torch.float16, 2, 66, 24, 16, 1, True, True, True, True, True, None),
    (torch.float32, 1, 60, 18, 16, 1, True, True, True, True, True, (1, 2, 0, 7, 8, 9, 1, 32, 0)),
    (torch.float32, 1, 530, 16, 16, 1, True, True, True, True, True, (255, 1, 1, 200, 73)),
    (torch.float32, 1, 530, 16, 16, 1, False, False, True, False, True, (256, 0, 256, 18)),
    (torch.float32, 1, 140, 66, 20, 1, True, True, True, True, True, (63, 1, 64, 0, 12)),
    (torch.bfloat16, 1, 290, 40, 16, 1, True, True, True, False, True, (0, 3, 100, 187)),
]


def run_scan(ts, cu, softplus, dy, dht):
    y, ht = sophia_b200.selective_scan(ts["x"], ts["dt"], ts["A"], ts["B"], ts["C"], ts["D"], ts["z"], ts["dt_bias"],
                                       dt_softplus=softplus, initial_state=ts["h0"], output_final_state=True,
                                       cu_seqlens=cu)
    leaves = [k for k, v in ts.items() if v is not None]
    return y, ht, dict(zip(leaves, torch.autograd.grad((y, ht), [ts[k] for k in leaves], (dy, dht))))


def reference_scan(ts, cu, softplus, dy, dht):
    r = doubles(ts)
    y, ht = ref.scan(r["x"], r["dt"], r["A"], r["B"], r["C"], r["D"], r["z"], r["dt_bias"], r["h0"], cu, softplus)
    leaves = [k for k, v in r.items() if v is not None]
    return y, ht, dict(zip(leaves, torch.autograd.grad((y, ht), [r[k] for k in leaves], (dy.double(), dht.double()))))


@gpu
@pytest.mark.parametrize("case", SCAN, ids=lambda c: "-".join(str(v).replace("torch.", "").replace(" ", "") for v in c))
def test_scan_forward_and_gradients(case):
    dtype, B, T, E, N, G, gate, skip, bias, state, softplus, docs = case
    ts, dy, dht = scan_tensors(dtype, B, T, E, N, G, gate, skip, bias, state, docs)
    cu = cu_of(docs)
    y, ht, grads = run_scan(ts, cu, softplus, dy, dht)
    ry, rht, want = reference_scan(ts, cu, softplus, dy, dht)
    assert y.dtype == dtype and ht.dtype == torch.float32
    close("y", y, ry, dtype)
    close("final_state", ht, rht, torch.float32)
    assert set(grads) == set(want)
    for k in want:
        close("d_" + k, grads[k], want[k], ts[k].dtype)
    assert sophia_b200._lib.device_error(reset=True) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [4, 16, 5, 48])
def test_sequences_start_and_end_at_every_place_of_a_segment(dtype, N):
    """Value by value: a few dozen outputs are too few for a bound on their mean rounding."""
    for tail in [(1,), (2,), (3,), (4,), (5,), (6,), (7,), (8,), (1, 1), (1, 1, 1), (2, 3, 1), (1, 0, 8)]:
        for T in (8, 21, 56):
            docs = (T - sum(tail), *tail) if T > sum(tail) else tail
            ts, dy, dht = scan_tensors(dtype, 1, sum(docs), 12, N, 1, True, True, True, True, docs)
            cu = cu_of(docs)
            y, ht, grads = run_scan(ts, cu, True, dy, dht)
            ry, rht, want = reference_scan(ts, cu, True, dy, dht)
            close_each("y", y, ry, dtype)
            close_each("final_state", ht, rht, torch.float32)
            for k in want:
                close_each("d_" + k, grads[k], want[k], ts[k].dtype)


SPANS = [  # few channels and many tokens: the tokens are cut into spans
    (torch.float32, 1, 1500, 8, 16, 1, True, None),
    (torch.float32, 2, 1111, 40, 5, 2, True, None),
    (torch.bfloat16, 1, 2049, 24, 16, 1, False, None),
    (torch.float32, 1, 1400, 8, 16, 1, True, (64, 1, 63, 127, 1, 0, 500, 2, 642)),
    (torch.bfloat16, 1, 1030, 16, 32, 1, True, (1, 1028, 1)),
    (torch.float16, 1, 777, 20, 8, 1, False, (255, 1, 521)),
    (torch.float32, 3, 600, 72, 64, 1, True, None),
]


@gpu
@pytest.mark.parametrize("case", SPANS, ids=lambda c: "-".join(str(v).replace("torch.", "").replace(" ", "") for v in c))
def test_scan_of_few_rows(case):
    dtype, B, T, E, N, G, state, docs = case
    ts, dy, dht = scan_tensors(dtype, B, T, E, N, G, True, True, True, state, docs)
    cu = cu_of(docs)
    y, ht, grads = run_scan(ts, cu, True, dy, dht)
    ry, rht, want = reference_scan(ts, cu, True, dy, dht)
    close("y", y, ry, dtype)
    close("final_state", ht, rht, torch.float32)
    for k in want:
        close("d_" + k, grads[k], want[k], ts[k].dtype)


@gpu
def test_spans_keep_infinities_and_growing_states():
    """A state that grows (positive rates) and one that is infinite cross the spans; a document behind
    them sees neither."""
    E, N, T = 8, 4, 1000
    rn = gen(5)
    x, Bm, Cm = rn(1, T, E), rn(1, T, N), rn(1, T, N)
    dt = torch.full((1, T, E), 0.02, device="cuda")
    A = torch.full((E, N), 0.5, device="cuda")
    y, _ = sophia_b200.selective_scan(x, dt, A, Bm, Cm, dt_softplus=False)
    want, _ = ref.scan(x.double(), dt.double(), A.double(), Bm[:, :, None].double(), Cm[:, :, None].double(), None, None,
                       None, None, None, False)
    assert torch.isfinite(y).all()
    assert ((y.double() - want).norm() <= 1e-4 * want.norm())
    x[:, 100, 3] = float("inf")
    cu = cu_of((700, 300))
    y, ht = sophia_b200.selective_scan(x, dt, -A, Bm, Cm, dt_softplus=False, cu_seqlens=cu, output_final_state=True)
    assert not torch.isfinite(y[:, 100:700, 3]).any() and not torch.isfinite(ht[0, 3]).any()
    assert torch.isfinite(y[:, :100]).all() and torch.isfinite(y[:, 700:]).all() and torch.isfinite(ht[1]).all()
    assert torch.isfinite(y[:, :, [0, 1, 2, 4, 5, 6, 7]]).all()


@gpu
def test_scan_without_softplus_takes_positive_steps():
    ts, dy, dht = scan_tensors(torch.float32, 2, 90, 24, 16, 1, True, True, False, True, None)
    ts["dt"] = (ts["dt"].detach().abs() * 0.1).requires_grad_()
    y, ht, grads = run_scan(ts, None, False, dy, dht)
    ry, rht, want = reference_scan(ts, None, False, dy, dht)
    close("y", y, ry, torch.float32)
    close("final_state", ht, rht, torch.float32)
    for k in want:
        close("d_" + k, grads[k], want[k], torch.float32)


@gpu
def test_a_step_of_zero_leaves_the_state():
    ts, _, _ = scan_tensors(torch.float32, 1, 40, 8, 16, 1, False, False, False, True, None)
    zero = torch.zeros(1, 40, 8, device="cuda")
    _, ht = sophia_b200.selective_scan(ts["x"].detach(), zero, ts["A"].detach(), ts["B"].detach(), ts["C"].detach(),
                                       dt_softplus=False, initial_state=ts["h0"].detach(), output_final_state=True)
    assert torch.equal(ht, ts["h0"].detach())


@gpu
def test_scan_gradient_agrees_with_differences():
    """Directional differences of the fp32 kernel's own loss: a central difference with
    step 2^-6 has a truncation error of order 2^-12 of the third derivative and a rounding
    error of 2^-24 |loss| / 2^-6; 2e-3 of the gradient's norm times the direction's covers both."""
    ts, dy, dht = scan_tensors(torch.float32, 1, 40, 8, 4, 1, True, True, True, True, None, seed=9)
    _, _, grads = run_scan(ts, None, True, dy, dht)

    def loss(t):
        with torch.no_grad():
            y, ht = sophia_b200.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"], t["z"], t["dt_bias"],
                                               initial_state=t["h0"], output_final_state=True)
            return float((y.double() * dy.double()).sum() + (ht.double() * dht.double()).sum())

    rn = gen(21)
    for k in ts:
        v = rn(*ts[k].shape)
        v = v / v.norm()
        step = 2.0 ** -6
        up, down = loss({**ts, k: ts[k].detach() + step * v}), loss({**ts, k: ts[k].detach() - step * v})
        slope = float((grads[k].double() * v.double()).sum())
        assert abs((up - down) / (2 * step) - slope) <= 2e-3 * float(grads[k].norm()), k


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,G", [(16, 1), (5, 2), (40, 1)])
def test_scan_steps_continue_a_prompt(dtype, N, G):
    E, T, T0 = 26, 30, 21
    ts, _, _ = scan_tensors(dtype, 3, T, E, N, G, True, True, True, True, None)
    ts = {k: v.detach() for k, v in ts.items()}
    args = lambda sl: [ts["x"][:, sl], ts["dt"][:, sl], ts["A"], ts["B"][:, sl], ts["C"][:, sl]]  # noqa: E731
    rest = lambda sl: [ts["D"], ts["z"][:, sl], ts["dt_bias"]]  # noqa: E731
    whole, final = sophia_b200.selective_scan(*args(slice(0, T)), *rest(slice(0, T)), initial_state=ts["h0"],
                                              output_final_state=True)
    _, state = sophia_b200.selective_scan(*args(slice(0, T0)), *rest(slice(0, T0)), initial_state=ts["h0"],
                                          output_final_state=True)
    pool = torch.full((5, E, N), 7.0, device="cuda")
    slots = torch.tensor([3, 1, 0], device="cuda", dtype=torch.int32)
    pool[slots.long()] = state
    for t in range(T0, T):
        y = sophia_b200.selective_scan_step(*args(t), pool, *rest(t), slots=slots)
        close("y", y, whole[:, t], dtype)
    close("state", pool[slots.long()], final, torch.float32)
    assert (pool[[2, 4]] == 7.0).all()


@gpu
def test_padding_rows_and_slots_past_the_pool():
    rn = gen(2)
    x, w = rn(4, 8), rn(8, 4)
    pool, slots = rn(2, 8, 3), torch.tensor([1, -1, 0, 5], device="cuda", dtype=torch.int32)
    before = pool.clone()
    y = sophia_b200.short_conv_step(x, pool, w, slots=slots)
    assert not y[1].any() and not y[3].any() and y[0].any() and y[2].any()
    assert torch.equal(pool[1, :, :2], before[1, :, 1:]) and torch.equal(pool[1, :, 2], x[0])
    assert sophia_b200._lib.device_error(reset=True) == 11
    state, A, b = rn(2, 8, 16), -torch.exp(rn(8, 16)), rn(4, 16)
    kept = state.clone()
    y = sophia_b200.selective_scan_step(x, x, A, b, b, state, slots=torch.tensor([-1, -7, 1, 2], device="cuda",
                                                                               dtype=torch.int32))
    assert not y[[0, 1, 3]].any() and y[2].any() and torch.equal(state[0], kept[0]) and not torch.equal(state, kept)
    assert sophia_b200._lib.device_error(reset=True) == 11


@gpu
def test_infinities_and_nan_stay_in_their_sequence_channel_and_past():
    docs = (20, 30, 25)
    cu = cu_of(docs)
    ts, dy, _ = scan_tensors(torch.float32, 1, 75, 12, 16, 1, True, True, True, False, docs)
    ts = {k: None if v is None else v.detach() for k, v in ts.items()}
    call = lambda x: sophia_b200.selective_scan(x, ts["dt"], ts["A"], ts["B"], ts["C"], ts["D"], ts["z"],  # noqa: E731
                                                ts["dt_bias"], cu_seqlens=cu, output_final_state=True)
    y, ht = call(ts["x"])
    for bad in (float("inf"), float("nan")):
        x = ts["x"].clone()
        x[0, 33, 4] = bad
        by, bht = call(x)
        touched = torch.zeros_like(y, dtype=torch.bool)
        touched[0, 33:50, 4] = True
        assert torch.equal(by[~touched], y[~touched]) and not torch.isfinite(by[touched]).any()
        assert torch.equal(bht[[0, 2]], ht[[0, 2]])
        xg = x.clone().requires_grad_()
        by, _ = call(xg)
        (dx,) = torch.autograd.grad(by, xg, dy)
        assert torch.isfinite(dx[0, :20]).all() and torch.isfinite(dx[0, 50:]).all()
        # a convolution: the taps reach three tokens on and not past the document
        w = gen(1)(12, 2)
        c0, _ = sophia_b200.short_conv(ts["x"], w, cu_seqlens=cu)
        c1, _ = sophia_b200.short_conv(x, w, cu_seqlens=cu)
        far = torch.ones_like(c0, dtype=torch.bool)
        far[0, 33:35, 4] = False
        assert torch.equal(c1[far], c0[far]) and not torch.isfinite(c1[0, 33, 4])


@gpu
def test_results_do_not_depend_on_the_call():
    ts, dy, dht = scan_tensors(torch.float32, 2, 300, 40, 16, 1, True, True, True, True, None)
    first = run_scan(ts, None, True, dy, dht)
    for _ in range(3):
        again = run_scan(ts, None, True, dy, dht)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        for k in first[2]:
            assert torch.equal(first[2][k], again[2][k]), k


@gpu
def test_packed_documents_equal_the_documents_alone():
    docs = (70, 1, 300, 129)
    cu = cu_of(docs)
    ts, _, _ = scan_tensors(torch.bfloat16, 1, 500, 32, 16, 1, True, True, True, True, docs)
    ts = {k: v.detach() for k, v in ts.items()}
    y, ht = sophia_b200.selective_scan(ts["x"], ts["dt"], ts["A"], ts["B"], ts["C"], ts["D"], ts["z"], ts["dt_bias"],
                                       initial_state=ts["h0"], output_final_state=True, cu_seqlens=cu)
    at = 0
    for i, n in enumerate(docs):
        sl = slice(at, at + n)
        y1, h1 = sophia_b200.selective_scan(*(ts[k][:, sl] for k in ("x", "dt")), ts["A"], ts["B"][:, sl],
                                            ts["C"][:, sl], ts["D"], ts["z"][:, sl], ts["dt_bias"],
                                            initial_state=ts["h0"][i:i + 1], output_final_state=True)
        close("y", y[:, sl], y1, torch.bfloat16)
        close("state", ht[i], h1[0], torch.float32)
        at += n


@gpu
def test_empty_tokens_pass_the_state_through():
    h0 = gen(4)(2, 6, 16).requires_grad_()
    e = torch.empty(2, 0, 6, device="cuda")
    bc = torch.empty(2, 0, 16, device="cuda")
    A = torch.full((6, 16), -1.0, device="cuda", requires_grad=True)
    y, ht = sophia_b200.selective_scan(e, e, A, bc, bc, initial_state=h0, output_final_state=True)
    assert y.shape == (2, 0, 6) and torch.equal(ht, h0)
    dh0, dA = torch.autograd.grad(ht, (h0, A), torch.ones_like(ht))
    assert (dh0 == 1).all() and not dA.any()
    c0 = gen(4)(2, 6, 3)
    w = torch.ones(6, 4, device="cuda", requires_grad=True)
    y, ct = sophia_b200.short_conv(e, w, initial_state=c0, output_final_state=True)
    assert torch.equal(ct, c0) and not torch.autograd.grad(y.sum(), w)[0].any()


@gpu
def test_mixed_types_expanded_rows_and_transposed_views():
    """Types promote to fp32; a broadcast gate and a view with no contiguous dimension are read right."""
    ts, dy, _ = scan_tensors(torch.float32, 2, 50, 16, 16, 1, True, True, True, False, None)
    x = ts["x"].detach().to(torch.bfloat16).requires_grad_()
    z = ts["z"].detach()[:, :1].requires_grad_()
    dt = ts["dt"].detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    y, _ = sophia_b200.selective_scan(x, dt, ts["A"], ts["B"], ts["C"], ts["D"], z.expand(2, 50, 16), ts["dt_bias"])
    dx, dz, ddt = torch.autograd.grad(y, (x, z, dt), dy.to(torch.bfloat16))
    r = doubles({**ts, "x": x, "z": z, "dt": dt})
    ry, _ = ref.scan(r["x"], r["dt"], r["A"], r["B"], r["C"], r["D"], r["z"].expand(2, 50, 16), r["dt_bias"], None,
                     None, True)
    wx, wz, wdt = torch.autograd.grad(ry, (r["x"], r["z"], r["dt"]), dy.to(torch.bfloat16).double())
    assert y.dtype == torch.bfloat16
    close("y", y, ry, torch.bfloat16)
    close("dx", dx, wx, torch.bfloat16)
    close("dz", dz, wz, torch.float32)
    close("ddt", ddt, wdt, torch.float32)


@gpu
def test_calls_follow_the_current_stream_and_fit_a_graph():
    ts, dy, dht = scan_tensors(torch.bfloat16, 1, 200, 32, 16, 1, True, True, True, True, None)
    ts = {k: v.detach() for k, v in ts.items()}
    call = lambda: sophia_b200.selective_scan(ts["x"], ts["dt"], ts["A"], ts["B"], ts["C"], ts["D"], ts["z"],  # noqa: E731
                                              ts["dt_bias"], initial_state=ts["h0"], output_final_state=True)
    want, _ = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = call()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@gpu
def test_a_malformed_table_is_reported():
    x, w = gen(1)(1, 12, 8), gen(2)(8, 4)
    bad = torch.tensor([0, 9, 4, 12], device="cuda", dtype=torch.int32)
    sophia_b200.short_conv(x, w, cu_seqlens=bad, output_final_state=True)
    assert sophia_b200._lib.device_error(reset=True) == 3


# --------------------------------------------------------------------------- refusals (no GPU)


def _meta(*s, dtype=torch.float32):
    return torch.empty(*s, device="meta", dtype=dtype)


def test_conv_refusals():
    x, w = _meta(2, 5, 8), _meta(8, 4)
    cases = [
        (ValueError, lambda: sophia_b200.short_conv(x, _meta(7, 4))),
        (ValueError, lambda: sophia_b200.short_conv(x, _meta(8))),
        (NotImplementedError, lambda: sophia_b200.short_conv(x, _meta(8, 5))),
        (ValueError, lambda: sophia_b200.short_conv(x, w, _meta(4))),
        (ValueError, lambda: sophia_b200.short_conv(x, w, activation="gelu")),
        (ValueError, lambda: sophia_b200.short_conv(x, w, initial_state=_meta(2, 8, 4))),
        (AssertionError, lambda: sophia_b200.short_conv(x, w, initial_state=_meta(2, 8, 3, dtype=torch.bfloat16))),
        (ValueError, lambda: sophia_b200.short_conv(x, w, cu_seqlens=_meta(3, dtype=torch.int32))),
        (ValueError, lambda: sophia_b200.short_conv(_meta(1, 5, 8), w, cu_seqlens=_meta(3))),
        (NotImplementedError, lambda: sophia_b200.short_conv(_meta(2, 5, 8, dtype=torch.float64), w)),
        (RuntimeError, lambda: sophia_b200.short_conv(torch.zeros(2, 5, 8), torch.zeros(8, 4))),
        (ValueError, lambda: sophia_b200.short_conv_step(_meta(3, 8), _meta(2, 8, 3), w)),
        (ValueError, lambda: sophia_b200.short_conv_step(_meta(3, 8), _meta(4, 8, 2), w)),
        (ValueError, lambda: sophia_b200.short_conv_step(_meta(3, 8), _meta(4, 8, 3), w, slots=_meta(3))),
        (NotImplementedError, lambda: sophia_b200.short_conv_step(_meta(3, 8).requires_grad_(), _meta(4, 8, 3), w)),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()


def test_scan_refusals():
    x, A, b = _meta(2, 5, 8), _meta(8, 16), _meta(2, 5, 16)
    good = dict(x=x, dt=x, A=A, B=b, C=b)
    cases = [
        (ValueError, dict(dt=_meta(2, 5, 7))),
        (ValueError, dict(A=_meta(7, 16))),
        (ValueError, dict(B=_meta(2, 5, 15))),
        (ValueError, dict(C=_meta(2, 4, 16))),
        (ValueError, dict(B=_meta(2, 5, 3, 16), C=_meta(2, 5, 3, 16))),
        (NotImplementedError, dict(A=_meta(8, 65), B=_meta(2, 5, 65), C=_meta(2, 5, 65))),
        (ValueError, dict(D=_meta(7))),
        (ValueError, dict(dt_bias=_meta(9))),
        (ValueError, dict(z=_meta(2, 5, 9))),
        (ValueError, dict(initial_state=_meta(3, 8, 16))),
        (AssertionError, dict(initial_state=_meta(2, 8, 16, dtype=torch.float16))),
        (ValueError, dict(cu_seqlens=_meta(3, dtype=torch.int32))),
        (NotImplementedError, dict(x=_meta(2, 5, 8, dtype=torch.int32))),
        (RuntimeError, {k: torch.zeros(v.shape) for k, v in good.items()}),
    ]
    for error, change in cases:
        with pytest.raises(error):
            sophia_b200.selective_scan(**{**good, **change})
    step = dict(x=_meta(3, 8), dt=_meta(3, 8), A=A, B=_meta(3, 16), C=_meta(3, 16), state=_meta(3, 8, 16))
    for error, change in [(ValueError, dict(state=_meta(2, 8, 16))), (ValueError, dict(state=_meta(3, 8, 15))),
                          (ValueError, dict(state=_meta(3, 8, 16, dtype=torch.bfloat16))),
                          (ValueError, dict(slots=_meta(2, dtype=torch.int32))),
                          (NotImplementedError, dict(dt=_meta(3, 8).requires_grad_()))]:
        with pytest.raises(error):
            sophia_b200.selective_scan_step(**{**step, **change})


def test_ops_trace_under_compile():
    """The custom ops' fakes and autograd formulas, without a GPU."""
    m = lambda *s, dt=torch.bfloat16: _meta(*s, dtype=dt).requires_grad_()  # noqa: E731
    f = lambda *s: m(*s, dt=torch.float32)  # noqa: E731

    def step(x, w, b, dt, A, B, C, D, z, bias, h0):
        c, _ = sophia_b200.short_conv(x, w, b)
        y, ht = sophia_b200.selective_scan(c, dt, A, B, C, D, z, bias, initial_state=h0, output_final_state=True)
        return y, ht

    args = (m(2, 70, 32), f(32, 4), f(32), m(2, 70, 32), f(32, 16), m(2, 70, 2, 16), m(2, 70, 2, 16), f(32), m(2, 70, 32),
            f(32), f(2, 32, 16))
    y, ht = torch.compile(step, backend="aot_eager", fullgraph=True)(*args)
    assert y.shape == (2, 70, 32) and y.dtype == torch.bfloat16 and ht.shape == (2, 32, 16)
    (y.float().sum() + ht.sum()).backward()
    for a in args:
        assert a.grad is not None and a.grad.shape == a.shape and a.grad.dtype == a.dtype
