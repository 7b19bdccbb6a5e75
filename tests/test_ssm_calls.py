"""How the state-space operators are called: grad modes, derivatives that they do not have, compilation
for changing lengths, and single tokens after long prompts."""

from __future__ import annotations

import contextlib

import pytest
import torch

import sophia_b200
from sophia_b200 import ssm

gpu = pytest.mark.gpu


def _meta(*s, dtype=torch.float32):
    return torch.empty(*s, device="meta", dtype=dtype)


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, scale=1.0, dtype=torch.float32: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)


MODES = {"grad": contextlib.nullcontext, "no_grad": torch.no_grad, "inference": torch.inference_mode}


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("parameters", [False, True])
def test_states_are_kept_for_a_backward_alone(monkeypatch, mode, parameters):
    """Parameters among the inputs are no reason to keep states where no graph is built."""
    asked = []

    def forward(x, dt, A, B, C, D, z, dt_bias, h0, cu, softplus, want_final, training):
        asked.append(training)
        return x.new_empty(x.shape), x.new_empty(0, dtype=torch.float32), x.new_empty(0, dtype=torch.uint8)

    monkeypatch.setattr(ssm, "_scan_fwd_impl", forward)
    leaf = (lambda t: torch.nn.Parameter(t)) if parameters else (lambda t: t)
    A, D, bias = leaf(_meta(8, 16)), leaf(_meta(8)), leaf(_meta(8))
    with MODES[mode]():
        x, b = _meta(2, 40, 8), _meta(2, 40, 16)
        y, _ = sophia_b200.selective_scan(x, x, A, b, b, D, None, bias)
    assert asked == [mode == "grad" and parameters]
    assert y.requires_grad == asked[0]


@gpu
@pytest.mark.parametrize("mode", ["no_grad", "inference"])
def test_a_prompt_allocates_no_checkpoints(mode):
    """The memory of a call with Parameters under no_grad: y, the final state and the spans' workspace,
    far less than the checkpoints of a training call."""
    B, T, E, N = 1, 2048, 512, 16
    rn = gen(1)
    x, z, dt, Bm, Cm = rn(B, T, E), rn(B, T, E), rn(B, T, E), rn(B, T, N), rn(B, T, N)
    A, D, bias = (torch.nn.Parameter(t) for t in (-torch.exp(rn(E, N)), rn(E), rn(E)))
    lib = sophia_b200._lib.load()
    saved = lib.kda_b200_scan_saved_bytes(B, T, E, N, 1)
    ws = lib.kda_b200_scan_workspace_bytes(B, T, E, N, 1, 0, 0)

    def peak(context):
        with context():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y, ht = sophia_b200.selective_scan(x, dt, A, Bm, Cm, D, z, bias, output_final_state=True)
            torch.cuda.synchronize()
            return torch.cuda.max_memory_allocated() - before, y.detach().clone(), ht.detach().clone()

    want = B * T * E * 4 + B * E * N * 4 + ws
    got, y, ht = peak(MODES[mode])
    # the allocator may hand out up to 1 MB more than each of the three large buffers needs
    assert got <= want + (3 << 20) < want + saved, (got, want, saved)
    trained, y1, h1 = peak(MODES["grad"])
    assert trained >= got + saved // 2
    assert torch.equal(y, y1) and torch.equal(ht, h1)


@gpu
@pytest.mark.parametrize("call", ["conv_step", "scan_step", "put_states", "clip", "clip_out", "clip_copy"])
def test_a_graph_notices_what_is_written_in_place(call):
    """A tensor that a graph saved and a call then rewrote: backward refuses, as behind torch's own in-place operations."""
    rn = gen(3)
    written = rn(4, 6, 3)
    w = rn(4, 6, 3).requires_grad_()
    loss = (w * written).sum()  # saves `written`
    x, slots = rn(4, 6), torch.arange(4, device="cuda", dtype=torch.int32)
    if call == "conv_step":
        sophia_b200.short_conv_step(x, written, rn(6, 4))
    elif call == "scan_step":
        sophia_b200.selective_scan_step(x, x, -torch.ones(6, 3, device="cuda"), rn(4, 3), rn(4, 3), written)
    elif call == "put_states":
        ssm.put_states(rn(4, 6, 3), written, slots)
    elif call == "clip":
        sophia_b200.clip_grad_norm_([written], 0.1)
    elif call == "clip_out":
        sophia_b200.clip_grad_norm_([rn(4, 6, 3)], 0.1, out=[written])
    else:
        sophia_b200.clip_grad_norm_([rn(4, 6, 3)], 0.1, out=[written.transpose(0, 1).contiguous().transpose(0, 1), ])
        sophia_b200.clip_grad_norm_([written, rn(6, 8)[:, ::2]], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@gpu
def test_inference_tensors_are_written():
    rn = gen(3)
    with torch.inference_mode():
        pool, grad = torch.zeros(4, 6, 3, device="cuda"), torch.ones(6, device="cuda")
        sophia_b200.short_conv_step(rn(4, 6), pool, rn(6, 4))
        sophia_b200.clip_grad_norm_([grad], 0.1)
        assert pool[:, :, 2].any() and float(grad[0]) < 0.1


def test_kept_states_have_the_size_that_the_library_asks_for():
    """What the traced form allocates is what the library computes, at every size."""
    lib = sophia_b200._lib.load()
    op = torch.ops.sophia_b200.selective_scan_fwd
    for b, T, E, N, G in [(1, 1, 1, 1, 1), (1, 0, 4, 4, 1), (2, 7, 3, 16, 1), (1, 8, 6, 5, 2), (3, 9, 8, 64, 4), (1, 257, 34, 33, 2)]:
        with torch._subclasses.FakeTensorMode():
            y, _, saved = op(torch.empty(b, T, E, device="cuda"), torch.empty(b, T, E, device="cuda"),
                             torch.empty(E, N, device="cuda"), torch.empty(b, T, G, N, device="cuda"),
                             torch.empty(b, T, G, N, device="cuda"), None, None, None, None, None, True, False, True)
        assert saved.numel() == lib.kda_b200_scan_saved_bytes(b, T, E, N, G) and y.shape == (b, T, E)


def test_changing_lengths_compile_once():
    """Training steps of other token counts run the code that the first ones compiled."""
    from torch._dynamo.testing import CompileCounterWithBackend

    counter = CompileCounterWithBackend("aot_eager")

    def step(x, w, dt, A, B, C):
        c, _ = sophia_b200.short_conv(x, w)
        return sophia_b200.selective_scan(c, dt, A, B, C)[0]

    run = torch.compile(step, backend=counter, fullgraph=True, dynamic=True)
    w, A = _meta(32, 4).requires_grad_(), _meta(32, 16).requires_grad_()
    for T in (70, 91, 128, 260, 33, 1000):
        x, dt, bc = _meta(2, T, 32).requires_grad_(), _meta(2, T, 32).requires_grad_(), _meta(2, T, 16).requires_grad_()
        y = run(x, w, dt, A, bc, bc)
        y.sum().backward()
        assert x.grad.shape == x.shape and bc.grad.shape == bc.shape
    assert counter.frame_count == 1


def _without_kernels(monkeypatch):
    """Both operators on meta tensors, their kernels replaced by allocations."""
    empty = lambda t, dtype=None: None if t is None else t.new_empty(t.shape, dtype=dtype or t.dtype)  # noqa: E731
    none = lambda x: x.new_empty(0, dtype=torch.float32)  # noqa: E731
    monkeypatch.setattr(ssm, "_conv_fwd_impl", lambda x, *r: (empty(x), none(x)))
    monkeypatch.setattr(ssm, "_conv_bwd_impl", lambda x, w, b, h0, cu, dy, dht, silu, want: (
        empty(x), empty(w), empty(b), none(x)))
    monkeypatch.setattr(ssm, "_scan_fwd_impl", lambda x, *r: (empty(x), none(x), x.new_empty(0, dtype=torch.uint8)))
    monkeypatch.setattr(ssm, "_scan_bwd_impl", lambda x, dt, A, B, C, D, z, bias, h0, cu, saved, dy, dht, sp, want: (
        empty(x), empty(dt), empty(A), empty(B), empty(C), empty(D), empty(z), empty(bias), none(x)))


@pytest.mark.parametrize("leaf", ["x", "weight", "dy"])
def test_second_derivatives_are_refused(monkeypatch, leaf):
    """A gradient penalty would count the gradient as a constant and lose its part of the loss silently."""
    _without_kernels(monkeypatch)
    g = {k: _meta(2, 9, 8) for k in ("x", "dy")}
    g["weight"] = _meta(8, 4)
    g[leaf].requires_grad_()
    for call in (lambda: sophia_b200.short_conv(g["x"] + 0, g["weight"], g["bias"])[0],
                 lambda: sophia_b200.selective_scan(g["x"] + 0, g["x"] + 0, -g["weight"], g["b"], g["b"], g["bias"])[0]):
        g["bias"], g["b"] = _meta(8).requires_grad_(), _meta(2, 9, 4)
        (db,) = torch.autograd.grad(call(), g["bias"], g["dy"], create_graph=True)
        assert db.requires_grad
        with pytest.raises(NotImplementedError, match="no second derivative"):
            (db.square().sum() + g[leaf].sum()).backward()


def test_first_derivatives_take_no_detour(monkeypatch):
    _without_kernels(monkeypatch)
    x, w, b = _meta(2, 9, 8).requires_grad_(), _meta(8, 4).requires_grad_(), _meta(2, 9, 4).requires_grad_()
    y = sophia_b200.selective_scan(sophia_b200.short_conv(x, w)[0], x, -w, b, b)[0]
    y.sum().backward()
    assert not any(t.grad.requires_grad for t in (x, w, b))


def test_forward_mode_is_refused():
    """Calls that go straight to a kernel would drop a dual number's tangent."""
    from torch.autograd import forward_ad

    x, w, pool, b = _meta(3, 8), _meta(8, 4), _meta(3, 8, 3), _meta(3, 16)
    scan = dict(x=x, dt=x, A=_meta(8, 16), B=b, C=b, state=_meta(3, 8, 16), D=_meta(8), z=x, dt_bias=_meta(8))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: sophia_b200.short_conv_step(dual(x), pool, w), lambda: sophia_b200.short_conv_step(x, dual(pool), w),
                 lambda: sophia_b200.short_conv_step(x, pool, dual(w)),
                 lambda: sophia_b200.short_conv_step(x, pool, w, dual(_meta(8))),
                 lambda: ssm.put_states(dual(pool), pool, _meta(3, dtype=torch.int32)),
                 lambda: sophia_b200.grad_norm([dual(torch.ones(3))]),
                 lambda: sophia_b200.clip_grad_norm_([torch.ones(3), dual(torch.ones(3))], 1.0)]
        calls += [lambda k=k: sophia_b200.selective_scan_step(**{**scan, k: dual(scan[k])}) for k in scan]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError):  # CUDA tensors only: plain ones in a dual level are not refused for it
            sophia_b200.grad_norm([torch.ones(3)])


@pytest.mark.parametrize("op", ["conv", "scan"])
def test_forward_mode_of_the_prompt_calls_is_refused(monkeypatch, op):
    from torch.autograd import forward_ad

    _without_kernels(monkeypatch)
    x, w, b = _meta(2, 9, 8), _meta(8, 4), _meta(2, 9, 4)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((NotImplementedError, RuntimeError)):
            sophia_b200.short_conv(d, w) if op == "conv" else sophia_b200.selective_scan(d, x, -w, b, b)


def test_single_tokens_compile():
    def step(x, pool, w, A, b, state):
        y = sophia_b200.short_conv_step(x, pool, w)
        return sophia_b200.selective_scan_step(y, x, A, b, b, state)

    args = (_meta(3, 8), _meta(4, 8, 3), _meta(8, 4), _meta(8, 16), _meta(3, 16), _meta(4, 8, 16))
    assert torch.compile(step, backend="aot_eager", fullgraph=True)(*args).shape == (3, 8)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,G", [(16, 1), (4, 1), (5, 2), (24, 1), (40, 1), (64, 2)])
def test_decoded_states_have_the_prompts_bits(dtype, N, G):
    """A hundred tokens one by one and in one call (too few for spans): the same arithmetic for every state, so
    the same bits, with slow decays, whose errors a state would gather over the tokens, among them."""
    T, E, rows = 100, 26, 3
    rn = gen(12)
    x, z, dt = rn(rows, T, E, dtype=dtype), rn(rows, T, E, dtype=dtype), rn(rows, T, E, scale=0.5, dtype=dtype)
    Bm, Cm = rn(rows, T, G, N, dtype=dtype), rn(rows, T, G, N, dtype=dtype)
    A, D, bias, h0 = -torch.exp(rn(E, N) - 1.0), rn(E), rn(E) - 4.0, rn(rows, E, N)
    y, want = sophia_b200.selective_scan(x, dt, A, Bm, Cm, D, z, bias, initial_state=h0, output_final_state=True)
    pool, slots = torch.zeros(5, E, N, device="cuda"), torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
    pool[slots.long()] = h0
    round_ = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    for t in range(T):
        out = sophia_b200.selective_scan_step(x[:, t], dt[:, t], A, Bm[:, t], Cm[:, t], pool, D, z[:, t], bias, slots=slots)
        # y sums the same 64 products at most in another order: 64 roundings of 2^-24 of their sizes' sum
        size = (Cm[:, t].double().abs().repeat_interleave(E // G, 1) * pool[slots.long()].double().abs()).sum(-1)
        size = (size + (D * x[:, t]).double().abs()) * z[:, t].double().abs()
        tol = 64 * 2.0 ** -24 * size + 2 * round_ * y[:, t].double().abs() + 2.0 ** -24
        assert ((out.double() - y[:, t].double()).abs() <= tol).all()
    assert torch.equal(pool[slots.long()], want) and not pool[[1, 3]].any()


@gpu
@pytest.mark.parametrize("W", [1, 2, 3, 4])
def test_fp16_convolution_steps_continue_a_prompt(W):
    rn = gen(6)
    x, w, b = rn(3, 30, 50, dtype=torch.float16), rn(50, W, scale=0.5), rn(50)
    whole, final = sophia_b200.short_conv(x, w, b, output_final_state=True)
    _, pool = sophia_b200.short_conv(x[:, :11], w, b, output_final_state=True)
    for t in range(11, 30):
        assert torch.equal(sophia_b200.short_conv_step(x[:, t], pool, w, b), whole[:, t])
    assert torch.equal(pool, final)


@gpu
@pytest.mark.parametrize("T,B", [(5, 2), (16, 1), (43, 2), (1203, 1)])  # ends inside a tile and at one; spans
def test_states_that_forget_at_once(T, B):
    """A rate of -inf: its decay is 0 for every step, so everything is as with a rate of -1e30, bit for bit; the
    places past a row's end (steps of 0) add nothing."""
    E, N = 20, 5
    rn = gen(8)
    x, dt, z, bc = rn(B, T, E), rn(B, T, E), rn(B, T, E), rn(B, T, 2 * N)
    dy, h0 = rn(B, T, E), rn(B, E, N)

    def run(rate):
        A = -torch.exp(gen(4)(E, N))
        A[::3, 1] = rate
        A[4] = rate
        ts = [t.detach().clone().requires_grad_() for t in (x, dt, A, bc[..., :N], bc[..., N:], z, h0)]
        y, ht = sophia_b200.selective_scan(*ts[:5], None, ts[5], initial_state=ts[6], output_final_state=True)
        return [y, ht, *torch.autograd.grad((y, ht), ts, (dy, torch.ones_like(ht)))], A, ts

    got, A, _ = run(float("-inf"))
    want, _, _ = run(-1e30)
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    pool = h0.clone()
    for t in range(min(T, 5)):
        sophia_b200.selective_scan_step(x[:, t], dt[:, t], A, bc[:, t, :N], bc[:, t, N:], pool, None, z[:, t])
    assert torch.isfinite(pool).all()


@gpu
def test_a_rate_that_is_not_a_number_shows():
    A = -torch.ones(4, 3, device="cuda")
    A[1, 2] = float("nan")
    rn = gen(1)
    x, b = rn(1, 9, 4), rn(1, 9, 3)
    y, _ = sophia_b200.selective_scan(x, x, A, b, b)
    assert torch.isnan(y[0, :, 1]).all() and torch.isfinite(y[0, :, [0, 2, 3]]).all()


@gpu
def test_an_infinite_gradient_leaves_infinite_sums():
    """dD = sum ds x and d dt_bias = sum d dt over the tokens: one infinite term makes them infinite, as the plain sum,
    where it is the only one; other channels stay finite."""
    E, N, T = 12, 4, 75
    rn = gen(2)
    x, dt, b, dy = rn(2, T, E), rn(2, T, E), rn(2, T, N), rn(2, T, E)
    z = rn(2, T, E)
    for at in (0, 33, T - 1):
        for value in (float("inf"), -float("inf")):
            bad = dy.clone()
            bad[1, at, 5] = value
            D, bias = rn(E).requires_grad_(), rn(E).requires_grad_()
            y, _ = sophia_b200.selective_scan(x, dt, -torch.ones(E, N, device="cuda"), b, b, D, z, bias)
            dD, dbias = torch.autograd.grad(y, (D, bias), bad)
            want = value * torch.sign(x[1, at, 5] * z[1, at, 5])
            assert dD[5] == want and not torch.isfinite(dbias[5])
            rest = [k for k in range(E) if k != 5]
            assert torch.isfinite(dD[rest]).all() and torch.isfinite(dbias[rest]).all()
