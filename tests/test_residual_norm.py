"""``residual_norm`` against a plain float64 statement of the formulas (``residual_reference.py``)
on the same inputs, gradients by autograd of that statement and by differences.

Tolerances, derived beforehand.  Kernels compute in fp32 and round once.
* Outputs stored in 16 bits: half a step, 2^-8 (bf16) or 2^-11 (fp16) of an element, plus the fp32 term.
* fp32: a row's sums of D <= 8192 squares or products have an error of at most D / (32 W) + 10 additions in a
  row (K V products a thread, five exchanges, W warps), 64 + 16 of them here: 80 2^-24 = 5e-6 of the sum of the
  magnitudes; the square root halves it.  The products around it add 12 roundings and two approximations of 2^-22:
  1.5e-6, 1e-5 in all.  A gradient is a difference of two terms, r (t - v r^2 mean(t v)), that may cancel (to nothing in
  a row of one channel): its error is that share of the terms, not of their difference.  Both are at most r |t|, as
  |v r| mean(|t v|) r <= |t| by Cauchy and Schwarz up to the row's largest.  So elements are within 2e-5 of the largest
  term of their row, which ``terms`` below bounds from the formulas.
* Sums over rows: the terms' errors above, and one rounding per row of a CTA and per CTA: 1e-5 of the largest sum or
  of the terms' root sum of squares, whichever is larger (terms may cancel).
* Dropped places are exact: the words are integers.
"""

from __future__ import annotations

import pytest
import torch

import sophia_b200
import residual_reference as ref

ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half a step of fp16's subnormals
gpu = pytest.mark.gpu
f32, bf16, f16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("residual", "branch", "weight", "branch_weight", "gate", "scale")


def terms(r, ups, p, eps):
    """Per row, the size of what the gradients are differences of."""
    u = r["branch"]
    rb = 1.0
    if r["branch_weight"] is not None:
        rb = 1 / (u.square().mean(-1, keepdim=True) + eps).sqrt()
        u = u * rb * r["branch_weight"]
    up = ups[0].double().abs()
    if len(ups) > 1:
        v = ref.residual_norm(*(r[k] for k in NAMES), 0, 0, 0, eps)[0]
        up = up + (ups[1].double() * r["weight"]).abs() / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    up = up.amax(-1, keepdim=True)
    down = up * (1 if r["scale"] is None else r["scale"].abs().max()) / (1 - p)
    size = {"d_residual": up, "d_gate": down * u.abs().amax(-1, keepdim=True)}
    size["d_branch"] = down * rb * (1 if r["branch_weight"] is None else r["branch_weight"].abs().max())
    return {k: t.detach() for k, t in size.items()}


def close(name, got, want, size=None):
    dtype = got.dtype
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, name
    if not want.numel():
        return
    assert torch.isfinite(got).all(), name
    if want.dim() == 1:
        assert (got - want).abs().max() <= (1e-5 + ROUND[dtype]) * want.abs().max() + 1e-12, name
        return
    size = want.abs().amax(-1, keepdim=True) if size is None else size
    tol = ROUND[dtype] * want.abs() + 2e-5 * size + TINY[dtype]
    assert ((got - want).abs() - tol).max() <= 0, f"{name}: {float((got - want).abs().max())} off"


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, scale=1.0, shift=0.0, dtype=f32: (torch.randn(*s, device="cuda", generator=g) * scale
                                                        + shift).to(dtype)


def inputs(rn, shape, wide, dtype, norm=True, post=True, gate=True, scale=True, pad=0):
    D = shape[-1]
    act = lambda d: rn(*shape[:-1], D + pad, dtype=d)[..., pad:]  # noqa: E731
    ts = {"residual": act(wide), "branch": act(dtype), "weight": rn(D, scale=0.2, shift=1.0) if norm else None,
          "branch_weight": rn(D, scale=0.2, shift=1.0) if post else None, "gate": act(dtype) if gate else None,
          "scale": rn(D, scale=0.5) if scale else None}
    return {k: None if v is None else v.detach().requires_grad_() for k, v in ts.items()}


def call(ts, **kw):
    return sophia_b200.residual_norm(ts["residual"], ts["branch"], ts["weight"], branch_weight=ts["branch_weight"],
                                     gate=ts["gate"], scale=ts["scale"], **kw)


def check(ts, rn, p=0.0, seed=None, offset=0, eps=1e-5):
    v, n = call(ts, dropout_p=p, seed=seed, offset=offset, eps=eps)
    r = {k: None if t is None else t.detach().double().requires_grad_() for k, t in ts.items()}
    rv, rn_ = ref.residual_norm(*(r[k] for k in NAMES), p, int(seed) if seed is not None else 0, offset, eps)
    assert v.dtype == ts["residual"].dtype
    close("stream", v, rv)
    outs, routs = [v], [rv]
    if n is not None:
        assert n.dtype == ts["branch"].dtype
        close("normed", n, rn_)
        outs.append(n), routs.append(rn_)
    ups = [rn(*o.shape, dtype=o.dtype) for o in outs]
    leaves = [k for k in NAMES if ts[k] is not None]
    got = torch.autograd.grad(outs, [ts[k] for k in leaves], ups)
    want = torch.autograd.grad(routs, [r[k] for k in leaves], [u.double() for u in ups])
    sizes = terms(r, ups, p, eps)
    for k, a, b in zip(leaves, got, want):
        assert a.dtype == ts[k].dtype
        close("d_" + k, a, b, sizes.get("d_" + k))


CASES = [  # shape, stream, branch, next norm, branch norm, gate, scale, p, elements beside the rows
    ((1, 1), f32, f32, True, True, True, True, 0.0, 0),
    ((3, 5), f32, f32, True, False, True, False, 0.3, 0),
    ((2, 3, 64), f32, bf16, True, True, True, True, 0.1, 0),
    ((2, 7, 8), bf16, bf16, True, True, False, True, 0.0, 8),
    ((1, 9, 1536), f32, bf16, True, True, True, True, 0.1, 8),
    ((3, 4, 1536), bf16, bf16, True, True, True, False, 0.5, 0),
    ((2, 3, 4096), bf16, bf16, True, True, False, True, 0.0, 0),
    ((1, 3, 8192), f16, f16, True, True, True, True, 0.2, 0),
    ((5, 8192), f32, f32, True, True, True, True, 0.2, 0),
    ((2, 8191), f32, bf16, True, True, True, True, 0.2, 1),
    ((2, 2, 1003), f32, f32, True, False, True, False, 0.2, 0),
    ((37, 1003), bf16, bf16, True, True, True, True, 0.1, 0),
    ((600, 72), f16, f16, False, True, True, True, 0.1, 0),
    ((33, 264), f32, f16, False, False, True, True, 0.0, 0),
    ((700, 96), f32, bf16, False, False, False, False, 0.0, 0),
    ((3, 130, 512), bf16, bf16, True, False, False, False, 0.0, 0),
    ((2, 3, 4, 100), f32, f32, True, True, True, True, 0.1, 4),
    ((40,), f32, f32, True, True, True, True, 0.1, 0),
    ((2000, 40), bf16, bf16, True, True, True, True, 0.1, 3),
    ((330, 7008), bf16, bf16, True, True, True, True, 0.1, 0),
    ((700, 4096), f32, bf16, True, True, True, True, 0.1, 0),
    ((5, 200, 520), f32, f32, True, True, True, True, 0.0, 4),
    ((40000, 64), bf16, bf16, True, True, True, True, 0.1, 0),
    ((9, 1000, 24), f32, f16, True, True, True, True, 0.1, 8),
]


@gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "").replace(" ", "") for v in c))
def test_forward_and_gradients(case):
    shape, wide, dtype, norm, post, gate, scale, p, pad = case
    rn = gen(17)
    check(inputs(rn, shape, wide, dtype, norm, post, gate, scale, pad), rn, p, 0x123456789ABCDEF if p else None, 41)


@gpu
@pytest.mark.parametrize("shape,dtype", [((900, 2043), bf16), ((650, 2501), bf16), ((1200, 131), f16), ((3, 211, 2047), f32)],
                         ids=str)
def test_odd_rows_many(shape, dtype):
    """More odd rows than run at once, at both widths of a thread: the column sums go over several rows of a group."""
    rn = gen(23)
    check(inputs(rn, shape, f32, dtype, True, True, True, True, 0), rn, 0.1, 77, 3)


@gpu
@pytest.mark.parametrize("shape,wide,dtype", [((400, 8192), f32, f32), ((310, 8192), f32, f16), ((1000, 4096), f32, f32)],
                         ids=str)
def test_widest_rows_many(shape, wide, dtype):
    """Rows of which shared memory holds one or two beside the parameters, more of them than there are SMs."""
    rn = gen(29)
    check(inputs(rn, shape, wide, dtype, True, True, True, True, 0), rn, 0.1, 78, 4)


def test_generator_known_answers():
    """The published vectors of Philox4x32-10, and the tensor form against the integers."""
    assert ref.philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ref.philox([ref.LOW] * 4, [ref.LOW] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    w = ref.words(5, 11, 0xFEDCBA9876543210, 7)
    for row, col in ((0, 0), (0, 10), (4, 3), (3, 8)):
        assert int(w[row, col]) == ref.philox([col // 4, row, 0, 7], [0x76543210, 0xFEDCBA98])[col % 4]


@gpu
@pytest.mark.parametrize("dtype,D", [(f32, 1003), (bf16, 1536), (f16, 40)])
def test_mask_is_the_generators(dtype, D):
    rows, p = 61, 0.37
    seed = torch.tensor([-(2 ** 62) + 12345], device="cuda")
    one = torch.ones(rows, D, device="cuda", dtype=dtype)
    v, _ = sophia_b200.residual_norm(torch.zeros_like(one), one, dropout_p=p, seed=seed, offset=2 ** 32 - 1)
    keep = ref.words(rows, D, int(seed) & (2 ** 64 - 1), 2 ** 32 - 1).cuda() >= round(p * 2 ** 32)
    assert torch.equal(v != 0, keep)
    assert torch.equal(v[keep], torch.full_like(v[keep], 1 / (1 - p)))
    again, _ = sophia_b200.residual_norm(torch.zeros_like(one), one, dropout_p=p, seed=int(seed), offset=2 ** 32 - 1)
    assert torch.equal(v, again)
    # another call number: another mask; kept within six standard deviations of the probability
    other, _ = sophia_b200.residual_norm(torch.zeros_like(one), one, dropout_p=p, seed=seed, offset=0)
    assert not torch.equal(v, other)
    for m in (v, other):
        assert abs((m != 0).double().mean().item() - (1 - p)) <= 6 * (p * (1 - p) / m.numel()) ** 0.5


@gpu
def test_probability_zero_and_one():
    rn = gen(1)
    ts = inputs(rn, (6, 96), f32, f32)
    base = call(ts)
    for a, b in zip(base, call(ts, dropout_p=0.0, seed=5)):
        assert torch.equal(a, b)
    v, _ = call(ts, dropout_p=1.0, seed=5)
    assert torch.equal(v, ts["residual"])
    d = torch.autograd.grad(v.sum(), [ts["residual"], ts["branch"], ts["gate"], ts["scale"]])
    assert (d[0] == 1).all() and not any(g.any() for g in d[1:])


@gpu
def test_what_is_dropped_may_be_anything():
    """Infinities and NaN in dropped places of an unnormed branch, and of its gate, touch nothing."""
    rn = gen(2)
    ts = inputs(rn, (8, 128), f32, f32, post=False)
    keep = ref.words(8, 128, 3, 0).cuda() >= round(0.4 * 2 ** 32)
    clean = call(ts, dropout_p=0.4, seed=3)
    ups = [torch.ones_like(t) for t in clean]
    want = torch.autograd.grad(clean, [ts[k] for k in NAMES if ts[k] is not None], ups)
    for bad in (float("nan"), float("inf")):
        dirty = dict(ts)
        for k in ("branch", "gate"):
            dirty[k] = torch.where(keep, ts[k].detach(), torch.full_like(ts[k], bad)).requires_grad_()
        got = call(dirty, dropout_p=0.4, seed=3)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        grads = torch.autograd.grad(got, [dirty[k] for k in NAMES if ts[k] is not None], ups)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


@gpu
def test_rows_do_not_touch_each_other():
    rn = gen(3)
    ts = inputs(rn, (9, 256), bf16, bf16)
    v, n = call(ts)
    dirty = {k: None if t is None else t.detach().clone() for k, t in ts.items()}
    dirty["branch"][4, 17] = float("nan")
    dv, dn = call(dirty)
    rest = torch.arange(9, device="cuda") != 4
    assert torch.equal(dv[rest], v[rest]) and torch.equal(dn[rest], n[rest]) and dn[4].isnan().all()


@gpu
def test_broadcast_gate_and_its_gradient():
    rn = gen(4)
    ts = inputs(rn, (3, 20, 192), f32, bf16)
    for shape in ((3, 1, 192), (192,), (1, 20, 192)):
        gate = rn(*shape, dtype=bf16).requires_grad_()
        some = dict(ts, gate=gate)
        v, n = call(some)
        up = [rn(*v.shape), rn(*n.shape, dtype=bf16)]
        (got,) = torch.autograd.grad((v, n), gate, up)
        r = {k: None if t is None else t.detach().double().requires_grad_() for k, t in some.items()}
        rv, rn_ = ref.residual_norm(*(r[k] for k in NAMES[:4]), r["gate"].expand(3, 20, 192), r["scale"], 0, 0, 0, 1e-5)
        (want,) = torch.autograd.grad((rv, rn_), r["gate"], [u.double() for u in up])
        close("stream", v, rv)
        # the kernel's gradient is rounded to bf16 for every token, then summed: 2^-8 of each of up to 60 terms
        terms = 60 * 2.0 ** -8 * 4.0
        assert got.shape == gate.shape and (got.double() - want).abs().max() <= terms


@gpu
def test_transposed_and_expanded_rows():
    rn = gen(5)
    base = inputs(rn, (4, 6, 128), f32, bf16)
    flip = {k: (t.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_() if t is not None and t.dim() == 3
                else t) for k, t in base.items()}
    assert not flip["branch"].is_contiguous()
    for a, b in zip(call(flip, dropout_p=0.2, seed=9), call(base, dropout_p=0.2, seed=9)):
        assert torch.equal(a, b)
    up = rn(6, 128).expand(4, 6, 128)
    a = torch.autograd.grad(call(flip)[0], flip["branch"], up)[0]
    b = torch.autograd.grad(call(base)[0], base["branch"], up.contiguous())[0]
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("which", [0, 1])
def test_one_output_alone(which):
    rn = gen(6)
    ts = inputs(rn, (5, 160), f32, bf16)
    r = {k: t.detach().double().requires_grad_() for k, t in ts.items()}
    out, want = call(ts)[which], ref.residual_norm(*(r[k] for k in NAMES), 0, 0, 0, 1e-5)[which]
    up = rn(5, 160, dtype=out.dtype)
    got = torch.autograd.grad(out, [ts[k] for k in NAMES], up, allow_unused=True)
    exp = torch.autograd.grad(want, [r[k] for k in NAMES], up.double(), allow_unused=True)
    for k, a, b in zip(NAMES, got, exp):
        close("d_" + k, a, torch.zeros_like(a) if b is None else b)


@gpu
def test_mixed_types():
    rn = gen(7)
    for wide, dtype, gate in ((bf16, f32, f32), (bf16, f16, f16), (f32, bf16, f32), (f16, bf16, bf16)):
        ts = inputs(rn, (7, 136), wide, dtype)
        ts["gate"] = rn(7, 136, dtype=gate).requires_grad_()
        check(ts, rn)


@gpu
def test_gradients_against_differences():
    """Central differences of step e = 1e-2 in fp32: e^2 f''' / 6 and 2^-24 |f| / e, 1e-3 of the directions' size."""
    rn = gen(8)
    ts = inputs(rn, (6, 72), f32, f32)
    up = rn(6, 72), rn(6, 72)

    def f(t):
        v, n = call(t, dropout_p=0.25, seed=11)
        return (v.double() * up[0]).sum() + (n.double() * up[1]).sum()

    grads = torch.autograd.grad(f(ts), [ts[k] for k in NAMES])
    for k, g in zip(NAMES, grads):
        d, e = rn(*ts[k].shape), 1e-2
        hi, lo = (dict(ts, **{k: ts[k].detach() + s * e * d}) for s in (1, -1))
        assert abs((f(hi) - f(lo)).item() / (2 * e) - (g * d).sum().item()) <= 2e-3 * (g.norm() * d.norm()).item(), k


@gpu
def test_no_rows():
    ts = inputs(gen(9), (0, 64), f32, bf16)
    v, n = call(ts)
    assert v.shape == n.shape == (0, 64)
    grads = torch.autograd.grad((v, n), [ts[k] for k in NAMES], (v.detach(), n.detach()))
    assert all(not g.any() for g in grads)


@gpu
def test_same_bits_and_no_grad():
    ts = inputs(gen(10), (300, 1536), f32, bf16)
    up = torch.ones(300, 1536, device="cuda"), torch.ones(300, 1536, device="cuda", dtype=bf16)
    runs = []
    for _ in range(3):
        out = call(ts, dropout_p=0.1, seed=2)
        runs.append((*out, *torch.autograd.grad(out, [ts[k] for k in NAMES], up)))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
    with torch.no_grad():
        quiet = call(ts, dropout_p=0.1, seed=2)
    assert quiet[0].grad_fn is None and all(torch.equal(a, b) for a, b in zip(quiet, runs[0]))


@gpu
def test_captured_step_draws_anew_with_its_seed():
    rn = gen(11)
    ts = inputs(rn, (64, 256), f32, bf16)
    seed = torch.tensor([1], device="cuda")
    leaves = [ts[k] for k in NAMES]
    up = rn(64, 256), rn(64, 256, dtype=bf16)

    def step():
        out = call(ts, dropout_p=0.3, seed=seed)
        return (*out, *torch.autograd.grad(out, leaves, up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for s in (1, 77):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


@gpu
def test_seed_changed_before_the_backward_is_noticed():
    ts = inputs(gen(12), (4, 64), f32, f32)
    seed = torch.tensor([1], device="cuda")
    v, _ = call(ts, dropout_p=0.3, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError):
        v.sum().backward()


@gpu
def test_compiled():
    ts = inputs(gen(13), (3, 20, 160), f32, bf16)
    seed = torch.tensor([5], device="cuda")
    fn = torch.compile(lambda t, s: call(t, dropout_p=0.2, seed=s), fullgraph=True)
    a, b = call(ts, dropout_p=0.2, seed=seed), fn(ts, seed)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    up = [torch.ones_like(t) for t in a]
    leaves = [ts[k] for k in NAMES]
    for x, y in zip(torch.autograd.grad(a, leaves, up), torch.autograd.grad(b, leaves, up)):
        assert torch.equal(x, y)


@gpu
def test_refusals():
    rn = gen(0)
    x, f = rn(4, 32), sophia_b200.residual_norm
    w = torch.ones(32, device="cuda")
    for bad in (dict(weight=w[:8]), dict(branch_weight=w[:8]), dict(scale=rn(4, 32)), dict(gate=rn(3, 32)),
                dict(gate=rn(4, 1)), dict(dropout_p=1.5, seed=1), dict(dropout_p=-0.1, seed=1), dict(dropout_p=0.5),
                dict(dropout_p=0.5, seed=torch.ones(2, device="cuda", dtype=torch.int64)),
                dict(dropout_p=0.5, seed=torch.ones(1, device="cuda")), dict(offset=-1), dict(offset=2 ** 32)):
        with pytest.raises(ValueError):
            f(x, x, **bad)
    with pytest.raises(ValueError):
        f(x, x[:2])
    with pytest.raises(NotImplementedError):
        f(rn(1, 8193), rn(1, 8193))
    with pytest.raises(NotImplementedError):
        f(x.double(), x.double())
    for bad in (dict(weight=w.cpu()), dict(dropout_p=0.5, seed=torch.ones(1, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            f(x, x, **bad)
    with pytest.raises(RuntimeError):
        f(x.cpu(), x.cpu())
    x.requires_grad_()
    (g,) = torch.autograd.grad(f(x, x, w)[0].sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError):
        g.sum().backward()


def converted(ts, kind):
    """The parameters as the kernels have to convert them: in bf16, or with a stride."""
    def one(t):
        t = t.detach()
        return (t.to(bf16) if kind == "bf16" else torch.stack([t, t + 1], -1)[:, 0]).requires_grad_()
    return {k: one(t) if k in ("weight", "branch_weight", "scale") else t for k, t in ts.items()}


@gpu
@pytest.mark.parametrize("kind", ["bf16", "strided"])
@pytest.mark.parametrize("shape,wide,dtype", [((1, 64), f32, bf16), ((2, 1536), bf16, bf16), ((8, 1003), f32, f32),
                                              ((700, 1536), f32, bf16), ((300, 2043), f32, f16)], ids=str)
def test_parameters_that_have_to_be_converted(kind, shape, wide, dtype):
    """Eager against the formulas, with allocations of the parameters' size before and after; captured with the same bits."""
    rn = gen(31)
    ts = converted(inputs(rn, shape, wide, dtype), kind)
    for _ in range(3):
        check(ts, rn, 0.1, 79, 5)
    leaves = [ts[k] for k in NAMES]
    up = rn(*shape, dtype=wide), rn(*shape, dtype=dtype)

    def step():
        out = call(ts, dropout_p=0.1, seed=79, offset=5)
        return (*out, *torch.autograd.grad(out, leaves, up))

    want = [t.detach() for t in step()]  # (no eager graph of the leaves lives while one is captured)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("shape", [(2, 3, 0, 8), (0, 3, 2, 8), (2, 0, 1, 4, 8), (0, 8), (2, 0, 8), (8,), (5, 8), (2, 3, 4, 8)], ids=str)
def test_any_leading_dimensions_as_three(shape):
    """The kernels' [B, T, D], of the same elements in the same order, also where there are none."""
    t = sophia_b200.residual._three(torch.arange(torch.Size(shape).numel()).reshape(shape))
    assert t.dim() == 3 and t.shape[-1] == 8 and torch.equal(t.flatten(), torch.arange(t.numel()))


@gpu
@pytest.mark.parametrize("shape", [(2, 3, 0, 8), (0, 3, 2, 8), (2, 0, 1, 4, 8)], ids=str)
def test_no_rows_of_more_dimensions(shape):
    ts = inputs(gen(9), shape, f32, bf16)
    v, n = call(ts, dropout_p=0.1, seed=3)
    assert v.shape == n.shape == shape
    grads = torch.autograd.grad((v, n), [ts[k] for k in NAMES], (v.detach(), n.detach()))
    assert all(g.shape == ts[k].shape and not g.any() for k, g in zip(NAMES, grads))


@gpu
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_gradient_of_a_broadcast_gate_term_by_term(dtype):
    """Every token's gradient is within the bounds above (2e-5 of its row's ``terms`` and half a step), and so their sum is
    within the sum of those bounds, for the terms that are summed, and one more rounding: half a step of the result."""
    rn = gen(33)
    ts = inputs(rn, (3, 20, 192), f32, dtype)
    for shape in ((3, 1, 192), (192,), (1, 20, 192)):
        gate = rn(*shape, dtype=dtype).requires_grad_()
        out = call(dict(ts, gate=gate))
        up = [rn(*out[0].shape), rn(*out[1].shape, dtype=dtype)]
        (got,) = torch.autograd.grad(out, gate, up)
        r = {k: None if t is None else t.detach().double() for k, t in dict(ts, gate=gate).items()}
        r["gate"] = r["gate"].expand(3, 20, 192).clone().requires_grad_()
        want = torch.autograd.grad(ref.residual_norm(*(r[k] for k in NAMES), 0, 0, 0, 1e-5), r["gate"], [u.double() for u in up])[0]
        each = ROUND[dtype] * want.abs() + 2e-5 * terms(r, up, 0.0, 1e-5)["d_gate"]
        total, bound = want.sum_to_size(shape), each.sum_to_size(shape)
        bound = bound + ROUND[dtype] * (total.abs() + bound)
        assert got.shape == gate.shape and ((got.double() - total).abs() <= bound).all()
