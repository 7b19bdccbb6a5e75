"""``grad_norm`` and ``clip_grad_norm_`` against the formula in float64.

Tolerances, derived beforehand: squares are summed in fp32 over at most 32
elements of a thread (relative error below 32 * 2^-24 = 2e-6, all terms positive) and in
fp64 from there, so the norm is within 1e-6; the factor adds three roundings, a scaled element
one more: 1.5e-6 relative in fp32.  In bf16 and fp16 a scaled element is the fp32 product with the
returned norm's factor, rounded once: equal bit for bit.
"""

from __future__ import annotations

import math

import pytest
import torch

import sophia_b200

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu

SHAPES = {
    "one": [(1,)],
    "odd": [(3, 5), (1,), (0,), (127,), (64, 33), (8192,), (8193,)],
    "large": [(1 << 20,), (1000, 1003)],
    "many": [(7 + i % 11,) for i in range(150)],
    "tables": [(3,)] * 2100,
}


def grads(name, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * 10.0 ** (i % 3 - 1)).to(dtype)
            for i, s in enumerate(SHAPES[name])]


def total(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(SHAPES))
def test_norm_and_in_place_clipping(name, dtype):
    ts = grads(name, dtype)
    want = total(ts)
    assert abs(float(sophia_b200.grad_norm(ts)) - want) <= 1e-6 * want
    for ratio in (0.3, 2.0):
        ts = grads(name, dtype)
        before = [t.double() for t in ts]
        norm = sophia_b200.clip_grad_norm_(ts, want * ratio)
        assert norm.shape == () and norm.dtype == torch.float32 and abs(float(norm) - want) <= 1e-6 * want
        k = min(1.0, want * ratio / (want + 1e-6))
        for a, b in zip(ts, before):
            if ratio > 1:
                assert torch.equal(a.double(), b)
            elif dtype == torch.float32:
                assert ((a.double() - b * k).abs() <= 1.5e-6 * (b * k).abs()).all()
            else:
                factor = torch.tensor(want * ratio, device="cuda", dtype=torch.float32) / (norm + 1e-6)
                assert torch.equal(a, (b.float() * factor).to(dtype))


@gpu
@pytest.mark.parametrize("ratio", [0.5, 3.0])
def test_other_outputs_types_and_addresses(ratio):
    """bf16 and fp16 gradients into the views of one fp32 buffer, end to end at any offset."""
    ts = [t if i % 2 else t.to(torch.float16) for i, t in enumerate(grads("odd", torch.bfloat16))]
    want = total(ts)
    flat = torch.full((sum(t.numel() for t in ts) + 1,), 9.0, device="cuda")
    outs = [v.view(t.shape) for v, t in zip(flat[1:].split([t.numel() for t in ts]), ts)]
    before = [t.clone() for t in ts]
    norm = sophia_b200.clip_grad_norm_(ts, want * ratio, out=outs)
    assert abs(float(norm) - want) <= 1e-6 * want and float(flat[0]) == 9.0
    k = min(1.0, want * ratio / (want + 1e-6))
    for t, b, o in zip(ts, before, outs):
        assert torch.equal(t, b)
        assert ((o.double() - b.double() * k).abs() <= 1.5e-6 * (b.double() * k).abs()).all()


@gpu
def test_views_with_holes_and_permuted_gradients():
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(40, 30, device="cuda", generator=g)
    ts = [base[:, 3:20], torch.randn(6, 7, 8, device="cuda", generator=g).permute(2, 0, 1)]
    before, want = [t.double().clone() for t in ts], total(ts)
    rest = base[:, 20:].clone()
    sophia_b200.clip_grad_norm_(ts, want / 4)
    for t, b in zip(ts, before):
        assert ((t.double() - b / 4).abs() <= 1e-5 * b.abs()).all()
    assert torch.equal(base[:, 20:], rest)


@gpu
def test_zero_infinite_and_nan_gradients():
    z = [torch.zeros(100, device="cuda")]
    assert float(sophia_b200.clip_grad_norm_(z, 1.0)) == 0 and not z[0].any()
    ts = [torch.ones(10, device="cuda"), torch.tensor([float("inf"), 1.0], device="cuda")]
    assert math.isinf(float(sophia_b200.clip_grad_norm_(ts, 1.0)))
    assert not ts[0].any() and torch.isnan(ts[1][0]) and ts[1][1] == 0
    ts = [torch.ones(10, device="cuda"), torch.tensor([float("nan")], device="cuda")]
    assert math.isnan(float(sophia_b200.clip_grad_norm_(ts, 1.0))) and torch.isnan(ts[0]).all()
    ts = grads("odd", torch.float32)
    keep = [t.clone() for t in ts]
    sophia_b200.clip_grad_norm_(ts, float("inf"))
    assert all(torch.equal(a, b) for a, b in zip(ts, keep))


@gpu
def test_the_norm_is_the_same_every_time():
    ts = grads("large", torch.bfloat16)
    first = sophia_b200.grad_norm(ts)
    for _ in range(4):
        assert torch.equal(sophia_b200.grad_norm(ts), first)


@gpu
def test_no_gradients():
    assert float(sophia_b200.grad_norm([])) == 0 and float(sophia_b200.clip_grad_norm_([], 1.0)) == 0
    assert float(sophia_b200.grad_norm([torch.empty(0, device="cuda")])) == 0


def test_refusals():
    t = torch.zeros(3)
    with pytest.raises(RuntimeError):
        sophia_b200.clip_grad_norm_([t], 1.0)
    with pytest.raises(RuntimeError):
        sophia_b200.grad_norm([t])
    with pytest.raises(NotImplementedError):
        sophia_b200.grad_norm([t.double()])
    with pytest.raises(ValueError):
        sophia_b200.grad_norm([None])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            sophia_b200.clip_grad_norm_([t], bad)
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([t], 1.0, eps=-1.0)


@gpu
def test_refusals_of_outputs():
    t = torch.zeros(3, device="cuda")
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([t, t], 1.0)
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([t], 1.0, out=[])
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([t], 1.0, out=[torch.zeros(4, device="cuda")])
    w = torch.nn.Parameter(torch.ones(3, device="cuda"))
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([w], 1.0)
    assert (w == 1).all()
