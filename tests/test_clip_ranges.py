"""``grad_norm`` and ``clip_grad_norm_`` over the whole range of their types, at any address and at the ends of chunks.

Tolerances, derived beforehand.  A thread sums at most 16384 / 256 = 64 squares in fp32, all terms positive:
a relative error below 64 * 2^-24 = 3.8e-6 of the sum, half of that in its root; sums that leave fp32's range are
fp64 and add nothing.  The root's rounding to fp32 adds 2^-24: the norm is within 2e-6.  The factor (a sum, a
division) adds three roundings of 2^-24, a scaled element one more and, where the factor itself is below 2^-126,
2^-150 absolute in it: 2.3e-6 of an element (those below 1e-37 left out) for factors above 1e-30.  In bf16 and fp16
a scaled element is the fp32 product with the returned norm's factor, rounded once: equal bit for bit.
"""

from __future__ import annotations

import math

import pytest
import torch

import sophia_b200

pytestmark = pytest.mark.gpu
CHUNK = 16384


def total(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def check(ts, dtype, max_norm, want):
    before = [t.clone() for t in ts]
    assert abs(float(sophia_b200.grad_norm(ts)) - want) <= 2e-6 * want
    norm = sophia_b200.clip_grad_norm_(ts, max_norm)
    assert abs(float(norm) - want) <= 2e-6 * want
    k = min(1.0, max_norm / (want + 1e-6))
    factor = torch.tensor(max_norm, device="cuda", dtype=torch.float32) / (norm + 1e-6)
    for a, b in zip(ts, before):
        if k == 1.0:
            assert torch.equal(a, b)
        elif dtype == torch.float32:
            exact = b.double() * k
            assert ((a.double() - exact).abs() <= 2.3e-6 * exact.abs() + 1e-37).all()
        else:
            assert torch.equal(a, (b.float() * factor).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [[1], [300, 16390], [40000]])
@pytest.mark.parametrize("values", ["1e20", "1e30", "one large", "1e-22", "1e-30", "small and zero", "small beside ordinary",
                                    "subnormal"])
def test_values_whose_squares_leave_fp32(dtype, sizes, values):
    """Finite gradients have a finite norm, tiny ones a norm that is not zero."""
    g = torch.Generator(device="cuda").manual_seed(7)
    ts = [torch.randn(n, device="cuda", generator=g).clamp(-4, 4) for n in sizes]
    ts = [t + t.sign() * 0.1 for t in ts]
    if values == "one large":
        ts[-1][-1] = 3e20
    elif values == "small and zero":
        ts = [t * 1e-24 * (torch.rand(t.shape, device="cuda", generator=g) < 0.1) for t in ts]
        ts[0][0] = 1e-24
    elif values == "small beside ordinary":
        ts = [torch.where(torch.rand(t.shape, device="cuda", generator=g) < 0.5, t * 1e-25, t) for t in ts]
    else:
        ts = [t * {"1e20": 1e20, "1e30": 1e30, "1e-22": 1e-22, "1e-30": 1e-30, "subnormal": 1e-39}[values] for t in ts]
    ts = [t.to(dtype) for t in ts]
    want = total(ts)
    check([t.clone() for t in ts], dtype, 1.0, want)
    check([t.clone() for t in ts], dtype, want * 0.4 + 1e-6 * 0.4, want)


def test_a_chunk_of_zeros_and_true_infinities():
    ts = [torch.zeros(3 * CHUNK, device="cuda"), torch.full((5,), 2.0, device="cuda")]
    assert abs(float(sophia_b200.grad_norm(ts)) - math.sqrt(20)) <= 2e-6 * math.sqrt(20)
    ts[0][CHUNK + 3] = float("inf")
    assert math.isinf(float(sophia_b200.grad_norm(ts)))
    ts[0][CHUNK + 3] = float("nan")
    assert math.isnan(float(sophia_b200.grad_norm(ts)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [CHUNK - 1, CHUNK, CHUNK + 1, 2 * CHUNK, 2 * CHUNK + 2049, 8191, 4096, 1024, 7])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_chunk_ends_at_any_address(dtype, n, offset):
    """Views of one flat bucket, end to end behind an odd size: most begin at no multiple of 16 bytes."""
    g = torch.Generator(device="cuda").manual_seed(n)
    flat = torch.randn(offset + n + 3 + n, device="cuda", generator=g).to(dtype)
    kept = flat.clone()
    ts = [flat[offset:offset + n], flat[offset + n + 3:]]
    want = total(ts)
    check(ts, dtype, want * 0.4, want)
    assert torch.equal(flat[:offset], kept[:offset]) and torch.equal(flat[offset + n:offset + n + 3],
                                                                     kept[offset + n:offset + n + 3])
    outs = [torch.empty(n + 1, device="cuda")[1:], torch.empty(n, device="cuda")]
    norm = sophia_b200.clip_grad_norm_(ts, 0.5, out=outs)
    factor = torch.tensor(0.5, device="cuda") / (norm + 1e-6)
    for t, o in zip(ts, outs):
        exact = t.double() * min(1.0, float(factor))
        assert ((o.double() - exact).abs() <= 1.2e-7 * exact.abs() + 1e-37).all()  # one rounding


def test_an_expanded_output_is_refused_before_anything_is_scaled():
    """autograd.grad of a sum returns a broadcast tensor: its elements share a place."""
    whole, base = torch.ones(10, device="cuda"), torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([whole, base.expand(5)], 0.1)
    with pytest.raises(ValueError):
        sophia_b200.clip_grad_norm_([whole, torch.ones(4, 3, device="cuda")], 0.1,
                                    out=[whole, torch.ones(4, 1, device="cuda").expand(4, 3)])
    assert (whole == 1).all() and float(base) == 1
    # as an input it is read like any other
    out = [torch.empty(10, device="cuda"), torch.empty(5, device="cuda")]
    norm = sophia_b200.clip_grad_norm_([whole, base.expand(5)], 0.1, out=out)
    assert abs(float(norm) - math.sqrt(15)) <= 2e-6 * math.sqrt(15)
    assert torch.equal(torch.cat(out), torch.ones(15, device="cuda") * (torch.tensor(0.1, device="cuda") / (norm + 1e-6)))
