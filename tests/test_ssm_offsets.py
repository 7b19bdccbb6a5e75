"""Offsets past 32 bits: the backward's partial sums of dB and dC with more channel groups than 2^31 floats hold."""

from __future__ import annotations

import pytest
import torch

import sophia_b200


@pytest.mark.gpu
def test_partial_sums_past_32_bits():
    """One token, a channel in each of 2^21 + 37 groups, 64 states: 8 x 2 x 64 floats a group, 2^31 of them and more.
    dB = C dy d x and dC = B dy d x are products of four fp32 factors: three roundings of 2^-24 on either side."""
    E, N = (1 << 21) + 37, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, dt, dy = rn(1, 1, E), rn(1, 1, E).abs() + 0.1, rn(1, 1, E)
    A = torch.full((1, N), -1.0, device="cuda").expand(E, N).contiguous()
    B, C = rn(1, 1, E, N).requires_grad_(), rn(1, 1, E, N).requires_grad_()
    y, _ = sophia_b200.selective_scan(x, dt, A, B, C, dt_softplus=False)
    dB, dC = torch.autograd.grad(y, (B, C), dy)
    scale = (dy * dt * x)[..., None]
    for got, other in ((dB, C.detach()), (dC, B.detach())):
        want = scale * other
        for part in range(0, E, 1 << 18):  # (in pieces: the whole takes a few GB)
            a, b = got[0, 0, part:part + (1 << 18)], want[0, 0, part:part + (1 << 18)]
            assert ((a - b).abs() <= 6 * 2.0 ** -24 * b.abs() + 1e-37).all()
