"""The state-space mixer block: its operators run together, in training and in serving.

Against the block written in float64 from elementary operations (the scan and the convolution of
``ssm_reference``), and against itself: prompts and single tokens give what one pass over
all of them gives, and clipped training lowers the loss.
"""

from __future__ import annotations

import os
import sys

import pytest
import torch
from torch.nn import functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import ssm_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


def block(dim=64, inner=96, state=16, std=0.08):
    from sophia_b200.ssm_mixer import SSMMixerBlock
    return SSMMixerBlock(dim, inner, state, dt_rank=12, std=std,
                         generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")


def exact(m, x, cu):
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    x = x.detach().double().requires_grad_()
    h = F.rms_norm(x, (m.dim,), p["in_norm"], m.eps)
    u, z = F.linear(h, p["w_xz"]).split(m.inner, dim=-1)
    u, _ = ref.conv(u, p["conv_weight"], p["conv_bias"], None, cu, True)
    low, B, C = F.linear(u, p["w_dbc"]).split([m.dt_rank, m.state, m.state], dim=-1)
    y, _ = ref.scan(u, F.linear(low, p["dt_up"]), -p["A_log"].exp(), B[:, :, None], C[:, :, None], p["D"], z,
                    p["dt_bias"], None, cu, True)
    return F.linear(y, p["o_proj"]), x, p


@pytest.mark.parametrize("docs", [None, (1, 40, 0, 29)])
def test_block_and_its_gradients(docs):
    """fp32 throughout.  The operators' own bound is 1e-5 of an output's norm; the block chains four
    projections and two operators and adds their errors, and TF32 is off: 2e-4 of each norm."""
    m = block()
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(2 if docs is None else 1, 70, m.dim, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(x.shape, device="cuda", generator=g)
    cu = None if docs is None else torch.tensor([0, 1, 41, 41, 70], device="cuda", dtype=torch.int32)
    y = m(x, cu)
    y.backward(dy)
    want, xx, p = exact(m, x, cu)
    want.backward(dy.double())
    assert (y.double() - want).norm() <= 2e-4 * want.norm()
    assert (x.grad.double() - xx.grad).norm() <= 2e-4 * xx.grad.norm()
    for n, t in m.named_parameters():
        assert (t.grad.double() - p[n].grad).norm() <= 2e-4 * p[n].grad.norm(), n


def test_prompts_and_single_tokens_give_the_whole_pass():
    m = block()
    lengths, more = [5, 1, 30], 6
    g = torch.Generator(device="cuda").manual_seed(9)
    seqs = [torch.randn(1, n + more, m.dim, device="cuda", generator=g) for n in lengths]
    with torch.no_grad():
        whole = [m(s) for s in seqs]
    pool = m.make_pool(5)
    slots = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
    prompt = torch.cat([s[:, :n] for s, n in zip(seqs, lengths)], 1)
    cu = torch.tensor([0, 5, 6, 36], device="cuda", dtype=torch.int32)
    y = m.prefill(prompt, cu, pool, slots)
    close = lambda a, b: (a - b).norm() <= 2e-4 * b.norm()  # noqa: E731
    assert close(y[0], torch.cat([w[0, :n] for w, n in zip(whole, lengths)]))
    padded = torch.cat([slots, torch.tensor([-1], device="cuda", dtype=torch.int32)])
    for t in range(more):
        x = torch.cat([s[:, n + t] for s, n in zip(seqs, lengths)] + [torch.ones(1, m.dim, device="cuda")])
        y = m.step(x, pool, padded)
        assert close(y[:3], torch.cat([w[:, n + t] for w, n in zip(whole, lengths)]))
        assert (y[3] == 0).all()
    assert (pool.scan[[1, 3]] == 0).all() and (pool.conv[[1, 3]] == 0).all()


def test_training_clips_and_learns():
    from sophia_b200.ssm_mixer import train_step
    m = block()
    g = torch.Generator(device="cuda").manual_seed(10)
    x = torch.randn(2, 64, m.dim, device="cuda", generator=g)
    target = x.roll(1, 1)  # the token before: the block has to remember
    target[:, 0] = 0
    opt = torch.optim.AdamW(m.parameters(), lr=3e-3, weight_decay=0.0)
    losses, norms = [], []
    for _ in range(60):
        loss, norm = train_step(m, opt, x, target, max_norm=0.05)
        after = torch.stack([p.grad.norm() for p in m.parameters()]).norm()
        # the clipped norm: fp32 gradients times a factor of fp32, a few roundings of 2^-24
        assert float(after) <= 0.05 * (1 + 1e-5) and (float(norm) > 0.05 or abs(float(after) - float(norm)) <= 1e-5 * float(norm))
        losses.append(float(loss))
        norms.append(float(norm))
    assert max(norms) > 0.05  # some steps were clipped
    assert losses[-1] < 0.5 * losses[0], (losses[0], losses[-1])
