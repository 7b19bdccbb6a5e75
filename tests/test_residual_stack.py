"""``RecurrentMixerBlock`` and ``ResidualStack``: the recurrence, its single-token step and
the residual norm run together, with the mixers that were there.

Tolerances: the blocks run in fp32 against the same formulas in float64.  cuBLAS products here sum at most 96 terms
(2^-24 each, 6e-6), the kernels' own bounds are 1e-5 of a tensor's largest value, and up to four layers pass
them on with gains around one: 2e-4 of the largest value of each output and gradient.
"""

from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

import recurrence_reference
import residual_reference
import ssm_reference
from sophia_b200 import clip_grad_norm_
from sophia_b200.mixer import KDAMixerBlock
from sophia_b200.recurrent_mixer import RecurrentMixerBlock, ResidualStack
from sophia_b200.ssm_mixer import SSMMixerBlock

gpu = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def recurrent(dim=64, inner=96, seed=0, **kw):
    return RecurrentMixerBlock(dim, inner, rank=16, std=0.15, generator=gen(seed), device="cuda", **kw)


def block_reference(b, p, x, cu=None):
    """RecurrentMixerBlock.mix in float64 with the parameters p."""
    xz = F.linear(x, p["w_xz"])
    x, z = xz.split(b.inner, dim=-1)
    x, _ = ssm_reference.conv(x, p["conv_weight"], p["conv_bias"], None, cu, False)
    decay, gate = F.linear(x, p["w_low"]).split(b.rank, dim=-1)
    y, _ = recurrence_reference.recurrence(x, F.linear(decay, p["decay_up"]), F.linear(gate, p["gate_up"]),
                                           -p["A_log"].exp(), z, p["decay_bias"], p["gate_bias"], None, cu)
    return F.linear(y, p["o_proj"])


def doubles(module):
    return {k: v.detach().double().requires_grad_() for k, v in module.named_parameters()}


def near(name, got, want, share=2e-4):
    assert (got.double() - want).abs().max() <= share * want.abs().max() + 1e-12, name


@gpu
def test_block_against_the_formulas():
    b = recurrent()
    x = torch.randn(1, 70, 64, device="cuda", generator=gen(1)).requires_grad_()
    cu = torch.tensor([0, 1, 40, 40, 70], device="cuda", dtype=torch.int32)
    up = torch.randn(1, 70, 64, device="cuda", generator=gen(2))
    for table in (None, cu):
        y = b(x, table)
        p, xd = doubles(b), x.detach().double().requires_grad_()
        want = block_reference(b, p, residual_reference.rms(xd, b.eps) * p["in_norm"], table)
        near("y", y, want)
        got = torch.autograd.grad(y, [x, *b.parameters()], up)
        exp = torch.autograd.grad(want, [xd, *p.values()], up.double())
        for name, a, e in zip(["x", *p], got, exp):
            near(name, a, e)


@gpu
def test_block_serves_what_it_trains():
    """Prompts packed in one call and single tokens afterwards give the outputs of the whole sequences."""
    b = recurrent(seed=3)
    lengths, extra = (5, 1, 33), 4
    xs = [torch.randn(1, n + extra, 64, device="cuda", generator=gen(n)) for n in lengths]
    with torch.no_grad():
        whole = [b(x)[0] for x in xs]
    pool = b.make_pool(6)
    for t in pool:
        t.fill_(float("nan"))
    slots = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 5, 6, 39], device="cuda", dtype=torch.int32)
    y = b.prefill(torch.cat([x[:, :n] for x, n in zip(xs, lengths)], 1), cu, pool, slots)
    for w, lo, n in zip(whole, cu.tolist(), lengths):
        near("prompt", y[0, lo:lo + n], w[:n].double())
    for t in range(extra):
        rows = torch.stack([x[0, n + t] for x, n in zip(xs, lengths)] + [xs[0][0, 0]])
        got = b.step(rows, pool, torch.cat([slots, slots.new_tensor([-1])]))
        near("token", got[:3], torch.stack([w[n + t] for w, n in zip(whole, lengths)]).double())
        assert not got[3].any()
    assert pool.state[[1, 3, 5]].isnan().all() and pool.conv[[1, 3, 5]].isnan().all()


def stack_reference(s, p, x, seed, cu=None):
    """A stack of RecurrentMixerBlocks in float64."""
    n = len(s.blocks)
    blocks = [{k[len(f"blocks.{i}."):]: v for k, v in p.items() if k.startswith(f"blocks.{i}.")} for i in range(n)]
    h = residual_reference.rms(x, s.eps) * blocks[0]["in_norm"]
    for i in range(n):
        after = blocks[i + 1]["in_norm"] if i + 1 < n else p["out_norm"]
        gate = F.linear(h, p[f"w_gates.{i}"]) if s.w_gates is not None else None
        x, h = residual_reference.residual_norm(x, block_reference(s.blocks[i], blocks[i], h, cu), after,
                                                p[f"post_norms.{i}"] if s.post_norms is not None else None, gate,
                                                p[f"scales.{i}"] if s.scales is not None else None,
                                                s.dropout_p if seed is not None else 0.0, seed or 0, i, s.eps)
    return x, h


@gpu
@pytest.mark.parametrize("kw,seed", [(dict(), None), (dict(gate=True, scale_init=0.5, dropout_p=0.2), 77),
                                     (dict(post_norm=False, scale_init=0.3), None)])
def test_stack_against_the_formulas(kw, seed):
    s = ResidualStack([recurrent(seed=i) for i in range(3)], generator=gen(9), **kw)
    x = torch.randn(2, 37, 64, device="cuda", generator=gen(5)).requires_grad_()
    out = s(x, seed=seed)
    p, xd = doubles(s), x.detach().double().requires_grad_()
    want = stack_reference(s, p, xd, seed)
    up = [torch.randn(2, 37, 64, device="cuda", generator=gen(6 + i)) for i in range(2)]
    for name, a, e in zip(("stream", "normed"), out, want):
        near(name, a, e)
    got = torch.autograd.grad(out, [x, *s.parameters()], up)
    exp = torch.autograd.grad(want, [xd, *p.values()], [u.double() for u in up])
    for name, a, e in zip(["x", *p], got, exp):
        near(name, a, e, 1e-3)  # gradients pass every layer twice


@gpu
def test_stack_of_all_mixers_trains_under_autocast():
    """The three mixers of the package around one stream: a step runs in bf16, every parameter gets a finite gradient, and
    the same seed gives the same step."""
    torch.manual_seed(0)
    blocks = [KDAMixerBlock(dim=128, heads=1, decay_rank=16, generator=gen(0), device="cuda"),
              SSMMixerBlock(dim=128, inner=128, state=8, dt_rank=16, generator=gen(1), device="cuda"),
              RecurrentMixerBlock(dim=128, inner=128, rank=16, generator=gen(2), device="cuda")]
    s = ResidualStack(blocks, gate=True, scale_init=0.5, dropout_p=0.1, generator=gen(3))
    x = torch.randn(2, 130, 128, device="cuda", generator=gen(4))
    seed = torch.tensor([3], device="cuda")
    runs = []
    for _ in range(2):
        s.zero_grad(set_to_none=True)
        with torch.autocast("cuda", torch.bfloat16):
            stream, normed = s(x, seed=seed)
            loss = (normed.float() - x).square().mean() + stream.float().square().mean()
        loss.backward()
        norm = clip_grad_norm_([p.grad for p in s.parameters()], 1.0)
        assert stream.dtype == torch.float32 and torch.isfinite(norm)
        runs.append([p.grad.clone() for p in s.parameters()])
    assert all(torch.isfinite(g).all() for g in runs[0])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    with torch.autocast("cuda", torch.bfloat16), torch.no_grad():
        assert not torch.equal(s(x, seed=seed + 1)[0], stream)


@gpu
def test_stack_serves_what_it_trains():
    s = ResidualStack([recurrent(seed=1), SSMMixerBlock(dim=64, inner=96, state=8, dt_rank=16, std=0.15, generator=gen(2),
                                                        device="cuda"), recurrent(seed=3)], scale_init=0.5, gate=True,
                      generator=gen(4))
    x = torch.randn(2, 20, 64, device="cuda", generator=gen(7))
    with torch.no_grad():
        stream, normed = s(x)
    pools = s.make_pools(4)
    slots = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 12, 24], device="cuda", dtype=torch.int32)
    got = s.prefill(x[:, :12].reshape(1, 24, 64), cu, pools, slots)
    near("prompt", got[0].reshape(2, 12, 64), stream[:, :12].double())
    for t in range(12, 20):
        a, b = s.step(x[:, t], pools, slots)
        near("stream", a, stream[:, t].double())
        near("normed", b, normed[:, t].double())


def test_stack_refusals():
    with pytest.raises(ValueError):
        ResidualStack([])
    with pytest.raises(ValueError):
        ResidualStack([RecurrentMixerBlock(8, 8, 2), RecurrentMixerBlock(16, 8, 2)])
    with pytest.raises(NotImplementedError):
        ResidualStack([KDAMixerBlock(dim=8, heads=1, decay_rank=2)]).make_pools(2)


def test_stack_refuses_blocks_of_another_eps():
    """Each block's own forward norms its input with the block's eps; a stack has one for all of its norms."""
    with pytest.raises(ValueError, match="eps"):
        ResidualStack([RecurrentMixerBlock(8, 8, 2), RecurrentMixerBlock(8, 8, 2, eps=1e-6)])
    assert ResidualStack([RecurrentMixerBlock(8, 8, 2, eps=1e-6), SSMMixerBlock(8, 8, eps=1e-6)]).eps == 1e-6


@gpu
def test_packed_stack_against_the_formulas():
    """Documents packed along T, one of them empty, one of a single token."""
    s = ResidualStack([recurrent(seed=i) for i in range(3)], scale_init=0.5, gate=True, dropout_p=0.2, generator=gen(9))
    cu = torch.tensor([0, 1, 20, 20, 37], device="cuda", dtype=torch.int32)
    x = torch.randn(1, 37, 64, device="cuda", generator=gen(5)).requires_grad_()
    out = s(x, cu, seed=78)
    p, xd = doubles(s), x.detach().double().requires_grad_()
    want = stack_reference(s, p, xd, 78, cu)
    up = [torch.randn(1, 37, 64, device="cuda", generator=gen(6 + i)) for i in range(2)]
    for name, a, e in zip(("stream", "normed"), out, want):
        near(name, a, e)
    got = torch.autograd.grad(out, [x, *s.parameters()], up)
    exp = torch.autograd.grad(want, [xd, *p.values()], [u.double() for u in up])
    for name, a, e in zip(["x", *p], got, exp):
        near(name, a, e, 1e-3)  # gradients pass every layer twice


@gpu
def test_packed_documents_in_a_stack_of_all_mixers():
    """Documents packed along T give what each gives alone, outputs and summed gradients, through every mixer of the
    package in fp32: the same sums, in matrix products of other heights."""
    blocks = [KDAMixerBlock(dim=128, heads=1, decay_rank=16, std=0.1, generator=gen(0), device="cuda"),
              SSMMixerBlock(dim=128, inner=128, state=8, dt_rank=16, std=0.1, generator=gen(1), device="cuda"),
              RecurrentMixerBlock(dim=128, inner=128, rank=16, std=0.1, generator=gen(2), device="cuda")]
    s = ResidualStack(blocks, scale_init=0.5)
    x = torch.randn(1, 133, 128, device="cuda", generator=gen(4)).requires_grad_()
    up = [torch.randn(1, 133, 128, device="cuda", generator=gen(6 + i)) for i in range(2)]
    bounds = [0, 33, 34, 133]
    cu = torch.tensor(bounds, device="cuda", dtype=torch.int32)
    spans = list(zip(bounds[:-1], bounds[1:]))
    for f in (blocks[0], lambda t, c=None: s(t, c)[0]):
        near("alone", f(x, cu), torch.cat([f(x[:, a:b].contiguous()) for a, b in spans], 1).double())
    out = s(x, cu)
    leaves = [x, *s.parameters()]
    got = torch.autograd.grad(out, leaves, up)
    alone = [s(x[:, a:b].contiguous()) for a, b in spans]
    flat = [t for pair in alone for t in pair]
    ups = [u[:, a:b].contiguous() for a, b in spans for u in up]
    want = torch.autograd.grad(flat, leaves, ups)
    for (name, _), a, e in zip([("x", None), *s.named_parameters()], got, want):
        near(name, a, e.double(), 1e-3)


def test_stack_refuses_another_number_of_pools():
    """Blocks without a pool would be left out of the stream silently."""
    s = ResidualStack([RecurrentMixerBlock(8, 8, 2), RecurrentMixerBlock(8, 8, 2)])
    pools, slots = s.make_pools(2), torch.zeros(1, dtype=torch.int32)
    for some in ([], pools[:1], [*pools, pools[0]]):
        with pytest.raises(ValueError, match="pools"):
            s.step(torch.zeros(1, 8), some, slots)
        with pytest.raises(ValueError, match="pools"):
            s.prefill(torch.zeros(1, 1, 8), torch.tensor([0, 1]), some, slots)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_pools_are_float32_for_parameters_in_16_bits(kind):
    s = ResidualStack([RecurrentMixerBlock(8, 8, 2), SSMMixerBlock(8, 8)]).to(kind)
    assert all(t.dtype == torch.float32 and not t.any() for pool in s.make_pools(3) for t in pool)


@gpu
def test_stack_in_16_bits_serves():
    """A model cast to bf16 as a whole: prompts and single tokens run, and continue each other's states.  One layer rounds
    about ten times (projections, convolution, gates, recurrence, norms), each by 2^-8 of its values, with gains around one,
    and what is compared went through two layers twice: 40 2^-8 of the largest value."""
    s = ResidualStack([recurrent(seed=1), recurrent(seed=2)], scale_init=0.5, gate=True, generator=gen(4)).bfloat16()
    x = torch.randn(2, 20, 64, device="cuda", generator=gen(7)).bfloat16()
    with torch.no_grad():
        stream, normed = s(x)
    pools = s.make_pools(4)
    slots = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 12, 24], device="cuda", dtype=torch.int32)
    got = s.prefill(x[:, :12].reshape(1, 24, 64), cu, pools, slots)
    assert got[0].dtype == got[1].dtype == torch.bfloat16
    near("prompt", got[1].reshape(2, 12, 64), normed[:, :12].double(), 40 * 2.0 ** -8)
    for t in range(12, 20):
        a, b = s.step(x[:, t], pools, slots)
        near("stream", a, stream[:, t].double(), 40 * 2.0 ** -8)
        near("normed", b, normed[:, t].double(), 40 * 2.0 ** -8)
