"""Prompts whose requests have no slot of the pool: padding, as in the single-token call."""

from __future__ import annotations

import pytest
import torch

from sophia_b200 import _lib
from sophia_b200.ssm import put_states
from sophia_b200.ssm_mixer import SSMMixerBlock

gpu = pytest.mark.gpu


@gpu
def test_padding_prompts_leave_the_pool():
    block = SSMMixerBlock(64, 96, 16, dt_rank=12, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(1, 20, 64, device="cuda", generator=g)
    cu = torch.tensor([0, 5, 5, 14, 20, 20], device="cuda", dtype=torch.int32)
    all_slots = torch.tensor([3, 0, 1, 4, 2], device="cuda", dtype=torch.int32)
    full = block.make_pool(5)
    y = block.prefill(x, cu, full, all_slots)
    for slots in ([3, -1, 1, 4, -1], [-1, -1, -1, -1, -1], [7, -1, 1, 5, 2]):
        for dtype in (torch.int32, torch.int64):
            pool = block.make_pool(5)
            pool.conv.fill_(2.0), pool.scan.fill_(2.0)
            assert torch.equal(block.prefill(x, cu, pool, torch.tensor(slots, device="cuda", dtype=dtype)), y)
            for part, whole in zip(pool, full):
                for r, s in enumerate(slots):
                    if 0 <= s < 5:
                        assert torch.equal(part[s], whole[all_slots[r]])
                rest = [k for k in range(5) if k not in slots]
                assert (part[rest] == 2.0).all()
            assert _lib.device_error(reset=True) == (11 if max(slots) > 4 else 0)


@gpu
@pytest.mark.parametrize("shape", [(1,), (7, 3), (96, 16), (2050, 64), (5, 0)])
def test_states_go_to_their_slots(shape):
    g = torch.Generator(device="cuda").manual_seed(1)
    new, pool = torch.randn(4, *shape, device="cuda", generator=g), torch.randn(9, *shape, device="cuda", generator=g)
    want, slots = pool.clone(), torch.tensor([8, -3, 0, 5], device="cuda", dtype=torch.int32)
    want[[8, 0, 5]] = new[[0, 2, 3]]
    put_states(new, pool, slots)
    assert torch.equal(pool, want)


@gpu
def test_many_rows_and_a_far_slot():
    new = torch.arange(70000, device="cuda", dtype=torch.float32).view(-1, 1)
    pool, slots = torch.zeros(70001, 1, device="cuda"), torch.arange(70000, 0, -1, device="cuda", dtype=torch.int32)
    put_states(new, pool, slots)
    assert torch.equal(pool[1:], new.flip(0)) and not pool[0].any()
    block = SSMMixerBlock(16, 8, 4, dt_rank=2, device="cuda")
    states = block.make_pool(2)
    block.prefill(torch.ones(1, 3, 16, device="cuda"), torch.tensor([0, 3], device="cuda", dtype=torch.int32), states,
                  torch.tensor([2 ** 32], device="cuda"))
    assert not states.conv.any() and not states.scan.any() and _lib.device_error(reset=True) == 11


@gpu
def test_prompts_compile():
    block = SSMMixerBlock(64, 96, 16, dt_rank=12, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    x = torch.randn(1, 20, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    cu = torch.tensor([0, 5, 14, 20], device="cuda", dtype=torch.int32)
    slots = torch.tensor([3, -1, 0], device="cuda", dtype=torch.int32)
    want, got = block.make_pool(5), block.make_pool(5)
    y = block.prefill(x, cu, want, slots)
    run = torch.compile(lambda a, b, c, d: block.prefill(a, b, c, d), backend="aot_eager", fullgraph=True)
    assert torch.equal(run(x, cu, got, slots), y)
    assert torch.equal(got.conv, want.conv) and torch.equal(got.scan, want.scan)


def test_refusals():
    meta = lambda *s, dtype=torch.float32: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    slots = meta(2, dtype=torch.int32)
    for new, pool, at in [(meta(2, 6, 3), meta(5, 6, 4), slots), (meta(3, 6, 3), meta(5, 6, 3), slots),
                          (meta(2, 6, 3), meta(5, 6, 3, dtype=torch.bfloat16), slots),
                          (meta(2, 6, 3), meta(5, 6, 3), meta(2, dtype=torch.int64))]:
        with pytest.raises(ValueError):
            put_states(new, pool, at)
