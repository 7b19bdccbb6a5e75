"""Prompts whose requests have no slot of the pool: padding, as in the single-token call."""

from __future__ import annotations

import pytest
import torch

from sophia_b200.ssm_mixer import SSMMixerBlock, SSMPool

INNER, TAPS, STATE = 6, 4, 3


@pytest.mark.parametrize("slots", [[2, 0, 3], [-1, 2, 0], [2, -1, -5], [-1, -1, 4], [-1, -2, -3], [5, 1, 6], [5, 5, 7],
                                   [4, -1, 9], [-1]])
def test_rows_without_a_slot_leave_the_pool(slots):
    """The block's prefill on the CPU, its operators' outputs given."""
    block = SSMMixerBlock(4, INNER, STATE, dt_rank=2, conv_kernel=TAPS)
    g = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rows = len(slots)
    y, conv, scan = rn(1, 7, 4), rn(rows, INNER, TAPS - 1), rn(rows, INNER, STATE)
    block._mix = lambda x, cu, want_state: (y, conv, scan)
    pool = SSMPool(rn(5, INNER, TAPS - 1), rn(5, INNER, STATE))
    want = [pool.conv.clone(), pool.scan.clone()]
    for r, s in enumerate(slots):
        if 0 <= s < 5:
            want[0][s], want[1][s] = conv[r], scan[r]
    cu = torch.tensor([0] * rows + [7], dtype=torch.int32)
    assert block.prefill(rn(1, 7, 4), cu, pool, torch.tensor(slots, dtype=torch.int32)) is y
    assert torch.equal(pool.conv, want[0]) and torch.equal(pool.scan, want[1])


def test_slots_of_another_number_are_refused():
    block = SSMMixerBlock(4, INNER, STATE, dt_rank=2, conv_kernel=TAPS)
    with pytest.raises(ValueError):
        block.prefill(torch.zeros(1, 7, 4), torch.tensor([0, 3, 7], dtype=torch.int32), block.make_pool(5),
                      torch.tensor([1, 2, 3], dtype=torch.int32))


@pytest.mark.gpu
def test_padding_prompts_on_the_gpu():
    block = SSMMixerBlock(64, 96, 16, dt_rank=12, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(1, 20, 64, device="cuda", generator=g)
    cu = torch.tensor([0, 5, 5, 14, 20, 20], device="cuda", dtype=torch.int32)
    all_slots = torch.tensor([3, 0, 1, 4, 2], device="cuda", dtype=torch.int32)
    full = block.make_pool(5)
    y = block.prefill(x, cu, full, all_slots)
    for slots in ([3, -1, 1, 4, -1], [-1, -1, -1, -1, -1], [7, -1, 1, 5, 2]):
        pool = block.make_pool(5)
        pool.conv.fill_(2.0), pool.scan.fill_(2.0)
        assert torch.equal(block.prefill(x, cu, pool, torch.tensor(slots, device="cuda", dtype=torch.int32)), y)
        for part, whole in zip(pool, full):
            for r, s in enumerate(slots):
                if 0 <= s < 5:
                    assert torch.equal(part[s], whole[all_slots[r]])
            rest = [k for k in range(5) if k not in slots]
            assert (part[rest] == 2.0).all()
