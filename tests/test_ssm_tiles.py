"""The scan's forward in both of its tile lengths: 16-bit calls of up to 8 and of more than 56 states take 32 tokens
where no SM gets a second CTA, else 16; spans, documents and ends inside a tile with each.  Tolerances as in ``test_ssm``."""

from __future__ import annotations

import pytest
import torch

from test_ssm import close, cu_of, reference_scan, run_scan, scan_tensors

pytestmark = pytest.mark.gpu

CASES = [  # dtype, B, T, E, N, G, documents
    (torch.bfloat16, 300, 37, 64, 8, 1, None),    # more CTAs than SMs: tiles of 16
    (torch.float16, 160, 65, 24, 5, 1, None),
    (torch.bfloat16, 170, 50, 8, 64, 1, None),
    (torch.float16, 90, 33, 20, 57, 2, None),
    (torch.bfloat16, 3, 95, 64, 8, 1, None),      # few: tiles of 32
    (torch.float16, 2, 61, 20, 60, 2, None),
    (torch.bfloat16, 2, 97, 40, 56, 1, None),     # two CTAs of 32 fit
    (torch.bfloat16, 1, 1500, 64, 8, 1, None),    # spans
    (torch.float16, 40, 260, 200, 7, 1, None),
    (torch.bfloat16, 1, 1400, 8, 64, 1, None),
    (torch.bfloat16, 1, 1400, 1200, 58, 1, None),
    (torch.bfloat16, 1, 1000, 640, 8, 2, (31, 1, 32, 0, 17, 15, 16, 33, 600, 255)),
    (torch.float16, 1, 400, 1300, 64, 1, (31, 1, 32, 0, 17, 15, 16, 33, 0, 255)),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c[:6]))
def test_tiles_of_both_lengths(case):
    dtype, B, T, E, N, G, docs = case
    ts, dy, dht = scan_tensors(dtype, B, T, E, N, G, True, True, True, True, docs)
    cu = cu_of(docs)
    y, ht, grads = run_scan(ts, cu, True, dy, dht)
    ry, rht, want = reference_scan(ts, cu, True, dy, dht)
    close("y", y, ry, dtype)
    close("final_state", ht, rht, torch.float32)
    for k in want:
        close("d_" + k, grads[k], want[k], ts[k].dtype)
