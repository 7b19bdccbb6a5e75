"""``short_conv`` where a thread walks many tokens: runs of 16 to 64 tokens forward and 32 to 256 backward,
which the run rule takes once there are enough threads for the GPU.  Rings wrap, groups without starts or ends
follow one another, and documents start and end at every place of a group and deep inside a run.

Tolerances as in ``test_ssm``, derived there for one value; sums over tokens (dw, dbias) add up to 256 terms in
order, then the runs': below (256 + 8 + T / 16 / 8) roundings of 2^-24 in the worst case, 3e-5 of the terms' size summed in
absolute value and about its square root, 1e-6 of the result, for terms of random sign.
"""

from __future__ import annotations

import pytest
import torch

import sophia_b200
import ssm_reference as ref
from test_ssm import close, cu_of, doubles, gen

pytestmark = pytest.mark.gpu

EVERY = tuple(n for k in range(36) for n in (k + 1, 70 - k)) + (0, 1, 1, 2, 0, 3, 1, 128, 5)  # 2697 tokens

CASES = [  # dtype, B, T, C, taps, state, silu, documents, backward's run
    (torch.bfloat16, 1, 700, 4096, 4, True, True, None, 32),
    (torch.float32, 2, 1500, 1024, 4, True, True, None, 32),
    (torch.bfloat16, 4, 1024, 4096, 4, False, True, None, 128),
    (torch.float16, 2, 2560, 4096, 4, True, True, None, 256),
    (torch.float32, 2, 2571, 4096, 4, True, False, None, 256),
    (torch.float32, 4, 700, 2049, 4, True, True, None, 64),   # one channel a thread
    (torch.bfloat16, 4, 701, 2049, 4, True, True, None, 64),  # and without the ring
    (torch.bfloat16, 2, 1309, 4096, 3, True, True, None, 128),
    (torch.float32, 2, 1309, 4096, 2, True, True, None, 128),
    (torch.bfloat16, 2, 1309, 4096, 1, True, True, None, 128),
    (torch.bfloat16, 1, sum(EVERY), 4096, 4, True, True, EVERY, 128),
    (torch.float32, 1, sum(EVERY), 4096, 4, True, True, EVERY, 128),
    (torch.float32, 1, sum(EVERY), 2049, 3, True, True, EVERY, 64),
    (torch.float16, 1, sum(EVERY), 4096, 2, False, True, EVERY, 128),
    (torch.bfloat16, 1, 5000, 4096, 4, True, True, (1, 2499, 0, 2, 3, 2495), 256),
]


@pytest.mark.parametrize("case", CASES,
                         ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c[:5]) + ("-docs" if c[7] else ""))
def test_long_runs(case):
    dtype, B, T, C, W, with_state, silu, docs, run = case
    rn, cu = gen(17), cu_of(docs)
    N = len(docs) if docs else B
    # the backward's partial sums tell the run that it takes
    size = lambda packed, backward: sophia_b200._lib.load().kda_b200_short_conv_workspace_bytes(  # noqa: E731
        B, T, C, W, packed, backward)
    sums = size(int(docs is not None), 1) - (size(1, 0) if docs else 0)
    assert sums == (B * ((T + run - 1) // run) * C * (W + 1) * 4 + 255) // 256 * 256
    ts = {"x": rn(B, T, C, dtype=dtype).requires_grad_(), "weight": rn(C, W, scale=0.5).requires_grad_(),
          "bias": rn(C, scale=0.2).requires_grad_(), "h0": rn(N, C, W - 1).requires_grad_() if with_state else None}
    y, ht = sophia_b200.short_conv(ts["x"], ts["weight"], ts["bias"], activation="silu" if silu else None,
                                   initial_state=ts["h0"], output_final_state=True, cu_seqlens=cu)
    dy, dht = rn(B, T, C, dtype=dtype), rn(N, C, W - 1)
    leaves = [k for k, v in ts.items() if v is not None]
    got = torch.autograd.grad((y, ht), [ts[k] for k in leaves], (dy, dht))
    r = doubles(ts)
    ry, rht = ref.conv(r["x"], r["weight"], r["bias"], r["h0"], cu, silu)
    want = torch.autograd.grad((ry, rht), [r[k] for k in leaves], (dy.double(), dht.double()), allow_unused=True)
    close("y", y, ry, dtype)
    close("final_state", ht, rht, torch.float32)
    for k, a, b in zip(leaves, got, want):
        close("d_" + k, a, torch.zeros_like(a) if b is None else b, ts[k].dtype)
    assert sophia_b200._lib.device_error(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_and_documents_give_the_same(dtype):
    """Long runs, short runs (a document alone) and packed rows agree bit for bit in y: a value's arithmetic
    does not depend on its place."""
    rn = gen(5)
    docs = (1300, 1, 700, 40, 2, 613)
    x, w, b = rn(1, sum(docs), 4096, dtype=dtype), rn(4096, 4, scale=0.5), rn(4096)
    y, ht = sophia_b200.short_conv(x, w, b, cu_seqlens=cu_of(docs), output_final_state=True)
    at = 0
    for i, n in enumerate(docs):
        y1, h1 = sophia_b200.short_conv(x[:, at:at + n, :64], w[:64], b[:64], output_final_state=True)
        assert torch.equal(y[:, at:at + n, :64], y1) and torch.equal(ht[i, :64], h1[0])
        at += n
