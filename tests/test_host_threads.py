"""Host threads in one operator at once, with sizes that want different amounts of shared memory of one and the same
kernel: no call depends on what another thread's call asked for.  (Calls of the library release the interpreter's lock;
each is repeated without Python in between, so that they do meet.)"""

from __future__ import annotations

import threading

import pytest
import torch

import sophia_b200
from sophia_b200 import _lib, recurrence, residual, ssm

gpu = pytest.mark.gpu
bf16 = torch.bfloat16


def in_threads(monkeypatch, module, calls, times=4000):
    """Each of `calls` in a thread and a stream of its own, every library call of theirs `times` times; the results are
    the ones that they have alone."""
    want = [f().detach() for f in calls]
    torch.cuda.synchronize()

    def repeat(fn, device, *args):
        stream = torch._C._cuda_getCurrentRawStream(device.index)
        rcs = {fn(*args, stream) for _ in range(times)}
        assert rcs == {0}, _lib.load().kda_b200_last_error().decode()

    monkeypatch.setattr(module, "_call", repeat)
    errors, got = [], [None] * len(calls)
    start = threading.Barrier(len(calls))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                got[i] = calls[i]()
        except Exception as e:  # noqa: BLE001 -- raised below, in the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, device="cuda", generator=g)


def rec(tokens, backward):
    rn = gen(tokens)
    ts = [rn(1, tokens, 64).to(bf16) for _ in range(4)]
    A = -torch.ones(64, device="cuda")

    def run():
        x = ts[0].detach().requires_grad_(backward)
        y = sophia_b200.gated_recurrence(x, ts[1], ts[2], A, ts[3])[0]
        return torch.autograd.grad(y, x, ts[0])[0] if backward else y
    return run


@gpu
@pytest.mark.parametrize("backward", [False, True])
def test_recurrence(monkeypatch, backward):
    in_threads(monkeypatch, recurrence, [rec(t, backward) for t in (60, 120, 250, 500)])


def norm(rows, backward):
    rn = gen(rows)
    x, o, gate, w = rn(rows, 1536).to(bf16), rn(rows, 1536).to(bf16), rn(rows, 1536).to(bf16), rn(1536)

    def run():
        leaf = o.detach().requires_grad_(backward)
        n = sophia_b200.residual_norm(x, leaf, w, gate=gate)[1]
        return torch.autograd.grad(n, leaf, x)[0] if backward else n
    return run


@gpu
@pytest.mark.parametrize("backward", [False, True])
def test_residual_norm(monkeypatch, backward):
    in_threads(monkeypatch, residual, [norm(r, backward) for r in (2, 500, 900, 1400)])


def scan(states, backward):
    rn = gen(states)
    ts = [rn(1, 40, 64).to(bf16) for _ in range(2)]
    B, C, A = rn(1, 40, 1, states).to(bf16), rn(1, 40, 1, states).to(bf16), -torch.ones(64, states, device="cuda")

    def run():
        x = ts[0].detach().requires_grad_(backward)
        y = sophia_b200.selective_scan(x, ts[1], A, B, C)[0]
        return torch.autograd.grad(y, x, ts[0])[0] if backward else y
    return run


@gpu
@pytest.mark.parametrize("backward", [False, True])
def test_selective_scan(monkeypatch, backward):
    in_threads(monkeypatch, ssm, [scan(n, backward) for n in (33, 40, 50, 63)])
