"""What a call hands the library by address lives until the library has it: the entry points of the recurrence and the
residual norm with their kernels' calls replaced, on the CPU, and parameters that have to be converted first."""

from __future__ import annotations

import types
import weakref

import pytest
import torch

from sophia_b200 import recurrence, residual

bf16 = torch.bfloat16


@pytest.fixture
def made(monkeypatch):
    """Every tensor that a conversion made, and whether all lived when the library was called."""
    seen = types.SimpleNamespace(refs=[], calls=[])  # of every call: the conversions before it

    def watch(module, name):
        real = getattr(module, name)

        def convert(t, *rest):
            out = real(t, *rest)
            if out is not None and out is not t:
                seen.refs.append(weakref.ref(out))
            return out
        monkeypatch.setattr(module, name, convert)

    def call(fn, device, *args):
        assert all(r() is not None for r in seen.refs), "a converted tensor is gone before the library is called"
        seen.calls.append(len(seen.refs))
        seen.refs.clear()

    class Lib:
        def __getattr__(self, name):
            return lambda *a: 4096

    for m in (recurrence, residual):
        watch(m, "_rows"), watch(m, "_param")
        monkeypatch.setattr(m, "_call", call)
    watch(recurrence, "_cu")
    monkeypatch.setattr(recurrence._lib, "load", Lib)
    return seen


def strided(*shape, dtype=torch.float32):
    """Last dimension not contiguous."""
    return torch.randn(*shape, 2).to(dtype)[..., 0]


@pytest.mark.parametrize("kind", ["bf16", "strided", "plain"])
def test_residual_norm_keeps_what_it_converts(made, kind):
    rows = (2, 3, 16)
    act = lambda: strided(*rows, dtype=bf16) if kind == "strided" else torch.randn(rows).to(bf16)  # noqa: E731
    par = {"bf16": lambda: torch.randn(16).to(bf16), "strided": lambda: strided(16), "plain": lambda: torch.randn(16)}[kind]
    x, o, g, w, wb, scale = act(), act(), act(), par(), par(), par()
    seed = torch.tensor([1])
    residual._fwd_impl(x, o, g, w, wb, scale, seed, 0, 0, 0.1, 1e-5, True)
    residual._bwd_impl(x, o, g, w, wb, scale, seed, torch.ones(6, 2), act(), act(), 0, 0, 0.1, 1e-5)
    assert made.calls == {"bf16": [3, 3], "strided": [6, 8], "plain": [0, 0]}[kind]


@pytest.mark.parametrize("kind", ["bf16", "strided"])
def test_recurrence_keeps_what_it_converts(made, kind):
    act = lambda: strided(1, 5, 8, dtype=bf16)  # noqa: E731
    par = (lambda *s: torch.randn(*s).to(bf16)) if kind == "bf16" else strided
    x, d, g, z, A, db, gb, h0 = act(), act(), act(), act(), par(8), par(8), par(8), strided(2, 8)
    cu = torch.tensor([0, 2, 5])
    recurrence._fwd_impl(x, d, g, A, z, db, gb, h0, cu, True, True)
    recurrence._bwd_impl(x, d, g, A, z, db, gb, h0, cu, torch.zeros(64, dtype=torch.uint8), act(), strided(2, 8), True)
    recurrence._step_impl(x[0], d[0], g[0], A, torch.zeros(9, 8), z[0], db, gb, None)
    assert made.calls == [9, 11, 7]
