"""The KDA layer's calls under the grad modes: activations are kept for a backward alone."""

from __future__ import annotations

import contextlib

import pytest
import torch

from sophia_b200 import kda_layer, ops

gpu = pytest.mark.gpu
MODES = {"grad": contextlib.nullcontext, "no_grad": torch.no_grad, "inference": torch.inference_mode}


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("parameters", [False, True])
def test_activations_are_kept_for_a_backward_alone(monkeypatch, mode, parameters):
    asked = []

    def forward(q, *rest):
        asked.append(rest[-1])
        return q.new_empty(q.shape), q.new_empty(0), q.new_empty(0, dtype=torch.uint8)

    monkeypatch.setattr(ops, "_kda_fwd_impl", forward)
    meta = lambda *s: torch.empty(*s, device="meta")  # noqa: E731
    leaf = torch.nn.Parameter if parameters else (lambda t: t)
    A_log, dt_bias = leaf(meta(2)), leaf(meta(256))
    with MODES[mode]():
        x, beta = meta(1, 70, 2, 128), meta(1, 70, 2)
        o, _ = ops._layer(x, x, x, x, beta, A_log, dt_bias, None, None, None, None, None, 1.0, -5.0, False)
    assert asked == [mode == "grad" and parameters]
    assert o.requires_grad == asked[0]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mode", ["no_grad", "inference"])
def test_parameters_under_no_grad_give_the_same_output_in_less_memory(mode, dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    rn = lambda *s, dt=dtype: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    B, T, H = 1, 1024, 4
    q, k, v, gate, beta = rn(B, T, H, 128), rn(B, T, H, 128), rn(B, T, H, 128), rn(B, T, H, 128), rn(B, T, H)
    A_log = torch.nn.Parameter(rn(H, dt=torch.float32).abs() * 0.3)
    dt_bias = torch.nn.Parameter(rn(H * 128, dt=torch.float32) * 0.1)
    taps = [torch.nn.Parameter(rn(H * 128, 4, dt=torch.float32) * 0.5) for _ in range(3)]

    def run(context):
        with context():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            o, ht = kda_layer(q, k, v, gate, beta, A_log, dt_bias, *taps, output_final_state=True)
            torch.cuda.synchronize()
            return torch.cuda.max_memory_allocated() - before, o.detach().clone(), ht.detach().clone()

    plain, o, ht = run(MODES[mode])
    trained, o1, h1 = run(MODES["grad"])
    assert torch.equal(o, o1) and torch.equal(ht, h1)
    assert plain < trained, (plain, trained)
