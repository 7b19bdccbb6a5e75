"""Plain float64 statement of the gated linear recurrence (test infrastructure): token
by token, one sequence at a time, differentiated by autograd."""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ssm_reference import spans


def recurrence(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu):
    """x, decay, gate, z [B, T, E] float64; returns (y, final state [sequences, E])."""
    E = x.shape[2]
    zero = x.new_zeros(())
    log_a = A * torch.sigmoid(decay + (zero if decay_bias is None else decay_bias))
    a = log_a.exp()
    fed = (-torch.expm1(2 * log_a)).sqrt() * torch.sigmoid(gate + (zero if gate_bias is None else gate_bias)) * x
    rows_a, rows_b = [r.unbind(0) for r in a.unbind(0)], [r.unbind(0) for r in fed.unbind(0)]
    ys, finals = {}, []
    for i, row, lo, hi in spans(x, cu):
        h = h0[i] if h0 is not None else x.new_zeros(E)
        out = []
        for t in range(lo, hi):
            h = rows_a[row][t] * h + rows_b[row][t]
            out.append(h)
        ys.setdefault(row, []).append(torch.stack(out) if out else x.new_zeros(0, E))
        finals.append(h)
    y = torch.stack([torch.cat(ys[r]) for r in sorted(ys)])
    return (y if z is None else y * F.silu(z)), torch.stack(finals)
