"""Plain float64 statements of the state-space operators (test infrastructure):
token by token, one sequence at a time, differentiated by autograd."""

from __future__ import annotations

import torch
import torch.nn.functional as F


def spans(x, cu):
    """(sequence, row, first, end) of every sequence."""
    if cu is None:
        return [(b, b, 0, x.shape[1]) for b in range(x.shape[0])]
    cu = [int(v) for v in cu]
    return [(i, 0, lo, hi) for i, (lo, hi) in enumerate(zip(cu, cu[1:]))]


def conv(x, weight, bias, h0, cu, silu):
    """x [B, T, C] float64; returns (y, final state [N, C, W-1])."""
    W = weight.shape[1]
    ys, finals = {}, []
    for i, row, lo, hi in spans(x, cu):
        past = h0[i].T if h0 is not None else x.new_zeros(W - 1, x.shape[2])
        seq = torch.cat([past, x[row, lo:hi]])
        n = hi - lo
        c = sum(weight[:, k] * seq[k:k + n] for k in range(W))
        c = c + (bias if bias is not None else 0)
        ys.setdefault(row, []).append(F.silu(c) if silu else c)
        finals.append(seq[n:].T)
    y = torch.stack([torch.cat(ys[r]) for r in sorted(ys)])
    return y, torch.stack(finals)


def scan(x, dt, A, B, C, D, z, dt_bias, h0, cu, softplus):
    """x [B, T, E], B and C [B, T, G, N], float64; returns (y, final state [sequences, E, N])."""
    E, N, G = x.shape[2], A.shape[1], B.shape[2]
    raw = dt + (dt_bias if dt_bias is not None else 0)
    d = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30)))) if softplus else raw
    group = torch.arange(E, device=x.device) // (E // G)
    ys, finals = {}, []
    for i, row, lo, hi in spans(x, cu):
        h = h0[i] if h0 is not None else x.new_zeros(E, N)
        out = []
        for t in range(lo, hi):
            h = torch.exp(d[row, t, :, None] * A) * h + (d[row, t] * x[row, t])[:, None] * B[row, t, group]
            out.append((h * C[row, t, group]).sum(1))
        y = torch.stack(out) if out else x.new_zeros(0, E)
        y = y + (D * x[row, lo:hi] if D is not None else 0)
        if z is not None:
            y = y * F.silu(z[row, lo:hi])
        ys.setdefault(row, []).append(y)
        finals.append(h)
    return torch.stack([torch.cat(ys[r]) for r in sorted(ys)]), torch.stack(finals)
