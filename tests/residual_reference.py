"""Plain float64 statement of the residual norm and of its dropout's generator (test infrastructure)."""

from __future__ import annotations

import torch

LOW = 0xFFFFFFFF


def philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) on Python integers."""
    x, k = list(counter), list(key)
    for _ in range(10):
        p, q = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [q >> 32 ^ x[1] ^ k[0], q & LOW, p >> 32 ^ x[3] ^ k[1], p & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return x


def words(rows, D, seed, offset):
    """[rows, D] words, in numpy-free tensor arithmetic: 32-bit halves in int64."""
    quads = (D + 3) // 4
    x = [torch.arange(quads).expand(rows, quads), torch.arange(rows)[:, None].expand(rows, quads),
         torch.zeros(rows, quads, dtype=torch.int64), torch.full((rows, quads), offset)]
    k = [seed & LOW, seed >> 32 & LOW]
    for _ in range(10):
        p, q = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57  # wrapped products, whose halves are right
        x = [(q >> 32 & LOW) ^ x[1] ^ k[0], q & LOW, (p >> 32 & LOW) ^ x[3] ^ k[1], p & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return torch.stack(x, -1).reshape(rows, 4 * quads)[:, :D]


def rms(a, eps):
    return a / (a.square().mean(-1, keepdim=True) + eps).sqrt()


def residual_norm(x, o, weight, branch_weight, gate, scale, p, seed, offset, eps):
    """float64 tensors [..., D]; returns (stream, normed or None)."""
    u = o if branch_weight is None else rms(o, eps) * branch_weight
    if gate is not None:
        u = u * torch.sigmoid(gate)
    if p > 0:
        D = o.shape[-1]
        keep = (words(o.numel() // D, D, seed, offset) >= round(p * 2 ** 32)).reshape(o.shape).to(o.device)
        u = torch.where(keep, u / (1 - p) if p < 1 else u * 0, torch.zeros_like(u))
    v = x + (u if scale is None else scale * u)
    return v, (None if weight is None else rms(v, eps) * weight)
