"""A state-space mixer block on the B200 kernels, for training and serving.

RMSNorm of the block input -> one projection to the channels x and their gate z
-> ``short_conv`` (+ SiLU) -> projections of x to a low-rank time step and to
B and C -> ``selective_scan`` (skip and gate included) -> out-projection: the
state-space counterpart of ``KDAMixerBlock``, whose conventions it follows
(fp32 parameters, cuBLAS for the projections, ``torch.autocast`` for bf16).

Serving keeps each request's state in a pool: ``prefill`` runs prompts (padded to no
common length: they are packed along one row) and writes their states to the
requests' slots, ``step`` advances each row of a batch by one token in its slot.
Training is ``forward`` and ``train_step``, which clips the gradients.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import nn
from torch.nn import functional as F

from .clip import clip_grad_norm_
from .mixer import _inverse_softplus
from .ssm import put_states, selective_scan, selective_scan_step, short_conv, short_conv_step


class SSMPool(NamedTuple):
    """The states of `slots` requests: the convolution's last inputs and the scan's state."""

    conv: torch.Tensor  # [slots, inner, taps - 1] float32
    scan: torch.Tensor  # [slots, inner, state] float32


class SSMMixerBlock(nn.Module):
    def __init__(self, dim: int = 1536, inner: int = 2048, state: int = 16, dt_rank: int = 128, conv_kernel: int = 4,
                 eps: float = 1e-5, dt_min: float = 1e-3, dt_max: float = 1e-1, dt_floor: float = 1e-4,
                 std: float = 0.02, generator: torch.Generator | None = None,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        self.dim, self.inner, self.state, self.dt_rank, self.taps, self.eps = dim, inner, state, dt_rank, conv_kernel, eps
        kw = {"device": device, "dtype": torch.float32}

        def normal(*shape):
            return nn.Parameter(torch.randn(*shape, generator=generator, **kw) * std)

        self.in_norm = nn.Parameter(torch.ones(dim, **kw))
        self.w_xz = normal(2 * inner, dim)
        self.conv_weight = normal(inner, conv_kernel)
        self.conv_bias = nn.Parameter(torch.zeros(inner, **kw))
        self.w_dbc = normal(dt_rank + 2 * state, inner)  # time step (low rank), B, C
        self.dt_up = normal(inner, dt_rank)
        u = torch.rand(inner, generator=generator, **kw)
        dt = torch.exp(u * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min)).clamp_min(dt_floor)
        self.dt_bias = nn.Parameter(_inverse_softplus(dt))
        self.A_log = nn.Parameter(torch.arange(1, state + 1, **kw).log().repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner, **kw))
        self.o_proj = normal(dim, inner)

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        return F.rms_norm(x, (self.dim,), self.in_norm.to(x.dtype), self.eps)

    def _in(self, h: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return F.linear(h, self.w_xz).split(self.inner, dim=-1)  # x and z, read in place

    def _dbc(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        low, B, C = F.linear(x, self.w_dbc).split([self.dt_rank, self.state, self.state], dim=-1)
        return F.linear(low, self.dt_up), B, C

    def _mix(self, h, cu_seqlens=None, want_state=False):
        x, z = self._in(h)
        x, conv = short_conv(x, self.conv_weight, self.conv_bias, output_final_state=want_state, cu_seqlens=cu_seqlens)
        dt, B, C = self._dbc(x)
        y, scan = selective_scan(x, dt, -self.A_log.exp(), B, C, self.D, z, self.dt_bias,
                                 output_final_state=want_state, cu_seqlens=cu_seqlens)
        return F.linear(y, self.o_proj), conv, scan

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
        """x [B, T, dim] -> [B, T, dim]; documents may be packed along T (B = 1, ``cu_seqlens``)."""
        return self.mix(self._norm(x), cu_seqlens)

    def mix(self, h: torch.Tensor, cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
        """The block behind its input norm: h [B, T, dim] -> [B, T, dim]."""
        return self._mix(h, cu_seqlens)[0]

    def make_pool(self, slots: int) -> SSMPool:
        """Zero states for `slots` requests, in float32 whatever the parameters' type."""
        new = lambda *s: self.in_norm.new_zeros(s, dtype=torch.float32)  # noqa: E731
        return SSMPool(new(slots, self.inner, self.taps - 1), new(slots, self.inner, self.state))

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, cu_seqlens: torch.Tensor, pool: SSMPool, slots: torch.Tensor) -> torch.Tensor:
        """Prompts packed along T: x [1, T, dim], cu_seqlens [R + 1], slots [R]; the requests' states go
        to their slots of the pool.  A negative slot marks a padding request, as in ``step``.  Returns [1, T, dim]."""
        return self.mix_prefill(self._norm(x), cu_seqlens, pool, slots)

    @torch.no_grad()
    def mix_prefill(self, h: torch.Tensor, cu_seqlens: torch.Tensor, pool: SSMPool, slots: torch.Tensor) -> torch.Tensor:
        """``prefill`` behind the input norm."""
        y, conv, scan = self._mix(h, cu_seqlens, want_state=True)
        if slots.dtype != torch.int32:
            slots = slots.clamp(-1, 2 ** 31 - 1).to(torch.int32)
        slots = slots.contiguous()
        put_states(conv, pool.conv, slots)
        put_states(scan, pool.scan, slots)
        return y

    @torch.no_grad()
    def step(self, x: torch.Tensor, pool: SSMPool, slots: torch.Tensor) -> torch.Tensor:
        """One token of each request: x [R, dim], slots int32 [R] (negative: a padding row) -> [R, dim]."""
        return self.mix_step(self._norm(x), pool, slots)

    @torch.no_grad()
    def mix_step(self, h: torch.Tensor, pool: SSMPool, slots: torch.Tensor) -> torch.Tensor:
        """``step`` behind the input norm."""
        x, z = self._in(h)
        x = short_conv_step(x, pool.conv, self.conv_weight, self.conv_bias, slots=slots)
        dt, B, C = self._dbc(x)
        y = selective_scan_step(x, dt, -self.A_log.exp(), B, C, pool.scan, self.D, z, self.dt_bias, slots=slots)
        return F.linear(y, self.o_proj)


def train_step(block: SSMMixerBlock, optimizer: torch.optim.Optimizer, x: torch.Tensor, target: torch.Tensor,
               max_norm: float = 1.0, cu_seqlens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One optimizer step on the mean squared error, gradients clipped to `max_norm`.  Returns
    (loss, gradient norm), both on the device."""
    optimizer.zero_grad(set_to_none=True)
    with torch.autocast("cuda", torch.bfloat16):
        y = block(x, cu_seqlens)
    loss = F.mse_loss(y.float(), target.float())
    loss.backward()
    norm = clip_grad_norm_([p.grad for p in block.parameters()], max_norm)
    optimizer.step()
    return loss.detach(), norm
