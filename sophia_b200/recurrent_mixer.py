"""A gated-recurrence mixer block on the B200 kernels, for training and serving, and a
stack of mixers joined by the residual norm.

``RecurrentMixerBlock``: RMSNorm of the block input -> one projection to the
channels x and their gate z -> ``short_conv`` -> low-rank projections of x to the decay's
and the input's gate -> ``gated_recurrence`` (output gate included) -> out-projection.
It follows ``SSMMixerBlock``'s conventions (fp32 parameters, cuBLAS for the
projections, ``torch.autocast`` for bf16, states of requests in a pool of slots).

``ResidualStack`` runs mixer blocks one after the other (``KDAMixerBlock``,
``SSMMixerBlock``, ``RecurrentMixerBlock``, in any order): between two of them
``residual_norm`` norms, gates, drops and scales a block's output, adds it to the
residual stream and norms the sum for the next block.
"""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch
from torch import nn
from torch.nn import functional as F

from .recurrence import gated_recurrence, gated_recurrence_step
from .residual import residual_norm
from .ssm import put_states, short_conv, short_conv_step


class RecurrentPool(NamedTuple):
    """The states of `slots` requests: the convolution's last inputs and the recurrence's state."""

    conv: torch.Tensor  # [slots, inner, taps - 1] float32
    state: torch.Tensor  # [slots, inner] float32


class RecurrentMixerBlock(nn.Module):
    def __init__(self, dim: int = 1536, inner: int = 2048, rank: int = 128, conv_kernel: int = 4, eps: float = 1e-5,
                 decay_min: float = 0.9, decay_max: float = 0.999, std: float = 0.02,
                 generator: torch.Generator | None = None, device: torch.device | str | None = None) -> None:
        super().__init__()
        self.dim, self.inner, self.rank, self.taps, self.eps = dim, inner, rank, conv_kernel, eps
        kw = {"device": device, "dtype": torch.float32}

        def normal(*shape):
            return nn.Parameter(torch.randn(*shape, generator=generator, **kw) * std)

        self.in_norm = nn.Parameter(torch.ones(dim, **kw))
        self.w_xz = normal(2 * inner, dim)
        self.conv_weight = normal(inner, conv_kernel)
        self.conv_bias = nn.Parameter(torch.zeros(inner, **kw))
        self.w_low = normal(2 * rank, inner)  # decay and input gate, low rank
        self.decay_up, self.gate_up = normal(inner, rank), normal(inner, rank)
        self.decay_bias = nn.Parameter(torch.zeros(inner, **kw))
        self.gate_bias = nn.Parameter(torch.zeros(inner, **kw))
        # a decay at a half-open gate spread over [decay_min, decay_max]: exp(A / 2)
        u = torch.rand(inner, generator=generator, **kw)
        self.A_log = nn.Parameter(torch.log(-2 * torch.log(decay_min + u * (decay_max - decay_min))))
        self.o_proj = normal(dim, inner)

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        return F.rms_norm(x, (self.dim,), self.in_norm.to(x.dtype), self.eps)

    def _in(self, h: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return F.linear(h, self.w_xz).split(self.inner, dim=-1)  # x and z, read in place

    def _gates(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        decay, gate = F.linear(x, self.w_low).split(self.rank, dim=-1)
        return F.linear(decay, self.decay_up), F.linear(gate, self.gate_up)

    def _mix(self, h, cu_seqlens=None, want_state=False):
        x, z = self._in(h)
        x, conv = short_conv(x, self.conv_weight, self.conv_bias, activation=None, output_final_state=want_state,
                             cu_seqlens=cu_seqlens)
        decay, gate = self._gates(x)
        y, state = gated_recurrence(x, decay, gate, -self.A_log.exp(), z, self.decay_bias, self.gate_bias,
                                    output_final_state=want_state, cu_seqlens=cu_seqlens)
        return F.linear(y, self.o_proj), conv, state

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
        """x [B, T, dim] -> [B, T, dim]; documents may be packed along T (B = 1, ``cu_seqlens``)."""
        return self.mix(self._norm(x), cu_seqlens)

    def mix(self, h: torch.Tensor, cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
        """The block behind its input norm: h [B, T, dim] -> [B, T, dim]."""
        return self._mix(h, cu_seqlens)[0]

    def make_pool(self, slots: int) -> RecurrentPool:
        """Zero states for `slots` requests, in float32 whatever the parameters' type."""
        new = lambda *s: self.in_norm.new_zeros(s, dtype=torch.float32)  # noqa: E731
        return RecurrentPool(new(slots, self.inner, self.taps - 1), new(slots, self.inner))

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, cu_seqlens: torch.Tensor, pool: RecurrentPool, slots: torch.Tensor) -> torch.Tensor:
        """Prompts packed along T: x [1, T, dim], cu_seqlens [R + 1], slots [R]; the requests' states go
        to their slots of the pool.  A negative slot marks a padding request, as in ``step``.  Returns [1, T, dim]."""
        return self.mix_prefill(self._norm(x), cu_seqlens, pool, slots)

    @torch.no_grad()
    def mix_prefill(self, h: torch.Tensor, cu_seqlens: torch.Tensor, pool: RecurrentPool,
                    slots: torch.Tensor) -> torch.Tensor:
        """``prefill`` behind the input norm."""
        y, conv, state = self._mix(h, cu_seqlens, want_state=True)
        if slots.dtype != torch.int32:
            slots = slots.clamp(-1, 2 ** 31 - 1).to(torch.int32)
        slots = slots.contiguous()
        put_states(conv, pool.conv, slots)
        put_states(state, pool.state, slots)
        return y

    @torch.no_grad()
    def step(self, x: torch.Tensor, pool: RecurrentPool, slots: torch.Tensor) -> torch.Tensor:
        """One token of each request: x [R, dim], slots int32 [R] (negative: a padding row) -> [R, dim]."""
        return self.mix_step(self._norm(x), pool, slots)

    @torch.no_grad()
    def mix_step(self, h: torch.Tensor, pool: RecurrentPool, slots: torch.Tensor) -> torch.Tensor:
        """``step`` behind the input norm."""
        x, z = self._in(h)
        x = short_conv_step(x, pool.conv, self.conv_weight, self.conv_bias, activation=None, slots=slots)
        decay, gate = self._gates(x)
        y = gated_recurrence_step(x, decay, gate, -self.A_log.exp(), pool.state, z, self.decay_bias, self.gate_bias,
                                  slots=slots)
        return F.linear(y, self.o_proj)


class ResidualStack(nn.Module):
    """Mixer blocks of one width around a residual stream:

        h = rms_norm(x) * blocks[0].in_norm
        for every block i:
            x, h = residual_norm(x, block.mix(h), next norm's weight, branch norm, gate, scale, dropout)

    The norm in front of a block is the block's own ``in_norm``, the one behind the last is ``out_norm``; all norms have
    the eps that the blocks share (blocks that differ in it are refused).  ``post_norm`` norms every block's output,
    ``gate`` multiplies it with a sigmoid of a projection of the block's input, ``scale_init`` gives each block a scale
    per channel that starts there.  ``forward`` returns (stream, normed stream)."""

    def __init__(self, blocks: Sequence[nn.Module], post_norm: bool = True, gate: bool = False,
                 scale_init: float | None = None, dropout_p: float = 0.0, std: float = 0.02,
                 generator: torch.Generator | None = None) -> None:
        super().__init__()
        if not blocks:
            raise ValueError("ResidualStack needs at least one block")
        dims = {b.dim for b in blocks}
        if len(dims) != 1:
            raise ValueError(f"ResidualStack: the blocks' widths differ: {sorted(dims)}")
        epss = {b.eps for b in blocks}
        if len(epss) != 1:  # one call norms a block's output and the next block's input
            raise ValueError(f"ResidualStack: the blocks' eps differ: {sorted(epss)}")
        self.dim, self.eps, self.dropout_p = blocks[0].dim, blocks[0].eps, dropout_p
        self.blocks = nn.ModuleList(blocks)
        like = blocks[0].in_norm

        def each(make):
            return nn.ParameterList([nn.Parameter(make()) for _ in blocks])

        self.out_norm = nn.Parameter(torch.ones_like(like))
        self.post_norms = each(lambda: torch.ones_like(like)) if post_norm else None
        self.scales = each(lambda: torch.full_like(like, scale_init)) if scale_init is not None else None
        self.w_gates = each(lambda: torch.randn(self.dim, self.dim, generator=generator, device=like.device,
                                                dtype=torch.float32) * std) if gate else None

    def _join(self, i: int, x, h, branch, seed):
        """The stream and the next block's input behind block i."""
        after = self.blocks[i + 1].in_norm if i + 1 < len(self.blocks) else self.out_norm
        return residual_norm(x, branch, after, branch_weight=None if self.post_norms is None else self.post_norms[i],
                             gate=None if self.w_gates is None else F.linear(h, self.w_gates[i]),
                             scale=None if self.scales is None else self.scales[i],
                             dropout_p=self.dropout_p if seed is not None else 0.0, seed=seed, offset=i, eps=self.eps)

    def _first(self, x):
        return F.rms_norm(x, (self.dim,), self.blocks[0].in_norm.to(x.dtype), self.eps)

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                seed: torch.Tensor | int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """x [B, T, dim]; documents may be packed along T (B = 1, ``cu_seqlens``).  Dropout needs a ``seed`` of every step's
        own (an int, or an int64 tensor on the device); without one nothing is dropped."""
        h = self._first(x)
        for i, block in enumerate(self.blocks):
            branch = block.mix(h) if cu_seqlens is None else block.mix(h, cu_seqlens)
            x, h = self._join(i, x, h, branch, seed)
        return x, h

    def make_pools(self, slots: int) -> list:
        """Zero states of every block for `slots` requests."""
        for b in self.blocks:
            if not hasattr(b, "mix_step"):
                raise NotImplementedError(f"{type(b).__name__} keeps no states in a pool")
        return [b.make_pool(slots) for b in self.blocks]

    def _with(self, pools):
        """The blocks with their pools."""
        if len(pools) != len(self.blocks):
            raise ValueError(f"ResidualStack: {len(pools)} pools for {len(self.blocks)} blocks")
        return enumerate(zip(self.blocks, pools))

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, cu_seqlens: torch.Tensor, pools: list,
                slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Prompts packed along T (x [1, T, dim]), their states to the requests' slots of every block's pool."""
        h = self._first(x)
        for i, (block, pool) in self._with(pools):
            x, h = self._join(i, x, h, block.mix_prefill(h, cu_seqlens, pool, slots), None)
        return x, h

    @torch.no_grad()
    def step(self, x: torch.Tensor, pools: list, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """One token of each request: x [R, dim]."""
        h = self._first(x)
        for i, (block, pool) in self._with(pools):
            x, h = self._join(i, x, h, block.mix_step(h, pool, slots), None)
        return x, h
