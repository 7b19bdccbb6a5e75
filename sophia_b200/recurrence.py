"""Gated linear recurrence: one state per channel, gates per token and channel.

``gated_recurrence`` is the recurrence of a mixer beside KDA and the selective
scan, for prompts and training (differentiable, packed documents, initial and
final states); ``gated_recurrence_step`` takes single tokens with their states in
a pool, for decoding.  Types, strides, errors and compilation are those of the
state-space operators (``ssm.py``).  The reference has no counterpart.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import RecArgs
from .ssm import (_IO, _call, _check_activations, _check_no_tangents, _check_params, _check_pool, _check_state, _cu,
                  _first_order, _needs_grad, _num_seqs, _param, _ptr, _rows)

__all__ = ["gated_recurrence", "gated_recurrence_step"]

TILE = {torch.float32: 32, torch.bfloat16: 64, torch.float16: 64}  # tokens between the states kept for a backward


def _new(t: Tensor) -> Tensor:
    """A contiguous tensor of t's shape and type."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _workspace(lib, x: Tensor, cu: Tensor | None, backward: bool) -> Tensor | None:
    """A prompt of plain rows needs none."""
    if cu is None and not backward:
        return None
    b, T, E = x.shape
    return x.new_empty(lib.kda_b200_recurrence_workspace_bytes(b, T, E, _IO[x.dtype], int(cu is not None), int(backward)),
                       dtype=torch.uint8)


def _inputs(x, decay, gate, z):
    return tuple(None if t is None else _rows(t, x.dtype) for t in (x, decay, gate, z))


def _args(rows, nseq, A, decay_bias, gate_bias, h0, cu):
    """The fields that both directions share."""
    x, decay, gate, z = rows
    b, T, E = x.shape
    xb, xt, _ = x.stride()
    db, dt, _ = decay.stride()
    gb, gt, _ = gate.stride()
    zb, zt, _ = (0, 0, 0) if z is None else z.stride()
    return RecArgs(b, T, E, nseq, _IO[x.dtype], 0, x.data_ptr(), decay.data_ptr(), gate.data_ptr(), _ptr(z), xb, xt, db, dt,
                   gb, gt, zb, zt, A.data_ptr(), _ptr(decay_bias), _ptr(gate_bias), _ptr(h0), _ptr(cu))


def _fwd_impl(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, want_final, training):
    """Returns (y, final state or empty, saved buffer or empty)."""
    b, T, E = x.shape
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    lib, io = _lib.load(), _IO[x.dtype]
    rows = _inputs(x, decay, gate, z)
    A, decay_bias, gate_bias, h0, cu = _param(A), _param(decay_bias), _param(gate_bias), _param(h0), _cu(cu_seqlens)
    y = _new(x)
    ht = x.new_empty((nseq, E) if want_final else 0, dtype=torch.float32)
    saved = x.new_empty(lib.kda_b200_recurrence_saved_bytes(b, T, E, io) if training else 0, dtype=torch.uint8)
    if b:
        ws = _workspace(lib, x, cu, False)
        a = _args(rows, nseq, A, decay_bias, gate_bias, h0, cu)
        a.y, a.ht, a.saved, a.saved_bytes = y.data_ptr(), ht.data_ptr(), saved.data_ptr(), saved.numel()
        _call(lib.kda_b200_recurrence_fwd, x.device, a, _ptr(ws), 0 if ws is None else ws.numel())
    return y, ht, saved


def _bwd_impl(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, saved, dy, dht, want_dh0):
    """Returns (dx, ddecay, dgate, dA, dz, ddecay_bias, dgate_bias, dh0); absent ones empty."""
    b, T, E = x.shape
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    lib = _lib.load()
    rows, dyr = _inputs(x, decay, gate, z), _rows(dy, x.dtype)
    Af, dbias, gbias, h, cu, dh = (_param(A), _param(decay_bias), _param(gate_bias), _param(h0), _cu(cu_seqlens),
                                   _param(dht))
    dx, ddecay, dgate = _new(x), _new(x), _new(x)
    dz = _new(x) if z is not None else x.new_empty(0)
    dA, ddb, dgb = (x.new_empty(E, dtype=torch.float32) for _ in range(3))
    dh0 = x.new_empty((nseq, E) if want_dh0 else 0, dtype=torch.float32)
    if b:
        ws = _workspace(lib, x, cu, True)
        a = _args(rows, nseq, Af, dbias, gbias, h, cu)
        a.saved, a.saved_bytes = saved.data_ptr(), saved.numel()
        a.dy, (a.dy_sb, a.dy_st, _) = dyr.data_ptr(), dyr.stride()
        a.dht, a.dx, a.ddecay, a.dgate, a.dz, a.dh0 = _ptr(dh), _ptr(dx), _ptr(ddecay), _ptr(dgate), _ptr(dz), _ptr(dh0)
        a.dA, a.ddecay_bias, a.dgate_bias = _ptr(dA), _ptr(ddb), _ptr(dgb)
        _call(lib.kda_b200_recurrence_bwd, x.device, a, ws.data_ptr(), ws.numel())
    else:
        dA.zero_(), ddb.zero_(), dgb.zero_()
    return dx, ddecay, dgate, dA, dz, ddb, dgb, dh0


@torch.library.custom_op("sophia_b200::gated_recurrence_fwd", mutates_args=(), device_types="cuda")
def _rec_fwd(x: Tensor, decay: Tensor, gate: Tensor, A: Tensor, z: Optional[Tensor], decay_bias: Optional[Tensor],
             gate_bias: Optional[Tensor], h0: Optional[Tensor], cu_seqlens: Optional[Tensor], want_final: bool,
             training: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _fwd_impl(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, want_final, training)


@_rec_fwd.register_fake
def _(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, want_final, training):
    b, T, E = x.shape
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    # kda_b200_recurrence_saved_bytes() in symbols: a size of its own per length would compile for every length
    nbytes = torch.sym_max(16, b * ((T + TILE[x.dtype] - 1) // TILE[x.dtype]) * E * 4) if training else 0
    return (x.new_empty((b, T, E)), x.new_empty((nseq, E) if want_final else (0,), dtype=torch.float32),
            x.new_empty((nbytes,), dtype=torch.uint8))


@torch.library.custom_op("sophia_b200::gated_recurrence_bwd", mutates_args=(), device_types="cuda")
def _rec_bwd(x: Tensor, decay: Tensor, gate: Tensor, A: Tensor, z: Optional[Tensor], decay_bias: Optional[Tensor],
             gate_bias: Optional[Tensor], h0: Optional[Tensor], cu_seqlens: Optional[Tensor], saved: Tensor, dy: Tensor,
             dht: Optional[Tensor], want_dh0: bool
             ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _bwd_impl(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, saved, dy, dht, want_dh0)


@_rec_bwd.register_fake
def _(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, saved, dy, dht, want_dh0):
    b, T, E = x.shape
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    act = lambda t: x.new_empty((b, T, E) if t is not None else (0,))  # noqa: E731
    f = lambda *s: x.new_empty(s, dtype=torch.float32)  # noqa: E731
    return act(x), act(x), act(x), f(E), act(z), f(E), f(E), f(nseq, E) if want_dh0 else f(0)


def _grads(ctx, dy, dht, bwd):
    x, decay, gate, A, z, decay_bias, gate_bias, h0, cu, saved = ctx.saved_tensors
    dht = None if dht is None or dht.numel() == 0 else dht
    dy = x.new_zeros(x.shape) if dy is None else dy
    dx, ddecay, dgate, dA, dz, ddb, dgb, dh0 = bwd(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu, saved, dy, dht,
                                                   h0 is not None)
    return (dx, ddecay, dgate, dA.to(A.dtype), None if z is None else dz,
            None if decay_bias is None else ddb.to(decay_bias.dtype),
            None if gate_bias is None else dgb.to(gate_bias.dtype), None if h0 is None else dh0)


def _setup(ctx, inputs, output):
    *tensors, _, training = inputs
    if not training:
        raise RuntimeError("gated_recurrence_fwd was called with training=False but autograd needs its backward")
    ctx.save_for_backward(*tensors, output[2])


_rec_fwd.register_autograd(lambda ctx, dy, dht, _s: (*_grads(ctx, dy, dht, _rec_bwd), None, None, None),
                           setup_context=_setup)


class _RecEager(torch.autograd.Function):
    """The eager path: the custom ops' implementation without their dispatch."""

    @staticmethod
    def forward(ctx, x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, want_final):
        y, ht, saved = _fwd_impl(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, want_final, True)
        ctx.save_for_backward(x, decay, gate, A, z, decay_bias, gate_bias, h0, cu_seqlens, saved)
        ctx.set_materialize_grads(False)
        return y, ht

    @staticmethod
    def backward(ctx, dy, dht):
        grads = _first_order("gated_recurrence", ctx, _grads(ctx, dy, dht, _bwd_impl), dy, dht)
        return (*grads, None, None)


def _check(what, x, dims, decay, gate, A, z, decay_bias, gate_bias) -> torch.dtype:
    io = _check_activations(what, x=x, decay=decay, gate=gate, z=z)
    shape = x.shape
    if x.dim() != len(dims):
        raise ValueError(f"{what}: x must have shape [{', '.join(dims)}], got {list(shape)}")
    for name, t in (("decay", decay), ("gate", gate), ("z", z)):
        if t is not None and t.shape != shape:
            raise ValueError(f"{what}: {name} must have x's shape {list(shape)}, got {list(t.shape)}")
    E = shape[-1]
    if E < 1:
        raise ValueError(f"{what}: x has no channels")
    _check_params(what, x.device, A=(A, (E,)), decay_bias=(decay_bias, (E,)), gate_bias=(gate_bias, (E,)))
    return io


def _promoted(io, *ts):
    return ts if all(t is None or t.dtype == io for t in ts) else tuple(None if t is None else t.to(io) for t in ts)


def gated_recurrence(x: Tensor, decay: Tensor, gate: Tensor, A: Tensor, z: Tensor | None = None,
                     decay_bias: Tensor | None = None, gate_bias: Tensor | None = None, *,
                     initial_state: Tensor | None = None, output_final_state: bool = False,
                     cu_seqlens: Tensor | None = None) -> tuple[Tensor, Tensor | None]:
    """Gated linear recurrence over tokens.  Per channel, with
    ``r = sigmoid(decay + decay_bias)`` and ``i = sigmoid(gate + gate_bias)``::

        a[t] = exp(A r[t])
        h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) i[t] x[t]
        y[t] = h[t] * silu(z[t])        (h[t] without z)

    x, decay, gate, z: ``[B, T, E]``, the gates as logits; A: ``[E]``, the rates
    themselves, not positive (a positive one gives NaN, -inf is the largest finite one);
    decay_bias, gate_bias: ``[E]``.  ``initial_state`` ``[sequences, E]`` float32; with ``cu_seqlens``
    (``[sequences + 1]``, B = 1) sequences are packed along T and the state restarts
    at each.  Returns ``(y, final_state | None)``, y in x's type; gradients reach every
    floating-point input.  Where 1 - a^2 is below fp32's normal range (1.2e-38) it
    counts as 0: nothing enters the state, and no gradient reaches the rate through the input."""
    what = "gated_recurrence"
    io = _check(what, x, ("B", "T", "E"), decay, gate, A, z, decay_bias, gate_bias)
    nseq = _num_seqs(what, x, cu_seqlens)
    _check_state(what, initial_state, (nseq, x.shape[2]), x.device)
    like = x.dtype
    x, decay, gate, z = _promoted(io, x, decay, gate, z)
    args = (x, decay, gate, A, z, decay_bias, gate_bias, initial_state, cu_seqlens, bool(output_final_state))
    training = _needs_grad(x, decay, gate, A, z, decay_bias, gate_bias, initial_state)
    if torch.compiler.is_compiling():
        y, ht, _ = _rec_fwd(*args, training)
    elif training:
        y, ht = _RecEager.apply(*args)
    else:
        _check_no_tangents(what, x, decay, gate, A, z, decay_bias, gate_bias, initial_state)
        y, ht, _ = _fwd_impl(*args, False)
    return (y if y.dtype == like else y.to(like)), (ht if output_final_state else None)


def _step_impl(x, decay, gate, A, state, z, decay_bias, gate_bias, slots):
    rows, E = x.shape
    xr, dr, gr, zr = _inputs(x, decay, gate, z)
    Af, db, gb = _param(A), _param(decay_bias), _param(gate_bias)
    y = x.new_empty((rows, E))
    a = RecArgs(1, 1, E, 1, _IO[x.dtype], rows, _ptr(xr), _ptr(dr), _ptr(gr), _ptr(zr), xr.stride(0), 0, dr.stride(0), 0,
                gr.stride(0), 0, zr.stride(0) if zr is not None else 0, 0, _ptr(Af), _ptr(db), _ptr(gb))
    a.y, a.state, a.slots, a.pool = _ptr(y), _ptr(state), _ptr(slots), state.shape[0]
    _call(_lib.load().kda_b200_recurrence_step, x.device, a)
    return y


@torch.library.custom_op("sophia_b200::gated_recurrence_step", mutates_args=("state",), device_types="cuda")
def _rec_step(x: Tensor, decay: Tensor, gate: Tensor, A: Tensor, state: Tensor, z: Optional[Tensor],
              decay_bias: Optional[Tensor], gate_bias: Optional[Tensor], slots: Optional[Tensor]) -> Tensor:
    return _step_impl(x, decay, gate, A, state, z, decay_bias, gate_bias, slots)


@_rec_step.register_fake
def _(x, decay, gate, A, state, z, decay_bias, gate_bias, slots):
    return x.new_empty(x.shape)


def gated_recurrence_step(x: Tensor, decay: Tensor, gate: Tensor, A: Tensor, state: Tensor, z: Tensor | None = None,
                          decay_bias: Tensor | None = None, gate_bias: Tensor | None = None, *,
                          slots: Tensor | None = None) -> Tensor:
    """One token of ``gated_recurrence`` for each of B requests.  x, decay, gate, z:
    ``[B, E]``; state: a pool ``[S, E]`` float32, updated in place; slots: int32 ``[B]``,
    each row's entry of the pool (row r uses entry r without it).  A negative slot
    marks a padding row: its y is 0 and no state is touched.  Two rows must not share
    a slot.  Inference only.  Returns y ``[B, E]`` in x's type."""
    what = "gated_recurrence_step"
    io = _check(what, x, ("B", "E"), decay, gate, A, z, decay_bias, gate_bias)
    _check_pool(what, state, (x.shape[1],), x.device, x.shape[0], slots)
    if _needs_grad(x, decay, gate, A, state, z, decay_bias, gate_bias):
        raise NotImplementedError(f"{what} has no backward; use gated_recurrence for training")
    _check_no_tangents(what, x, decay, gate, A, state, z, decay_bias, gate_bias)
    like = x.dtype
    x, decay, gate, z = _promoted(io, x, decay, gate, z)
    if torch.compiler.is_compiling():
        y = _rec_step(x, decay, gate, A, state, z, decay_bias, gate_bias, slots)
    else:
        y = _step_impl(x, decay, gate, A, state, z, decay_bias, gate_bias, slots)
        increment_version(state)
    return y if y.dtype == like else y.to(like)
