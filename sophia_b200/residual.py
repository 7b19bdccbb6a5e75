"""What stands between two mixers of a stack: norms behind and in front of a block,
its gate, dropout and residual scale, fused into one pass over the tokens.

``residual_norm`` takes the residual stream and a block's output and returns the
new stream and what the next block reads.  It sits beside ``gated_rms_norm``, the
norm inside the KDA mixer; types, strides, errors and compilation are those of the
state-space operators (``ssm.py``).  The reference keeps a plain pre-norm in front
of every block (``ml/runtime/model/blocks.py:51-87``).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib
from ._lib import NormArgs
from .ssm import (_IO, _call, _check_activations, _check_no_tangents, _check_params, _first_order, _needs_grad, _param, _ptr,
                  _rows)

__all__ = ["residual_norm"]

MAX_WIDTH = 8192


def _args(x, o, gate, w, wb, scale, seed, seed_value, offset, p, eps):
    b, t, D = x.shape
    xb, xt, _ = x.stride()
    ob, ot, _ = o.stride()
    gb, gt, _ = (0, 0, 0) if gate is None else gate.stride()
    return NormArgs(b, t, D, _IO[o.dtype], _IO[x.dtype], offset, x.data_ptr(), o.data_ptr(), _ptr(gate), xb, xt, ob, ot, gb,
                    gt, _ptr(w), _ptr(wb), _ptr(scale), _ptr(seed), seed_value & (2 ** 64 - 1), p, eps)


def _new(t: Tensor) -> Tensor:
    """A contiguous tensor of t's shape and type."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _fwd_impl(x, o, gate, weight, branch_weight, scale, seed, seed_value, offset, p, eps, training):
    """x, o, gate [B, T, D].  Returns (stream, next block's input or empty, reciprocal roots or empty)."""
    xr, orr, gr = _rows(x, x.dtype), _rows(o, o.dtype), None if gate is None else _rows(gate, o.dtype)
    w, wb, sc = _param(weight), _param(branch_weight), _param(scale)  # (held: the arguments are addresses)
    a = _args(xr, orr, gr, w, wb, sc, seed, seed_value, offset, p, eps)
    v = _new(x)
    n = _new(o) if weight is not None else o.new_empty(0)
    rstd = x.new_empty((x.shape[0] * x.shape[1], 2) if training else 0, dtype=torch.float32)
    a.v, a.n, a.rstd = v.data_ptr(), n.data_ptr(), rstd.data_ptr()
    _call(_lib.load().kda_b200_norm_fwd, x.device, a)
    return v, n, rstd


def _sum_of(t: Tensor | None, x: Tensor) -> Tensor:
    """Where the gradient of a parameter goes: float32, empty where there is no parameter."""
    if t is not None and t.dtype == torch.float32:
        return _new(t)
    return x.new_empty(0 if t is None else t.shape, dtype=torch.float32)


def _bwd_impl(x, o, gate, weight, branch_weight, scale, seed, rstd, dv, dn, seed_value, offset, p, eps):
    """Returns (dx, do, dgate, dweight, dbranch_weight, dscale); absent ones empty."""
    lib = _lib.load()
    xr, orr, gr = _rows(x, x.dtype), _rows(o, o.dtype), None if gate is None else _rows(gate, o.dtype)
    w, wb, sc = _param(weight), _param(branch_weight), _param(scale)
    a = _args(xr, orr, gr, w, wb, sc, seed, seed_value, offset, p, eps)
    dvr = None if dv is None else _rows(dv, x.dtype)
    dnr = None if dn is None else _rows(dn, o.dtype)
    dx, do = _new(x), _new(o)
    dgate = _new(o) if gate is not None else o.new_empty(0)
    dw, dwb, dscale = _sum_of(weight, x), _sum_of(branch_weight, x), _sum_of(scale, x)
    ws = x.new_empty(lib.kda_b200_norm_workspace_bytes(a.B, a.T, a.D, a.dtype), dtype=torch.uint8)
    a.rstd = rstd.data_ptr()
    if dvr is not None:
        a.dv, (a.dv_sb, a.dv_st, _) = dvr.data_ptr(), dvr.stride()
    if dnr is not None:
        a.dn, (a.dn_sb, a.dn_st, _) = dnr.data_ptr(), dnr.stride()
    a.dx, a.d_o, a.dgate, a.dw, a.dwb, a.dscale = (t.data_ptr() for t in (dx, do, dgate, dw, dwb, dscale))
    _call(lib.kda_b200_norm_bwd, x.device, a, ws.data_ptr(), ws.numel())
    return dx, do, dgate, dw, dwb, dscale


@torch.library.custom_op("sophia_b200::residual_norm_fwd", mutates_args=(), device_types="cuda")
def _norm_fwd(x: Tensor, o: Tensor, gate: Optional[Tensor], weight: Optional[Tensor], branch_weight: Optional[Tensor],
              scale: Optional[Tensor], seed: Optional[Tensor], seed_value: int, offset: int, p: float, eps: float,
              training: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _fwd_impl(x, o, gate, weight, branch_weight, scale, seed, seed_value, offset, p, eps, training)


@_norm_fwd.register_fake
def _(x, o, gate, weight, branch_weight, scale, seed, seed_value, offset, p, eps, training):
    return (x.new_empty(x.shape), o.new_empty(o.shape if weight is not None else (0,)),
            x.new_empty((x.shape[0] * x.shape[1], 2) if training else (0,), dtype=torch.float32))


@torch.library.custom_op("sophia_b200::residual_norm_bwd", mutates_args=(), device_types="cuda")
def _norm_bwd(x: Tensor, o: Tensor, gate: Optional[Tensor], weight: Optional[Tensor], branch_weight: Optional[Tensor],
              scale: Optional[Tensor], seed: Optional[Tensor], rstd: Tensor, dv: Optional[Tensor], dn: Optional[Tensor],
              seed_value: int, offset: int, p: float, eps: float
              ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _bwd_impl(x, o, gate, weight, branch_weight, scale, seed, rstd, dv, dn, seed_value, offset, p, eps)


@_norm_bwd.register_fake
def _(x, o, gate, weight, branch_weight, scale, seed, rstd, dv, dn, seed_value, offset, p, eps):
    col = lambda t: x.new_empty((0,) if t is None else (x.shape[2],), dtype=torch.float32)  # noqa: E731
    return (x.new_empty(x.shape), o.new_empty(o.shape), o.new_empty(o.shape if gate is not None else (0,)), col(weight),
            col(branch_weight), col(scale))


def _grads(ctx, dv, dn, bwd):
    x, o, gate, weight, branch_weight, scale, seed, rstd = ctx.saved_tensors
    dn = None if dn is None or weight is None else dn
    dx, do, dgate, dw, dwb, dscale = bwd(x, o, gate, weight, branch_weight, scale, seed, rstd, dv, dn, *ctx.numbers)
    return (dx, do, None if gate is None else dgate, None if weight is None else dw.to(weight.dtype),
            None if branch_weight is None else dwb.to(branch_weight.dtype), None if scale is None else dscale.to(scale.dtype))


def _setup(ctx, inputs, output):
    *tensors, seed_value, offset, p, eps, training = inputs
    if not training:
        raise RuntimeError("residual_norm_fwd was called with training=False but autograd needs its backward")
    ctx.save_for_backward(*tensors, output[2])
    ctx.numbers = (seed_value, offset, p, eps)


_norm_fwd.register_autograd(lambda ctx, dv, dn, _r: (*_grads(ctx, dv, dn, _norm_bwd), *[None] * 6), setup_context=_setup)


class _NormEager(torch.autograd.Function):
    """The eager path: the custom ops' implementation without their dispatch."""

    @staticmethod
    def forward(ctx, x, o, gate, weight, branch_weight, scale, seed, seed_value, offset, p, eps):
        v, n, rstd = _fwd_impl(x, o, gate, weight, branch_weight, scale, seed, seed_value, offset, p, eps, True)
        ctx.save_for_backward(x, o, gate, weight, branch_weight, scale, seed, rstd)
        ctx.numbers = (seed_value, offset, p, eps)
        ctx.set_materialize_grads(False)
        return v, n

    @staticmethod
    def backward(ctx, dv, dn):
        grads = _first_order("residual_norm", ctx, _grads(ctx, dv, dn, _bwd_impl), dv, dn)
        return (*grads, *[None] * 5)


def _seed_of(seed, device):
    """(device tensor or None, value)"""
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"seed must be an int or an int64 tensor of one element, got {seed.dtype} {list(seed.shape)}")
        if seed.device != device:
            raise RuntimeError(f"residual_norm: the seed is on {seed.device}, the activations on {device}")
        return seed, 0
    if not isinstance(seed, int):
        raise ValueError("dropout needs a seed: an int or an int64 tensor of one element on the activations' device")
    value = seed & (2 ** 64 - 1)
    return None, value - 2 ** 64 if value >= 2 ** 63 else value


def _three(t: Tensor | None) -> Tensor | None:
    """[..., D] as [B, T, D], a view where the strides allow one."""
    if t is None or t.dim() == 3:
        return t
    if t.dim() < 3:
        return t.reshape(1, -1, t.shape[-1]) if t.dim() == 1 else t.unsqueeze(0)
    return t.flatten(0, -3)  # (reshape(-1, ...) has no answer where a dimension is 0)


def residual_norm(residual: Tensor, branch: Tensor, weight: Tensor | None = None, *, branch_weight: Tensor | None = None,
                  gate: Tensor | None = None, scale: Tensor | None = None, dropout_p: float = 0.0,
                  seed: Tensor | int | None = None, offset: int = 0, eps: float = 1e-5
                  ) -> tuple[Tensor, Tensor | None]:
    """Adds a block's output to the residual stream and norms the sum for the next block::

        u = branch                     (rms_norm(branch) * branch_weight with branch_weight)
        u = u * sigmoid(gate)          (with gate)
        u = dropout(u)                 (with dropout_p > 0)
        stream = residual + scale * u
        normed = rms_norm(stream) * weight

    with ``rms_norm(a) = a / sqrt(mean(a^2) + eps)`` over the last dimension, D <= 8192.
    residual, branch: ``[..., D]``; gate: logits of branch's shape, or ``[..., D]`` whose
    leading dimensions broadcast to it; weight, branch_weight, scale: ``[D]``.  The residual may be
    float32 beside a 16-bit branch.  Returns ``(stream, normed)``: the stream in residual's type,
    normed in branch's, or None without weight.

    Dropout needs a ``seed``, an int or an int64 tensor of one element on the device, which a
    captured step may change between replays (but not between a call and its backward).
    ``offset`` (below 2^32) numbers the calls that share a seed.  Element (row, channel) is
    dropped where its 32 bits of Philox4x32-10 -- key: the seed, counter: (channel // 4, row, row
    >> 32, offset) -- are below ``dropout_p 2^32``; the others are divided by ``1 - dropout_p``.
    The mask is never stored.  Gradients reach every floating-point tensor."""
    what = "residual_norm"
    if residual.shape != branch.shape:
        raise ValueError(f"{what}: branch must have residual's shape {list(residual.shape)}, got {list(branch.shape)}")
    if branch.dim() < 1 or branch.shape[-1] < 1:
        raise ValueError(f"{what}: the tensors must have shape [..., D] with D >= 1, got {list(branch.shape)}")
    _check_activations(what, x=residual, branch=branch, gate=gate)
    D = branch.shape[-1]
    if D > MAX_WIDTH:
        raise NotImplementedError(f"{what}: at most {MAX_WIDTH} channels are supported, got {D}")
    if gate is not None and gate.shape != branch.shape:
        if gate.dim() > branch.dim() or gate.dim() < 1 or gate.shape[-1] != D:
            raise ValueError(f"{what}: gate must broadcast to {list(branch.shape)} over its leading dimensions, "
                             f"got {list(gate.shape)}")
        try:
            gate = gate.expand(branch.shape)
        except RuntimeError:
            raise ValueError(f"{what}: gate must broadcast to {list(branch.shape)} over its leading dimensions, "
                             f"got {list(gate.shape)}") from None
    _check_params(what, branch.device, weight=(weight, (D,)), branch_weight=(branch_weight, (D,)), scale=(scale, (D,)))
    if not 0.0 <= dropout_p <= 1.0:
        raise ValueError(f"dropout_p must be in [0, 1], got {dropout_p}")
    if not 0 <= offset < 2 ** 32:
        raise ValueError(f"offset must be in [0, 2^32), got {offset}")
    seed, value = _seed_of(seed, branch.device) if dropout_p > 0 else (None, 0)
    io = branch.dtype if gate is None or gate.dtype == branch.dtype else torch.promote_types(branch.dtype, gate.dtype)
    wide = residual.dtype if residual.dtype == io else torch.float32
    if io != torch.float32 and residual.dtype not in (io, torch.float32):  # bf16 beside fp16
        io = torch.float32
    shape = branch.shape
    x = residual if residual.dtype == wide else residual.to(wide)
    o = branch if branch.dtype == io else branch.to(io)
    g = gate if gate is None or gate.dtype == io else gate.to(io)
    if branch.dim() != 3:
        x, o, g = _three(x), _three(o), _three(g)
    args = (x, o, g, weight, branch_weight, scale, seed, value, offset, float(dropout_p), float(eps))
    training = _needs_grad(residual, branch, weight, branch_weight, gate, scale)
    if torch.compiler.is_compiling():
        v, n, _ = _norm_fwd(*args, training)
    elif training:
        v, n = _NormEager.apply(*args)
    else:
        _check_no_tangents(what, residual, branch, weight, branch_weight, gate, scale)
        v, n, _ = _fwd_impl(*args, False)
    if v.shape != shape:
        v = v.reshape(shape)
    if v.dtype != residual.dtype:
        v = v.to(residual.dtype)
    if weight is None:
        return v, None
    if n.shape != shape:
        n = n.reshape(shape)
    return v, (n if n.dtype == branch.dtype else n.to(branch.dtype))
