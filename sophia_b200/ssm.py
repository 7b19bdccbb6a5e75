"""State-space operators: the short causal convolution and the selective scan.

``short_conv`` and ``selective_scan`` are the two kernels of a state-space
mixer, for prompts and training (differentiable, packed documents, initial and
final states); ``short_conv_step`` and ``selective_scan_step`` take single tokens
with their states in a pool, for decoding.  They sit beside the KDA mixer and
keep its manner: one shared library behind a C ABI, ``torch.library`` custom ops
under ``torch.compile`` and a plain ``autograd.Function`` in eager mode, errors as
``ValueError`` / ``NotImplementedError`` / ``KdaError``, no other implementation
behind them.  The reference has no counterpart (its mixers are KDA and attention).

Activations may be float32, bfloat16 or float16 and strided (a slice of a wider
projection is read in place, as long as its last dimension is contiguous);
mixed types are promoted.  Arithmetic, parameters and states are float32.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import ScanArgs

__all__ = ["short_conv", "short_conv_step", "selective_scan", "selective_scan_step"]

_IO = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_STATE = 64
MAX_TAPS = 4
SAVED_EVERY = 8  # tokens between the states that the scan keeps for its backward


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()  # 0 (NULL) where there is nothing


def _call(fn, device: torch.device, *args) -> None:
    """A library call on the current stream of the tensors' device."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)))


def _rows(t: Tensor, dtype: torch.dtype) -> Tensor:
    """An activation as the kernels read it: its type, and a contiguous last dimension."""
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(t: Tensor | None) -> Tensor | None:
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.float().contiguous()


def _cu(cu_seqlens: Tensor | None) -> Tensor | None:
    if cu_seqlens is None or (cu_seqlens.dtype == torch.int32 and cu_seqlens.is_contiguous()):
        return cu_seqlens
    return cu_seqlens.to(torch.int32).contiguous()


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _check_no_tangents(what: str, *tensors: Tensor | None) -> None:
    """Refuses forward-mode differentiation, whose tangents a kernel called directly would drop."""
    if forward_ad._current_level < 0:  # no dual numbers anywhere
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


class _FirstOrder(torch.autograd.Function):
    """Gradients of a backward under ``create_graph``: they depend on the inputs, but how is not provided."""

    @staticmethod
    def forward(ctx, what, count, *tensors):
        ctx.what = what
        return tuple(None if t is None else t.view_as(t) for t in tensors[:count])

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError(f"{ctx.what} has no second derivative")


def _first_order(what: str, ctx, grads: tuple, *dys: Tensor | None) -> tuple:
    """The gradients as they are, or, where a graph of them is built, so that differentiating them is refused; they
    would count as constants otherwise."""
    if not torch.is_grad_enabled():
        return grads
    depend = (*dys, *ctx.saved_tensors)
    return _FirstOrder.apply(what, len(grads), *grads, *depend)


def _check_activations(what: str, **tensors) -> torch.dtype:
    """All on one CUDA device and of supported types; returns the promoted type."""
    first = tensors["x"]
    dtype, device = first.dtype, first.device
    if device.type != "cuda" and device.type != "meta":
        raise RuntimeError(f"{what} runs on the CUDA kernels only: its tensors must be CUDA tensors")
    for name, t in tensors.items():
        if t is None:
            continue
        if t.dtype not in _IO:
            raise NotImplementedError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
        if t.dtype != dtype:
            dtype = torch.promote_types(dtype, t.dtype)
        if t.device != device:
            raise RuntimeError(f"{what}: tensors are on {device} and {t.device}")
    return dtype


def _check_params(what: str, device: torch.device, **tensors) -> None:
    for name, (t, shape) in tensors.items():
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise ValueError(f"{what}: {name} must have shape {list(shape)}, got {list(t.shape)}")
        if t.device != device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the activations on {device}")
        if not t.is_floating_point():
            raise NotImplementedError(f"{what}: {name} must be a floating-point tensor, got {t.dtype}")


def _check_state(what: str, state: Tensor | None, shape: tuple, device: torch.device) -> None:
    if state is None:
        return
    if tuple(state.shape) != shape:
        raise ValueError(f"{what}: initial_state must have shape {list(shape)}, got {list(state.shape)}")
    assert state.dtype == torch.float32, "initial_state must be in float32."
    if state.device != device:
        raise RuntimeError(f"{what}: initial_state is on {state.device}, the activations on {device}")


def _num_seqs(what: str, x: Tensor, cu_seqlens: Tensor | None) -> int:
    if cu_seqlens is None:
        return x.shape[0]
    if x.shape[0] != 1:
        raise ValueError(f"The batch size is expected to be 1 rather than {x.shape[0]} when using `cu_seqlens`.")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: cu_seqlens must be an int32 or int64 tensor of at least two entries")
    if cu_seqlens.device != x.device:
        raise RuntimeError(f"{what}: cu_seqlens is on {cu_seqlens.device}, the activations on {x.device}")
    return cu_seqlens.shape[0] - 1


def _check_pool(what: str, state: Tensor, inner: tuple, device: torch.device, rows: int, slots: Tensor | None) -> None:
    if state.dim() != 1 + len(inner) or tuple(state.shape[1:]) != inner:
        raise ValueError(f"{what}: the states must have shape {['pool', *inner]}, got {list(state.shape)}")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{what}: the states must be a contiguous float32 tensor (they are updated in place)")
    if state.device != device:
        raise RuntimeError(f"{what}: the states are on {state.device}, the activations on {device}")
    if slots is None:
        if rows > state.shape[0]:
            raise ValueError(f"{what}: {rows} rows but {state.shape[0]} states")
        return
    if tuple(slots.shape) != (rows,) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be a contiguous int32 tensor [{rows}]")
    if slots.device != device:
        raise RuntimeError(f"{what}: slots are on {slots.device}, the activations on {device}")


def _put_states_impl(new, pool, slots):
    rows = new.shape[0]
    _call(_lib.load().kda_b200_put_states, new.device,
          _ptr(new), _ptr(slots), rows, new.numel() // max(1, rows), pool.shape[0], _ptr(pool))


@torch.library.custom_op("sophia_b200::put_states", mutates_args=("pool",), device_types="cuda")
def _put_states(new: Tensor, pool: Tensor, slots: Tensor) -> None:
    _put_states_impl(new, pool, slots)


def put_states(new: Tensor, pool: Tensor, slots: Tensor) -> None:
    """Row r of ``new``, final states of a prompt call, to ``pool[slots[r]]``; padding rows as in the single-token
    calls, with their states nowhere."""
    _check_pool("put_states", pool, tuple(new.shape[1:]), new.device, new.shape[0], slots)
    if _needs_grad(new, pool):
        raise NotImplementedError("put_states has no backward")
    _check_no_tangents("put_states", new, pool)
    if torch.compiler.is_compiling():
        _put_states(_param(new), pool, slots)
    else:
        _put_states_impl(_param(new), pool, slots)
        increment_version(pool)


# --------------------------------------------------------------------------- convolution


def _conv_fwd_impl(x, weight, bias, h0, cu_seqlens, silu, want_final):
    B, T, C = x.shape
    W = weight.shape[1]
    N = B if cu_seqlens is None else cu_seqlens.shape[0] - 1
    lib = _lib.load()
    xr = _rows(x, x.dtype)
    w, b, h, cu = _param(weight), _param(bias), _param(h0), _cu(cu_seqlens)
    y = x.new_empty((B, T, C))
    ht = x.new_empty((N, C, W - 1) if want_final else 0, dtype=torch.float32)
    ws = x.new_empty(lib.kda_b200_short_conv_workspace_bytes(B, T, C, W, int(cu is not None), 0), dtype=torch.uint8)
    if B:
        _call(lib.kda_b200_short_conv_fwd, x.device,
              _ptr(xr), xr.stride(0), xr.stride(1), _ptr(w), _ptr(b), _ptr(h), _ptr(cu), B, T, C, W, N, _IO[x.dtype],
              int(silu), _ptr(y), _ptr(ht), _ptr(ws), ws.numel())
    return y, ht


def _conv_bwd_impl(x, weight, bias, h0, cu_seqlens, dy, dht, silu, want_dh0):
    B, T, C = x.shape
    W = weight.shape[1]
    N = B if cu_seqlens is None else cu_seqlens.shape[0] - 1
    lib = _lib.load()
    xr, dyr = _rows(x, x.dtype), _rows(dy, x.dtype)
    w, b, h, cu, dh = _param(weight), _param(bias), _param(h0), _cu(cu_seqlens), _param(dht)
    dx = x.new_empty((B, T, C))
    dw = x.new_empty((C, W), dtype=torch.float32)
    db = x.new_empty(C if bias is not None else 0, dtype=torch.float32)
    dh0 = x.new_empty((N, C, W - 1) if want_dh0 else 0, dtype=torch.float32)
    ws = x.new_empty(lib.kda_b200_short_conv_workspace_bytes(B, T, C, W, int(cu is not None), 1), dtype=torch.uint8)
    if B:
        _call(lib.kda_b200_short_conv_bwd, x.device,
              _ptr(xr), xr.stride(0), xr.stride(1), _ptr(w), _ptr(b), _ptr(h), _ptr(cu), B, T, C, W, N, _IO[x.dtype],
              int(silu), _ptr(dyr), dyr.stride(0), dyr.stride(1), _ptr(dh), _ptr(dx), _ptr(dw), _ptr(db), _ptr(dh0),
              _ptr(ws), ws.numel())
    else:
        dw.zero_(), db.zero_()
    return dx, dw, db, dh0


@torch.library.custom_op("sophia_b200::short_conv_fwd", mutates_args=(), device_types="cuda")
def _conv_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], h0: Optional[Tensor], cu_seqlens: Optional[Tensor],
              silu: bool, want_final: bool) -> tuple[Tensor, Tensor]:
    return _conv_fwd_impl(x, weight, bias, h0, cu_seqlens, silu, want_final)


@_conv_fwd.register_fake
def _(x, weight, bias, h0, cu_seqlens, silu, want_final):
    B, T, C = x.shape
    N = B if cu_seqlens is None else cu_seqlens.shape[0] - 1
    ht = x.new_empty((N, C, weight.shape[1] - 1) if want_final else (0,), dtype=torch.float32)
    return x.new_empty((B, T, C)), ht


@torch.library.custom_op("sophia_b200::short_conv_bwd", mutates_args=(), device_types="cuda")
def _conv_bwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], h0: Optional[Tensor], cu_seqlens: Optional[Tensor],
              dy: Tensor, dht: Optional[Tensor], silu: bool, want_dh0: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    return _conv_bwd_impl(x, weight, bias, h0, cu_seqlens, dy, dht, silu, want_dh0)


@_conv_bwd.register_fake
def _(x, weight, bias, h0, cu_seqlens, dy, dht, silu, want_dh0):
    B, T, C = x.shape
    N = B if cu_seqlens is None else cu_seqlens.shape[0] - 1
    f = lambda *s: x.new_empty(s, dtype=torch.float32)  # noqa: E731
    return (x.new_empty((B, T, C)), f(C, weight.shape[1]), f(C) if bias is not None else f(0),
            f(N, C, weight.shape[1] - 1) if want_dh0 else f(0))


def _conv_grads(ctx, dy, dht, bwd):
    x, weight, bias, h0, cu = ctx.saved_tensors
    dht = None if dht is None or dht.numel() == 0 else dht
    dy = x.new_zeros(x.shape) if dy is None else dy
    dx, dw, db, dh0 = bwd(x, weight, bias, h0, cu, dy, dht, ctx.silu, h0 is not None)
    return (dx, dw.to(weight.dtype), None if bias is None else db.to(bias.dtype),
            None if h0 is None else dh0, None, None, None)


def _conv_setup(ctx, inputs, output):
    x, weight, bias, h0, cu, silu, _ = inputs
    ctx.save_for_backward(x, weight, bias, h0, cu)
    ctx.silu = silu


_conv_fwd.register_autograd(lambda ctx, dy, dht: _conv_grads(ctx, dy, dht, _conv_bwd), setup_context=_conv_setup)


class _ConvEager(torch.autograd.Function):
    """The eager path: the custom ops' implementation without their dispatch."""

    @staticmethod
    def forward(ctx, x, weight, bias, h0, cu_seqlens, silu, want_final):
        ctx.save_for_backward(x, weight, bias, h0, cu_seqlens)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return _conv_fwd_impl(x, weight, bias, h0, cu_seqlens, silu, want_final)

    @staticmethod
    def backward(ctx, dy, dht):
        return _first_order("short_conv", ctx, _conv_grads(ctx, dy, dht, _conv_bwd_impl), dy, dht)


def _check_taps(what: str, weight: Tensor, C: int) -> int:
    if weight.dim() != 2 or weight.shape[0] != C:
        raise ValueError(f"{what}: weight must have shape {[C, 'taps']}, got {list(weight.shape)}")
    if not 1 <= weight.shape[1] <= MAX_TAPS:
        raise NotImplementedError(f"{what}: 1 to {MAX_TAPS} taps are supported, got {weight.shape[1]}")
    return weight.shape[1]


def _check_activation(activation: str | None) -> bool:
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return activation == "silu"


def short_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str | None = "silu",
               initial_state: Tensor | None = None, output_final_state: bool = False,
               cu_seqlens: Tensor | None = None) -> tuple[Tensor, Tensor | None]:
    """Causal depthwise convolution over tokens with an optional SiLU:
    ``c[t] = bias + sum_k weight[:, k] x[t - (W-1) + k]``, ``y = silu(c)``.

    x: ``[B, T, C]``; weight: ``[C, W]``, 1 <= W <= 4 (the oldest tap first, as
    ``CausalDepthwiseConv1d.weight``); bias: ``[C]``.  ``initial_state``
    ``[N, C, W-1]`` float32 holds the inputs before each sequence's first token, oldest
    first (zeros without it), and the returned final state the last ones.  With
    ``cu_seqlens`` (``[N+1]``, B = 1) sequences are packed along T.  Returns
    ``(y, final_state | None)``; gradients reach x, weight, bias and
    initial_state."""
    silu = _check_activation(activation)
    _check_activations("short_conv", x=x)
    if x.dim() != 3:
        raise ValueError(f"short_conv: x must have shape [B, T, C], got {list(x.shape)}")
    W = _check_taps("short_conv", weight, x.shape[2])
    N = _num_seqs("short_conv", x, cu_seqlens)
    C = x.shape[2]
    _check_params("short_conv", x.device, weight=(weight, (C, W)), bias=(bias, (C,)))
    _check_state("short_conv", initial_state, (N, C, W - 1), x.device)
    fn = _conv_fwd if torch.compiler.is_compiling() else _ConvEager.apply
    y, ht = fn(x, weight, bias, initial_state, cu_seqlens, silu, bool(output_final_state))
    return y, (ht if output_final_state else None)


def _conv_step_impl(x, conv_state, weight, bias, slots, silu):
    rows, C = x.shape
    xr = _rows(x, x.dtype)
    w, b = _param(weight), _param(bias)
    y = x.new_empty((rows, C))
    _call(_lib.load().kda_b200_short_conv_step, x.device,
          _ptr(xr), xr.stride(0), _ptr(w), _ptr(b), _ptr(conv_state), _ptr(slots), rows, C, weight.shape[1],
          conv_state.shape[0], _IO[x.dtype], int(silu), _ptr(y))
    return y


@torch.library.custom_op("sophia_b200::short_conv_step", mutates_args=("conv_state",), device_types="cuda")
def _conv_step(x: Tensor, conv_state: Tensor, weight: Tensor, bias: Optional[Tensor], slots: Optional[Tensor],
               silu: bool) -> Tensor:
    return _conv_step_impl(x, conv_state, weight, bias, slots, silu)


@_conv_step.register_fake
def _(x, conv_state, weight, bias, slots, silu):
    return x.new_empty(x.shape)


def short_conv_step(x: Tensor, conv_state: Tensor, weight: Tensor, bias: Tensor | None = None, *,
                    activation: str | None = "silu", slots: Tensor | None = None) -> Tensor:
    """One token of ``short_conv`` for each of B requests.  x: ``[B, C]``;
    conv_state: a pool ``[S, C, W-1]`` float32 of last inputs, updated in place;
    slots: int32 ``[B]``, each row's entry of the pool (row r uses entry r without
    it).  A negative slot marks a padding row: its y is 0 and no state is touched.
    Two rows must not share a slot.  Inference only.  Returns y ``[B, C]``."""
    silu = _check_activation(activation)
    _check_activations("short_conv_step", x=x)
    if x.dim() != 2:
        raise ValueError(f"short_conv_step: x must have shape [B, C], got {list(x.shape)}")
    rows, C = x.shape
    W = _check_taps("short_conv_step", weight, C)
    device = x.device
    _check_params("short_conv_step", device, weight=(weight, (C, W)), bias=(bias, (C,)))
    _check_pool("short_conv_step", conv_state, (C, W - 1), device, rows, slots)
    if _needs_grad(x, weight, bias, conv_state):
        raise NotImplementedError("short_conv_step has no backward; use short_conv for training")
    _check_no_tangents("short_conv_step", x, conv_state, weight, bias)
    if torch.compiler.is_compiling():
        return _conv_step(x, conv_state, weight, bias, slots, silu)
    y = _conv_step_impl(x, conv_state, weight, bias, slots, silu)
    increment_version(conv_state)  # written in place: a graph that saved it has to notice
    return y


# --------------------------------------------------------------------------- scan


def _scan_inputs(io, x, dt, B, C, z):
    return tuple(None if t is None else _rows(t, io) for t in (x, dt, B, C, z))


def _scan_fwd_impl(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, softplus, want_final, training):
    """Returns (y in the activations' type, final state or empty, saved buffer or empty)."""
    b, T, E = x.shape
    N, G = A.shape[1], B.shape[2]
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    lib = _lib.load()
    xr, dtr, Br, Cr, zr = _scan_inputs(x.dtype, x, dt, B, C, z)
    Af, Df, bf, h, cu = _param(A), _param(D), _param(dt_bias), _param(h0), _cu(cu_seqlens)
    y = x.new_empty((b, T, E))
    ht = x.new_empty((nseq, E, N) if want_final else 0, dtype=torch.float32)
    saved = x.new_empty(lib.kda_b200_scan_saved_bytes(b, T, E, N, G) if training else 0, dtype=torch.uint8)
    ws = x.new_empty(lib.kda_b200_scan_workspace_bytes(b, T, E, N, G, int(cu is not None), 0), dtype=torch.uint8)
    if b:
        a = ScanArgs(b, T, E, N, G, nseq, _IO[x.dtype], int(softplus), _ptr(xr), _ptr(dtr), _ptr(zr), _ptr(Br),
                     _ptr(Cr), xr.stride(0), xr.stride(1), dtr.stride(0), dtr.stride(1),
                     *((zr.stride(0), zr.stride(1)) if zr is not None else (0, 0)),
                     Br.stride(0), Br.stride(1), Br.stride(2), Cr.stride(0), Cr.stride(1), Cr.stride(2), _ptr(Af),
                     _ptr(Df), _ptr(bf), _ptr(h), _ptr(cu), _ptr(y), _ptr(ht), _ptr(saved), saved.numel())
        _call(lib.kda_b200_selective_scan_fwd, x.device, a, _ptr(ws), ws.numel())
    return y, ht, saved


def _scan_bwd_impl(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, saved, dy, dht, softplus, want_dh0):
    """Returns (dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dh0); absent ones empty."""
    b, T, E = x.shape
    N, G = A.shape[1], B.shape[2]
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    lib = _lib.load()
    io = x.dtype
    xr, dtr, Br, Cr, zr = _scan_inputs(io, x, dt, B, C, z)
    dyr = _rows(dy, io)
    Af, Df, bf, h, cu, dh = _param(A), _param(D), _param(dt_bias), _param(h0), _cu(cu_seqlens), _param(dht)
    new = lambda shape, dtype=torch.float32: x.new_empty(shape, dtype=dtype)  # noqa: E731
    dx, ddt = new((b, T, E), io), new((b, T, E), io)
    dz = new((b, T, E) if z is not None else (0,), io)
    dB, dC = new((b, T, G, N), io), new((b, T, G, N), io)
    dA, dD, dbias = new((E, N)), new((E,) if D is not None else (0,)), new((E,) if dt_bias is not None else (0,))
    dh0 = new((nseq, E, N) if want_dh0 else (0,))
    ws = x.new_empty(lib.kda_b200_scan_workspace_bytes(b, T, E, N, G, int(cu is not None), 1), dtype=torch.uint8)
    if b:
        a = ScanArgs(b, T, E, N, G, nseq, _IO[io], int(softplus), _ptr(xr), _ptr(dtr), _ptr(zr), _ptr(Br),
                     _ptr(Cr), xr.stride(0), xr.stride(1), dtr.stride(0), dtr.stride(1),
                     *((zr.stride(0), zr.stride(1)) if zr is not None else (0, 0)),
                     Br.stride(0), Br.stride(1), Br.stride(2), Cr.stride(0), Cr.stride(1), Cr.stride(2), _ptr(Af),
                     _ptr(Df), _ptr(bf), _ptr(h), _ptr(cu), None, None, _ptr(saved), saved.numel(),
                     _ptr(dyr), dyr.stride(0), dyr.stride(1), _ptr(dh), _ptr(dx), _ptr(ddt), _ptr(dz), _ptr(dB),
                     _ptr(dC), _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dh0))
        _call(lib.kda_b200_selective_scan_bwd, x.device, a, _ptr(ws), ws.numel())
    else:
        dA.zero_(), dD.zero_(), dbias.zero_()
    return dx, ddt, dA, dB, dC, dD, dz, dbias, dh0


@torch.library.custom_op("sophia_b200::selective_scan_fwd", mutates_args=(), device_types="cuda")
def _scan_fwd(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor],
              dt_bias: Optional[Tensor], h0: Optional[Tensor], cu_seqlens: Optional[Tensor], softplus: bool,
              want_final: bool, training: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _scan_fwd_impl(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, softplus, want_final, training)


@_scan_fwd.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, softplus, want_final, training):
    b, T, E = x.shape
    N = A.shape[1]
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    # kda_b200_scan_saved_bytes() in symbols: a size of its own per length would compile for every length
    nbytes = torch.sym_max(16, b * ((T + SAVED_EVERY - 1) // SAVED_EVERY) * E * N * 4) if training else 0
    return (x.new_empty((b, T, E)), x.new_empty((nseq, E, N) if want_final else (0,), dtype=torch.float32),
            x.new_empty((nbytes,), dtype=torch.uint8))


@torch.library.custom_op("sophia_b200::selective_scan_bwd", mutates_args=(), device_types="cuda")
def _scan_bwd(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor],
              dt_bias: Optional[Tensor], h0: Optional[Tensor], cu_seqlens: Optional[Tensor], saved: Tensor, dy: Tensor,
              dht: Optional[Tensor], softplus: bool, want_dh0: bool
              ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _scan_bwd_impl(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, saved, dy, dht, softplus, want_dh0)


@_scan_bwd.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, saved, dy, dht, softplus, want_dh0):
    b, T, E = x.shape
    N = A.shape[1]
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    act = lambda t: x.new_empty(t.shape if t is not None else (0,))  # noqa: E731
    f = lambda *s: x.new_empty(s, dtype=torch.float32)  # noqa: E731
    return (act(x), act(dt), f(E, N), act(B), act(C), f(E) if D is not None else f(0), act(z),
            f(E) if dt_bias is not None else f(0), f(nseq, E, N) if want_dh0 else f(0))


def _scan_grads(ctx, dy, dht, bwd):
    x, dt, A, B, C, D, z, dt_bias, h0, cu, saved = ctx.saved_tensors
    dht = None if dht is None or dht.numel() == 0 else dht
    dy = x.new_zeros(x.shape) if dy is None else dy
    dx, ddt, dA, dB, dC, dD, dz, dbias, dh0 = bwd(x, dt, A, B, C, D, z, dt_bias, h0, cu, saved, dy, dht, ctx.softplus,
                                                  h0 is not None)
    return (dx, ddt, dA.to(A.dtype), dB, dC, None if D is None else dD.to(D.dtype), None if z is None else dz,
            None if dt_bias is None else dbias.to(dt_bias.dtype), None if h0 is None else dh0)


def _scan_setup(ctx, inputs, output):
    *tensors, softplus, _, training = inputs
    if not training:
        raise RuntimeError("selective_scan_fwd was called with training=False but autograd needs its backward")
    ctx.save_for_backward(*tensors, output[2])
    ctx.softplus = softplus


_scan_fwd.register_autograd(lambda ctx, dy, dht, _s: (*_scan_grads(ctx, dy, dht, _scan_bwd), None, None, None, None),
                            setup_context=_scan_setup)


class _ScanEager(torch.autograd.Function):
    """The eager path: the custom ops' implementation without their dispatch."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, softplus, want_final, grad_mode):
        # (the caller's grad mode: it is off in here, and ctx.needs_input_grad follows requires_grad alone)
        training = grad_mode and any(ctx.needs_input_grad)
        y, ht, saved = _scan_fwd_impl(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, softplus, want_final, training)
        if training:
            ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, h0, cu_seqlens, saved)
            ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, ht

    @staticmethod
    def backward(ctx, dy, dht):
        grads = _first_order("selective_scan", ctx, _scan_grads(ctx, dy, dht, _scan_bwd_impl), dy, dht)
        return (*grads, None, None, None, None)


def _check_scan(what, x, dt, A, B, C, D, z, dt_bias):
    """Shapes of a scan (rows [..., E], B and C [..., G, N]); returns (E, N)."""
    lead, E = tuple(x.shape[:-1]), x.shape[-1]
    for name, t in (("dt", dt), ("z", z)):
        if t is not None and tuple(t.shape) != tuple(x.shape):
            raise ValueError(f"{what}: {name} must have x's shape {list(x.shape)}, got {list(t.shape)}")
    if A.dim() != 2 or A.shape[0] != E or A.shape[1] < 1:
        raise ValueError(f"{what}: A must have shape {[E, 'N']}, got {list(A.shape)}")
    N = A.shape[1]
    if N > MAX_STATE:
        raise NotImplementedError(f"{what}: at most {MAX_STATE} states per channel are supported, got {N}")
    for name, t in (("B", B), ("C", C)):
        if tuple(t.shape[:-2]) != lead or t.dim() != len(lead) + 2 or t.shape[-1] != N or t.shape[-2] != B.shape[-2]:
            raise ValueError(f"{what}: {name} must have shape {[*lead, 'groups', N]} or {[*lead, N]}, "
                             f"got {list(t.shape)}")
    if E < 1 or B.shape[-2] < 1 or E % B.shape[-2]:
        raise ValueError(f"{what}: {B.shape[-2]} groups do not divide {E} channels")
    _check_params(what, x.device, A=(A, (E, N)), D=(D, (E,)), dt_bias=(dt_bias, (E,)))
    return E, N


def selective_scan(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None,
                   z: Tensor | None = None, dt_bias: Tensor | None = None, *, dt_softplus: bool = True,
                   initial_state: Tensor | None = None, output_final_state: bool = False,
                   cu_seqlens: Tensor | None = None) -> tuple[Tensor, Tensor | None]:
    """Selective state space scan over tokens.  Per channel e and state n, with
    ``d = softplus(dt + dt_bias)`` (``dt + dt_bias`` without ``dt_softplus``)::

        h[t] = exp(d[t] A) h[t-1] + d[t] x[t] B[t]
        y[t] = (sum_n C[t] h[t] + D x[t]) * silu(z[t])

    x, dt, z: ``[B, T, E]``; A: ``[E, N]`` (the decay rates themselves, negative in
    use), N <= 64; B, C: ``[B, T, N]`` or ``[B, T, G, N]`` for G groups of channels; D,
    dt_bias: ``[E]``.  ``initial_state`` ``[sequences, E, N]`` float32; with
    ``cu_seqlens`` (``[sequences + 1]``, B = 1) sequences are packed along T and the
    state restarts at each.  Returns ``(y, final_state | None)``, y in x's type;
    gradients reach every floating-point input."""
    what = "selective_scan"
    io = _check_activations(what, x=x, dt=dt, B=B, C=C, z=z)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must have shape [B, T, E], got {list(x.shape)}")
    B = B.unsqueeze(2) if B.dim() == 3 else B
    C = C.unsqueeze(2) if C.dim() == 3 else C
    E, N = _check_scan(what, x, dt, A, B, C, D, z, dt_bias)
    nseq = _num_seqs(what, x, cu_seqlens)
    _check_state(what, initial_state, (nseq, E, N), x.device)
    like = x.dtype
    if x.dtype != io or dt.dtype != io or B.dtype != io or C.dtype != io or (z is not None and z.dtype != io):
        x, dt, B, C, z = (t if t is None else t.to(io) for t in (x, dt, B, C, z))
    args = (x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens, bool(dt_softplus), bool(output_final_state))
    if torch.compiler.is_compiling():
        y, ht, _ = _scan_fwd(*args, _needs_grad(x, dt, A, B, C, D, z, dt_bias, initial_state))
    else:
        y, ht = _ScanEager.apply(*args, torch.is_grad_enabled())
    return (y if y.dtype == like else y.to(like)), (ht if output_final_state else None)


def _scan_step_impl(x, dt, A, B, C, state, D, z, dt_bias, slots, softplus):
    rows, E = x.shape
    N, G = A.shape[1], B.shape[1]
    xr, dtr, Br, Cr, zr = _scan_inputs(x.dtype, x, dt, B, C, z)
    Af, Df, bf = _param(A), _param(D), _param(dt_bias)
    y = x.new_empty((rows, E))
    a = ScanArgs(1, 1, E, N, G, 1, _IO[x.dtype], int(softplus), _ptr(xr), _ptr(dtr), _ptr(zr), _ptr(Br), _ptr(Cr),
                 xr.stride(0), 0, dtr.stride(0), 0, zr.stride(0) if zr is not None else 0, 0,
                 Br.stride(0), 0, Br.stride(1), Cr.stride(0), 0, Cr.stride(1), _ptr(Af), _ptr(Df), _ptr(bf))
    a.y, a.state, a.slots, a.rows, a.pool = _ptr(y), _ptr(state), _ptr(slots), rows, state.shape[0]
    _call(_lib.load().kda_b200_selective_scan_step, x.device, a)
    return y


@torch.library.custom_op("sophia_b200::selective_scan_step", mutates_args=("state",), device_types="cuda")
def _scan_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Optional[Tensor],
               z: Optional[Tensor], dt_bias: Optional[Tensor], slots: Optional[Tensor], softplus: bool) -> Tensor:
    return _scan_step_impl(x, dt, A, B, C, state, D, z, dt_bias, slots, softplus)


@_scan_step.register_fake
def _(x, dt, A, B, C, state, D, z, dt_bias, slots, softplus):
    return x.new_empty(x.shape)


def selective_scan_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None = None,
                        z: Tensor | None = None, dt_bias: Tensor | None = None, *, dt_softplus: bool = True,
                        slots: Tensor | None = None) -> Tensor:
    """One token of ``selective_scan`` for each of B requests.  x, dt, z:
    ``[B, E]``; B, C: ``[B, N]`` or ``[B, G, N]``; state: a pool ``[S, E, N]`` float32,
    updated in place; slots: int32 ``[B]``, each row's entry of the pool (row r
    uses entry r without it).  A negative slot marks a padding row: its y is 0 and
    no state is touched.  Two rows must not share a slot.  Inference only.
    Returns y ``[B, E]`` in x's type."""
    what = "selective_scan_step"
    io = _check_activations(what, x=x, dt=dt, B=B, C=C, z=z)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must have shape [B, E], got {list(x.shape)}")
    B = B.unsqueeze(1) if B.dim() == 2 else B
    C = C.unsqueeze(1) if C.dim() == 2 else C
    E, N = _check_scan(what, x, dt, A, B, C, D, z, dt_bias)
    _check_pool(what, state, (E, N), x.device, x.shape[0], slots)
    if _needs_grad(x, dt, A, B, C, D, z, dt_bias, state):
        raise NotImplementedError(f"{what} has no backward; use selective_scan for training")
    _check_no_tangents(what, x, dt, A, B, C, state, D, z, dt_bias)
    like = x.dtype
    if x.dtype != io or dt.dtype != io or B.dtype != io or C.dtype != io or (z is not None and z.dtype != io):
        x, dt, B, C, z = (t if t is None else t.to(io) for t in (x, dt, B, C, z))
    if torch.compiler.is_compiling():
        y = _scan_step(x, dt, A, B, C, state, D, z, dt_bias, slots, bool(dt_softplus))
    else:
        y = _scan_step_impl(x, dt, A, B, C, state, D, z, dt_bias, slots, bool(dt_softplus))
        increment_version(state)
    return y if y.dtype == like else y.to(like)
