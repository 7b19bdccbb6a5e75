"""Global gradient norm and clipping, between the gradient all-reduce and the
optimizer: ``grad_norm`` and ``clip_grad_norm_`` take any number of gradient
tensors of any supported types in two kernel launches (two for every 1024 tensors),
without a host wait (a training step stays capturable).  The reference clips in its trainer with torch's
own utility.
"""

from __future__ import annotations

import math
from array import array
from typing import Iterable, Sequence

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import GradArgs
from .ssm import _IO, _call, _check_no_tangents

__all__ = ["grad_norm", "clip_grad_norm_"]


def _list(what: str, grads) -> tuple[list[Tensor], torch.device | None, bytes]:
    """The tensors, their one device and their types."""
    ts = [grads] if isinstance(grads, Tensor) else list(grads)
    for kind in set(map(type, ts)):
        if not issubclass(kind, Tensor):
            raise ValueError(f"{what} takes gradient tensors, got {kind.__name__}")
    try:
        types = bytes([_IO[t.dtype] for t in ts])
    except KeyError as e:
        raise NotImplementedError(f"{what}: gradients must be float32, bfloat16 or float16, got {e.args[0]}") from None
    _check_no_tangents(what, *ts)
    if len(set(map(Tensor.get_device, ts))) > 1:
        raise RuntimeError(f"{what}: gradients are on several devices")
    device = ts[0].device if ts else None
    if device is not None and device.type != "cuda":
        raise RuntimeError(f"{what} runs on the CUDA kernels only: gradients must be CUDA tensors")
    return ts, device, types


def _dense(t: Tensor) -> bool:
    """Whether the tensor's elements fill one run of memory, in whatever order."""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((st, s) for st, s in zip(t.stride(), t.shape) if s != 1):
        if stride != at:
            return False
        at *= size
    return True


def _launch(ts: list[Tensor], types: bytes, out: list[Tensor] | None, out_types: bytes | None, max_norm: float,
            eps: float, at: list[int] | None = None, sizes: list[int] | None = None) -> Tensor:
    """``at``, ``sizes``: the outputs' addresses and element counts, where the caller has them."""
    norm = ts[0].new_empty((), dtype=torch.float32)
    lib = _lib.load()
    ws = norm.new_empty(lib.kda_b200_grad_workspace_bytes(len(ts)), dtype=torch.uint8)
    numel = array("q", map(Tensor.numel, ts) if sizes is None else sizes)
    dst = None if out is None else array("Q", map(Tensor.data_ptr, out) if at is None else at)
    src = dst if dst is not None and out is ts else array("Q", map(Tensor.data_ptr, ts))
    addr = lambda a: None if a is None else a.buffer_info()[0]  # noqa: E731
    args = GradArgs(len(ts), addr(src), addr(dst), addr(numel), types, out_types, max_norm, eps, norm.data_ptr())
    _call(lib.kda_b200_grad_clip, norm.device, args, ws.data_ptr(), ws.numel())
    return norm


def grad_norm(grads: Tensor | Iterable[Tensor]) -> Tensor:
    """``sqrt(sum g^2)`` over all elements of all tensors (float32, bfloat16 or
    float16, any mix), as a 0-d float32 CUDA tensor; 0 on an empty list is on the
    current device.  No host wait.  The result does not depend on timing: sums have a
    fixed order (which the sizes, the addresses modulo 16 bytes and the number of SMs decide).  Squares do not
    overflow or vanish: the norm is right wherever float32 can hold it.  Not differentiable: the norm has no
    graph."""
    with torch.no_grad():
        ts, _, types = _list("grad_norm", grads)
        if not ts:
            return torch.zeros((), device="cuda", dtype=torch.float32)
        return _launch([t if _dense(t) else t.contiguous() for t in ts], types, None, None, 0.0, 0.0)


def clip_grad_norm_(grads: Tensor | Iterable[Tensor], max_norm: float, *, eps: float = 1e-6,
                    out: Sequence[Tensor] | Tensor | None = None) -> Tensor:
    """Scales the gradients by ``min(1, max_norm / (norm + eps))``, ``norm``
    their global 2-norm, and returns the norm (0-d float32 CUDA tensor, before
    clipping).  It takes the gradients themselves, not the parameters that hold them.  In place
    by default; with ``out``, tensors of the gradients' shapes and of any
    supported type (an optimizer's float32 gradients), every element of which is
    written, the gradients stay as they are.  ``out[i] is grads[i]`` is allowed; otherwise no two
    tensors may overlap.  A NaN norm makes the scaled gradients NaN, an infinite one 0 (and
    NaN where a gradient is infinite), as the formula says; there is no host wait to look."""
    what = "clip_grad_norm_"
    max_norm, eps = float(max_norm), float(eps)
    if math.isnan(max_norm) or max_norm < 0 or not eps >= 0:
        raise ValueError(f"{what}: max_norm and eps must be >= 0, got {max_norm} and {eps}")
    with torch.no_grad():
        ts, device, types = _list(what, grads)
        outs, out_device, out_types = (ts, device, types) if out is None else _list(what, out)
        if len(outs) != len(ts):
            raise ValueError(f"{what}: {len(ts)} gradients but {len(outs)} outputs")
        if not ts:
            return torch.zeros((), device="cuda", dtype=torch.float32)
        if outs is not ts:
            for g, o in zip(ts, outs):
                if g.shape != o.shape:
                    raise ValueError(f"{what}: an output of shape {list(o.shape)} for a gradient of {list(g.shape)}")
            if out_device != device:
                raise RuntimeError(f"{what}: gradients and outputs are on different devices")
        at, sizes = list(map(Tensor.data_ptr, outs)), list(map(Tensor.numel, outs))
        if len(set(at)) != len(at) and len({a for a, n in zip(at, sizes) if n}) != len(sizes) - sizes.count(0):
            raise ValueError(f"{what}: one tensor is named twice")
        if any(o.requires_grad for o in outs):
            raise ValueError(f"{what} scales gradients; a tensor that requires grad (a parameter?) is not one")
        if all(map(Tensor.is_contiguous, ts)) and (outs is ts or all(map(Tensor.is_contiguous, outs))):
            norm = _launch(ts, types, outs, out_types, max_norm, eps, at, sizes)
            increment_version(outs)  # written in place: a graph that saved one has to notice
            return norm
        src, dst, back = list(ts), list(outs), []
        for i, (g, o) in enumerate(zip(ts, outs)):
            if g.is_contiguous() and o.is_contiguous():
                continue
            if g.stride() == o.stride() and _dense(g):  # the same order of elements in both
                continue
            if any(st == 0 and n > 1 for st, n in zip(o.stride(), o.shape)):  # an expanded tensor
                raise ValueError(f"{what}: an output of shape {list(o.shape)} holds several elements in one place")
            src[i] = g.contiguous()
            if not o.is_contiguous():
                dst[i] = torch.empty(o.shape, device=o.device, dtype=o.dtype)
                back.append(i)
        norm = _launch(src, types, dst, out_types, max_norm, eps)
        increment_version(outs)
        for i in back:
            outs[i].copy_(dst[i])
        return norm
