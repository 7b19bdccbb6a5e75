"""ctypes binding of ``libkda_b200.so`` (declarations: ``include/kda_b200.h``).

The library is loaded from the package directory.  There is no fallback: if
the library is missing or fails to load, every op raises.
"""

from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_int64, c_size_t, c_void_p, c_char_p
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libkda_b200.so"

KDA_OK = 0
KDA_ERR_INVALID = 1
KDA_ERR_UNSUPPORTED = 2
KDA_ERR_CUDA = 3



class ScanArgs(ctypes.Structure):
    """``kda_b200_scan_args``."""

    _fields_ = ([(n, c_int64) for n in ("B", "T")]
                + [(n, ctypes.c_int32) for n in ("E", "N", "G", "nseq", "dtype", "softplus")]
                + [(n, c_void_p) for n in ("x", "dt", "z", "B_", "C_")]
                + [(n, c_int64) for n in ("x_sb", "x_st", "dt_sb", "dt_st", "z_sb", "z_st", "B_sb", "B_st", "B_sg",
                                          "C_sb", "C_st", "C_sg")]
                + [(n, c_void_p) for n in ("A", "D", "dt_bias", "h0", "cu_seqlens", "y", "ht", "saved")]
                + [("saved_bytes", c_size_t), ("dy", c_void_p), ("dy_sb", c_int64), ("dy_st", c_int64)]
                + [(n, c_void_p) for n in ("dht", "dx", "ddt", "dz", "dB", "dC", "dA", "dD", "ddt_bias", "dh0", "state",
                                           "slots")]
                + [("rows", ctypes.c_int32), ("pool", ctypes.c_int32)])


class RecArgs(ctypes.Structure):
    """``kda_b200_recurrence_args``."""

    _fields_ = ([(n, c_int64) for n in ("B", "T")]
                + [(n, ctypes.c_int32) for n in ("E", "nseq", "dtype", "rows")]
                + [(n, c_void_p) for n in ("x", "decay", "gate", "z")]
                + [(n, c_int64) for n in ("x_sb", "x_st", "decay_sb", "decay_st", "gate_sb", "gate_st", "z_sb", "z_st")]
                + [(n, c_void_p) for n in ("A", "decay_bias", "gate_bias", "h0", "cu_seqlens", "y", "ht", "saved")]
                + [("saved_bytes", c_size_t), ("dy", c_void_p), ("dy_sb", c_int64), ("dy_st", c_int64)]
                + [(n, c_void_p) for n in ("dht", "dx", "ddecay", "dgate", "dz", "dA", "ddecay_bias", "dgate_bias", "dh0",
                                           "state", "slots")]
                + [("pool", ctypes.c_int32)])


class NormArgs(ctypes.Structure):
    """``kda_b200_norm_args``."""

    _fields_ = ([(n, c_int64) for n in ("B", "T")]
                + [(n, ctypes.c_int32) for n in ("D", "dtype", "stream_dtype")] + [("offset", ctypes.c_uint32)]
                + [(n, c_void_p) for n in ("x", "o", "gate")]
                + [(n, c_int64) for n in ("x_sb", "x_st", "o_sb", "o_st", "gate_sb", "gate_st")]
                + [(n, c_void_p) for n in ("w", "wb", "scale", "seed_ptr")]
                + [("seed", ctypes.c_uint64), ("dropout_p", ctypes.c_double), ("eps", c_float)]
                + [(n, c_void_p) for n in ("v", "n", "rstd", "dv", "dn")]
                + [(n, c_int64) for n in ("dv_sb", "dv_st", "dn_sb", "dn_st")]
                + [(n, c_void_p) for n in ("dx", "d_o", "dgate", "dw", "dwb", "dscale")])


class GradArgs(ctypes.Structure):
    """``kda_b200_grad_args`` (host arrays; the types as bytes objects)."""

    _fields_ = [("count", c_int64), ("in_", c_void_p), ("out", c_void_p), ("numel", c_void_p), ("in_type", c_char_p),
                ("out_type", c_char_p), ("max_norm", c_float), ("eps", c_float), ("norm", c_void_p)]


# every symbol the header declares, with its ctypes signature
SIGNATURES = {
    "kda_b200_version": ([], c_char_p),
    "kda_b200_last_error": ([], c_char_p),
    "kda_b200_saved_bytes": ([c_int64, c_int, c_int, c_int], c_size_t),
    "kda_b200_fwd_workspace_bytes": ([c_int64, c_int, c_int, c_int, c_int], c_size_t),
    "kda_b200_bwd_workspace_bytes": ([c_int64, c_int, c_int, c_int], c_size_t),
    "kda_b200_fwd": ([c_void_p] * 12 + [c_int] * 5 + [c_float, c_float]
                     + [c_void_p, c_void_p, c_void_p, c_size_t, c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_bwd": ([c_void_p] * 12 + [c_int] * 5 + [c_float, c_float]
                     + [c_void_p, c_size_t] + [c_void_p] * 13 + [c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_f32_saved_bytes": ([c_int64, c_int, c_int], c_size_t),
    "kda_b200_f32_fwd_workspace_bytes": ([c_int64, c_int, c_int, c_int], c_size_t),
    "kda_b200_f32_bwd_workspace_bytes": ([c_int64, c_int, c_int], c_size_t),
    "kda_b200_fwd_f32": ([c_void_p] * 12 + [c_int] * 5 + [c_float, c_float]
                         + [c_void_p, c_void_p, c_void_p, c_size_t, c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_bwd_f32": ([c_void_p] * 12 + [c_int] * 5 + [c_float, c_float]
                         + [c_void_p, c_size_t] + [c_void_p] * 13 + [c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_recurrent": ([c_void_p] * 9 + [c_int] * 6 + [c_float, c_float] + [c_void_p] * 3, c_int),
    "kda_b200_decode": ([c_void_p] * 13 + [c_int] * 6 + [c_float, c_float] + [c_void_p] * 3, c_int),
    "kda_b200_doc_cu_seqlens": ([c_void_p, c_int64, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p], c_int),
    "kda_b200_chunk_table": ([c_void_p, c_int, c_int64, c_void_p, c_void_p, c_void_p, c_void_p], c_int),
    "kda_b200_device_error": ([c_int], c_int),
    "kda_b200_debug_set_input_wait_polls": ([ctypes.c_uint], c_int),
    "kda_b200_debug_set_state_wait": ([ctypes.c_uint, c_int], c_int),
    "kda_b200_fwd_noalloc": ([c_void_p] * 12 + [c_int] * 5 + [c_float, c_float] + [c_void_p, c_void_p, c_void_p],
                             c_int),
    "kda_b200_timing_enable": ([c_int], c_int),
    "kda_b200_timing_reset": ([], c_int),
    "kda_b200_timing_read": ([c_int, c_void_p, c_void_p, c_void_p], c_int),
    "kda_b200_gated_norm_workspace_bytes": ([c_int64, c_int], c_size_t),
    "kda_b200_gated_norm_fwd": ([c_void_p, c_void_p, c_void_p, c_int64, c_int, c_float, c_int, c_void_p, c_void_p],
                                c_int),
    "kda_b200_gated_norm_bwd": ([c_void_p] * 4 + [c_int64, c_int, c_float, c_int] + [c_void_p] * 4
                                + [c_size_t, c_void_p], c_int),
    "kda_b200_short_conv_workspace_bytes": ([c_int64, c_int64] + [c_int] * 4, c_size_t),
    "kda_b200_short_conv_fwd": ([c_void_p, c_int64, c_int64] + [c_void_p] * 4 + [c_int64, c_int64] + [c_int] * 5
                                + [c_void_p, c_void_p, c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_short_conv_bwd": ([c_void_p, c_int64, c_int64] + [c_void_p] * 4 + [c_int64, c_int64] + [c_int] * 5
                                + [c_void_p, c_int64, c_int64] + [c_void_p] * 5 + [c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_short_conv_step": ([c_void_p, c_int64] + [c_void_p] * 4 + [c_int] * 6 + [c_void_p, c_void_p], c_int),
    "kda_b200_put_states": ([c_void_p, c_void_p, c_int, c_int64, c_int, c_void_p, c_void_p], c_int),
    "kda_b200_scan_saved_bytes": ([c_int64, c_int64] + [c_int] * 3, c_size_t),
    "kda_b200_scan_workspace_bytes": ([c_int64, c_int64] + [c_int] * 5, c_size_t),
    "kda_b200_selective_scan_fwd": ([ctypes.POINTER(ScanArgs), c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_selective_scan_bwd": ([ctypes.POINTER(ScanArgs), c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_selective_scan_step": ([ctypes.POINTER(ScanArgs), c_void_p], c_int),
    "kda_b200_recurrence_saved_bytes": ([c_int64, c_int64] + [c_int] * 2, c_size_t),
    "kda_b200_recurrence_workspace_bytes": ([c_int64, c_int64] + [c_int] * 4, c_size_t),
    "kda_b200_recurrence_fwd": ([ctypes.POINTER(RecArgs), c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_recurrence_bwd": ([ctypes.POINTER(RecArgs), c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_recurrence_step": ([ctypes.POINTER(RecArgs), c_void_p], c_int),
    "kda_b200_norm_workspace_bytes": ([c_int64, c_int64] + [c_int] * 2, c_size_t),
    "kda_b200_norm_fwd": ([ctypes.POINTER(NormArgs), c_void_p], c_int),
    "kda_b200_norm_bwd": ([ctypes.POINTER(NormArgs), c_void_p, c_size_t, c_void_p], c_int),
    "kda_b200_grad_workspace_bytes": ([c_int64], c_size_t),
    "kda_b200_grad_clip": ([ctypes.POINTER(GradArgs), c_void_p, c_size_t, c_void_p], c_int),
}

_lib = None


class KdaError(RuntimeError):
    """A non-OK status from the CUDA library."""


def load() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"KDA CUDA library not built ({LIB_PATH}); run `python -m sophia_b200.build`")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (args, res) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    _lib = lib
    return lib


def check(rc: int) -> None:
    if rc == KDA_OK:
        return
    msg = load().kda_b200_last_error().decode()
    if rc in (KDA_ERR_INVALID,):
        raise ValueError(msg)
    if rc == KDA_ERR_UNSUPPORTED:
        raise NotImplementedError(msg)
    raise KdaError(msg)


def timing_enable(on: bool) -> None:
    load().kda_b200_timing_enable(int(on))


def timing_reset() -> None:
    load().kda_b200_timing_reset()


def timing_read() -> dict[str, tuple[int, float]]:
    """{kernel name: (launches, total ms)} since the last reset."""
    n = 32
    names = (ctypes.c_char_p * n)()
    launches = (ctypes.c_int * n)()
    ms = (ctypes.c_float * n)()
    rc = load().kda_b200_timing_read(n, ctypes.cast(names, c_void_p), ctypes.cast(launches, c_void_p),
                                     ctypes.cast(ms, c_void_p))
    if rc <= 0:
        raise KdaError(load().kda_b200_last_error().decode())
    return {names[i].decode(): (launches[i], ms[i]) for i in range(rc)}


def device_error(reset: bool = True) -> int:
    """Nonzero when a tensor-core kernel hit a bounded-wait timeout (synchronises)."""
    return int(load().kda_b200_device_error(int(reset)))
