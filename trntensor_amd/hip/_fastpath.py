"""Loader of the host launch table (``csrc/tt_fastpath.cpp``) and of the
serving operators' host path (``csrc/tt_serving_host.cpp``), one extension.

The table keeps, per (subscripts, operand sizes, strides, dtype, device), the
tt_gemm_packed parameter block of a two-operand contraction that runs as one
GEMM launch, so a repeat einsum call costs one lookup, one allocation and one
library call in C++. It calls the entry point of the already loaded
libtrntensor_hip.so by address. When the table is not built (or cannot be
loaded), einsum keeps its launchers in a Python dict instead: the same
launches through ctypes, a few microseconds more per call.
"""

from __future__ import annotations

import ctypes
import importlib.util
import os

from . import _lib

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib", "fastpath", "tt_fastpath.so")

_module = None
_table = None
_rows = None
_error: str | None = None
_tried = False


def _addr(fn) -> int:
    return ctypes.cast(fn, ctypes.c_void_p).value


def module():
    """The extension (loaded on first use), or None with the reason in error()."""
    global _module, _error, _tried
    if _tried:
        return _module
    _tried = True
    if _lib.load() is None:
        _error = _lib.load_error()
        return None
    if not os.path.exists(PATH):
        _error = f"{PATH} is not built"
        return None
    try:
        spec = importlib.util.spec_from_file_location("tt_fastpath", PATH)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        for name in ("LaunchTable", "Q4Host", "CacheHost", "RowsHost", "Fp8Host"):
            getattr(mod, name)
        _module = mod
    except (ImportError, OSError, AttributeError) as exc:
        _error = f"cannot load {PATH}: {exc}"
    return _module


def table(max_entries: int):
    """The process's LaunchTable (created on first use), or None with the reason in error()."""
    global _table
    if _table is None:
        mod = module()
        if mod is not None:
            lib = _lib.load()
            _table = mod.LaunchTable(_addr(lib.tt_gemm_packed), _addr(lib.tt_last_error), _addr(lib.tt_status_string),
                                     max_entries)
    return _table


def serving_entries() -> list[int]:
    """The library's entry points that the serving operators' host path calls, by address."""
    lib = _lib.load()
    return [_addr(fn) for fn in (lib.tt_q4_matmul, lib.tt_kv_append, lib.tt_kv_attention_workspace_bytes,
                                 lib.tt_kv_attention, lib.tt_last_error, lib.tt_status_string, lib.tt_fp8_quantize,
                                 lib.tt_rms_norm, lib.tt_fp8_matmul, lib.tt_fp8_gated_workspace_bytes,
                                 lib.tt_fp8_gated_matmul)]


def rows_host():
    """The process's RowsHost (created on first use), or None with the reason in error()."""
    global _rows
    if _rows is None:
        mod = module()
        if mod is not None:
            _rows = mod.RowsHost(serving_entries())
    return _rows


def error() -> str | None:
    return _error
