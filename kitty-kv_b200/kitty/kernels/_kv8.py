"""ctypes binding of ``libkitty_kv8.so`` (the C ABI in ``include/kitty_kv8.h``).

Loaded on first use, like ``libkitty_b200.so``: a missing library or one of another
ABI version raises ``RuntimeError``, there is no fallback.  The operators themselves go
through :func:`ops`, which checks the tensors in C++ and runs the entry points on the
current torch stream of the tensors' device, whichever device is the current one; the
structs here are for callers that bind the C ABI themselves.
"""

from __future__ import annotations

import ctypes
import os
import threading
from pathlib import Path
from typing import Optional

import torch

from ._lib import c_f32, c_i32, c_i64, c_ptr, c_size

ABI_VERSION = 1
LIB_NAME = "libkitty_kv8.so"
_LIB_PATH = Path(os.environ.get("KITTY_KV8_LIB", Path(__file__).resolve().parent.parent / LIB_NAME))

ERROR_NAMES = {1: "invalid argument", 2: "unsupported", 3: "CUDA error", 4: "workspace"}

# Sticky device error bits (kitty_kv8_error_flags).
ERRORS = {1 << 1: "page number outside the pool or the block table", 1 << 2: "row offsets out of order or range",
          1 << 3: "slot out of range or repeated in one write", 1 << 4: "length negative or past the block table, "
          "or tokens read past it", 1 << 5: "position past the rotary table"}


class Cache(ctypes.Structure):
    _fields_ = [("key_codes", c_ptr), ("value_codes", c_ptr), ("key_scale", c_ptr), ("value_scale", c_ptr),
                ("tail_k", c_ptr), ("tail_v", c_ptr), ("block_table", c_ptr), ("lengths", c_ptr),
                ("bt_s_slot", c_i64), ("pages", c_i64), ("slots", c_i32), ("max_pages", c_i32),
                ("num_heads", c_i32), ("head_dim", c_i32), ("page_size", c_i32), ("code", c_i32), ("dtype", c_i32)]


class WriteArgs(ctypes.Structure):
    _fields_ = [("cache", Cache), ("key", c_ptr), ("value", c_ptr), ("k_s_row", c_i64), ("k_s_head", c_i64),
                ("v_s_row", c_i64), ("v_s_head", c_i64), ("row_offsets", c_ptr), ("seq_map", c_ptr), ("n", c_i32),
                ("rows", c_i32)]


class ReadArgs(ctypes.Structure):
    _fields_ = [("cache", Cache), ("key", c_ptr), ("value", c_ptr), ("row_offsets", c_ptr), ("first", c_ptr),
                ("seq_map", c_ptr), ("n", c_i32), ("rows", c_i32)]


class AttentionArgs(ctypes.Structure):
    _fields_ = [("cache", Cache), ("q", c_ptr), ("q_s_seq", c_i64), ("q_s_head", c_i64), ("out", c_ptr),
                ("out_s_seq", c_i64), ("out_s_head", c_i64), ("seq_map", c_ptr), ("batch", c_i32),
                ("num_q_heads", c_i32), ("sm_scale", c_f32), ("workspace", c_ptr), ("workspace_bytes", c_size)]


class QkNormRopeArgs(ctypes.Structure):
    _fields_ = [("q", c_ptr), ("k", c_ptr), ("q_out", c_ptr), ("k_out", c_ptr),
                ("q_s_row", c_i64), ("q_s_head", c_i64), ("k_s_row", c_i64), ("k_s_head", c_i64),
                ("qo_s_row", c_i64), ("qo_s_head", c_i64), ("ko_s_row", c_i64), ("ko_s_head", c_i64),
                ("q_weight", c_ptr), ("k_weight", c_ptr), ("positions", c_ptr), ("table", c_ptr),
                ("table_rows", c_i64), ("rows", c_i32), ("num_q_heads", c_i32), ("num_k_heads", c_i32),
                ("head_dim", c_i32), ("rot", c_i32), ("interleaved", c_i32), ("positions64", c_i32),
                ("weight_f32", c_i32), ("dtype", c_i32), ("eps", c_f32)]


STRUCTS = {0: Cache, 1: WriteArgs, 2: ReadArgs, 3: AttentionArgs, 4: QkNormRopeArgs}
SIGNATURES = {
    "kitty_kv8_abi_version": (ctypes.c_int, []),
    "kitty_kv8_last_error": (ctypes.c_char_p, []),
    "kitty_kv8_args_size": (c_size, [ctypes.c_int]),
    "kitty_kv8_error_flags": (ctypes.c_int, [ctypes.POINTER(ctypes.c_uint32), ctypes.c_int]),
    "kitty_kv8_write": (ctypes.c_int, [ctypes.POINTER(WriteArgs), c_ptr]),
    "kitty_kv8_read": (ctypes.c_int, [ctypes.POINTER(ReadArgs), c_ptr]),
    "kitty_kv8_attention_workspace_size": (ctypes.c_int, [ctypes.POINTER(AttentionArgs), ctypes.POINTER(c_size)]),
    "kitty_kv8_attention": (ctypes.c_int, [ctypes.POINTER(AttentionArgs), c_ptr]),
    "kitty_qk_norm_rope": (ctypes.c_int, [ctypes.POINTER(QkNormRopeArgs), c_ptr]),
}

_lib: Optional[ctypes.CDLL] = None
_lock = threading.Lock()


def library_path() -> Path:
    return _LIB_PATH


def load() -> ctypes.CDLL:
    """Load the library (once), bind every signature and check the ABI."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not _LIB_PATH.exists():
            raise RuntimeError(f"Kitty CUDA library not found at {_LIB_PATH}. Build it with "
                               "`python kitty-kv_b200/build.py` (there is no CPU fallback).")
        lib = ctypes.CDLL(str(_LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if lib.kitty_kv8_abi_version() != ABI_VERSION:
            raise RuntimeError(f"{_LIB_PATH} has ABI version {lib.kitty_kv8_abi_version()}, expected {ABI_VERSION}")
        for kind, st in STRUCTS.items():
            if lib.kitty_kv8_args_size(kind) != ctypes.sizeof(st):
                raise RuntimeError(f"struct layout mismatch for {st.__name__}: library "
                                   f"{lib.kitty_kv8_args_size(kind)} bytes, binding {ctypes.sizeof(st)}")
        _lib = lib
        return lib


def check(rc: int, what: str) -> None:
    if rc:
        msg = load().kitty_kv8_last_error().decode(errors="replace")
        raise RuntimeError(f"{what} failed ({ERROR_NAMES.get(rc, rc)}): {msg}")


_ops = None


def ops():
    """The module that calls the entry points with torch tensors (``csrc/kv8/kv8_torch.cpp``)."""
    global _ops
    if _ops is None:
        load()
        try:
            from . import _kv8_torch
        except ImportError as e:
            raise RuntimeError("Kitty's torch module for the 8-bit cache cannot be loaded. Build it with "
                               f"`python kitty-kv_b200/build.py` (there is no CPU fallback): {e}") from e
        _ops = _kv8_torch
    return _ops


def error_flags(device: torch.device, clear: bool = True) -> int:
    v = ctypes.c_uint32(0)
    with torch.cuda.device(device):
        check(load().kitty_kv8_error_flags(ctypes.byref(v), int(clear)), "kitty_kv8_error_flags")
    return v.value
