"""ctypes binding of libkrk_attn.so (C ABI declared in include/krk_attn.h).

Like the GEMM library's binding it loads once, checks the ABI version and the
struct layouts, and has no fallback: a missing library is an ImportError.
"""

from __future__ import annotations

import ctypes
import struct
import threading
from pathlib import Path

import torch  # noqa: F401  (must be loaded before the HIP library)

from ._lib import KrkError

LIB_PATH = Path(__file__).resolve().parent.parent / "libkrk_attn.so"

KRK_ATTN_ERR_HIP = -5

_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f = ctypes.c_float
_size = ctypes.c_size_t


class Cache(ctypes.Structure):
    """``krk_cache``: a [sequences, slots, heads, head_dim] tensor."""

    _fields_ = [("p", _p), ("seq", _i64), ("slot", _i64), ("head", _i64)]


class AttnShape(ctypes.Structure):
    """``krk_attn_shape``."""

    _fields_ = [(n, _int) for n in ("B", "R", "heads", "kv_heads", "head_dim", "capacity", "window", "sinks", "prefix",
                                    "scored")]


class AttnArgs(ctypes.Structure):
    """``krk_attn_args``."""

    _fields_ = [("q", _p), ("q_row", _i64), ("k", Cache), ("v", Cache), ("kp", Cache), ("vp", Cache), ("prefix", _int),
                ("scale", _f), ("lens", _p), ("tree", _p), ("out", _p), ("out_row", _i64), ("lse", _p),
                ("scores", _p), ("sc_seq", _i64), ("sc_head", _i64), ("scores_out", _p), ("so_seq", _i64),
                ("so_head", _i64)]


class RopeArgs(ctypes.Structure):
    """``krk_rope_args``."""

    _fields_ = [("qkv", _p), ("qkv_row", _i64), ("q_norm", _p), ("k_norm", _p), ("eps", _f), ("table", _p),
                ("table_rows", _int), ("positions", _p), ("lens", _p), ("q_out", _p), ("q_row", _i64), ("k", Cache),
                ("v", Cache), ("B", _int), ("R", _int), ("heads", _int), ("kv_heads", _int), ("head_dim", _int),
                ("capacity", _int)]


class EvictArgs(ctypes.Structure):
    """``krk_evict_args``."""

    _fields_ = [("k", Cache), ("v", Cache), ("k_out", Cache), ("v_out", Cache), ("scores", _p), ("sc_seq", _i64),
                ("sc_head", _i64), ("scores_out", _p), ("so_seq", _i64), ("so_head", _i64), ("lens", _p),
                ("lens_out", _p), ("keep", _p), ("B", _int), ("kv_heads", _int), ("head_dim", _int),
                ("capacity", _int), ("budget", _int), ("sinks", _int), ("recent", _int)]


class AttnPlan(ctypes.Structure):
    """``krk_attn_plan_t``."""

    _fields_ = [(n, _int) for n in ("rows", "splits", "prefix_rows", "prefix_splits")]

    def as_dict(self) -> dict:
        return {name: getattr(self, name) for name, _ in self._fields_}


_ptr = ctypes.POINTER

#: Every function the header declares, with (restype, argtypes).  The calls of
#: a step take their structs as packed bytes (:data:`PACK`) or by reference.
SIGNATURES = {
    "krk_attn_bf16": (_int, [_p, _p, _p, _size, _p]),
    "krk_attn_workspace_bytes": (_size, [_ptr(AttnShape)]),
    "krk_attn_check": (_int, [_ptr(AttnShape)]),
    "krk_attn_plan": (_int, [_ptr(AttnShape), _ptr(AttnPlan)]),
    "krk_qk_norm_rope_bf16": (_int, [_p, _p]),
    "krk_cache_evict_bf16": (_int, [_p, _p]),
    "krk_attn_abi_version": (_int, []),
    "krk_attn_struct_size": (_size, [_int]),
    "krk_attn_last_error": (ctypes.c_char_p, []),
}

#: The ABI this binding was written against (KRK_ATTN_ABI_VERSION) and its structs, in the header's order.
ABI_VERSION = 1
STRUCTS = (AttnShape, AttnArgs, RopeArgs, EvictArgs, AttnPlan)

_CODES = {_p: "P", _i64: "q", _int: "i", _f: "f"}


def _packer(cls) -> struct.Struct:
    """The struct's layout for ``pack``: its fields in order, nested caches
    flattened.  One call fills it, where setting a ctypes field costs as much
    as reading a tensor's pointer."""
    fmt = ""
    for _, t in cls._fields_:
        fmt += "".join(_CODES[u] for _, u in t._fields_) if t is Cache else _CODES[t]
    s = struct.Struct("@" + fmt + "0P")
    if s.size != ctypes.sizeof(cls):
        raise ImportError(f"{cls.__name__}: packed {s.size} bytes, laid out {ctypes.sizeof(cls)}")
    return s


PACK = {cls: _packer(cls).pack for cls in (AttnArgs, RopeArgs, EvictArgs)}

_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load (once) and return the library.  Raises ImportError if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise ImportError(
                    f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                    "or `python kernel-rush-kawk_amd/build_lib.py` (there is no fallback)")
            lib = ctypes.CDLL(str(LIB_PATH))
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            abi = lib.krk_attn_abi_version()
            sizes = [lib.krk_attn_struct_size(i) for i in range(len(STRUCTS))]
            mine = [ctypes.sizeof(s) for s in STRUCTS]
            if abi != ABI_VERSION or sizes != mine:
                raise ImportError(f"{LIB_PATH}: ABI version {abi} with structs of {sizes} bytes; this binding expects "
                                  f"version {ABI_VERSION} and {mine} (rebuild the library or update the binding)")
            _lib = lib
    return _lib


def last_error() -> str:
    return load().krk_attn_last_error().decode(errors="replace")


def check(rc: int) -> None:
    """Raise for a non-zero return code: ValueError for argument errors, KrkError for runtime errors."""
    if rc == 0:
        return
    msg = last_error()
    if rc == KRK_ATTN_ERR_HIP:
        raise KrkError(rc, msg)
    raise ValueError(f"krk error {rc}: {msg}")
