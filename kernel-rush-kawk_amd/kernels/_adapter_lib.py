"""ctypes binding of libkrk_adapter.so (C ABI declared in include/krk_adapter.h)."""

from __future__ import annotations

import ctypes
from pathlib import Path

from ._binding import I64, INT, P, SIZE, Library, packer

LIB_PATH = Path(__file__).resolve().parent.parent / "libkrk_adapter.so"
SLICES = 4


class Shape(ctypes.Structure):
    """``krk_adapter_shape``."""

    _fields_ = [(n, INT) for n in ("rows", "N", "K", "rank", "silu", "slices")] + [("widths", INT * SLICES)]


class Args(ctypes.Structure):
    """``krk_adapter_args``."""

    _fields_ = [("x", P), ("ldx", I64), ("a", P), ("a_adapter", I64), ("a_row", I64), ("b", P), ("b_adapter", I64), ("b_row", I64),
                ("scale", P), ("index", P), ("y", P), ("ldy", I64), ("out", P), ("ldo", I64), ("adapters", INT)]


_ptr = ctypes.POINTER

#: Every function the header declares, with (restype, argtypes).
SIGNATURES = {
    "krk_adapter_bf16": (INT, [P, P, P, SIZE, P]),
    "krk_adapter_workspace_bytes": (SIZE, [_ptr(Shape)]),
    "krk_adapter_check": (INT, [_ptr(Shape)]),
    "krk_adapter_abi_version": (INT, []),
    "krk_adapter_struct_size": (SIZE, [INT]),
    "krk_adapter_last_error": (ctypes.c_char_p, []),
}

#: The ABI this binding was written against (KRK_ADAPTER_ABI_VERSION) and its structs, in the header's order.
ABI_VERSION = 1
STRUCTS = (Shape, Args)
LIB = Library(LIB_PATH, "krk_adapter_", ABI_VERSION, STRUCTS, SIGNATURES)
PACK = packer(Args)
