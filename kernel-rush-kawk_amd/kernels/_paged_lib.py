"""ctypes binding of libkrk_paged.so (C ABI declared in include/krk_paged.h)."""

from __future__ import annotations

import ctypes
from pathlib import Path

from ._binding import F32, I64, INT, P, SIZE, Library, packer

LIB_PATH = Path(__file__).resolve().parent.parent / "libkrk_paged.so"


class PageStepArgs(ctypes.Structure):
    """``krk_page_step_args``."""

    _fields_ = [("lens", P), ("keep", P), ("fresh", P), ("labels", P), ("table", P), ("table_row", I64), ("free_pages", P),
                ("free_count", P), ("starts", P), ("keys", P), ("slots", P), ("positions", P), ("owner", P), ("B", INT),
                ("rows", INT), ("pages", INT), ("page_size", INT), ("width", INT)]


class Pages(ctypes.Structure):
    """``krk_pages``: a [pages, page_size, heads, head_dim] tensor."""

    _fields_ = [("p", P), ("page", I64), ("slot", I64), ("head", I64)]


class RopeArgs(ctypes.Structure):
    """``krk_paged_rope_args``."""

    _fields_ = [("qkv", P), ("qkv_row", I64), ("q_norm", P), ("k_norm", P), ("eps", F32), ("table", P), ("table_rows", INT),
                ("slots", P), ("positions", P), ("q_out", P), ("q_row", I64), ("k", Pages), ("v", Pages), ("rows", INT),
                ("heads", INT), ("kv_heads", INT), ("head_dim", INT), ("pages", INT), ("page_size", INT)]


class Shape(ctypes.Structure):
    """``krk_paged_shape``."""

    _fields_ = [(n, INT) for n in ("B", "rows", "heads", "kv_heads", "head_dim", "page_size", "width", "window", "sinks")]


class AttnArgs(ctypes.Structure):
    """``krk_paged_attn_args``."""

    _fields_ = [("q", P), ("q_row", I64), ("k", Pages), ("v", Pages), ("pages", INT), ("scale", F32), ("table", P),
                ("table_row", I64), ("starts", P), ("keys", P), ("out", P), ("out_row", I64), ("lse", P)]


_ptr = ctypes.POINTER

#: Every function the header declares, with (restype, argtypes).  The calls of a step
#: take their structs as packed bytes or by reference.
SIGNATURES = {
    "krk_page_step": (INT, [P, P]),
    "krk_paged_rope_bf16": (INT, [P, P]),
    "krk_paged_attn_bf16": (INT, [P, P, P, SIZE, P]),
    "krk_paged_workspace_bytes": (SIZE, [_ptr(Shape)]),
    "krk_paged_check": (INT, [_ptr(Shape)]),
    "krk_paged_abi_version": (INT, []),
    "krk_paged_struct_size": (SIZE, [INT]),
    "krk_paged_last_error": (ctypes.c_char_p, []),
}

#: The ABI this binding was written against (KRK_PAGED_ABI_VERSION) and its structs, in the header's order.
ABI_VERSION = 1
STRUCTS = (PageStepArgs, RopeArgs, Shape, AttnArgs)
LIB = Library(LIB_PATH, "krk_paged_", ABI_VERSION, STRUCTS, SIGNATURES)
PACK_STEP, PACK_ROPE, PACK_ATTN = (packer(t) for t in (PageStepArgs, RopeArgs, AttnArgs))
