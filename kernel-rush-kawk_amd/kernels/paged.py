"""The paged key/value cache on MI355X: a step over many requests of different
lengths, whose keys lie in pages of one pool.

* :class:`PageTables` — pages given back and taken for a step's new rows, on the
  GPU; each request's page table, each row's slot, position and owner;
* :func:`paged_qk_norm_rope` — per-head RMSNorm of q and k, rotary embedding, and
  the rows' k and v written into their slots;
* :class:`PagedAttention` — attention of every request's new rows over its pages:
  one token of some, drafts or a prompt's chunk of others, in one call.

They stand beside :mod:`kernels.attention`, whose caches hold one run of slots per
sequence (the reference has no paged cache).

A step has ``B`` requests; request b brings rows ``starts[b] .. starts[b + 1] - 1``
of the step's rows (none when it is idle), and rows behind ``starts[B]`` belong to
nobody.  Position t of a request is slot ``t % page_size`` of page ``table[b, t //
page_size]``.  Pools are ``[pages, page_size, kv_heads, head_dim]`` bf16 tensors of any
strides whose last one is 1; page sizes are powers of two from 8.

Calls launch on torch's current stream, never synchronise, and may be captured in a
graph; lengths are read on the GPU when the kernels run, so one graph serves all of
them.  An object's calls are ordered on one stream.  Building an object waits until
its memory is filled (and is refused while a graph is captured); a graph that holds
its calls needs the object as long as it is replayed.  All compute runs in
libkrk_paged.so; there is no fallback.
"""

from __future__ import annotations

import ctypes

import torch

from ._binding import Owner, blocks, index_of, ints, plain, refuse_capture, rows as _rows
from ._paged_lib import LIB, PACK_ATTN, PACK_ROPE, PACK_STEP, Shape

__all__ = ["PageTables", "PagedAttention", "paged_qk_norm_rope", "paged_workspace_bytes"]

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_byref = ctypes.byref


class PageTables(Owner):
    """Page tables of ``B`` requests over a pool of ``pages`` pages of ``page_size``
    slots, for steps of up to ``rows`` rows; ``width`` pages a request at most.

    State, on the GPU: ``lens`` (int32 ``[B]``, cached keys), ``table`` (int32 ``[B,
    width]``), and the stack of free pages, ``free`` (int32 ``[pages]``) up to
    ``count`` (int32 ``[1]``).  At first every page is free, page 0 on top.  With
    ``managed=False`` there is no stack: the caller fills ``table``.

    :meth:`step` leaves what a step's operators take: ``starts`` (int32 ``[B + 1]``),
    ``keys`` (int32 ``[B]``), and by row ``slots``, ``positions`` and ``owner``
    (int32 ``[rows]``; -1 for rows without a slot).
    """

    def __init__(self, B: int, rows: int, pages: int, page_size: int, width: int, device, *, managed: bool = True):
        ints(B=B, rows=rows, pages=pages, page_size=page_size, width=width)
        # What every step would be refused for is refused here.
        LIB.check(LIB.load().krk_paged_check(_byref(Shape(B, rows, 1, 1, 128, page_size, width, 0, 0))))
        if not 1 <= pages <= ((1 << 31) - 1) // page_size:
            raise ValueError(f"pages={pages} of {page_size} slots: needs 1 or more, and fewer than 2^31 slots")
        refuse_capture(device)
        self.B, self.rows, self.pages, self.page_size, self.width, self.managed = B, rows, pages, page_size, width, bool(managed)

        def zeros(*shape):
            return torch.zeros(shape, dtype=_I32, device=device)

        self.lens, self.table = zeros(B), zeros(B, width)
        self.free = torch.arange(pages - 1, -1, -1, dtype=_I32, device=device) if managed else None
        self.count = torch.full((1,), pages, dtype=_I32, device=device) if managed else None
        self.starts, self.keys = zeros(B + 1), zeros(B)
        self.slots, self.positions, self.owner = (torch.full((rows,), -1, dtype=_I32, device=device) for _ in range(3))
        own = (self.lens, self.table, self.starts, self.keys, self.slots, self.positions, self.owner)
        super().__init__(device, own + ((self.free, self.count) if managed else ()))

    def step(self, new: torch.Tensor, *, keep: torch.Tensor | None = None, labels: torch.Tensor | None = None) -> None:
        """Cut request b to its first ``keep[b]`` keys (None: none is cut) and give it
        ``new[b]`` rows more, request after request (both int32 ``[B]`` on the GPU).
        ``owner`` becomes each row's ``labels[b]`` (int32 ``[B]``; None: b itself).

        Pages that a cut empties are free for this step already.  A request whose
        rows end behind ``rows``, pass the table's width, or need pages that the
        stack does not hold gets none: its rows have no slot, ``keys[b]`` is 0 and
        ``lens[b]`` what it was cut to."""
        index = index_of("new", new)
        own = self.lens.get_device()
        if index != own:
            raise ValueError(f"new is on {new.device}; these tables are on {self.lens.device}")
        B = (self.B,)
        args = PACK_STEP(
            self.lens.data_ptr(), 0 if keep is None else plain("keep", keep, index, _I32, B), plain("new", new, index, _I32, B),
            0 if labels is None else plain("labels", labels, index, _I32, B), self.table.data_ptr(), self.width,
            self.free.data_ptr() if self.managed else 0, self.count.data_ptr() if self.managed else 0, self.starts.data_ptr(),
            self.keys.data_ptr(), self.slots.data_ptr(), self.positions.data_ptr(), self.owner.data_ptr(), self.B, self.rows,
            self.pages, self.page_size, self.width)
        self.outlive(index)
        LIB.launch(LIB.load().krk_page_step, index, args)


def paged_qk_norm_rope(qkv: torch.Tensor, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None, eps: float,
                       table: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Normalise and rotate the q and k heads of ``qkv`` and write k and v into the
    rows' slots (:func:`kernels.attention.qk_norm_rope` over pages).

    ``qkv`` is ``[rows, (heads + 2 * kv_heads) * head_dim]``: q heads, k heads, v heads;
    kv_heads, head_dim, pages and page_size are those of the pools ``k`` and ``v``.
    Each q and k head becomes ``x * rsqrt(mean(x * x) + eps) * gain`` (``q_norm``,
    ``k_norm``; None for both: no norm), then its halves ``(a, b)`` become ``(a cos - b
    sin, b cos + a sin)`` with row ``positions[row]`` of ``table``
    (:func:`kernels.attention.rope_table`).  fp32 inside, one rounding.

    Returns the q heads, ``[rows, heads * head_dim]``: in ``q_out``, which may be
    ``qkv[:, :heads * head_dim]`` itself, or a new tensor.  Rows whose slot is outside
    the pool, or whose position is outside the table, leave ``q_out`` and the pools as
    they were."""
    index = index_of("qkv", qkv)
    if not 0.0 <= eps <= 3e38:
        raise ValueError(f"eps={eps} must be finite and >= 0")
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be a [pages, page_size, kv_heads, head_dim] tensor")
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a [positions, head_dim] tensor")
    shape = k.shape
    pages, size, KV, D = shape
    if qkv.dim() != 2 or D < 1 or qkv.shape[0] < 1 or qkv.shape[1] % D:
        raise ValueError(f"qkv must be [rows, (heads + 2 * kv_heads) * head_dim] for pools of shape {tuple(shape)}, "
                         f"got {tuple(qkv.shape)}")
    M, cols = qkv.shape
    heads = cols // D - 2 * KV
    if heads < 1:
        raise ValueError(f"qkv of {cols} columns has no q heads beside {KV} k and {KV} v heads of {D}")
    if q_out is None:
        q_out = qkv.new_empty((M, heads * D))
    n = table.shape[0]
    args = PACK_ROPE(
        *_rows("qkv", qkv, index, (M, cols)), 0 if q_norm is None else plain("q_norm", q_norm, index, _BF16, (D,)),
        0 if k_norm is None else plain("k_norm", k_norm, index, _BF16, (D,)), eps, plain("table", table, index, _F32, (n, D)), n,
        plain("slots", slots, index, _I32, (M,)), plain("positions", positions, index, _I32, (M,)),
        *_rows("q_out", q_out, index, (M, heads * D)), *blocks("k", k, index, shape), *blocks("v", v, index, shape), M, heads, KV, D,
        pages, size)
    LIB.launch(LIB.load().krk_paged_rope_bf16, index, args)
    return q_out


def _shape(B, rows, heads, kv_heads, head_dim, page_size, width, window, sinks) -> Shape:
    """The library's description of a shape that it takes (ValueError for others)."""
    ints(B=B, rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, width=width, window=window,
         sinks=sinks)
    shape = Shape(B, rows, heads, kv_heads, head_dim, page_size, width, window, sinks)
    LIB.check(LIB.load().krk_paged_check(_byref(shape)))
    return shape


def paged_workspace_bytes(B: int, rows: int, heads: int, kv_heads: int, head_dim: int, page_size: int, width: int, *,
                          window: int = 0, sinks: int = 0) -> int:
    """Bytes of workspace that a :class:`PagedAttention` of this shape needs."""
    return int(LIB.load().krk_paged_workspace_bytes(_byref(_shape(B, rows, heads, kv_heads, head_dim, page_size, width, window, sinks))))


class PagedAttention(Owner):
    """Attention of a step's rows over their requests' pages, for a fixed shape:
    ``f(q, k, v, table, starts, keys) -> out``.

    Request b's rows are its last: row i of n has position ``keys[b] - n + i`` and sees
    every key up to itself; with ``window`` the ``window`` last of them, and the first
    ``sinks`` positions as well.  Query head h reads key/value head ``h // (heads //
    kv_heads)``.  ``scale`` is ``head_dim ** -0.5`` unless given.

    The workspace (:func:`paged_workspace_bytes`) belongs to the object, or is
    ``workspace``: zero-filled uint8 memory that objects may share if all their calls
    are ordered on one stream.  Results are deterministic.
    """

    def __init__(self, B: int, rows: int, heads: int, kv_heads: int, head_dim: int, page_size: int, width: int, device, *,
                 window: int = 0, sinks: int = 0, scale: float | None = None, workspace: torch.Tensor | None = None):
        self._shape = _shape(B, rows, heads, kv_heads, head_dim, page_size, width, window, sinks)
        if scale is not None and not 1e-45 < scale <= 2.3e38:  # as an fp32, and times log2(e)
            raise ValueError(f"scale={scale} must be positive and at most 2.3e38")
        self.B, self.rows, self.heads, self.kv_heads, self.head_dim = B, rows, heads, kv_heads, head_dim
        self.page_size, self.width, self.window, self.sinks = page_size, width, window, sinks
        self.scale = float(head_dim ** -0.5 if scale is None else scale)
        nbytes = int(LIB.load().krk_paged_workspace_bytes(_byref(self._shape)))
        self._q_shape = (rows, heads * head_dim)
        refuse_capture(device)
        if workspace is None:
            if nbytes:
                workspace = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        elif workspace.dtype is not torch.uint8 or workspace.numel() < nbytes or not workspace.is_contiguous():
            raise ValueError(f"workspace must be {nbytes} contiguous bytes (uint8) or more, got {workspace.dtype} {tuple(workspace.shape)}")
        elif workspace.device.type != torch.device(device).type or torch.device(device).index not in (None, workspace.device.index):
            raise ValueError(f"workspace on {workspace.device}; this object is built on {device}")
        self.workspace = workspace
        super().__init__(device, () if workspace is None else (workspace,))

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, keys: torch.Tensor,
            out: torch.Tensor, *, lse: torch.Tensor | None = None) -> torch.Tensor:
        """Allocation-free form: write into ``out`` (``[rows, heads * head_dim]``), and
        with ``lse`` (``[rows, heads]`` fp32) the log of each softmax's sum.  Rows
        behind ``starts[B]`` are left as they were."""
        index = index_of("q", q)
        if not isinstance(k, torch.Tensor) or k.dim() != 4:
            raise ValueError("k must be a [pages, page_size, kv_heads, head_dim] tensor")
        pages = k.shape[0]
        pool = (pages, self.page_size, self.kv_heads, self.head_dim)
        args = PACK_ATTN(
            *_rows("q", q, index, self._q_shape), *blocks("k", k, index, pool), *blocks("v", v, index, pool), pages, self.scale,
            *_rows("table", table, index, (self.B, self.width), _I32), plain("starts", starts, index, _I32, (self.B + 1,)),
            plain("keys", keys, index, _I32, (self.B,)), *_rows("out", out, index, self._q_shape),
            0 if lse is None else plain("lse", lse, index, _F32, (self.rows, self.heads)))
        ws = self.workspace
        if ws is None:
            LIB.launch(LIB.load().krk_paged_attn_bf16, index, _byref(self._shape), args, 0, 0)
        elif ws.get_device() == index:
            self.outlive(index)
            LIB.launch(LIB.load().krk_paged_attn_bf16, index, _byref(self._shape), args, ws.data_ptr(), ws.numel())
        else:
            raise ValueError(f"operands on {q.device}; this object was built on {self.device}")
        return out

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                 keys: torch.Tensor, *, lse: torch.Tensor | None = None) -> torch.Tensor:
        """``softmax(scale * q k^T) v`` as a new ``[rows, heads * head_dim]`` tensor, zeros
        in rows behind ``starts[B]``.

        ``q`` may be the first columns of the qkv rows.  ``table`` (int32 ``[B,
        width]``), ``starts`` and ``keys`` as :class:`PageTables` keeps them."""
        index_of("q", q)
        out = torch.zeros(self._q_shape, dtype=_BF16, device=q.device)
        return self.run(q, k, v, table, starts, keys, out, lse=lse)
