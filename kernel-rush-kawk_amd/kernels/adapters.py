"""Low-rank adapters of many requests beside one shared projection on MI355X.

:class:`LowRankAdapters` adds ``scale[i] * (x A_i^T) B_i^T`` to a projection's output,
with i each row's own adapter, or none (the reference has no adapters).  Calls launch
on torch's current stream, never synchronise, and may be captured in a graph; an
object's calls are ordered on one stream; it is built before a graph is captured, and a
graph that holds its calls needs it as long as it is replayed.  All compute runs in libkrk_adapter.so; there is no fallback.
"""

from __future__ import annotations

import ctypes

import torch

from ._adapter_lib import LIB, PACK, SLICES, Shape
from ._binding import Owner, blocks, index_of, ints, plain, refuse_capture, rows as _rows

__all__ = ["LowRankAdapters"]

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_byref = ctypes.byref


class LowRankAdapters(Owner):
    """Adapters of rank ``rank`` for a projection of ``rows`` rows, ``[rows, K] -> [rows,
    N]``: ``f(x, a, b, index, y) -> y + scale[i] * (x a[i].T) b[i].T``, i = index[row].

    ``slices``: the widths of the parts of y that have first factors of their own (q, k
    and v of a fused projection); None: one.  ``silu``: y is ``[gate, up]`` side by side
    (1 slice, or 2 of ``N // 2``) and the result ``silu(gate) * up``, ``[rows, N // 2]``.
    """

    def __init__(self, rows: int, N: int, K: int, rank: int, device, *, slices: tuple | list | None = None, silu: bool = False):
        widths = [N] if slices is None else list(slices)
        if not 1 <= len(widths) <= SLICES:
            raise ValueError(f"slices={slices!r}: 1 to {SLICES} widths")
        ints(rows=rows, N=N, K=K, rank=rank, **{f"slices[{i}]": w for i, w in enumerate(widths)})
        self._shape = Shape(rows, N, K, rank, int(bool(silu)), len(widths), (ctypes.c_int * SLICES)(*widths))
        LIB.check(LIB.load().krk_adapter_check(_byref(self._shape)))
        self.rows, self.N, self.K, self.rank, self.silu, self.widths = rows, N, K, rank, bool(silu), tuple(widths)
        self.out_cols = N // 2 if silu else N
        refuse_capture(device)
        self.workspace = torch.empty(int(LIB.load().krk_adapter_workspace_bytes(_byref(self._shape))), dtype=torch.uint8, device=device)
        super().__init__(device, (self.workspace,))

    def run(self, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor, y: torch.Tensor, out: torch.Tensor, *,
            scale: torch.Tensor | None = None) -> torch.Tensor:
        """Allocation-free form: write into ``out``, which may be ``y`` itself (not with
        ``silu``)."""
        gpu = index_of("x", x)
        if not isinstance(a, torch.Tensor) or a.dim() != 3 or a.shape[0] < 1:
            raise ValueError("a must be an [adapters, slices * rank, K] tensor")
        n = a.shape[0]
        M, K, N = self.rows, self.K, self.N
        args = PACK(
            *_rows("x", x, gpu, (M, K)), *blocks("a", a, gpu, (n, len(self.widths) * self.rank, K)),
            *blocks("b", b, gpu, (n, N, self.rank)), 0 if scale is None else plain("scale", scale, gpu, _F32, (n,)),
            plain("index", index, gpu, _I32, (M,)), *_rows("y", y, gpu, (M, N)), *_rows("out", out, gpu, (M, self.out_cols)), n)
        ws = self.workspace
        if ws.get_device() != gpu:
            raise ValueError(f"operands on {x.device}; this object was built on {self.device}")
        self.outlive(gpu)
        LIB.launch(LIB.load().krk_adapter_bf16, gpu, _byref(self._shape), args, ws.data_ptr(), ws.numel())
        return out

    def __call__(self, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor, y: torch.Tensor, *,
                 scale: torch.Tensor | None = None) -> torch.Tensor:
        """The result as a new tensor.

        ``a`` ``[adapters, slices * rank, K]`` and ``b`` ``[adapters, N, rank]`` (bf16; of
        smaller ranks, padded with zeros), ``scale`` fp32 ``[adapters]`` (None: 1),
        ``index`` int32 ``[rows]``: a row's adapter, none where it is outside 0 ..
        adapters - 1."""
        index_of("x", x)
        out = torch.empty((self.rows, self.out_cols), dtype=_BF16, device=x.device)
        return self.run(x, a, b, index, y, out, scale=scale)
