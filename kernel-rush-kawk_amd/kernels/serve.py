"""Serving many requests at once: the model-wide state of a step over requests of
different lengths (:mod:`kernels.paged`) with adapters of their own
(:mod:`kernels.adapters`).

:class:`kernels.step.GemmStep` runs both: :class:`PagedCache` between the qkv and o
projections of each layer, as :class:`kernels.cache.DecodeCache` does for sequences of
one length, and :class:`AdapterSet` behind each projection (reference data flow of
``run_layers``, engine/model.py:181-214).
"""

from __future__ import annotations

import torch

from . import attention as A
from . import paged as P
from ._binding import refuse_capture
from .adapters import LowRankAdapters

_BF16, _I32 = torch.bfloat16, torch.int32
_ALL = 2 ** 31 - 1


class PagedCache:
    """Pages of k and v for up to ``B`` requests in each layer of the model ``m``
    (``m.cfg`` and ``m.layers`` as :func:`kernels.step.synthetic_model` builds them), for
    steps of up to ``rows`` rows: ``pages`` pages of ``page_size`` slots, shared by all
    requests and numbered alike in all layers.

    A step's projections and logits run over all ``rows``, whatever its plan brings.

    A step is planned by :meth:`schedule`, on the host, which refuses what does not fit;
    :meth:`begin` then moves pages, tables and lengths on, on the device, so a captured
    step serves every plan.  The host's own count of each request's keys
    (:attr:`lens`) is what the next step starts from: rows of a step that failed, and
    those that :meth:`rollback` or :meth:`reset` took off, give their pages back when
    it begins.

    ``labels`` (int32 ``[B]`` on the GPU) is each request's adapter, -1 for none, as
    :meth:`reset` leaves it; by row it is ``tables.owner``.  ``window``, ``sinks``: sliding-window attention in every layer.
    """

    def __init__(self, m, B: int, rows: int, pages: int, page_size: int = 64, *, width: int | None = None, window: int = 0,
                 sinks: int = 0, max_positions: int | None = None):
        cfg, dev = m.cfg, m.device
        refuse_capture(dev)
        width = pages if width is None else width
        self.m, self.B, self.rows, self.pages, self.page_size, self.width = m, B, rows, pages, page_size, width
        self.heads, self.kv_heads, self.head_dim = cfg.heads, cfg.kv_heads, cfg.head_dim
        self.attention = P.PagedAttention(B, rows, cfg.heads, cfg.kv_heads, cfg.head_dim, page_size, width, dev, window=window,
                                          sinks=sinks)
        self.tables = P.PageTables(B, rows, pages, page_size, width, dev)
        shape = (len(m.layers), pages, page_size, cfg.kv_heads, cfg.head_dim)
        self.k, self.v = (list(torch.zeros(shape, dtype=_BF16, device=dev)) for _ in "kv")
        self.max_positions = min(width, pages) * page_size if max_positions is None else max_positions
        self.table = A.rope_table(self.max_positions, cfg.head_dim, cfg.theta, dev)
        self.new, self.keep = (torch.zeros(B, dtype=_I32, device=dev) for _ in range(2))
        self.labels = torch.full((B,), -1, dtype=_I32, device=dev)
        self.lens = [0] * B       # keys of each request, on the host
        self._plan: list | None = None  # new rows of the scheduled step
        A.filled(self.new.device)  # steps may run on another stream

    def _pages_of(self, n: int) -> int:
        return -(-n // self.page_size)

    def schedule(self, new: list) -> list:
        """Plan the next step: ``new[b]`` rows of request b.  Its first row's place among
        the step's rows is returned for each request.  ValueError, and nothing
        changes, where the rows, a request's pages or positions, or all pages together
        do not fit."""
        new = [int(n) for n in new]
        if len(new) != self.B or min(new) < 0:
            raise ValueError(f"schedule needs a row count for each of {self.B} requests, got {new}")
        if sum(new) > self.rows:
            raise ValueError(f"{sum(new)} rows for steps of up to {self.rows}")
        for b, n in enumerate(new):
            if n and self.lens[b] + n > min(self.max_positions, self.width * self.page_size):
                raise ValueError(f"request {b}: {n} rows behind {self.lens[b]} keys pass its {self.width} pages of {self.page_size} "
                                 f"or the rotary table's {self.max_positions} positions")
        need = sum(self._pages_of(have + n) for have, n in zip(self.lens, new))
        if need > self.pages:
            raise ValueError(f"the step needs {need} of {self.pages} pages")
        both = torch.tensor([new, self.lens], dtype=_I32)
        self.new.copy_(both[0])
        self.keep.copy_(both[1])
        self._plan = new
        return [sum(new[:b]) for b in range(self.B)]

    def check(self, M: int) -> None:
        """ValueError for a step that this cache does not serve."""
        if M != self.rows:
            raise ValueError(f"M={M} rows for a paged cache of steps of {self.rows}")

    def planned(self) -> None:
        """RuntimeError unless a step is scheduled."""
        if self._plan is None:
            raise RuntimeError("schedule() first")

    def begin(self) -> None:
        """The step starts: pages, tables, slots and positions, on the device."""
        self.tables.step(self.new, keep=self.keep, labels=self.labels)

    def attend(self, i: int, qkv: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """Layer ``i`` between its qkv and o projections: q and k normed and rotated (q
        in place), k and v written into their pages, attention into ``out``.  Rows of
        no request are left as they are."""
        layer, t = self.m.layers[i], self.tables
        q = qkv[:, :self.heads * self.head_dim]
        P.paged_qk_norm_rope(qkv, layer.q_norm, layer.k_norm, self.m.cfg.eps, self.table, t.slots, t.positions, self.k[i], self.v[i],
                             q_out=q)
        return self.attention.run(q, self.k[i], self.v[i], t.table, t.starts, t.keys, out)

    def commit(self) -> None:
        """The scheduled step's rows are cached."""
        self.lens = [have + n for have, n in zip(self.lens, self._plan)]
        self._plan = None

    def rollback(self, rows: list) -> None:
        """Forget the last ``rows[b]`` keys of each request: the rejected rows of a
        verified draft."""
        if len(rows) != self.B or any(not 0 <= n <= have for n, have in zip(rows, self.lens)):
            raise ValueError(f"rollback needs 0 .. keys rows for each of {self.B} requests, got {list(rows)}")
        self.lens = [have - int(n) for have, n in zip(self.lens, rows)]
        self._plan = None

    def reset(self, b: int | None = None) -> None:
        """Forget request ``b`` (None: all): its pages are free for the next step, and the
        next request in its place has no adapter until its label is written."""
        for i in range(self.B) if b is None else [b]:
            self.lens[i] = 0
        self.labels[slice(None) if b is None else b] = -1
        self._plan = None

    def idle(self) -> None:
        """No rows for any request, on the device: what a step is captured with."""
        self.new.zero_()
        self.keep.fill_(_ALL)
        self._plan = None


#: Projections that adapters can stand behind, by their names in ``decode_matmuls``.
TARGETS = ("qkv", "o", "gu", "d")


class AdapterSet:
    """``adapters`` adapters of rank ``rank`` for the projections ``targets`` ("qkv", "o",
    "gu": gate and up, "d": down) of each layer of the model ``m``.

    ``a[target][layer]`` (``[adapters, slices * rank, K]``) and ``b[target][layer]``
    (``[adapters, N, rank]``) hold the factors, zeros at first; the slices are q, k and v of
    "qkv", gate and up of "gu".  ``scale`` is fp32 ``[adapters]``, ones at first.
    """

    def __init__(self, m, adapters: int, rank: int, targets: tuple = TARGETS):
        if not targets or any(t not in TARGETS for t in targets) or len(set(targets)) != len(targets):
            raise ValueError(f"targets={targets!r}: some of {TARGETS}")
        if adapters < 1:
            raise ValueError(f"adapters={adapters} must be >= 1")
        cfg, dev = m.cfg, m.device
        refuse_capture(dev)
        D = cfg.head_dim
        q, kv, I = cfg.heads * D, cfg.kv_heads * D, cfg.intermediate
        widths = {"qkv": (q, kv, kv), "o": (cfg.hidden,), "gu": (I, I), "d": (cfg.hidden,)}
        depth = {"qkv": cfg.hidden, "o": q, "gu": cfg.hidden, "d": I}
        self.m, self.adapters, self.rank, self.targets = m, adapters, rank, tuple(targets)
        self.widths, self.depth = ({t: d[t] for t in targets} for d in (widths, depth))
        for t in targets:
            self.operator(t, 1)  # ValueError for a rank that no call takes

        def zeros(*shape):
            return [torch.zeros((adapters, *shape), dtype=_BF16, device=dev) for _ in m.layers]

        self.a = {t: zeros(len(widths[t]) * rank, depth[t]) for t in targets}
        self.b = {t: zeros(sum(widths[t]), rank) for t in targets}
        self.scale = torch.ones(adapters, device=dev)
        A.filled(self.scale.device)

    def operator(self, target: str, rows: int) -> LowRankAdapters:
        """The operator of ``target`` for ``rows`` rows."""
        w = self.widths[target]
        return LowRankAdapters(rows, sum(w), self.depth[target], self.rank, self.m.device, slices=w, silu=target == "gu")
