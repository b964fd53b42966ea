"""The key/value cache of a decode step: every layer's k and v, and the cache
operators of :mod:`kernels.attention` over them.

:class:`DecodeCache` is what :class:`kernels.step.GemmStep` calls between the
qkv and the o projection of each layer (reference data flow of ``run_layers``,
engine/model.py:181-214: ``mm["qkv"]``, ``qk_norm_rope_cache``, ``attention``,
``mm["o"]``).
"""

from __future__ import annotations

import torch

from . import attention as A

_BF16 = torch.bfloat16


class DecodeCache:
    """``capacity`` slots of k and v for ``B`` sequences in each layer of the
    model ``m`` (``m.cfg`` and ``m.layers`` as :func:`kernels.step.synthetic_model`
    builds them; each layer's ``q_norm`` and ``k_norm`` gains).

    * ``window``, ``sinks``: sliding-window attention in every layer;
    * ``prefix``: one ``(k, v)`` pair of ``[keys, kv_heads, head_dim]`` tensors
      per layer, shared by all sequences; own positions follow it;
    * ``scored``: each key's accumulated attention weight is kept
      (``scores[layer]``, ``[B, kv_heads, capacity]``), for :meth:`evict`.

    ``lens`` (int32 ``[B]``) counts the cached slots and ``seen`` the tokens a
    sequence has had (its next position): they differ after an eviction.  Each
    step's :meth:`begin` moves both on by its rows, on the device, so a captured
    step continues from replay to replay.  The host keeps its own count, to
    refuse a step that would not fit.
    """

    def __init__(self, m, B: int, capacity: int, *, window: int = 0, sinks: int = 0, prefix: list | None = None,
                 scored: bool = False, max_positions: int | None = None):
        cfg, dev = m.cfg, m.device
        self.m, self.B, self.capacity, self.window, self.sinks, self.scored = m, B, capacity, window, sinks, scored
        self.heads, self.kv_heads, self.head_dim = cfg.heads, cfg.kv_heads, cfg.head_dim
        if prefix is not None and len(prefix) != len(m.layers):
            raise ValueError(f"prefix: {len(prefix)} pairs for {len(m.layers)} layers")
        self.prefix = prefix
        self.prefix_keys = 0 if prefix is None else prefix[0][0].shape[0]
        # What every step would be refused for is refused here.
        A.workspace_bytes(B, 1, cfg.heads, cfg.kv_heads, cfg.head_dim, capacity, window=window, sinks=sinks,
                          prefix=self.prefix_keys, scored=scored)
        for i, pair in enumerate(prefix or ()):
            run = (self.prefix_keys, cfg.kv_heads, cfg.head_dim)
            if len(pair) != 2 or any(t.dtype is not _BF16 or t.shape != run or t.device.type != dev.type for t in pair):
                raise ValueError(f"prefix of layer {i}: needs a bf16 k and v of shape {run} on {dev}, as layer 0 has")
        shape = (B, capacity, cfg.kv_heads, cfg.head_dim)
        # One tensor, so that accept() moves the rows of all layers at once.
        self._kv = torch.zeros((2, len(m.layers), *shape), dtype=_BF16, device=dev)
        self.k, self.v = list(self._kv[0]), list(self._kv[1])
        self.scores = [torch.zeros((B, cfg.kv_heads, capacity), device=dev) for _ in m.layers] if scored else None
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)
        self.seen = torch.zeros(B, dtype=torch.int32, device=dev)
        self.max_positions = self.prefix_keys + 4 * capacity if max_positions is None else max_positions
        self.table = A.rope_table(self.max_positions, cfg.head_dim, cfg.theta, dev)
        self._host = [[0, 0] for _ in range(B)]  # slots and tokens of each sequence
        self._ops: dict = {}
        self._workspace: torch.Tensor | None = None
        self._evictions: dict = {}
        self._rows = 0
        self._positions = self._tree = None
        A.filled(self.lens.device)  # steps may run on another stream

    def _op(self, R: int) -> A.CacheAttention:
        """The attention of ``R`` rows per sequence.  Its calls are ordered by the
        cache itself, so all row counts share one workspace.  One that needs more
        takes at least twice as much: earlier ones, whose addresses graphs may
        hold, add up to less than the last."""
        if R not in self._ops:
            kw = dict(window=self.window, sinks=self.sinks, prefix=self.prefix_keys, scored=self.scored)
            shape = self.B, R, self.heads, self.kv_heads, self.head_dim, self.capacity
            need, have = A.workspace_bytes(*shape, **kw), 0 if self._workspace is None else self._workspace.numel()
            if need > have:
                self._workspace = A.zero_workspace(max(need, 2 * have), self.lens.device)
            self._ops[R] = A.CacheAttention(*shape, self.lens.device, workspace=self._workspace if need else None, **kw)
        return self._ops[R]

    def check(self, R: int, tree: torch.Tensor | None = None) -> None:
        """ValueError for a step of ``R`` rows per sequence that no cache of this
        shape takes, or for ``tree`` masks that it does not."""
        self._op(R)
        if tree is None:
            return
        if self.scored:
            raise ValueError("scores are kept for accepted rows only: a draft tree's rows may still be rejected")
        if R > 64 or 0 < self.window < R:
            raise ValueError(f"tree masks need R <= 64 and a window of 0 or >= R, got R={R} window={self.window}")
        if not isinstance(tree, torch.Tensor) or tree.dtype is not torch.int64 or tree.shape != (self.B, R):
            raise ValueError(f"tree must be an int64 tensor of shape {(self.B, R)}")
        if tree.device != self.lens.device or not tree.is_contiguous():
            raise ValueError(f"tree must be contiguous and on {self.lens.device}, got {tree.device} and strides {tree.stride()}")

    def reserve(self, R: int) -> None:
        """Count ``R`` more rows of every sequence on the host; ValueError where
        they do not fit."""
        for slots, tokens in self._host:
            if slots + R > self.capacity:
                raise ValueError(f"{R} more rows do not fit: a sequence has {slots} of {self.capacity} slots")
            if self.prefix_keys + tokens + R > self.max_positions:
                raise ValueError(f"{R} more rows pass the {self.max_positions} positions of the rotary table")
        for c in self._host:
            c[0] += R
            c[1] += R

    def begin(self, R: int, tree: torch.Tensor | None = None, reserve: bool = True) -> None:
        """A step of ``R`` rows per sequence starts: ``lens`` and ``seen`` move
        on, and the rows' positions follow (``tree``: ancestor masks, int64
        ``[B, R]``; a node's position is its depth below the first row's).  A
        step that is refused leaves the cache as it was."""
        self.check(R, tree)
        if reserve:
            self.reserve(R)
        dev = self.lens.device
        if tree is None:
            depth = torch.arange(R, dtype=torch.int32, device=dev)
        else:
            bits = tree[..., None] >> torch.arange(R, device=dev) & 1
            depth = bits.sum(dim=-1).int() - 1
        self._positions = ((self.seen + self.prefix_keys)[:, None] + depth).reshape(self.B * R)
        self.lens.add_(R)
        self.seen.add_(R)
        self._tree, self._rows, self._current = tree, R, self._op(R)

    def attend(self, i: int, qkv: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """Layer ``i`` between its qkv and o projections: q and k normed and
        rotated (q in place), k and v appended, attention into ``out``."""
        if not self._rows:
            raise RuntimeError("begin() first")
        layer, k, v = self.m.layers[i], self.k[i], self.v[i]
        q = qkv[:, :self.heads * self.head_dim]
        A.qk_norm_rope(qkv, layer.q_norm, layer.k_norm, self.m.cfg.eps, self.table, self.lens, k, v,
                       positions=self._positions, q_out=q)
        return self._current.run(q, k, v, self.lens, out, prefix=None if self.prefix is None else self.prefix[i],
                                 tree=self._tree, scores=self.scores[i] if self.scored else None)

    def evict(self, budget: int, *, sinks: int = 0, recent: int = 0) -> list:
        """Cut every layer's cache down to ``budget`` slots per sequence and
        head by the scores; the kept slots of each layer (int32 ``[B, kv_heads,
        budget]``).  Positions go on from ``seen``."""
        if not self.scored:
            raise ValueError("evict() needs a cache built with scored=True")
        if self.window:
            raise ValueError("a sliding window goes by slots: it does not go with evict()")
        key = (budget, sinks, recent)
        if key not in self._evictions:
            self._evictions[key] = A.CacheEviction(self.B, self.kv_heads, self.head_dim, self.capacity, budget,
                                                   self.lens.device, sinks=sinks, recent=recent)
        op, kept, after = self._evictions[key], [], torch.empty_like(self.lens)
        for i in range(len(self.k)):
            keep = torch.empty((self.B, self.kv_heads, budget), dtype=torch.int32, device=self.lens.device)
            kept.append(op.run(self.k[i], self.v[i], self.scores[i], self.lens, keep, after))
            self.scores[i][:, :, budget:].zero_()  # slots that new rows will take
        self.lens.copy_(after)
        for c in self._host:
            c[0] = min(c[0], budget)
        return kept

    def accept(self, R: int, paths: list) -> None:
        """End a draft tree's step of ``R`` rows: of each sequence's last ``R``
        slots the nodes ``paths[b]`` stay (ascending; from the root, each the
        parent of the next) and become its next slots in every layer; the rest
        is forgotten.  A node's position is its depth, so what stays is what a
        step of those rows alone would have cached.  Until this or
        :meth:`rollback`, later rows see every node."""
        if self.scored:
            raise ValueError("a scored cache takes no draft trees: rollback() forgets its last rows")
        paths = [list(p) for p in paths]
        if R < 1 or len(paths) != self.B or any(c[0] < R for c in self._host):
            raise ValueError(f"accept needs a path for each of {self.B} sequences and {R} >= 1 slots in each")
        for p in paths:
            if any(not 0 <= i < R for i in p) or any(a >= b for a, b in zip(p, p[1:])):
                raise ValueError(f"a path is ascending rows 0 .. {R - 1}, got {p}")
        moves = [(b * self.capacity + c[0] - R + j, b * self.capacity + c[0] - R + i)
                 for b, (c, p) in enumerate(zip(self._host, paths)) for j, i in enumerate(p) if i != j]
        if moves:
            to, at = torch.tensor(moves, device=self.lens.device).T
            rows = self._kv.view(2 * len(self.k), self.B * self.capacity, self.kv_heads, self.head_dim)
            rows[:, to] = rows[:, at]
        self.rollback([R - len(p) for p in paths])

    def rollback(self, rows: list) -> None:
        """Forget the last ``rows[b]`` slots of each sequence: the rejected rows
        of a verified draft, behind the accepted ones (:meth:`accept` where the
        accepted nodes of a tree are not its first).  What they added to the
        scores of the keys before them stays."""
        if len(rows) != self.B or any(not 0 <= n <= c[0] for n, c in zip(rows, self._host)):
            raise ValueError(f"rollback needs 0 .. slots rows for each of {self.B} sequences, got {list(rows)}")
        self._rows = 0
        less = torch.tensor(rows, dtype=torch.int32, device=self.lens.device)
        self.lens.sub_(less)
        self.seen.sub_(less)
        for c, n in zip(self._host, rows):
            c[0] -= n
            c[1] -= n
        if self.scored:  # the slots' next rows start at zero
            free = torch.arange(self.capacity, device=self.lens.device) >= self.lens[:, None, None]
            for s in self.scores:
                s.masked_fill_(free, 0.0)

    def reset(self, b: int | None = None) -> None:
        """Forget sequence ``b`` (None: all): its slots are free again."""
        at = slice(None) if b is None else b
        for t in (self.lens, self.seen, *(self.scores or ())):
            t[at] = 0
        for c in self._host if b is None else [self._host[b]]:
            c[0] = c[1] = 0

    def _state(self) -> tuple:
        return [list(c) for c in self._host], [t.clone() for t in (self.lens, self.seen, *(self.scores or ()))]

    def _restore(self, state: tuple) -> None:
        self._rows = 0
        self._host = [list(c) for c in state[0]]
        for t, s in zip((self.lens, self.seen, *(self.scores or ())), state[1]):
            t.copy_(s)
