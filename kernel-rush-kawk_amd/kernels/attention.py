"""The cache operators of a decode step on MI355X: what runs between the qkv
projection and the o projection.

* :func:`qk_norm_rope` — per-head RMSNorm of q and k, rotary embedding, and the
  new rows' k and v written into the cache (reference ``qk_norm_rope_cache``,
  engine/kernels/rope.py:147), with :func:`rope_table`;
* :class:`CacheAttention` — attention of R new rows of each of B sequences over
  their cache (reference ``DecodeAttention``, engine/kernels/attention.py:153):
  causal, with a sliding window and sinks, with a draft tree's ancestor masks,
  over a prefix that the whole batch shares, and with each key's attention
  weight added to its score;
* :class:`CacheEviction` — the cache cut down to a budget of slots per head, by
  those scores.

Caches are ``[B, capacity, kv_heads, head_dim]`` bf16 tensors of any strides
whose last one is 1 (a ``[B, kv_heads, capacity, head_dim]`` cache is passed as
its ``transpose(1, 2)``).  ``lens`` is an int32 ``[B]`` tensor on the GPU: each
sequence's cached keys, the call's own R rows among them and last.  Row
``b * R + i`` lies in slot ``lens[b] - R + i``; rows without a slot (a sequence
shorter than R, an idle one) are padding and give zeros.

Calls launch on torch's current stream, never synchronise, and may be captured
in a graph; an object's workspace is its own, so its calls are ordered on one
stream.  All compute runs in libkrk_attn.so; there is no fallback.
"""

from __future__ import annotations

import ctypes

import torch

from . import _attn_lib as _lib
from ._attn_lib import AttnArgs, AttnPlan, AttnShape, Cache, EvictArgs, RopeArgs

__all__ = ["CacheAttention", "CacheEviction", "qk_norm_rope", "rope_table"]

_BF16 = torch.bfloat16
_byref = ctypes.byref


def _launch(fn, index: int, *args) -> None:
    """``fn(*args, stream)`` on GPU ``index`` and torch's current stream there."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _on(index: int, name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.get_device() != index or not t.is_cuda:
        raise ValueError(f"{name} must be on the operands' GPU, got {t.device}")


def _index(name: str, t: torch.Tensor) -> int:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor, got device {t.device}")
    return t.get_device()


def _cache(name: str, t: torch.Tensor, index: int, B: int | None, slots: int | None, kv_heads: int, dim: int) -> tuple:
    """The fields of ``krk_cache`` for a [B, slots, kv_heads, dim] tensor (B
    None: a [slots, kv_heads, dim] one), checked."""
    _on(index, name, t)
    want = (slots, kv_heads, dim) if B is None else (B, slots, kv_heads, dim)
    if t.dtype is not _BF16 or t.dim() != len(want) or any(w is not None and s != w for s, w in zip(t.shape, want)):
        raise ValueError(f"{name} must be bfloat16 of shape {want}, got {t.dtype} {tuple(t.shape)}")
    st = t.stride()
    if st[-1] != 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous, got strides {st}")
    return (t.data_ptr(), 0, *st[:2]) if B is None else (t.data_ptr(), *st[:3])


def _rows(name: str, t: torch.Tensor, index: int, rows: int, cols: int) -> tuple:
    _on(index, name, t)
    if t.dtype is not _BF16 or t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols:
        raise ValueError(f"{name} must be bfloat16 of shape ({rows}, {cols}), got {t.dtype} {tuple(t.shape)}")
    row, one = t.stride()
    if one != 1 and cols > 1:
        raise ValueError(f"{name} rows must be contiguous (stride(1) == 1), got strides {t.stride()}")
    return t.data_ptr(), row if rows > 1 else max(row, cols)


def _plain(name: str, t: torch.Tensor, index: int, dtype: torch.dtype, shape: tuple) -> int:
    """The address of a contiguous tensor of this type and shape."""
    _on(index, name, t)
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()}")
    return t.data_ptr()


def _scores(name: str, t: torch.Tensor, index: int, B: int, kv_heads: int, slots: int, more: bool = False) -> tuple:
    _on(index, name, t)
    if (t.dtype is not torch.float32 or t.dim() != 3 or t.shape[:2] != (B, kv_heads)
            or not (t.shape[2] == slots or more and t.shape[2] > slots)):
        raise ValueError(f"{name} must be float32 of shape ({B}, {kv_heads}, {slots}), got {t.dtype} {tuple(t.shape)}")
    seq, head, one = t.stride()
    if one != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: the scores of a head must be contiguous, got strides {t.stride()}")
    return t.data_ptr(), seq, head


def rope_table(positions: int, head_dim: int, theta: float, device) -> torch.Tensor:
    """``[positions, head_dim]`` fp32: cosines, then sines, of the angles
    ``position * theta ** (-2 i / head_dim)``, taken in 64 bits."""
    if positions < 1 or head_dim < 2 or head_dim % 2:
        raise ValueError(f"rope_table needs positions >= 1 and an even head_dim, got {positions} and {head_dim}")
    freq = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device)


def qk_norm_rope(qkv: torch.Tensor, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None, eps: float,
                 table: torch.Tensor, lens: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                 positions: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Normalise and rotate the q and k heads of ``qkv`` and append k and v to
    the cache.

    ``qkv`` is ``[B * R, (heads + 2 * kv_heads) * head_dim]``: q heads, k heads,
    v heads, as the fused projection leaves them; B, kv_heads and head_dim are
    those of the cache ``k``, ``v``.  Each q and k head becomes
    ``x * rsqrt(mean(x * x) + eps) * gain`` (``q_norm``, ``k_norm``; None for
    both: no norm), then its halves ``(a, b)`` become ``(a cos - b sin, b cos +
    a sin)`` with row ``position`` of ``table`` (:func:`rope_table`): the row's
    slot, or ``positions`` (int32 ``[B * R]``), as a draft tree's rows or a
    shared prefix need them.  fp32 inside, one rounding.

    Returns the q heads, ``[B * R, heads * head_dim]``: in ``q_out``, which may
    be ``qkv[:, :heads * head_dim]`` itself, or a new tensor.  k and v go to
    the rows' slots.  Rows without a slot, or whose position is outside the
    table, leave ``q_out`` and the cache as they were."""
    index = _index("qkv", qkv)
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be a [B, capacity, kv_heads, head_dim] tensor")
    B, cap, KV, D = k.shape
    if qkv.dim() != 2 or B < 1 or D < 1 or qkv.shape[0] < 1 or qkv.shape[0] % B or qkv.shape[1] % D:
        raise ValueError(f"qkv must be [B * R, (heads + 2 * kv_heads) * head_dim] for a cache of shape {tuple(k.shape)}, "
                         f"got {tuple(qkv.shape)}")
    M, cols = qkv.shape
    heads = cols // D - 2 * KV
    if heads < 1:
        raise ValueError(f"qkv of {cols} columns has no q heads beside {KV} k and {KV} v heads of {D}")
    a = RopeArgs()
    a.qkv, a.qkv_row = _rows("qkv", qkv, index, M, cols)
    a.k = _cache("k", k, index, B, cap, KV, D)
    a.v = _cache("v", v, index, B, cap, KV, D)
    if q_norm is not None:
        a.q_norm = _plain("q_norm", q_norm, index, _BF16, (D,))
    if k_norm is not None:
        a.k_norm = _plain("k_norm", k_norm, index, _BF16, (D,))
    a.eps = eps
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a [positions, head_dim] tensor")
    a.table, a.table_rows = _plain("table", table, index, torch.float32, (table.shape[0], D)), table.shape[0]
    a.lens = _plain("lens", lens, index, torch.int32, (B,))
    if positions is not None:
        a.positions = _plain("positions", positions, index, torch.int32, (M,))
    if q_out is None:
        q_out = torch.empty((M, heads * D), dtype=_BF16, device=qkv.device)
    a.q_out, a.q_row = _rows("q_out", q_out, index, M, heads * D)
    if M == 1 and a.q_out == a.qkv:
        a.q_row = a.qkv_row  # one row in place: its stride is of no matter
    a.B, a.R, a.heads, a.kv_heads, a.head_dim, a.capacity = B, M // B, heads, KV, D, cap
    _launch(_lib.load().krk_qk_norm_rope_bf16, index, _byref(a))
    return q_out


class CacheAttention:
    """Attention of ``R`` new rows of each of ``B`` sequences over their cache,
    for a fixed shape: ``f(q, k, v, lens) -> out``.

    Query head h reads key/value head ``h // (heads // kv_heads)``.  The row at
    position p sees every key up to itself; with ``window`` the ``window`` last
    of them, and the first ``sinks`` positions as well.  ``prefix`` is the most
    keys of a prefix that all sequences share; the cache's slot s then has
    position ``prefix keys + s``.  ``scored`` objects update their keys' scores.
    ``scale`` is ``head_dim ** -0.5`` unless given.

    The workspace belongs to the object.  Results are deterministic.
    """

    def __init__(self, B: int, R: int, heads: int, kv_heads: int, head_dim: int, capacity: int, device, *,
                 window: int = 0, sinks: int = 0, prefix: int = 0, scored: bool = False, scale: float | None = None):
        self.B, self.R, self.heads, self.kv_heads, self.head_dim = B, R, heads, kv_heads, head_dim
        self.capacity, self.window, self.sinks, self.prefix, self.scored = capacity, window, sinks, prefix, bool(scored)
        self.device = torch.device(device)
        self.scale = float(head_dim ** -0.5 if scale is None else scale)
        self._shape = AttnShape(B, R, heads, kv_heads, head_dim, capacity, window, sinks, prefix, int(self.scored))
        lib = _lib.load()
        _lib.check(lib.krk_attn_check(_byref(self._shape)))
        nbytes = int(lib.krk_attn_workspace_bytes(_byref(self._shape)))
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None

    @property
    def plan(self) -> dict:
        """How the library cuts this shape's work (``krk_attn_plan_t``)."""
        out = AttnPlan()
        _lib.check(_lib.load().krk_attn_plan(_byref(self._shape), _byref(out)))
        return out.as_dict()

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor, out: torch.Tensor, *,
            prefix: tuple | None = None, tree: torch.Tensor | None = None, scores: torch.Tensor | None = None,
            scores_out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
        """Allocation-free form: write into ``out`` (``[B * R, heads *
        head_dim]``), and with ``lse`` (``[B * R, heads]`` fp32) the log of each
        softmax's sum."""
        B, M, KV, D, cap = self.B, self.B * self.R, self.kv_heads, self.head_dim, self.capacity
        index = _index("q", q)
        a = AttnArgs()
        a.q, a.q_row = _rows("q", q, index, M, self.heads * D)
        a.out, a.out_row = _rows("out", out, index, M, self.heads * D)
        a.k = _cache("k", k, index, B, cap, KV, D)
        a.v = _cache("v", v, index, B, cap, KV, D)
        a.lens = _plain("lens", lens, index, torch.int32, (B,))
        a.scale = self.scale
        if prefix is not None:
            kp, vp = prefix
            if not isinstance(kp, torch.Tensor) or kp.dim() != 3:
                raise ValueError("prefix must be a pair of [keys, kv_heads, head_dim] tensors")
            n = kp.shape[0]
            if n > self.prefix:
                raise ValueError(f"a prefix of {n} keys; this object was built for up to {self.prefix}")
            if n:
                a.kp = _cache("prefix k", kp, index, None, n, KV, D)
            _on(index, "prefix v", vp)
            if n or vp.shape != kp.shape:
                a.vp = _cache("prefix v", vp, index, None, n, KV, D)
            a.prefix = n
        if tree is not None:
            a.tree = _plain("tree", tree, index, torch.int64, (B, self.R))
        if lse is not None:
            a.lse = _plain("lse", lse, index, torch.float32, (M, self.heads))
        if self.scored:
            if scores is None:
                raise ValueError("this object updates scores: give scores=")
            a.scores, a.sc_seq, a.sc_head = _scores("scores", scores, index, B, KV, cap)
            if scores_out is None:
                a.scores_out, a.so_seq, a.so_head = a.scores, a.sc_seq, a.sc_head
            else:
                a.scores_out, a.so_seq, a.so_head = _scores("scores_out", scores_out, index, B, KV, cap)
        elif scores is not None or scores_out is not None:
            raise ValueError("scores are kept by objects built with scored=True")
        ws = self.workspace
        if ws is None:
            _launch(_lib.load().krk_attn_bf16, index, _byref(self._shape), _byref(a), 0, 0)
        else:
            if ws.get_device() != index:
                raise ValueError(f"operands on {q.device}; this object was built on {self.device}")
            _launch(_lib.load().krk_attn_bf16, index, _byref(self._shape), _byref(a), ws.data_ptr(), ws.numel())
        return out

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor, *,
                 prefix: tuple | None = None, tree: torch.Tensor | None = None, scores: torch.Tensor | None = None,
                 scores_out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
        """``out = softmax(scale * q k^T) v`` as a new ``[B * R, heads *
        head_dim]`` tensor.

        ``q`` ``[B * R, heads * head_dim]`` may be the first columns of the qkv
        rows.  ``prefix=(kp, vp)``: the shared keys and values, ``[keys,
        kv_heads, head_dim]``.  ``tree`` (int64 ``[B, R]``, R <= 64): bit j of
        row i says whether the row sees the call's own row j; its position is
        then that of the first row plus its set bits less one.  ``scores``
        (``[B, kv_heads, capacity]`` fp32): each cached key's weight, summed over
        rows and the query heads of its group, is added; into ``scores_out``
        where given (slots below ``lens``)."""
        _index("q", q)
        out = torch.empty((self.B * self.R, self.heads * self.head_dim), dtype=_BF16, device=q.device)
        return self.run(q, k, v, lens, out, prefix=prefix, tree=tree, scores=scores, scores_out=scores_out, lse=lse)


class CacheEviction:
    """Cuts a cache down to ``budget`` slots per sequence and head by the keys'
    scores, for a fixed shape.

    Where a sequence has more than ``budget`` keys, its first ``sinks`` and last
    ``recent`` slots stay, and of the others those with the highest scores
    (equal scores: the lower slot first; NaN counts as the highest).  Kept slots
    keep their order and become slots 0, 1, ...
    """

    def __init__(self, B: int, kv_heads: int, head_dim: int, capacity: int, budget: int, device, *, sinks: int = 0,
                 recent: int = 0):
        if not 1 <= budget <= capacity:
            raise ValueError(f"budget={budget} must be 1 .. capacity={capacity}")
        if sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"sinks={sinks} and recent={recent} must be >= 0 and together at most budget={budget}")
        if B < 1 or kv_heads < 1 or head_dim not in (64, 128):
            raise ValueError(f"B={B} and kv_heads={kv_heads} must be >= 1 and head_dim={head_dim} 64 or 128")
        self.B, self.kv_heads, self.head_dim, self.capacity, self.budget = B, kv_heads, head_dim, capacity, budget
        self.sinks, self.recent = sinks, recent
        self.device = torch.device(device)

    def run(self, k: torch.Tensor, v: torch.Tensor, scores: torch.Tensor, lens: torch.Tensor, keep: torch.Tensor,
            lens_out: torch.Tensor, out: tuple | None = None) -> torch.Tensor:
        """Allocation-free form: the kept slots into ``keep`` (int32 ``[B,
        kv_heads, budget]``, ascending, -1 behind the last), the new lengths into
        ``lens_out`` (which may be ``lens``).  ``out=(k, v, scores)`` receives the
        kept rows (at least ``budget`` slots each; what lies behind them is left
        as it was); without it the cache is compacted in place."""
        B, KV, D, cap = self.B, self.kv_heads, self.head_dim, self.capacity
        index = _index("k", k)
        a = EvictArgs()
        a.k = _cache("k", k, index, B, cap, KV, D)
        a.v = _cache("v", v, index, B, cap, KV, D)
        a.scores, a.sc_seq, a.sc_head = _scores("scores", scores, index, B, KV, cap)
        if out is None:
            a.k_out, a.v_out = a.k, a.v
            a.scores_out, a.so_seq, a.so_head = a.scores, a.sc_seq, a.sc_head
        else:
            ko, vo, so = out
            a.k_out = _cache("out k", ko, index, B, None, KV, D)
            a.v_out = _cache("out v", vo, index, B, None, KV, D)
            if min(ko.shape[1], vo.shape[1]) < self.budget:
                raise ValueError(f"out k and v must have at least {self.budget} slots, got {ko.shape[1]} and {vo.shape[1]}")
            a.scores_out, a.so_seq, a.so_head = _scores("out scores", so, index, B, KV, self.budget, more=True)
        a.lens = _plain("lens", lens, index, torch.int32, (B,))
        a.lens_out = _plain("lens_out", lens_out, index, torch.int32, (B,))
        a.keep = _plain("keep", keep, index, torch.int32, (B, KV, self.budget))
        a.B, a.kv_heads, a.head_dim, a.capacity = B, KV, D, cap
        a.budget, a.sinks, a.recent = self.budget, self.sinks, self.recent
        _launch(_lib.load().krk_cache_evict_bf16, index, _byref(a))
        return keep

    def __call__(self, k: torch.Tensor, v: torch.Tensor, scores: torch.Tensor, lens: torch.Tensor,
                 out: tuple | None = None) -> tuple:
        """``(keep, new lens)`` as new tensors (:meth:`run`)."""
        _index("k", k)
        dev = k.device
        keep = torch.empty((self.B, self.kv_heads, self.budget), dtype=torch.int32, device=dev)
        lens_out = torch.empty((self.B,), dtype=torch.int32, device=dev)
        self.run(k, v, scores, lens, keep, lens_out, out)
        return keep, lens_out
