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
stream.  Building an object waits until its workspace is filled (and is refused
while a graph is captured), so its first call may come on any stream; a graph that
holds its calls needs the object as long as it is replayed.  All compute runs in libkrk_attn.so; there is no fallback.
"""

from __future__ import annotations

import ctypes

import torch

from . import _attn_lib as _lib
from ._attn_lib import AttnArgs, AttnPlan, AttnShape, EvictArgs, RopeArgs

__all__ = ["CacheAttention", "CacheEviction", "qk_norm_rope", "rope_table", "workspace_bytes"]

_BF16 = torch.bfloat16
_byref = ctypes.byref
_PACK_ATTN, _PACK_ROPE, _PACK_EVICT = (_lib.PACK[t] for t in (AttnArgs, RopeArgs, EvictArgs))


# One eager call of a decode step's operators is bound by the host (their
# kernels take 3-10 us at one row): each property of an operand is read once,
# in one expression that a good operand passes, and only one that fails it is
# looked at again for the message.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice
_NO_CACHE = (0, 0, 0, 0)


def _ints(**sizes) -> None:
    """Sizes that fit the structs' ints (which would take others modulo 2^32)."""
    for name, n in sizes.items():
        if not isinstance(n, int) or not -1 << 31 <= n < 1 << 31:
            raise ValueError(f"{name} must be an int of 32 bits, got {n!r}")


def _launch(fn, index: int, *args) -> None:
    """``fn(*args, stream)`` on GPU ``index`` and torch's current stream there."""
    stream = _raw_stream(index)
    if _current() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _index(name: str, t: torch.Tensor) -> int:
    """The GPU that a call's first operand is on."""
    if isinstance(t, torch.Tensor):
        index = t.get_device()
        if index >= 0 and t.is_cuda:
            return index
        raise ValueError(f"{name} must be a GPU tensor, got device {t.device}")
    raise ValueError(f"{name} must be a torch.Tensor")


def _refuse(name: str, t, index: int, dtype: torch.dtype, shape: tuple, layout: str):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.get_device() != index or not t.is_cuda:
        raise ValueError(f"{name} must be on the operands' GPU, got {t.device}")
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    raise ValueError(f"{name}: {layout}, got strides {t.stride()}")


def _cache(name: str, t: torch.Tensor, index: int, shape: tuple) -> tuple:
    """The fields of ``krk_cache`` for a [sequences, slots, kv_heads, head_dim] tensor."""
    if isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.shape == shape and t.get_device() == index:
        seq, slot, head, one = t.stride()
        if one == 1:
            return t.data_ptr(), seq, slot, head
    _refuse(name, t, index, _BF16, shape, "the elements of a head must be contiguous")


def _prefix(name: str, t: torch.Tensor, index: int, shape: tuple) -> tuple:
    """The same for a [keys, kv_heads, head_dim] tensor."""
    if isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.shape == shape and t.get_device() == index:
        slot, head, one = t.stride()
        if one == 1:
            return t.data_ptr(), 0, slot, head
    _refuse(name, t, index, _BF16, shape, "the elements of a head must be contiguous")


def _rows(name: str, t: torch.Tensor, index: int, shape: tuple) -> tuple:
    """Address and row stride of a [rows, columns] bf16 tensor."""
    if isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.shape == shape and t.get_device() == index:
        row, one = t.stride()
        if one == 1:
            return t.data_ptr(), row
    _refuse(name, t, index, _BF16, shape, "rows must be contiguous")


def _plain(name: str, t: torch.Tensor, index: int, dtype: torch.dtype, shape: tuple) -> int:
    """The address of a contiguous tensor of this type and shape."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index
            and t.is_contiguous()):
        return t.data_ptr()
    _refuse(name, t, index, dtype, shape, "it must be contiguous")


def _scores(name: str, t: torch.Tensor, index: int, shape: tuple, more: bool = False) -> tuple:
    """Address and strides of [sequences, heads, slots] scores (``more``: or more slots)."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.get_device() == index and t.dim() == 3:
        if t.shape == shape or more and t.shape[:2] == shape[:2] and t.shape[2] > shape[2]:
            seq, head, one = t.stride()
            if one == 1 or t.shape[2] == 1:
                return t.data_ptr(), seq, head
    _refuse(name, t, index, torch.float32, shape, "the scores of a head must be contiguous")


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
    if not 0.0 <= eps <= 3e38:
        raise ValueError(f"eps={eps} must be finite and >= 0")
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be a [B, capacity, kv_heads, head_dim] tensor")
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a [positions, head_dim] tensor")
    shape = k.shape
    B, cap, KV, D = shape
    if qkv.dim() != 2 or B < 1 or D < 1 or qkv.shape[0] < 1 or qkv.shape[0] % B or qkv.shape[1] % D:
        raise ValueError(f"qkv must be [B * R, (heads + 2 * kv_heads) * head_dim] for a cache of shape {tuple(shape)}, "
                         f"got {tuple(qkv.shape)}")
    M, cols = qkv.shape
    heads = cols // D - 2 * KV
    if heads < 1:
        raise ValueError(f"qkv of {cols} columns has no q heads beside {KV} k and {KV} v heads of {D}")
    if q_out is None:
        q_out = qkv.new_empty((M, heads * D))
    x, x_row = _rows("qkv", qkv, index, (M, cols))
    q, q_row = _rows("q_out", q_out, index, (M, heads * D))
    n = table.shape[0]
    args = _PACK_ROPE(
        x, x_row,
        0 if q_norm is None else _plain("q_norm", q_norm, index, _BF16, (D,)),
        0 if k_norm is None else _plain("k_norm", k_norm, index, _BF16, (D,)),
        eps, _plain("table", table, index, torch.float32, (n, D)), n,
        0 if positions is None else _plain("positions", positions, index, torch.int32, (M,)),
        _plain("lens", lens, index, torch.int32, (B,)), q, q_row,
        *_cache("k", k, index, shape), *_cache("v", v, index, shape), B, M // B, heads, KV, D, cap)
    _launch(_lib.load().krk_qk_norm_rope_bf16, index, args)
    return q_out


def _attn_shape(B, R, heads, kv_heads, head_dim, capacity, window, sinks, prefix, scored) -> AttnShape:
    """The library's description of a shape that it takes (ValueError for others)."""
    _ints(B=B, R=R, heads=heads, kv_heads=kv_heads, head_dim=head_dim, capacity=capacity, window=window, sinks=sinks,
          prefix=prefix)
    shape = AttnShape(B, R, heads, kv_heads, head_dim, capacity, window, sinks, prefix, int(bool(scored)))
    _lib.check(_lib.load().krk_attn_check(_byref(shape)))
    return shape


def workspace_bytes(B: int, R: int, heads: int, kv_heads: int, head_dim: int, capacity: int, *, window: int = 0,
                    sinks: int = 0, prefix: int = 0, scored: bool = False) -> int:
    """Bytes of workspace that a :class:`CacheAttention` of this shape needs."""
    shape = _attn_shape(B, R, heads, kv_heads, head_dim, capacity, window, sinks, prefix, scored)
    return int(_lib.load().krk_attn_workspace_bytes(_byref(shape)))


def filled(device: torch.device) -> None:
    """Wait for the current stream, on which memory of an object was just filled:
    its calls may come on any other."""
    if device.type == "cuda":
        torch.cuda.current_stream(device).synchronize()


def zero_workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Zero-filled memory, ready for calls on every stream when this returns."""
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a workspace is filled when its object is built: build it before the capture")
    ws = torch.zeros(nbytes, dtype=torch.uint8, device=device)
    filled(device)
    return ws


class CacheAttention:
    """Attention of ``R`` new rows of each of ``B`` sequences over their cache,
    for a fixed shape: ``f(q, k, v, lens) -> out``.

    Query head h reads key/value head ``h // (heads // kv_heads)``.  The row at
    position p sees every key up to itself; with ``window`` the ``window`` last
    of them, and the first ``sinks`` positions as well.  ``prefix`` is the most
    keys of a prefix that all sequences share; the cache's slot s then has
    position ``prefix keys + s``.  ``scored`` objects update their keys' scores.
    ``scale`` is ``head_dim ** -0.5`` unless given.

    The workspace (:func:`workspace_bytes`) belongs to the object, or is
    ``workspace``: zero-filled uint8 memory that objects of one B and kv_heads may
    share if all their calls are ordered on one stream.  A scored object without a
    window keeps q.k there for up to 16 rows a key/value head: ``4 * B * R * heads
    * capacity`` bytes.  Results are deterministic.
    """

    def __init__(self, B: int, R: int, heads: int, kv_heads: int, head_dim: int, capacity: int, device, *,
                 window: int = 0, sinks: int = 0, prefix: int = 0, scored: bool = False, scale: float | None = None,
                 workspace: torch.Tensor | None = None):
        self._shape = _attn_shape(B, R, heads, kv_heads, head_dim, capacity, window, sinks, prefix, scored)
        if scale is not None and not 1e-45 < scale <= 2.3e38:  # as an fp32, and times log2(e)
            raise ValueError(f"scale={scale} must be positive and at most 2.3e38")
        self.B, self.R, self.heads, self.kv_heads, self.head_dim = B, R, heads, kv_heads, head_dim
        self.capacity, self.window, self.sinks, self.prefix, self.scored = capacity, window, sinks, prefix, bool(scored)
        self.device = torch.device(device)
        self.scale = float(head_dim ** -0.5 if scale is None else scale)
        nbytes = int(_lib.load().krk_attn_workspace_bytes(_byref(self._shape)))
        self._q_shape = (B * R, heads * head_dim)
        self._cache_shape = (B, capacity, kv_heads, head_dim)
        if workspace is None:
            workspace = zero_workspace(nbytes, self.device) if nbytes else None
        elif workspace.dtype is not torch.uint8 or workspace.numel() < nbytes or not workspace.is_contiguous():
            raise ValueError(f"workspace must be {nbytes} contiguous bytes (uint8) or more, got {workspace.dtype} {tuple(workspace.shape)}")
        elif workspace.device.type != self.device.type or self.device.index not in (None, workspace.device.index):
            raise ValueError(f"workspace on {workspace.device}; this object is built on {self.device}")
        self.workspace = workspace
        self._streams: set = set()  # whose work the workspace outlives

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
        index = _index("q", q)
        B, shape = self.B, self._cache_shape
        kp = vp = _NO_CACHE
        n = 0
        if prefix is not None:
            kp, vp = prefix
            if not isinstance(kp, torch.Tensor) or kp.dim() != 3:
                raise ValueError("prefix must be a pair of [keys, kv_heads, head_dim] tensors")
            n = kp.shape[0]
            if n > self.prefix:
                raise ValueError(f"a prefix of {n} keys; this object was built for up to {self.prefix}")
            run = (n, self.kv_heads, self.head_dim)
            kp, vp = _prefix("prefix k", kp, index, run), _prefix("prefix v", vp, index, run)
        sc = so = (0, 0, 0)
        if self.scored:
            if scores is None:
                raise ValueError("this object updates scores: give scores=")
            run = (B, self.kv_heads, self.capacity)
            sc = so = _scores("scores", scores, index, run)
            if scores_out is not None:
                so = _scores("scores_out", scores_out, index, run)
        elif scores is not None or scores_out is not None:
            raise ValueError("scores are kept by objects built with scored=True")
        args = _PACK_ATTN(
            *_rows("q", q, index, self._q_shape), *_cache("k", k, index, shape), *_cache("v", v, index, shape),
            *kp, *vp, n, self.scale, _plain("lens", lens, index, torch.int32, (B,)),
            0 if tree is None else _plain("tree", tree, index, torch.int64, (B, self.R)),
            *_rows("out", out, index, self._q_shape),
            0 if lse is None else _plain("lse", lse, index, torch.float32, (B * self.R, self.heads)), *sc, *so)
        ws = self.workspace
        if ws is None:
            _launch(_lib.load().krk_attn_bf16, index, _byref(self._shape), args, 0, 0)
        elif ws.get_device() == index:
            if _raw_stream(index) not in self._streams:
                self._outlive(index)
            _launch(_lib.load().krk_attn_bf16, index, _byref(self._shape), args, ws.data_ptr(), ws.numel())
        else:
            raise ValueError(f"operands on {q.device}; this object was built on {self.device}")
        return out

    def _outlive(self, index: int) -> None:
        """The workspace's memory is not given to others before the current
        stream is through with it, also where the object goes first.  (Of a
        captured graph only its owner knows when it runs last.)"""
        if not torch.cuda.is_current_stream_capturing():
            self.workspace.record_stream(torch.cuda.current_stream(index))
            self._streams.add(_raw_stream(index))

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor, *,
                 prefix: tuple | None = None, tree: torch.Tensor | None = None, scores: torch.Tensor | None = None,
                 scores_out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
        """``out = softmax(scale * q k^T) v`` as a new ``[B * R, heads *
        head_dim]`` tensor.

        ``q`` ``[B * R, heads * head_dim]`` may be the first columns of the qkv
        rows.  ``prefix=(kp, vp)``: the shared keys and values, ``[keys,
        kv_heads, head_dim]``.  ``tree`` (int64 ``[B, R]``, R <= 64): bit j of
        row i says whether the row sees the call's own row j; its position is
        then that of the sequence's first row plus its set bits less one.  ``scores``
        (``[B, kv_heads, capacity]`` fp32): each cached key's weight, summed over
        rows and the query heads of its group, is added; into ``scores_out``
        where given (slots below ``lens``)."""
        _index("q", q)
        out = torch.empty(self._q_shape, dtype=_BF16, device=q.device)
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
        _ints(B=B, kv_heads=kv_heads, head_dim=head_dim, capacity=capacity, budget=budget, sinks=sinks, recent=recent)
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
        index = _index("k", k)
        B, KV, D, cap, n = self.B, self.kv_heads, self.head_dim, self.capacity, self.budget
        shape, run = (B, cap, KV, D), (B, KV, cap)
        kc, vc, sc = _cache("k", k, index, shape), _cache("v", v, index, shape), _scores("scores", scores, index, run)
        if out is None:
            ko, vo, so = kc, vc, sc
        else:
            ko, vo, so = out
            for name, t in (("out k", ko), ("out v", vo)):
                if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[1] < n:
                    raise ValueError(f"{name} must be a [{B}, {n} or more, {KV}, {D}] tensor")
            ko = _cache("out k", ko, index, (B, ko.shape[1], KV, D))
            vo = _cache("out v", vo, index, (B, vo.shape[1], KV, D))
            so = _scores("out scores", so, index, (B, KV, n), more=True)
        args = _PACK_EVICT(
            *kc, *vc, *ko, *vo, *sc, *so, _plain("lens", lens, index, torch.int32, (B,)),
            _plain("lens_out", lens_out, index, torch.int32, (B,)), _plain("keep", keep, index, torch.int32, (B, KV, n)),
            B, KV, D, cap, n, self.sinks, self.recent)
        _launch(_lib.load().krk_cache_evict_bf16, index, args)
        return keep

    def __call__(self, k: torch.Tensor, v: torch.Tensor, scores: torch.Tensor, lens: torch.Tensor,
                 out: tuple | None = None) -> tuple:
        """``(keep, new lens)`` as new tensors (:meth:`run`)."""
        _index("lens", lens)
        keep, lens_out = lens.new_empty((self.B, self.kv_heads, self.budget)), lens.new_empty((self.B,))
        self.run(k, v, scores, lens, keep, lens_out, out)
        return keep, lens_out
