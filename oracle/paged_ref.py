"""64-bit oracle of the paged cache and of low-rank adapters (TEST INFRASTRUCTURE
ONLY): page tables one request at a time in plain Python, attention through
:mod:`oracle.attn_ref` over each request's gathered pages, adapters from their
definition, with the bounds that the tests hold the kernels to."""

from __future__ import annotations

import torch

from . import attn_ref as A64
from .attn_ref import BF16_HALF, FP32_HALF

F64 = torch.float64


class Tables:
    """Page tables as lists of ints: the state of ``PageTables`` and its step."""

    def __init__(self, B, rows, pages, page_size, width, managed=True):
        self.B, self.rows, self.pages, self.P, self.width, self.managed = B, rows, pages, page_size, width, managed
        self.lens = [0] * B
        self.table = [[0] * width for _ in range(B)]
        self.free = list(range(pages - 1, -1, -1))
        self.count = pages

    def _need(self, n):
        return -(-n // self.P)

    def step(self, new, keep=None, labels=None):
        full = self.width * self.P
        old = [min(max(n, 0), full) for n in self.lens]
        cut = [n if keep is None else min(n, max(keep[b], 0)) for b, n in enumerate(old)]
        back = [self.table[b][i] for b in range(self.B) for i in range(self._need(cut[b]), self._need(old[b]))]
        if self.managed:
            for page in reversed(back):
                self.free[self.count] = page
                self.count += 1
        top, at, wanted = self.count, 0, 0
        self.starts, self.keys, self.slots, self.positions, self.owner = [0], [], [], [], []
        for b in range(self.B):
            n = max(new[b], 0)
            fits = n > 0 and at + n <= self.rows and cut[b] + n <= full
            need = self._need(cut[b] + n) - self._need(cut[b]) if fits and self.managed else 0
            wanted += need
            ok = fits and (need == 0 or wanted <= top)
            if ok:
                for i in range(need):
                    self.count -= 1
                    self.table[b][self._need(cut[b]) + i] = self.free[self.count]
            for i in range(n):
                if at + i >= self.rows:
                    break
                pos = cut[b] + i
                page = self.table[b][pos // self.P] if ok else -1
                live = 0 <= page < self.pages
                self.slots.append(page * self.P + pos % self.P if live else -1)
                self.positions.append(pos if live else -1)
                self.owner.append((b if labels is None else labels[b]) if live else -1)
            at += n
            self.starts.append(min(at, self.rows))
            self.lens[b] = cut[b] + n if ok else cut[b]
            self.keys.append(self.lens[b] if ok or n == 0 else 0)
        for rest in (self.slots, self.positions, self.owner):
            rest += [-1] * (self.rows - len(rest))


def gather(pool, table_row, n, P):
    """The first n keys of a request, [n, heads, D], from a [pages, P, heads, D] pool (bad entries: the pool's last page)."""
    at = torch.arange(n)
    ids = torch.as_tensor(table_row)[at // P].long()
    ids = torch.where((ids < 0) | (ids >= pool.shape[0]), pool.shape[0] - 1, ids)
    return pool[ids, at % P]


def attention(q, k, v, table, starts, keys, *, heads, window=0, sinks=0, scale=None):
    """(out [rows, heads, D], lse [rows, heads], tolerance of both) in 64 bits; rows of no
    request are NaN in ``out`` and the tolerances."""
    rows, P, KV, D = q.shape[0], k.shape[1], k.shape[2], k.shape[3]
    G = heads // KV
    out = torch.full((rows, heads, D), float("nan"), dtype=F64)
    lse = torch.full((rows, heads), float("nan"), dtype=F64)
    tol, ltol = out.clone(), lse.clone()
    full = len(table[0]) * P
    for b, (s, e) in enumerate(zip(starts, starts[1:])):
        n, L = e - s, min(max(keys[b], 0), full)
        if n == 0:
            continue
        kk, vv = (gather(t, table[b], max(L, 1), P)[None] for t in (k, v))
        o, l, _, size, top = A64.attention(q[s:e], kk, vv, [L], heads=heads, R=n, window=window, sinks=sinks, scale=scale)
        half = 2.0 ** -8 if n * G > 64 else 2.0 ** -16
        out[s:e], lse[s:e] = o[0], l[0]
        tol[s:e] = A64.attention_tolerance(o, size, top, D, L, half)[0]
        ltol[s:e] = (A64.score_error(top, D) + (L + 32) * FP32_HALF + 4 * FP32_HALF * torch.where(l.isfinite(), l.abs(), 0))[0]
    return out, lse, tol, ltol


def adapters(x, a, b, index, y, scale, widths, rank, silu=False):
    """(out, tolerance) in 64 bits.  The bound counts: fp32 sums over K, products x A^T in
    two bf16 parts (2^-16), fp32 sums over 2 * rank products and with y, and one rounding
    to bf16; silu: (|gate| + 8) roundings of its exponential and quotient."""
    x, a, b, y = (t.detach().cpu().to(F64) for t in (x, a, b, y))
    K = x.shape[1]
    out, err = y.clone(), FP32_HALF * y.abs()
    for m, i in enumerate(index.tolist()):
        if not 0 <= i < a.shape[0]:
            continue
        f = 1.0 if scale is None else float(scale[i])
        col = 0
        for s, w in enumerate(widths):
            ai, bi = a[i, s * rank:(s + 1) * rank], b[i, col:col + w]
            h, size = ai @ x[m], ai.abs() @ x[m].abs()
            off = (K + 16) * FP32_HALF * size + (2.0 ** -16 + 2 * FP32_HALF) * h.abs()
            out[m, col:col + w] += f * (bi @ h)
            err[m, col:col + w] += abs(f) * (bi.abs() @ (off + (2 * rank + 4) * FP32_HALF * (h.abs() + off)))
            err[m, col:col + w] += FP32_HALF * out[m, col:col + w].abs()
            col += w
    if silu:
        half = out.shape[1] // 2
        g, u, eg, eu = out[:, :half], out[:, half:], err[:, :half], err[:, half:]
        s = g * torch.sigmoid(g)
        out = s * u
        err = 1.1 * eg * (u.abs() + eu) + s.abs() * eu + (g.abs() + 8) * FP32_HALF * out.abs()
    return out, BF16_HALF * (out.abs() + err) + err + 1e-38
