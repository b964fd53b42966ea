"""64-bit oracle of the cache operators (TEST INFRASTRUCTURE ONLY): rotary
embedding, cache attention and eviction from their definitions, one sequence
and head at a time, with the bounds that the tests hold the kernels to."""

from __future__ import annotations

import math

import torch

F64 = torch.float64
BF16_HALF = 2.0 ** -8   # half a step of bf16, relative
FP32_HALF = 2.0 ** -24  # half a step of fp32, relative


def visible(prefix: int, length: int, R: int, window: int, sinks: int, tree=None) -> torch.Tensor:
    """[R, prefix + length] booleans of one sequence (tree: its R ints)."""
    n = prefix + length
    seen = torch.zeros((R, n), dtype=torch.bool)
    first = n - R
    for i in range(R):
        if length - R + i < 0:
            continue
        if tree is None:
            pos, own = first + i, set()
            top = pos
        else:  # of the call's own rows, those that have a slot
            own = {first + j for j in range(R) if tree[i] >> j & 1 and length - R + j >= 0}
            cached = prefix + max(0, length - R)
            pos, top = cached + len(own) - 1, cached - 1
        for t in range(n):
            near = t <= top and (window == 0 or t > pos - window or t < sinks)
            seen[i, t] = near or t in own
    return seen


def attention(q, k, v, lens, *, heads, R, window=0, sinks=0, prefix=None, tree=None, scale=None, seen=None):
    """(out, lse, weights, size, top) in 64 bits on the CPU: ``out`` [B, R, heads, D],
    ``lse`` [B, R, heads], ``weights`` [B, kv_heads, capacity] (summed over rows
    and the group), ``size`` = sum of p |v| per output, ``top`` [B, R, heads] the
    largest sum of scale |q_d k_d| among visible keys (for error bounds)."""
    B, cap, KV, D = k.shape
    G = heads // KV
    scale = D ** -0.5 if scale is None else scale
    q = q.detach().cpu().to(F64).view(B, R, heads, D)
    k, v = k.detach().cpu(), v.detach().cpu()
    P = 0 if prefix is None else prefix[0].shape[0]
    out, size = torch.zeros((B, R, heads, D), dtype=F64), torch.zeros((B, R, heads, D), dtype=F64)
    lse = torch.full((B, R, heads), -math.inf, dtype=F64)
    top = torch.zeros((B, R, heads), dtype=F64)
    weights = torch.zeros((B, KV, cap), dtype=F64)
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        sight = visible(P, n, R, window, sinks, None if tree is None else [int(x) & (1 << 64) - 1 for x in tree[b]])
        for h in range(KV):
            kk, vv = k[b, :n, h].to(F64), v[b, :n, h].to(F64)
            if P:
                kk = torch.cat([prefix[0][:, h].cpu().to(F64), kk])
                vv = torch.cat([prefix[1][:, h].cpu().to(F64), vv])
            for i in range(R):
                at = sight[i].nonzero()[:, 0]
                if len(at) == 0:
                    continue
                x = kk[at] @ q[b, i, h * G:(h + 1) * G].T * scale  # keys x G
                m = x.max(dim=0).values
                e = (x - m).exp()
                l = e.sum(dim=0)
                p = e / l
                out[b, i, h * G:(h + 1) * G] = p.T @ vv[at]
                size[b, i, h * G:(h + 1) * G] = p.T @ vv[at].abs()
                lse[b, i, h * G:(h + 1) * G] = m + l.log()
                top[b, i, h * G:(h + 1) * G] = (kk[at].abs() @ q[b, i, h * G:(h + 1) * G].abs().T * scale).max(dim=0).values
                own = at >= P
                weights[b, h].index_add_(0, at[own] - P, p[own].sum(dim=1))
    return out, lse, weights, size, top


def score_error(top, D):
    """How far a score may be off: D products of exact bf16 operands summed in
    fp32 (each partial sum at most `top`), scaled, and its distance from the
    maximum taken and multiplied once more (4 further roundings)."""
    return (D + 8) * FP32_HALF * (top + 1)


def attention_tolerance(out, size, top, D, keys, weight_half):
    """Bound on |kernel - out|: the rounding to bf16; the weights' own rounding
    (``weight_half`` relative: 2^-16 where they are carried in two bf16 parts,
    2^-8 in one); each weight's error from its score (numerator and sum, so
    twice) and from exp2 (2 units); fp32 sums over `keys` terms."""
    rel = weight_half + 2 * score_error(top, D) + (2 * keys + 16) * FP32_HALF
    return BF16_HALF * out.abs() * (1 + rel.unsqueeze(-1)) + size * rel.unsqueeze(-1) * 1.01 + 1e-38


def rope(qkv, q_norm, k_norm, eps, theta, positions, heads, kv_heads, D):
    """(q, k, v) in 64 bits: [M, heads, D], [M, kv_heads, D], [M, kv_heads, D]."""
    M = qkv.shape[0]
    x = qkv.detach().cpu().to(F64).view(M, heads + 2 * kv_heads, D)
    freq = theta ** (-torch.arange(0, D, 2, dtype=F64) / D)
    ang = positions.cpu().to(F64)[:, None, None] * freq
    cos, sin = ang.cos(), ang.sin()

    def turn(y, gain):
        if gain is not None:
            y = y / (y.square().mean(dim=-1, keepdim=True) + eps).sqrt() * gain.detach().cpu().to(F64)
        a, b = y[..., :D // 2], y[..., D // 2:]
        size = torch.cat([(a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()], dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1), size

    return turn(x[:, :heads], q_norm), turn(x[:, heads:heads + kv_heads], k_norm), x[:, heads + kv_heads:]


def evict(scores, lens, budget, sinks, recent):
    """Kept slots per sequence and head, ascending (lists of ints)."""
    B, KV, cap = scores.shape
    s = scores.detach().cpu()

    def rank(x):  # NaN above +inf, -0 equal to +0
        return (1, 0.0) if math.isnan(x) else (0, x + 0.0)

    kept = []
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        row = []
        for h in range(KV):
            if n <= budget:
                row.append(list(range(n)))
                continue
            stay = set(range(sinks)) | set(range(n - recent, n))
            rest = [i for i in range(n) if i not in stay]
            vals = s[b, h].tolist()
            rest.sort(key=lambda i: (tuple(-c for c in rank(vals[i])), i))
            row.append(sorted(stay | set(rest[:budget - sinks - recent])))
        kept.append(row)
    return kept
