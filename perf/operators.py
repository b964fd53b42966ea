"""Performance cases of the key/value cache operators of a decode step.

Each case is one pass through one operator, as a serving loop calls it between
the qkv projection and the o projection (head layouts: Qwen3-4B's 32 query and
8 key/value heads of 128, its tensor-parallel shards, and a few generic ones).

Kinds:

* ``rope``    per-head RMSNorm of q and k, rotary embedding, and the new rows'
              k and v written into the cache.
* ``attn``    attention of R new rows of each of B sequences over their cache:
              causal, with a sliding window behind which a few first tokens
              (sinks) stay visible, or with the ancestor masks of a draft tree.
* ``prefix``  the same for a batch whose sequences share one long prefix, kept
              once.
* ``scored``  attention that also adds each cached key's attention weight,
              summed over rows and query heads of its group, to its score.
* ``evict``   the cache cut down to a budget of slots per head: first tokens
              and most recent ones stay, and of the rest the highest scores.

Sequence b of a case has ``len - (b * 7919) % (spread + 1)`` cached keys, the
call's own rows among them.  Cases are plain numbers; every tensor comes from
the seed.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False  # True: the framework's kernels; False: the plain forms

DEV = "cuda:0"
BF16 = torch.bfloat16
EPS = 1e-6
THETA = 1e6
_PKG = str(Path(__file__).resolve().parent.parent / "kernel-rush-kawk_amd")


def _kernels():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from kernels import attention

    return attention


# ------------------------------------------------------------------ cases
def _case(kind, B, R, len_, heads=32, kv_heads=8, dim=128, spread=0, window=0, sinks=0, prefix=0, tree=False, budget=0,
          recent=0):
    return {"kind": kind, "B": B, "R": R, "len": len_, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "spread": spread, "window": window, "sinks": sinks, "prefix": prefix, "tree": tree, "budget": budget,
            "recent": recent}


def listed():
    named = {
        # One sequence's decode step: one new row.
        "rope_b1": _case("rope", 1, 1, 1000),
        # A prompt batch of 4 x 2048 rows filling its cache.
        "rope_prompt": _case("rope", 4, 2048, 2048),
        # One sequence's decode step over a short chat: latency.
        "decode_b1": _case("attn", 1, 1, 1000),
        # A ragged batch deep into long documents, window of 4096 behind 4 sinks.
        "decode_window_b32": _case("attn", 32, 1, 32000, spread=30000, window=4096, sinks=4),
        # Verification of 4 sequences' draft trees of 16 nodes.
        "tree_b4": _case("attn", 4, 16, 2011, spread=700, tree=True),
        # A long prompt with a sliding window.
        "prompt_window": _case("attn", 1, 8192, 8192, window=2048, sinks=4),
        # 16 chats under one system prompt.
        "prefix_b16": _case("prefix", 16, 1, 300, spread=250, prefix=2000),
        # 64 questions over one long document.
        "prefix_b64": _case("prefix", 64, 1, 1000, spread=900, prefix=32768),
        # Decode that keeps the keys' scores.
        "scored_b8": _case("scored", 8, 1, 8000, spread=3000),
        # The last 32 rows of a prompt score its keys before it is cut down.
        "scored_prompt_tail": _case("scored", 2, 32, 16000, spread=1),
        # One short cache cut in half.
        "evict_b1": _case("evict", 1, 1, 1024, budget=512, sinks=4, recent=64),
        # A batch of long prompts cut down to 4096 slots.
        "evict_b8": _case("evict", 8, 1, 32768, spread=9000, budget=4096, sinks=4, recent=256),
    }
    return [dict(c, name=n) for n, c in named.items()]


#: (query heads, key/value heads, head size): Qwen3-4B, its shards over 2, 4 and 8 GPUs, and other common groupings.
_LAYOUTS = [(32, 8, 128), (32, 8, 128), (16, 4, 128), (8, 2, 128), (4, 1, 128), (16, 16, 64), (24, 8, 64), (40, 8, 128)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "attn", "prefix", "prefix", "scored", "evict"])
    heads, kv_heads, dim = rng.choice(_LAYOUTS)
    B = _log_int(rng, 1, 64)
    c = dict(heads=heads, kv_heads=kv_heads, dim=dim)
    if kind == "rope":
        R = _log_int(rng, 1, 8192 // B)
        return _case(kind, B, R, R + rng.randint(0, 2000), spread=rng.choice([0, 500]) if R < 64 else 0, **c)
    if kind == "evict":
        B = min(B, 16)
        L = _log_int(rng, 300, 32768)
        budget = _log_int(rng, 64, max(65, L // 2))
        return _case(kind, B, 1, L, spread=rng.randint(0, L // 2), budget=budget, sinks=rng.randint(0, 8),
                     recent=rng.randint(0, budget // 2), **c)
    form = rng.choice(["decode", "decode", "tree", "prompt"]) if kind == "attn" else rng.choice(["decode", "rows"])
    tree = form == "tree" or (kind == "prefix" and form == "rows")
    R = 1 if form == "decode" else rng.randint(2, 32) if form == "prompt" and B > 16 else rng.randint(2, 64)
    if form == "prompt":
        B = min(B, 4)
        R = _log_int(rng, 65, 3500 // B)
        L = R + rng.choice([0, rng.randint(1, 1500 // B)])
    else:
        B = min(B, max(1, 512 // R))
        L = R + _log_int(rng, 16, max(32, min(32000, (1 << 19) // B)))
    spread = 0 if form == "prompt" else rng.randint(0, (L - R) // 2)
    window = rng.choice([0, 0, _log_int(rng, 64, 8192)]) if kind != "scored" else 0
    sinks = rng.choice([0, 1, 4, 16]) if window else 0
    prefix = _log_int(rng, 100, min(32768, (1 << 25) // (B * R * heads))) if kind == "prefix" else 0
    return _case(kind, B, R, L, spread=spread, window=window, sinks=sinks, prefix=prefix, tree=tree, **c)


def _lens(c):
    return [max(c["R"], c["len"] - (b * 7919) % (c["spread"] + 1)) for b in range(c["B"])]


def _tree_rows(c):
    """For each sequence its rows' ancestor sets (bit j of row i: node j is an
    ancestor of node i or i itself); node 0 is the root of all."""
    if not c["tree"]:
        return None
    rng = random.Random(c["B"] * 1000 + c["R"])
    rows = []
    for _ in range(c["B"]):
        masks = [1]
        for i in range(1, c["R"]):
            masks.append(masks[rng.randrange(max(0, i - 8), i)] | 1 << i)
        rows.append(masks)
    return rows


# ----------------------------------------------------------------- inputs
def _inputs(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(BF16)

    B, R, H, KV, D = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"]
    cap = c["len"] + 24  # slots of the cache: room for the next rows
    s = {"case": c, "lens": torch.tensor(_lens(c), dtype=torch.int32, device=DEV)}
    if c["kind"] == "rope":
        s["qkv"] = rnd(B * R, (H + 2 * KV) * D)
        s["q_norm"], s["k_norm"] = (torch.randn(D, generator=g, device=DEV).mul_(0.1).add_(1).to(BF16) for _ in "qk")
        s["k"], s["v"] = (torch.zeros((B, cap, KV, D), dtype=BF16, device=DEV) for _ in "kv")
        # Cosines and sines of every position, from 64 bits: a model's program computes them once.
        angle = torch.arange(cap, dtype=torch.float64, device=DEV)[:, None] * (
            THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D))
        s["table"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["q"] = torch.empty((B * R, H * D), dtype=BF16, device=DEV)
        return s
    # Normed keys and queries: scores of a head spread over a few units, values around a small mean.
    s["k"] = rnd(B, cap, KV, D)
    s["v"] = rnd(B, cap, KV, D).add_(0.05)
    if c["kind"] in ("scored", "evict"):
        # Accumulated attention weights: a heavy tail, and keys that no row has looked at yet.
        w = torch.randn((B, KV, cap), generator=g, device=DEV).mul_(2).exp_()
        s["scores"] = torch.where(torch.rand((B, KV, cap), generator=g, device=DEV) < 0.1, torch.zeros_like(w), w)
        s["scores_out"] = torch.zeros((B, KV, cap if c["kind"] == "scored" else c["budget"]), device=DEV)
    if c["kind"] == "evict":
        s["k_out"], s["v_out"] = (torch.zeros((B, c["budget"], KV, D), dtype=BF16, device=DEV) for _ in "kv")
        return s
    # q as the qkv projection leaves it: the first columns of its rows.
    s["q"] = rnd(B * R, (H + 2 * KV) * D)[:, :H * D]
    s["tree"] = None
    if c["tree"]:
        signed = [[m - (1 << 64) if m >> 63 else m for m in rows] for rows in _tree_rows(c)]
        s["tree"] = torch.tensor(signed, dtype=torch.int64, device=DEV)
    if c["kind"] == "prefix":
        s["kp"], s["vp"] = rnd(c["prefix"], KV, D), rnd(c["prefix"], KV, D).add_(0.05)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the objects that a serving loop builds once per shape: they own the workspaces
        c, A = case, _kernels()
        B, R, H, KV, D, cap = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"], c["len"] + 24
        if c["kind"] == "evict":
            s["op"] = A.CacheEviction(B, KV, D, cap, c["budget"], DEV, sinks=c["sinks"], recent=c["recent"])
        elif c["kind"] != "rope":
            s["op"] = A.CacheAttention(B, R, H, KV, D, cap, DEV, window=c["window"], sinks=c["sinks"],
                                       prefix=c["prefix"], scored=c["kind"] == "scored")
        else:
            s["op"] = A.qk_norm_rope
    return s


# ------------------------------------------------------------------ plain
def _plain_rope(s):
    c = s["case"]
    B, R, H, KV, D = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"]
    slot = s["lens"].long()[:, None] - R + torch.arange(R, device=DEV)
    cos, sin = s["table"][slot].view(B, R, 1, D).split(D // 2, dim=-1)
    q, k, v = s["qkv"].view(B, R, H + 2 * KV, D).split([H, KV, KV], dim=2)

    def turned(x, gain):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * gain.float()
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(BF16)

    rows = torch.arange(B, device=DEV)[:, None]
    s["k"][rows, slot] = turned(k, s["k_norm"])
    s["v"][rows, slot] = v
    return {"q": turned(q, s["q_norm"]).view(B * R, H * D), "k": s["k"], "v": s["v"]}


def _visible(s):
    """[B, R, prefix + len]: which keys each row sees."""
    c = s["case"]
    R, P, L = c["R"], c["prefix"], c["len"]
    lens = s["lens"].long()[:, None]
    key = torch.arange(P + L, device=DEV)[None, None, :]
    first = (P + lens - R)[..., None]
    if s["tree"] is None:
        row = first + torch.arange(R, device=DEV)[:, None]
        seen = key <= row
    else:
        bits = s["tree"][..., None] >> torch.arange(R, device=DEV) & 1
        row = first + bits.sum(dim=-1, keepdim=True) - 1
        node = (key - first).clamp(0, R - 1).expand(-1, R, -1)
        seen = (key < first) | (key < first + R) & (bits.gather(2, node) > 0)
    if c["window"]:
        near = (key < c["sinks"]) | (key > row - c["window"])
        seen = seen & (near if s["tree"] is None else near | (key >= first))
    return seen


def _plain_attention(s):
    c = s["case"]
    B, R, H, KV, D, P, L = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"], c["prefix"], c["len"]
    G = H // KV
    q = s["q"].float().reshape(B, R, KV, G, D).permute(0, 2, 1, 3, 4)  # B KV R G D
    k = s["k"][:, :L].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][:, :L].float().permute(0, 2, 1, 3).contiguous()
    a = q.reshape(B, KV, R * G, D) @ k
    if P:
        qs = q.permute(1, 0, 2, 3, 4).reshape(KV, B * R * G, D)
        kp = s["kp"].float().permute(1, 2, 0).contiguous()
        vp = s["vp"].float().permute(1, 0, 2).contiguous()
        a = torch.cat([(qs @ kp).view(KV, B, R * G, P).transpose(0, 1), a], dim=-1)
    a = (a * D ** -0.5).view(B, KV, R, G, P + L).masked_fill_(~_visible(s)[:, None, :, None, :], -math.inf)
    a = a - a.amax(dim=-1, keepdim=True).clamp(min=-3e38)
    a = a.exp_()
    total = a.sum(dim=-1, keepdim=True)
    a = torch.where(total > 0, a / total, torch.zeros_like(a)).view(B, KV, R * G, P + L)
    o = a[..., P:] @ v
    if P:
        o = o + (a[..., :P].transpose(0, 1).reshape(KV, B * R * G, P) @ vp).view(KV, B, R * G, D).transpose(0, 1)
    o = o.view(B, KV, R, G, D).permute(0, 2, 1, 3, 4).reshape(B * R, H * D).to(BF16)
    if c["kind"] != "scored":
        return o
    live = torch.arange(L, device=DEV) < s["lens"][:, None, None]
    s["scores_out"][:, :, :L] = torch.where(live, s["scores"][:, :, :L] + a.sum(dim=2), s["scores_out"][:, :, :L])
    return {"out": o, "scores": s["scores_out"]}


def _plain_evict(s):
    c = s["case"]
    L, n = c["len"], c["budget"]
    lens = s["lens"].long()[:, None, None]
    slot = torch.arange(L, device=DEV)[None, None, :]
    score = s["scores"][:, :, :L]
    stays = (slot < c["sinks"]) | (slot >= lens - c["recent"]) | (lens <= n)
    rank = torch.where(stays, torch.full_like(score, math.inf), score)
    rank = torch.where(slot < lens, rank, torch.full_like(score, -1.0))
    keep = rank.sort(dim=-1, descending=True, stable=True).indices[..., :n]
    keep = torch.where(keep < lens, keep, L).sort(dim=-1).values
    live = keep < L
    at = torch.where(live, keep, 0)
    rows = torch.arange(c["B"], device=DEV)[:, None, None]
    head = torch.arange(c["kv_heads"], device=DEV)[None, :, None]
    some = live[..., None]
    s["k_out"].copy_(torch.where(some, s["k"][rows, at, head], 0).transpose(1, 2))
    s["v_out"].copy_(torch.where(some, s["v"][rows, at, head], 0).transpose(1, 2))
    s["scores_out"].copy_(torch.where(live, score.gather(2, at), 0))
    return {"keep": torch.where(live, keep, -1).int(), "lens": s["lens"].clamp(max=n), "k": s["k_out"],
            "v": s["v_out"], "scores": s["scores_out"]}


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return _plain_rope(s) if kind == "rope" else _plain_evict(s) if kind == "evict" else _plain_attention(s)
    op = s["op"]
    if kind == "rope":
        op(s["qkv"], s["q_norm"], s["k_norm"], EPS, s["table"], s["lens"], s["k"], s["v"], q_out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if kind == "evict":
        keep, lens = op(s["k"], s["v"], s["scores"], s["lens"], out=(s["k_out"], s["v_out"], s["scores_out"]))
        return {"keep": keep, "lens": lens, "k": s["k_out"], "v": s["v_out"], "scores": s["scores_out"]}
    if kind == "scored":
        o = op(s["q"], s["k"], s["v"], s["lens"], scores=s["scores"], scores_out=s["scores_out"])
        return {"out": o, "scores": s["scores_out"]}
    if kind == "prefix":
        return op(s["q"], s["k"], s["v"], s["lens"], prefix=(s["kp"], s["vp"]), tree=s["tree"])
    return op(s["q"], s["k"], s["v"], s["lens"], tree=s["tree"])


# ------------------------------------------------------------- accounting
def _seen_counts(c):
    """(visible row-key pairs of one query head, keys of each kind that some
    row sees: the sequences' own, the prefix's)."""
    R, P, W, S = c["R"], c["prefix"], c["window"], c["sinks"]
    trees = _tree_rows(c)
    pairs, keys, prefix_from = 0, 0, P
    for b, n in enumerate(_lens(c)):
        first = P + n - R  # position of the sequence's first row
        lowest = P + n
        for i in range(R):
            at = first + (bin(trees[b][i]).count("1") - 1 if trees else i)
            lo = max(0, at - W + 1) if W else 0
            if trees:
                lo = min(lo, first)
                pairs += first - lo + bin(trees[b][i]).count("1") + min(S, lo)
            else:
                pairs += at + 1 - lo + min(S, lo)
            lowest = min(lowest, lo)
        keys += P + n - max(lowest, P) + max(0, min(S, lowest) - P)
        prefix_from = min(prefix_from, lowest)
    return pairs, keys, P - prefix_from + min(S, prefix_from, P) if P else 0


def work(case):
    c = case
    B, R, H, KV, D = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rope":
        row = (H + 2 * KV) * D
        return {"bytes": B * R * (4 * row + 4 * D) + 4 * D + 4 * B, "flops": 8 * B * R * (H + KV) * D}
    if c["kind"] == "evict":
        kept = sum(min(n, c["budget"]) for n in _lens(c))
        # Scores of all slots, then the kept rows in and out, their scores and indices.
        return {"bytes": KV * (4 * sum(_lens(c)) + kept * (8 * D + 4 + 4)) + 8 * B, "flops": KV * sum(_lens(c))}
    pairs, keys, prefix = _seen_counts(c)
    w = {"bytes": 4 * B * R * H * D + 4 * (keys + prefix) * KV * D, "flops": 4 * pairs * H * D}
    if c["kind"] == "scored":
        w["bytes"] += 8 * KV * sum(_lens(c))
    return w


# ---------------------------------------------------------------- 64 bits
def _exact_rope(s):
    c = s["case"]
    B, R, H, KV, D = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"]
    k, v = s["k"].double(), s["v"].double()
    freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    q = torch.empty((B * R, H * D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(c)):
        x = s["qkv"][b * R:(b + 1) * R].double().view(R, H + 2 * KV, D)
        angle = torch.arange(n - R, n, dtype=torch.float64, device=DEV)[:, None, None] * freq
        turn = torch.polar(torch.ones_like(angle), angle)
        for part, gain, heads in ((0, s["q_norm"], H), (1, s["k_norm"], KV)):
            y = x[:, part * H:part * H + heads]
            y = y / (y.square().mean(dim=-1, keepdim=True) + EPS).sqrt() * gain.double()
            z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
            y = torch.cat([z.real, z.imag], dim=-1)
            if part == 0:
                q[b * R:(b + 1) * R] = y.reshape(R, H * D)
            else:
                k[b, n - R:n] = y
        v[b, n - R:n] = x[:, H + KV:]
    return {"q": q, "k": k, "v": v}


def _exact_attention(s):
    c = s["case"]
    B, R, H, KV, D, P = c["B"], c["R"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    G = H // KV
    out = torch.empty((B, R, H, D), dtype=torch.float64, device=DEV)
    scores = s["scores_out"].double() if c["kind"] == "scored" else None
    trees = _tree_rows(c)
    for b, n in enumerate(_lens(c)):
        at = torch.arange(P + n, device=DEV)[None, :]
        row = torch.arange(P + n - R, P + n, device=DEV)[:, None]
        hide = at > row
        if trees:
            anc = torch.tensor([[not m >> j & 1 for j in range(R)] for m in trees[b]], device=DEV)
            hide = torch.cat([torch.zeros((R, P + n - R), dtype=torch.bool, device=DEV), anc], dim=1)
            row = P + n - R + (~anc).sum(dim=1, keepdim=True) - 1
        if c["window"]:
            far = (row - at >= c["window"]) & (at >= c["sinks"])
            hide = hide | (far & (at < P + n - R) if trees else far)
        for h in range(KV):
            k, v = s["k"][b, :n, h].double(), s["v"][b, :n, h].double()
            if P:
                k, v = torch.cat([s["kp"][:, h].double(), k]), torch.cat([s["vp"][:, h].double(), v])
            for j in range(h * G, h * G + G):
                x = s["q"][b * R:(b + 1) * R, j * D:(j + 1) * D].double() @ k.t().contiguous() / math.sqrt(D)
                x = x.masked_fill(hide, -math.inf)
                x = (x - torch.logsumexp(x, dim=1, keepdim=True)).exp()
                out[b, :, j] = x @ v
                if scores is not None:
                    scores[b, h, :n] += x.sum(dim=0)
            if scores is not None:
                scores[b, h, :n] += s["scores"][b, h, :n].double()
    out = out.view(B * R, H * D)
    return out if scores is None else {"out": out, "scores": scores}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "evict":
        return None  # rows moved as they are: compared value by value
    return _exact_rope(s) if case["kind"] == "rope" else _exact_attention(s)
