"""Performance cases of serving many requests at once: page tables, the paged
key/value cache and its attention, and low-rank adapters.

Each case is one pass through one operator, as a serving loop calls it for a
step over requests of different lengths: some decode one token, some verify a
few drafted ones, some bring in a chunk of a prompt (sizes: Qwen3-4B's 32 query
and 8 key/value heads of 128, its projections, and a few generic ones).

Kinds:

* ``tables``  pages given back and taken for the step's new tokens; each
              request's page table, each row's slot, position and label.
* ``write``   per-head RMSNorm of q and k, rotary embedding, and the rows' k and
              v written into their pages.
* ``attn``    attention of every request's new rows over its pages: causal, with
              a sliding window behind which a few first tokens stay visible.
* ``adapt``   each row's low-rank adapter added to a projection's output, whose
              columns fall into slices with their own first factor, or which a
              SiLU gate follows.

Requests 0 .. chunks - 1 of a case bring in about ``chunk`` rows each, the others
``R`` rows, and with ``idle`` every seventh none.  Request b has ``len - (b * 7919)
% (spread + 1)`` keys, its new rows among them.  Cases are plain numbers; every
tensor comes from the seed.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False  # True: the framework's kernels; False: the plain forms

DEV = "cuda:0"
BF16 = torch.bfloat16
I32 = torch.int32
EPS = 1e-6
THETA = 1e6
_PKG = str(Path(__file__).resolve().parent.parent / "kernel-rush-kawk_amd")


def _kernels():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import kernels

    return kernels


# ------------------------------------------------------------------ cases
def _case(kind, B=0, R=1, len_=0, chunks=0, chunk=0, spread=0, idle=False, restart=0, page=16, heads=32, kv_heads=8, dim=128,
          window=0, sinks=0, pad=0, M=0, N=0, K=0, rank=0, adapters=0, run=1, slices=1, silu=False):
    return {"kind": kind, "B": B, "R": R, "len": len_, "chunks": chunks, "chunk": chunk, "spread": spread, "idle": idle,
            "restart": restart, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window,
            "sinks": sinks, "pad": pad, "M": M, "N": N, "K": K, "rank": rank, "adapters": adapters, "run": run,
            "slices": slices, "silu": silu}


def listed():
    named = {
        # A decode step of 64 requests.
        "tables_decode_b64": _case("tables", 64, 1, 4000, spread=3800, pad=0),
        # A full step: finished requests replaced by new prompts, other prompts going on, the rest decoding.
        "tables_mixed_b256": _case("tables", 256, 1, 6000, chunks=12, chunk=800, spread=5000, idle=True, restart=8, pad=40),
        # The rows of a decode step.
        "write_b32": _case("write", 32, 1, 3000, spread=2900),
        # A chunk of a prompt beside decoding requests.
        "write_chunk": _case("write", 33, 1, 4100, chunks=1, chunk=4064, spread=36, pad=5),
        # One request's decode step over a short chat: latency.
        "decode_b1": _case("attn", 1, 1, 1000),
        # Decoding requests of very different lengths, one of them idle now and then.
        "decode_ragged_b64": _case("attn", 64, 1, 16000, spread=15700, idle=True, pad=3),
        # Eight requests' drafts of 16 tokens verified, over large pages.
        "verify_b8": _case("attn", 8, 16, 3500, spread=2500, page=64),
        # A chunk of a long prompt.
        "chunk_long": _case("attn", 1, 1, 16384, chunks=1, chunk=2048),
        # Two prompts' chunks beside decoding requests, with a sliding window.
        "mixed_window": _case("attn", 50, 1, 9000, chunks=2, chunk=1100, spread=7000, window=4096, sinks=4, page=32, pad=7),
        # The qkv projection of a decode step over 16 adapters.
        "adapt_qkv_b32": _case("adapt", M=32, N=6144, K=2560, rank=16, adapters=16, slices=3),
        # Gate and up of a verification step, SiLU behind them.
        "adapt_gate_up_b64": _case("adapt", M=64, N=19456, K=2560, rank=32, adapters=8, run=16, slices=2, silu=True),
        # The down projection of prompts' chunks of a few adapters.
        "adapt_down_chunk": _case("adapt", M=4096, N=2560, K=9728, rank=64, adapters=6, run=900),
    }
    return [dict(c, name=n) for n, c in named.items()]


#: (query heads, key/value heads, head size): Qwen3-4B, its shards, and other common groupings.
_LAYOUTS = [(32, 8, 128), (32, 8, 128), (8, 2, 128), (4, 1, 128), (16, 16, 64), (24, 8, 64), (40, 8, 128)]
#: (columns, slices, SiLU) and K: Qwen3-4B's projections and a smaller model's.
_PROJECTIONS = [(6144, 3, False, 2560), (2560, 1, False, 4096), (19456, 2, True, 2560), (2560, 1, False, 9728),
                (1536, 3, False, 1024), (1024, 1, False, 2816)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attn", "attn", "attn", "attn", "adapt", "adapt"])
    if kind == "adapt":
        N, slices, silu, K = rng.choice(_PROJECTIONS)
        M = _log_int(rng, 1, 4096)
        return _case(kind, M=M, N=N, K=K, rank=rng.choice([8, 16, 24, 32, 64]), adapters=_log_int(rng, 1, 16),
                     run=_log_int(rng, 1, max(2, M)), slices=slices, silu=silu)
    heads, kv_heads, dim = rng.choice(_LAYOUTS)
    c = dict(heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 16, 32, 64, 128]), pad=rng.choice([0, 1, 9]),
             idle=rng.random() < 0.3)
    B = _log_int(rng, 1, 256 if kind == "tables" else 64)
    form = rng.choice(["decode", "decode", "verify", "chunk"])
    R = rng.randint(2, 24) if form == "verify" else 1
    chunks = min(B, rng.randint(1, 3)) if form == "chunk" else 0
    if kind != "attn":
        chunk = _log_int(rng, 20, 2000) if chunks else 0
        L = max(chunk, R) + _log_int(rng, 16, 4000)
        restart = min(chunks, rng.randint(0, 2)) if kind == "tables" else 0
        return _case(kind, B, R, L, chunks=chunks, chunk=chunk, spread=rng.randint(0, L // 2), restart=restart, **c)
    chunk = _log_int(rng, 20, 1600 // chunks) if chunks else 0
    L = max(chunk, R) + _log_int(rng, 16, min(14000, (1 << 19) // B))
    window = rng.choice([0, 0, _log_int(rng, 64, 4096)])
    return _case(kind, B, R, L, chunks=chunks, chunk=chunk, spread=rng.randint(0, L // 2), window=window,
                 sinks=rng.choice([0, 1, 4, 16]) if window else 0, **c)


def _new(c):
    """Each request's new rows."""
    n = []
    for b in range(c["B"]):
        if b < c["chunks"]:
            n.append(c["chunk"] - (b * 1009) % (c["chunk"] // 4 + 1))
        else:
            n.append(0 if c["idle"] and b % 7 == 6 else c["R"])
    return n


def _lens(c):
    """Each request's keys, the new rows among them (a restarted request's: before it was cut)."""
    return [max(n, c["len"] - (b * 7919) % (c["spread"] + 1)) for b, n in enumerate(_new(c))]


def _rows(c):
    return sum(_new(c)) + c["pad"]


def _starts(c):
    at = [0]
    for n in _new(c):
        at.append(at[-1] + n)
    return at


# ----------------------------------------------------------------- inputs
def _pages(c):
    """(pages of the pool, pages of the longest request's table row)."""
    P = c["page"]
    used = sum(-(-n // P) for n in _lens(c))
    return used + used // 8 + c["B"] + 4, -(-c["len"] // P) + 2


def _inputs(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(BF16)

    if c["kind"] == "adapt":
        M, N, K, r = c["M"], c["N"], c["K"], c["rank"]
        s = {"case": c, "x": rnd(M, K), "y": rnd(M, N)}
        s["a"] = rnd(c["adapters"], c["slices"] * r, K, scale=K ** -0.5)
        s["b"] = rnd(c["adapters"], N, r, scale=0.1)
        s["scale"] = 16.0 / r * (1 + torch.rand(c["adapters"], generator=g, device=DEV))
        # Runs of rows (a request's) with one adapter, or none (-1).
        ids = torch.randint(-1, c["adapters"], (-(-M // c["run"]),), generator=g, device=DEV)
        s["index"] = ids[torch.arange(M, device=DEV) // c["run"]].to(I32)
        s["out"] = torch.zeros((M, N // 2 if c["silu"] else N), dtype=BF16, device=DEV)
        return s
    B, H, KV, D, P, M = c["B"], c["heads"], c["kv_heads"], c["dim"], c["page"], _rows(c)
    pages, width = _pages(c)
    new, lens, starts = _new(c), _lens(c), _starts(c)
    # A pool in long use: every request's pages lie anywhere in it.
    order = torch.randperm(pages, generator=g, device=DEV).to(I32)
    s = {"case": c, "pages": pages, "width": width}
    held = lens if c["kind"] != "tables" else [n - k if b >= c["restart"] else n for b, (n, k) in enumerate(zip(lens, new))]
    flat, first = [], 0
    for n in held:
        need = -(-n // P)
        flat += [(first + i if i < need else -1) for i in range(width)]
        first += need
    at = torch.tensor(flat, device=DEV).view(B, width)
    s["table"] = torch.where(at >= 0, order[at.clamp(min=0)], torch.zeros_like(order[:1]))
    s["new"] = torch.tensor(new, dtype=I32, device=DEV)
    if c["kind"] == "tables":
        s["lens"] = torch.tensor(held, dtype=I32, device=DEV)
        # Restarted requests lose all their keys, the others what an earlier step's rows had added.
        s["keep"] = torch.tensor([0 if b < c["restart"] else n for b, n in enumerate(held)], dtype=I32, device=DEV)
        s["labels"] = torch.randint(-1, 16, (B,), generator=g, device=DEV).to(I32)
        s["free"] = torch.cat([order[first:].flip(0), order.new_zeros(first)])
        s["count"] = torch.tensor([pages - first], dtype=I32, device=DEV)
        return s
    s["starts"] = torch.tensor(starts, dtype=I32, device=DEV)
    s["keys"] = torch.tensor(lens, dtype=I32, device=DEV)
    s["qkv"] = rnd(M, (H + 2 * KV) * D)
    if c["kind"] == "write":
        s["q_norm"], s["k_norm"] = (torch.randn(D, generator=g, device=DEV).mul_(0.1).add_(1).to(BF16) for _ in "qk")
        s["k"], s["v"] = (torch.zeros((pages, P, KV, D), dtype=BF16, device=DEV) for _ in "kv")
        # Cosines and sines of every position, from 64 bits: a model's program computes them once.
        angle = torch.arange(c["len"], dtype=torch.float64, device=DEV)[:, None] * (
            THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D))
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["q"] = torch.zeros((M, H * D), dtype=BF16, device=DEV)
        where = [(b, n - k + i) for b, (n, k) in enumerate(zip(lens, new)) for i in range(k)]
        b, pos = torch.tensor(where, device=DEV).T
        pad = torch.full((c["pad"],), -1, device=DEV)
        s["positions"] = torch.cat([pos, pad]).to(I32)
        s["slots"] = torch.cat([s["table"][b, pos // P] * P + pos % P, pad]).to(I32)
        return s
    # Normed keys and queries: scores of a head spread over a few units, values around a small mean.
    s["q"] = s.pop("qkv")[:, :H * D]
    s["k"] = rnd(pages, P, KV, D)
    s["v"] = rnd(pages, P, KV, D).add_(0.05)
    s["out"] = torch.zeros((M, H * D), dtype=BF16, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    c, A = case, _kernels()  # the objects that a serving loop builds once: they own the workspaces and the tables
    if c["kind"] == "tables":
        op = s["op"] = A.PageTables(c["B"], _rows(c), s["pages"], c["page"], s["width"], DEV)
        for name in ("lens", "table", "free", "count"):
            getattr(op, name).copy_(s[name])
    elif c["kind"] == "attn":
        s["op"] = A.PagedAttention(c["B"], _rows(c), c["heads"], c["kv_heads"], c["dim"], c["page"], s["width"], DEV,
                                   window=c["window"], sinks=c["sinks"])
    elif c["kind"] == "adapt":
        widths = (c["N"] // 2,) * 2 if c["silu"] else (c["N"] * 2 // 3, c["N"] // 6, c["N"] // 6) if c["slices"] == 3 else None
        s["op"] = A.LowRankAdapters(c["M"], c["N"], c["K"], c["rank"], DEV, slices=widths, silu=c["silu"])
    else:
        s["op"] = A.paged_qk_norm_rope
    return s


# ------------------------------------------------------------------ plain
def _plain_tables(s):
    c = s["case"]
    P, W, M, pages, B = c["page"], s["width"], _rows(c), s["pages"], c["B"]
    old = s["lens"].long().clamp(0, W * P)
    cut = torch.minimum(old, s["keep"].long().clamp(min=0))
    had, held = (old + P - 1) // P, (cut + P - 1) // P
    i = torch.arange(W, device=DEV)[None, :]
    # Given back: pushed so that the first request's first page ends on top.
    gone = (i >= held[:, None]) & (i < had[:, None])
    top = s["count"].long() + gone.sum()
    spot = top - gone.view(-1).cumsum(0).view(B, W)
    free = torch.cat([s["free"], s["free"].new_zeros(1)])
    free.scatter_(0, torch.where(gone, spot, pages).view(-1), s["table"].view(-1))
    free = free[:pages]
    # Taken from the top, in the requests' order.
    n = s["new"].long().clamp(min=0)
    end = n.cumsum(0)
    start = end - n
    fits = (n > 0) & (end <= M) & (cut + n <= W * P)
    need = torch.where(fits, (cut + n + P - 1) // P - held, 0)
    taken = need.cumsum(0)
    ok = fits & ((need == 0) | (taken <= top))
    need = torch.where(ok, need, 0)
    j = i - held[:, None]
    page = free[(top - 1 - (taken - need)[:, None] - j).clamp(0, pages - 1)]
    table = torch.where((j >= 0) & (j < need[:, None]), page, s["table"])
    lens = torch.where(ok, cut + n, cut)
    r = torch.arange(M, device=DEV)
    b = torch.searchsorted(end, r, right=True).clamp(max=B - 1)
    live = (r < end[-1]) & ok[b]
    pos = torch.where(live, cut[b] + r - start[b], 0)
    slot = table[b, pos // P] * P + pos % P
    s["lens"].copy_(lens)
    s["table"].copy_(table)
    s["free"].copy_(free)
    s["count"].copy_(top - need.sum())
    return {"lens": s["lens"], "table": s["table"], "free": s["free"], "count": s["count"],
            "starts": torch.cat([start, end[-1:]]).clamp(max=M).to(I32),
            "keys": torch.where(ok | (n == 0), lens, 0).to(I32), "slots": torch.where(live, slot, -1).to(I32),
            "positions": torch.where(live, pos, -1).to(I32), "owner": torch.where(live, s["labels"][b], -1).to(I32)}


def _plain_write(s):
    c = s["case"]
    H, KV, D, n = c["heads"], c["kv_heads"], c["dim"], sum(_new(c))
    slot, pos = s["slots"][:n].long(), s["positions"][:n].long()
    cos, sin = s["cos_sin"][pos].view(n, 1, D).split(D // 2, dim=-1)
    q, k, v = s["qkv"][:n].view(n, H + 2 * KV, D).split([H, KV, KV], dim=1)

    def turned(x, gain):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * gain.float()
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(BF16)

    s["k"].view(-1, KV, D)[slot] = turned(k, s["k_norm"])
    s["v"].view(-1, KV, D)[slot] = v
    s["q"][:n] = turned(q, s["q_norm"]).view(n, H * D)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _groups(c):
    """Requests of the same number of new rows, and that number."""
    g = {}
    for b, n in enumerate(_new(c)):
        if n:
            g.setdefault(n, []).append(b)
    return g


def _plain_attention(s):
    c = s["case"]
    H, KV, D, P, W, S = c["heads"], c["kv_heads"], c["dim"], c["page"], c["window"], c["sinks"]
    G, lens, starts = H // KV, _lens(c), _starts(c)
    for n, bs in _groups(c).items():
        X, L = len(bs), max(lens[b] for b in bs)
        at = torch.tensor(bs, device=DEV)
        pages = s["table"][at, :-(-L // P)].long()
        k = s["k"][pages].view(X, -1, KV, D)[:, :L].float().permute(0, 2, 3, 1).contiguous()
        v = s["v"][pages].view(X, -1, KV, D)[:, :L].float().permute(0, 2, 1, 3).contiguous()
        rows = (s["starts"][at].long()[:, None] + torch.arange(n, device=DEV)).view(-1)
        q = s["q"][rows].float().view(X, n, KV, G, D).permute(0, 2, 1, 3, 4).reshape(X, KV, n * G, D)
        a = q @ k
        key = torch.arange(L, device=DEV)
        row = (s["keys"][at].long()[:, None] - n + torch.arange(n, device=DEV))[..., None]  # X n 1
        seen = key <= row
        if W:
            seen = seen & ((key < S) | (key > row - W))
        a = (a * D ** -0.5).view(X, KV, n, G, L).masked_fill_(~seen[:, None, :, None, :], -math.inf)
        a = (a - a.amax(dim=-1, keepdim=True)).exp_()
        a = (a / a.sum(dim=-1, keepdim=True)).view(X, KV, n * G, L)
        o = (a @ v).view(X, KV, n, G, D).permute(0, 2, 1, 3, 4).reshape(X * n, H * D)
        s["out"][rows] = o.to(BF16)
    return s["out"]


def _widths(c):
    N = c["N"]
    return [N // 2, N // 2] if c["silu"] else [N * 2 // 3, N // 6, N // 6] if c["slices"] == 3 else [N]


def _plain_adapters(s):
    c = s["case"]
    r, n, S = c["rank"], c["adapters"], c["slices"]
    # All adapters' first factors at once; every row keeps its own adapter's part.
    mine = torch.arange(n, device=DEV) == s["index"][:, None]
    gain = torch.where(mine, s["scale"], 0.0)
    h = (s["x"].float() @ s["a"].view(n * S * r, -1).float().t()).view(-1, n, S, r) * gain[:, :, None, None]
    out, col = [], 0
    for i, w in enumerate(_widths(c)):
        b = s["b"][:, col:col + w].float().transpose(1, 2).reshape(n * r, w)
        out.append(s["y"][:, col:col + w].float() + h[:, :, i].reshape(-1, n * r) @ b)
        col += w
    y = torch.cat(out, dim=1)
    if c["silu"]:
        gate, up = y.split(c["N"] // 2, dim=1)
        y = gate / (1 + (-gate).exp()) * up
    s["out"].copy_(y)
    return s["out"]


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return {"tables": _plain_tables, "write": _plain_write, "attn": _plain_attention, "adapt": _plain_adapters}[kind](s)
    op = s["op"]
    if kind == "tables":
        op.step(s["new"], keep=s["keep"], labels=s["labels"])
        return {"lens": op.lens, "table": op.table, "free": op.free, "count": op.count, "starts": op.starts, "keys": op.keys,
                "slots": op.slots, "positions": op.positions, "owner": op.owner}
    if kind == "write":
        op(s["qkv"], s["q_norm"], s["k_norm"], EPS, s["cos_sin"], s["slots"], s["positions"], s["k"], s["v"], q_out=s["q"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if kind == "attn":
        return op.run(s["q"], s["k"], s["v"], s["table"], s["starts"], s["keys"], s["out"])
    return op.run(s["x"], s["a"], s["b"], s["index"], s["y"], s["out"], scale=s["scale"])


# ------------------------------------------------------------- accounting
def _pairs(c):
    """(visible row-key pairs of one query head, keys that some row sees)."""
    W, S = c["window"], c["sinks"]
    pairs = keys = 0
    for n, L in zip(_new(c), _lens(c)):
        for i in range(n):
            at = L - n + i
            lo = max(0, at - W + 1) if W else 0
            pairs += at + 1 - lo + min(S, lo)
        if n:
            lo = max(0, L - n - W + 1) if W else 0
            keys += L - lo + min(S, lo)
    return pairs, keys


def work(case):
    c = case
    if c["kind"] == "adapt":
        M, N, K, r = c["M"], c["N"], c["K"], c["rank"]
        used = min(c["adapters"], -(-M // c["run"]))
        out = N // 2 if c["silu"] else N
        return {"bytes": 2 * (M * (K + N + out) + used * r * (c["slices"] * K + N)) + 4 * M,
                "flops": 2 * M * r * (c["slices"] * K + N) + M * N}
    rows, P = sum(_new(c)), c["page"]
    if c["kind"] == "tables":
        moved = sum(-(-n // P) for n in _new(c)) + sum(-(-n // P) for n in _lens(c)[:c["restart"]])
        return {"bytes": 28 * c["B"] + 8 * moved + 12 * _rows(c), "flops": 10 * _rows(c)}
    H, KV, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "write":
        row = (H + 2 * KV) * D
        return {"bytes": rows * (4 * row + 4 * D + 8) + 4 * D, "flops": 8 * rows * (H + KV) * D}
    pairs, keys = _pairs(c)
    return {"bytes": 4 * rows * H * D + 4 * keys * KV * D + 4 * keys // P, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------- 64 bits
def _exact_write(s):
    c = s["case"]
    H, KV, D, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    k, v, q = s["k"].double(), s["v"].double(), s["q"].double()
    freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    row = 0
    for b, (n, L) in enumerate(zip(_new(c), _lens(c))):
        if not n:
            continue
        pos = torch.arange(L - n, L, device=DEV)
        page, slot = s["table"][b].long()[pos // P], pos % P
        x = s["qkv"][row:row + n].double().view(n, H + 2 * KV, D)
        angle = pos.double()[:, None, None] * freq
        turn = torch.polar(torch.ones_like(angle), angle)
        for first, heads, gain in ((0, H, s["q_norm"]), (H, KV, s["k_norm"])):
            y = x[:, first:first + heads]
            y = y / (y.square().mean(dim=-1, keepdim=True) + EPS).sqrt() * gain.double()
            z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
            y = torch.cat([z.real, z.imag], dim=-1)
            if first == 0:
                q[row:row + n] = y.reshape(n, H * D)
            else:
                k[page, slot] = y
        v[page, slot] = x[:, H + KV:]
        row += n
    return {"q": q, "k": k, "v": v}


def _exact_attention(s):
    c = s["case"]
    H, KV, D, P, W, S = c["heads"], c["kv_heads"], c["dim"], c["page"], c["window"], c["sinks"]
    G, M = H // KV, _rows(c)
    out = s["out"].double().view(M, H, D)
    row = 0
    for b, (n, L) in enumerate(zip(_new(c), _lens(c))):
        if not n:
            continue
        key = torch.arange(L, device=DEV)
        page, slot = s["table"][b].long()[key // P], key % P
        far = torch.arange(L - n, L, device=DEV)[:, None] - key
        hide = far < 0
        if W:
            hide = hide | (far >= W) & (key >= S)
        for h in range(KV):
            k, v = s["k"][page, slot, h].double(), s["v"][page, slot, h].double()
            for j in range(h * G, h * G + G):
                x = s["q"][row:row + n, j * D:(j + 1) * D].double() @ k.t().contiguous() / math.sqrt(D)
                x = x.masked_fill(hide, -math.inf)
                out[row:row + n, j] = (x - torch.logsumexp(x, dim=1, keepdim=True)).exp() @ v
        row += n
    return out.view(M, H * D)


def _exact_adapters(s):
    c = s["case"]
    r, y = c["rank"], s["y"].double()
    for i in range(c["adapters"]):
        rows = (s["index"] == i).nonzero()[:, 0]
        if not len(rows):
            continue
        x, col = s["x"][rows].double(), 0
        for part, w in enumerate(_widths(c)):
            h = x @ s["a"][i, part * r:(part + 1) * r].double().t().contiguous()
            y[rows, col:col + w] += s["scale"][i].double() * (h @ s["b"][i, col:col + w].double().t().contiguous())
            col += w
    if not c["silu"]:
        return y
    half = c["N"] // 2
    return y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    s = _inputs(case, seed)
    return {"write": _exact_write, "attn": _exact_attention, "adapt": _exact_adapters}[case["kind"]](s)
