"""The cache operators on the GPU against the 64-bit oracle: rotary embedding
and cache write, attention (decode rows, draft trees, prompts, windows and
sinks, shared prefixes, scores), eviction, and a run of them together."""

from __future__ import annotations

import math

import pytest
import torch

from kernels import attention as A
from oracle import attn_ref as R64

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def say(*a):
    print(*a, flush=True)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rnd(g, *shape, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g) * scale + shift).to(BF)


def tree_masks(g, B, R):
    """Random draft trees: node i > 0 hangs under an earlier node."""
    rows = []
    for _ in range(B):
        masks = [1]
        for i in range(1, R):
            masks.append(masks[int(torch.randint(0, i, (1,), generator=g))] | 1 << i)
        rows.append([m - (1 << 64) if m >> 63 else m for m in masks])
    return torch.tensor(rows, dtype=torch.int64)


def poison(t, lens):
    """NaN and infinities in the slots at and behind each sequence's length."""
    for b, n in enumerate(lens):
        n = max(0, min(n, t.shape[1]))
        t[b, n::2] = math.nan
        t[b, n + 1::2] = math.inf
    return t


def close(got, ref, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    fin = ref.isfinite()
    assert torch.equal(got[~fin & ~ref.isnan()], ref[~fin & ~ref.isnan()]), f"{what}: other infinities"
    err = (got - ref).abs()
    bad = (err > tol) & fin
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                           f"{float((err / tol)[fin].max()):.2f} times")


def weight_half(op):
    """Relative rounding of the weights: one bf16 part in workgroups of 128 rows, else two."""
    return 2.0 ** -8 if max(op.plan["rows"], op.plan["prefix_rows"]) >= 128 else 2.0 ** -16


def check_attention(dev, seed, B, R, heads, kv, D, cap, lens, window=0, sinks=0, tree=False, prefix=0, built_prefix=None,
                    scored=False, layout="slots", scale=None, spread=1.0):
    g = gen(seed)
    qkv = rnd(g, B * R, (heads + 2 * kv) * D, scale=spread)
    shape = (B, cap, kv, D) if layout == "slots" else (B, kv, cap, D)
    k, v = rnd(g, *shape), rnd(g, *shape, shift=0.05)
    if layout != "slots":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    poison(k, lens), poison(v, lens)
    masks = tree_masks(g, B, R) if tree else None
    shared = (rnd(g, prefix, kv, D), rnd(g, prefix, kv, D, shift=0.05)) if prefix else None
    was = torch.rand((B, kv, cap), generator=g) if scored else None
    say("attention", seed, B, R, heads, kv, D, cap, lens, window, sinks, tree, prefix, scored, layout)
    op = A.CacheAttention(B, R, heads, kv, D, cap, dev, window=window, sinks=sinks,
                          prefix=prefix if built_prefix is None else built_prefix, scored=scored, scale=scale)
    q = qkv[:, :heads * D]
    qd = qkv.to(dev)[:, :heads * D]
    kd, vd = (t.to(dev) if layout == "slots" else t.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for t in (k, v))
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    lse = torch.empty((B * R, heads), device=dev)
    kw = {}
    if scored:
        kw = dict(scores=was.to(dev), scores_out=torch.full_like(was, -7.0).to(dev))
    out = op(qd, kd, vd, ln, prefix=None if shared is None else tuple(t.to(dev) for t in shared),
             tree=None if masks is None else masks.to(dev), lse=lse, **kw)
    torch.cuda.synchronize()
    ref, rlse, w, size, top = R64.attention(q, k, v, lens, heads=heads, R=R, window=window, sinks=sinks, prefix=shared,
                                            tree=None if masks is None else masks.tolist(), scale=scale)
    keys = prefix + cap
    tol = R64.attention_tolerance(ref, size, top, D, keys, weight_half(op))
    close(out.view(ref.shape), ref, tol, "out")
    err = R64.score_error(top, D) + (keys + 32) * R64.FP32_HALF + 4 * R64.FP32_HALF * torch.where(rlse.isfinite(), rlse.abs(), 0)
    close(lse.view(rlse.shape), rlse, err, "lse")
    if scored:
        live = torch.arange(cap)[None, None, :] < torch.tensor(lens).clamp(0, cap)[:, None, None]
        want = torch.where(live, was.double() + w, torch.full_like(w, -7.0))
        rel = 2 * float(R64.score_error(top, D).max()) + (keys + 64) * R64.FP32_HALF
        close(kw["scores_out"], want, w * rel + (R + 4) * R64.FP32_HALF * want.abs() + 1e-30, "scores")
    return op


DECODE = [
    # B, R, heads, kv, D, cap, lens
    (1, 1, 32, 8, 128, 40, [1]),
    (1, 1, 32, 8, 128, 1, [1]),
    (3, 1, 32, 8, 128, 300, [0, 33, 300]),
    (2, 1, 8, 2, 64, 1025, [1025, 31]),
    (2, 1, 16, 16, 64, 200, [32, 64]),
    (1, 1, 24, 1, 128, 500, [333]),
    (4, 1, 40, 8, 128, 65, [64, 65, 2, -5]),
    (2, 3, 8, 8, 128, 130, [129, 2]),
    (2, 7, 12, 4, 64, 777, [700, 5]),
    (1, 16, 32, 8, 128, 2000, [1987]),
    (5, 2, 4, 1, 128, 96, [96, 1, 2, 3, 1000]),
]


@pytest.mark.parametrize("case", range(len(DECODE)))
@pytest.mark.parametrize("layout", ["slots", "heads"])
def test_decode(device, case, layout):
    check_attention(device, 100 + case, *DECODE[case], layout=layout)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 0), (33, 40), (100, 4), (5000, 9)])
@pytest.mark.parametrize("R", [1, 5])
def test_window_and_sinks(device, window, sinks, R):
    check_attention(device, 200 + window + sinks, 3, R, 8, 2, 128, 400, [400, 211, 3], window=window, sinks=sinks)


@pytest.mark.parametrize("B,R,heads,kv,D,cap,lens,window,sinks", [
    (1, 64, 8, 2, 128, 200, [180], 0, 0),
    (2, 16, 32, 8, 128, 500, [499, 16], 0, 0),
    (2, 64, 4, 4, 64, 300, [64, 270], 70, 2),
    (3, 5, 8, 2, 128, 90, [90, 5, 3], 6, 1),
    (1, 1, 8, 2, 128, 90, [50], 0, 0),
    (4, 64, 8, 2, 128, 70, [1, 63, 0, 70], 0, 0),
    (2, 33, 16, 2, 64, 300, [300, 20], 40, 3),
])
def test_tree(device, B, R, heads, kv, D, cap, lens, window, sinks):
    check_attention(device, 300 + R, B, R, heads, kv, D, cap, lens, window=window, sinks=sinks, tree=True)


@pytest.mark.parametrize("B,R,heads,kv,D,cap,lens,window,sinks", [
    (1, 100, 4, 1, 128, 100, [100], 0, 0),
    (1, 257, 8, 2, 128, 300, [290], 0, 0),
    (2, 130, 4, 4, 64, 150, [150, 77], 0, 0),
    (1, 300, 8, 2, 128, 300, [300], 40, 3),
    (1, 500, 2, 1, 64, 700, [700], 33, 70),
    (2, 200, 6, 2, 128, 256, [256, 0], 128, 4),
])
def test_prompt(device, B, R, heads, kv, D, cap, lens, window, sinks):
    check_attention(device, 400 + R, B, R, heads, kv, D, cap, lens, window=window, sinks=sinks)


@pytest.mark.parametrize("B,R,heads,kv,D,cap,lens,window,sinks,tree,scored", [
    (1, 70, 8, 2, 128, 2600, [2500], 0, 0, False, False),
    (2, 40, 8, 2, 128, 2000, [1990, 701], 0, 0, False, True),
    (1, 100, 8, 4, 64, 3000, [2900], 1500, 70, False, True),
    (1, 64, 8, 2, 128, 2100, [2033], 0, 0, True, False),
    (2, 64, 8, 4, 128, 2100, [2033, 70], 1900, 2, True, False),
])
def test_many_rows_in_key_ranges(device, B, R, heads, kv, D, cap, lens, window, sinks, tree, scored):
    op = check_attention(device, 450 + R, B, R, heads, kv, D, cap, lens, window=window, sinks=sinks, tree=tree, scored=scored)
    assert op.plan["rows"] == 128 and op.plan["splits"] > 1


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_nonfinite_values_in_key_ranges(device, what):
    """As below, with the keys of 128-row workgroups in several ranges: values
    at a window's edge and among the new rows."""
    g = gen(710)
    R, heads, kv, D, cap, n, window = 80, 8, 2, 128, 2400, 2303, 2000
    q, k, v = rnd(g, R, heads * D), rnd(g, 1, cap, kv, D), rnd(g, 1, cap, kv, D)
    for at in (250, 300, 1200, 2270):
        v[0, at, at // 300 % 2, at % 7::16] = what
    op = A.CacheAttention(1, R, heads, kv, D, cap, device, window=window)
    assert op.plan["rows"] == 128 and op.plan["splits"] > 1
    say("nonfinite in ranges", what)
    lens = torch.tensor([n], dtype=torch.int32)
    out = op(q.to(device), k.to(device), v.to(device), lens.to(device)).cpu().view(1, R, heads, D).double()
    ref, _, _, size, top = R64.attention(q, k, v, lens, heads=heads, R=R, window=window)
    fin = size.isfinite()
    tol = torch.where(fin, R64.attention_tolerance(torch.where(fin, ref, 0), torch.where(fin, size, 0), top, D, cap, weight_half(op)), 1.0)
    close(out, ref, tol, "out")


@pytest.mark.parametrize("B,R,heads,kv,D,cap,lens,prefix,built,window,sinks,tree", [
    (1, 1, 8, 2, 128, 40, [3], 1, None, 0, 0, False),
    (16, 1, 8, 2, 128, 60, list(range(1, 60, 4))[:15] + [0], 333, None, 0, 0, False),
    (3, 4, 32, 8, 128, 50, [50, 4, 2], 100, 128, 0, 0, True),
    (5, 1, 16, 16, 64, 70, [1, 30, 64, 65, 70], 96, None, 50, 3, False),
    (2, 3, 8, 2, 128, 70, [70, 9], 64, None, 20, 100, False),
    (2, 2, 8, 2, 128, 70, [70, 9], 0, 64, 0, 0, False),
    (7, 9, 10, 2, 128, 64, [64, 9, 10, 33, 31, 8, 0], 65, None, 64, 0, False),
    (3, 7, 8, 2, 128, 40, [5, 40, 7], 20, None, 9, 2, True),
    (40, 1, 32, 8, 128, 33, [1 + b % 33 for b in range(40)], 300, None, 0, 0, False),
    (6, 8, 16, 4, 64, 100, [100, 8, 60, 9, 7, 50], 500, None, 77, 5, True),
    (2, 40, 8, 2, 128, 64, [64, 45], 130, None, 0, 0, False),
    (70, 1, 16, 8, 64, 200, [1 + 53 * b % 200 for b in range(69)] + [0], 500, None, 0, 0, False),
    (64, 2, 8, 4, 128, 150, [2 + 37 * b % 149 for b in range(63)] + [1], 333, 400, 60, 5, False),
    (33, 4, 8, 8, 128, 300, [4 + 41 * b % 297 for b in range(33)], 70, None, 0, 0, True),
])
def test_shared_prefix(device, B, R, heads, kv, D, cap, lens, prefix, built, window, sinks, tree):
    check_attention(device, 500 + B, B, R, heads, kv, D, cap, lens, prefix=prefix, built_prefix=built, window=window,
                    sinks=sinks, tree=tree)


@pytest.mark.parametrize("B,R,heads,kv,D,cap,lens,window,sinks,tree", [
    (2, 1, 32, 8, 128, 700, [700, 45], 0, 0, False),
    (3, 1, 8, 8, 64, 129, [129, 0, 1], 0, 0, False),
    (2, 32, 8, 2, 128, 300, [300, 17], 0, 0, False),
    (2, 9, 8, 2, 128, 200, [200, 30], 25, 4, False),
    (1, 20, 8, 2, 64, 150, [140], 0, 0, True),
    (2, 4, 8, 2, 128, 150, [140, 2], 0, 0, True),
    (1, 90, 8, 4, 128, 300, [260], 0, 0, False),
    (1, 300, 4, 4, 64, 400, [333], 50, 70, False),
])
def test_scores(device, B, R, heads, kv, D, cap, lens, window, sinks, tree):
    check_attention(device, 600 + R, B, R, heads, kv, D, cap, lens, window=window, sinks=sinks, tree=tree, scored=True)


def test_scores_in_place_and_a_sum_of_weights(device):
    """In place, each call adds its rows' total weight: one per row and query head."""
    g = gen(650)
    B, R, heads, kv, D, cap = 2, 3, 8, 2, 128, 260
    op = A.CacheAttention(B, R, heads, kv, D, cap, device, scored=True)
    q, k, v = rnd(g, B * R, heads * D).to(device), rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    lens = torch.tensor([260, 100], dtype=torch.int32, device=device)
    s = torch.zeros((B, kv, cap), device=device)
    for n in range(1, 4):
        op(q, k, v, lens, scores=s)
        total = s.sum(dim=-1).cpu().double()
        want = float(n * R * heads // kv)
        # Each of the weights is off by at most 2^-16 relative (scores of a few units, fp32 sums).
        assert ((total - want).abs() <= want * 2.0 ** -16).all(), total
    assert (s[1, :, 100:] == 0).all()


@pytest.mark.parametrize("spread", [0.0, 1.0, 30.0])
def test_flat_and_peaked_scores(device, spread):
    """Equal scores, ordinary ones, and a softmax that one key dominates."""
    check_attention(device, 660, 2, 2, 8, 2, 128, 150, [150, 70], spread=spread)
    check_attention(device, 661, 1, 200, 4, 2, 128, 250, [250], spread=spread)


@pytest.mark.parametrize("R", [1, 20, 150])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e9])
def test_huge_scores(device, R, size):
    """Scores of up to 10^19: the highest key takes all of a row's weight, in the
    outputs and the scores."""
    g = gen(675)
    heads, kv, D, cap = 4, 2, 128, 300
    q, k, v = rnd(g, R, heads * D, scale=size), rnd(g, 1, cap, kv, D, scale=size / 10), rnd(g, 1, cap, kv, D)
    say("huge scores", R, size)
    op = A.CacheAttention(1, R, heads, kv, D, cap, device, scored=True)
    s = torch.zeros((1, kv, cap), device=device)
    out = op(q.to(device), k.to(device), v.to(device), torch.tensor([cap], dtype=torch.int32, device=device), scores=s)
    kh = k[0].double().repeat_interleave(heads // kv, dim=1)
    dots = torch.einsum("rhd,thd->rht", q.view(R, heads, D).double(), kh)
    dots[~(torch.arange(cap)[None] <= torch.arange(cap - R, cap)[:, None])[:, None].expand(R, heads, cap)] = -math.inf
    two = dots.topk(2, dim=-1)
    # fp32 sums of 128 products of up to (4 * size) * (4 * size / 10): off by less than 2^-9 of size^2 each.
    clear = two.values[..., 0] - two.values[..., 1] > size * size * 2.0 ** -8 + 1000
    assert clear.float().mean() > 0.9
    want = v[0].repeat_interleave(heads // kv, dim=1)[two.indices[..., 0], torch.arange(heads)]
    assert torch.equal(out.cpu().view(R, heads, D)[clear], want[clear])
    assert out.isfinite().all() and abs(float(s.sum()) - R * heads) <= 1e-3 * R * heads


@pytest.mark.parametrize("R", [1, 4, 150])
def test_other_scales(device, R):
    check_attention(device, 670, 1, R, 8, 2, 64, 300, [222], scale=1.0)
    check_attention(device, 671, 1, R, 8, 2, 64, 300, [222], scale=1e-4)


@pytest.mark.parametrize("R,window,bad", [(6, 0, 60), (6, 20, 50), (100, 0, 90), (100, 30, 60), (6, 0, 3), (100, 0, 3)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_nonfinite_values_reach_only_rows_that_see_them(device, R, window, bad, what):
    """v of one cached key holds NaN or an infinity: rows that see the key get
    it, the others are those of a finite cache."""
    g = gen(700 + R)
    heads, kv, D, cap, n = 8, 2, 128, 128, 110
    q, k, v = rnd(g, R, heads * D), rnd(g, 1, cap, kv, D), rnd(g, 1, cap, kv, D)
    at = n - R + bad if R == 100 and bad > 10 else bad
    at = min(at, n - 1)
    v[0, at, 1, 5::16] = what
    op = A.CacheAttention(1, R, heads, kv, D, cap, device, window=window)
    say("nonfinite", R, window, bad, what)
    lens = torch.tensor([n], dtype=torch.int32)
    out = op(q.to(device), k.to(device), v.to(device), lens.to(device)).cpu().view(1, R, heads, D).double()
    ref, _, _, size, top = R64.attention(q, k, v, lens, heads=heads, R=R, window=window)
    fin = size.isfinite()
    tol = torch.where(fin, R64.attention_tolerance(torch.where(fin, ref, 0), torch.where(fin, size, 0), top, D, cap, weight_half(op)), 1.0)
    assert ref.isfinite().all() == (not R64.visible(0, n, R, window, 0)[:, at].any())
    close(out, ref, tol, "out")


@pytest.mark.parametrize("R", [2, 100])
def test_nonfinite_keys_and_queries(device, R):
    """A NaN in q makes its own row and head NaN; one in k the rows that see it."""
    g = gen(720)
    heads, kv, D, cap, n = 4, 2, 128, 128, 120
    q, k, v = rnd(g, R, heads * D), rnd(g, 1, cap, kv, D), rnd(g, 1, cap, kv, D)
    op = A.CacheAttention(1, R, heads, kv, D, cap, device)
    lens = torch.tensor([n], dtype=torch.int32)
    q[0, D + 3] = math.nan
    k[0, n - 1, 1, 7] = math.nan
    out = op(q.to(device), k.to(device), v.to(device), lens.to(device)).cpu().view(R, heads, D)
    nan = torch.zeros((R, heads), dtype=torch.bool)
    nan[0, 1] = True
    nan[R - 1, 2:] = True
    assert torch.equal(out.isnan().all(dim=-1), nan) and torch.equal(out.isnan().any(dim=-1), nan)


def test_offsets_past_32_bits(device):
    """A cache whose slots lie 128 KB apart: its last keys are past 2^32 bytes
    and 2^31 elements."""
    slots, step, kv, D = 36000, 65536, 2, 128
    base = torch.zeros((slots - 1) * step + kv * 2 * D, dtype=BF, device=device)
    view = lambda off: torch.as_strided(base, (1, slots, kv, D), (0, step, 2 * D, 1), off)
    k, v = view(0), view(D)
    g = gen(730)
    heads, n = 8, slots
    near = 64
    k[0, -near:] = rnd(g, near, kv, D).to(device)
    v[0, -near:] = rnd(g, near, kv, D).to(device)
    q = rnd(g, 1, heads * D)
    lens = torch.tensor([n], dtype=torch.int32, device=device)
    say("offsets past 32 bits")
    op = A.CacheAttention(1, 1, heads, kv, D, slots, device, window=near)
    out = op(q.to(device), k, v, lens)
    ref, _, _, size, top = R64.attention(q, k[:, -near:].cpu(), v[:, -near:].cpu(), [near], heads=heads, R=1)
    close(out.view(ref.shape), ref, R64.attention_tolerance(ref, size, top, D, near, weight_half(op)), "out")
    kk, vv = k[:, -near:].clone(), v[:, -near:].clone()
    budget = 100
    score = torch.zeros((1, kv, slots), device=device)
    score[:, :, -near:] = 1.0
    ko, vo, so = (torch.zeros((1, budget, kv, D), dtype=BF, device=device) for _ in "kv"), None, None
    ko, vo = ko
    so = torch.zeros((1, kv, budget), device=device)
    keep, _ = A.CacheEviction(1, kv, D, slots, budget, device)(k, v, score, lens, out=(ko, vo, so))
    assert torch.equal(ko[:, -near:], kk) and torch.equal(vo[:, -near:], vv)
    assert torch.equal(keep[0, 0].cpu(), torch.cat([torch.arange(budget - near), torch.arange(slots - near, slots)]).int())


# ------------------------------------------------------------------- rope
@pytest.mark.parametrize("B,R,heads,kv,D,lens,norm,inplace,explicit", [
    (1, 1, 32, 8, 128, [1], True, False, False),
    (3, 5, 32, 8, 128, [5, 40, 3], True, False, False),
    (2, 33, 6, 2, 64, [33, 60], True, True, False),
    (2, 7, 4, 4, 64, [60, 0], False, False, True),
    (1, 60, 5, 1, 128, [60], True, True, True),
])
@pytest.mark.parametrize("layout", ["slots", "heads"])
def test_rope(device, B, R, heads, kv, D, lens, norm, inplace, explicit, layout):
    g = gen(800 + R)
    cap, theta, eps = 64, 1e6, 1e-6
    qkv = rnd(g, B * R, (heads + 2 * kv) * D)
    qn, kn = (rnd(g, D, scale=0.1, shift=1.0) for _ in "qk")
    shape = (B, cap, kv, D) if layout == "slots" else (B, kv, cap, D)
    k, v = (torch.full(shape, 9.0, dtype=BF, device=device) for _ in "kv")
    if layout != "slots":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    table = A.rope_table(5000, D, theta, device)
    slots = torch.tensor([n - R + i for n in lens for i in range(R)])
    pos = torch.randint(0, 5000, (B * R,), generator=g) if explicit else slots.clamp(min=0)
    if explicit:
        pos[0] = 4999
        pos[B * R // 2] = 5000  # outside the table: left as it was
        pos[-1] = -1
    ok = (slots >= 0) & (pos >= 0) & (pos < 5000)
    x = qkv.to(device)
    q_out = x[:, :heads * D] if inplace else torch.full((B * R, heads * D), 9.0, dtype=BF, device=device)
    before = q_out.clone()
    got = A.qk_norm_rope(x, qn.to(device) if norm else None, kn.to(device) if norm else None, eps, table,
                         torch.tensor(lens, dtype=torch.int32, device=device), k, v,
                         positions=pos.int().to(device) if explicit else None, q_out=q_out)
    assert got is q_out
    (rq, sq), (rk, sk), rv = R64.rope(qkv, qn if norm else None, kn if norm else None, eps, theta, pos, heads, kv, D)
    # fp32: the norm (D sums, root, two products), the table's rounding, two products and a sum; then bf16.
    rel = (D + 16) * R64.FP32_HALF
    tol = lambda r, s: R64.BF16_HALF * r.abs() * 1.01 + s * rel
    q = got.view(B * R, heads, D)
    close(q[ok], rq[ok], tol(rq, sq)[ok], "q")
    assert torch.equal(q[~ok], before.view(B * R, heads, D)[~ok])
    want_k, want_v = torch.full((B, cap, kv, D), 9.0, dtype=torch.float64), torch.full((B, cap, kv, D), 9.0, dtype=torch.float64)
    tk = torch.zeros((B, cap, kv, D), dtype=torch.float64)
    for m in range(B * R):
        if ok[m]:
            want_k[m // R, slots[m]], want_v[m // R, slots[m]] = rk[m], rv[m]
            tk[m // R, slots[m]] = tol(rk, sk)[m]
    close(k, want_k, tk + 1e-30, "k")
    assert torch.equal(v.cpu().double(), want_v)


# ------------------------------------------------------------------ evict
def some_scores(g, B, kv, cap, kind):
    if kind == "ties":
        return torch.randint(0, 3, (B, kv, cap), generator=g).float()
    s = torch.randn((B, kv, cap), generator=g)
    if kind == "special":
        s[..., ::7] = math.nan
        s[..., 1::9] = math.inf
        s[..., 2::9] = -math.inf
        s[..., 3::5] = 0.0
        s[..., 4::5] = -0.0
        s[..., 5::11] = 1e-42
    if kind == "close":  # the keys differ in their last bits only
        s = torch.ones_like(s) + torch.randint(0, 40, s.shape, generator=g) * 2.0 ** -23
    return s


EVICT = [
    # B, kv, D, cap, budget, sinks, recent, lens
    (1, 8, 128, 100, 40, 4, 10, [100]),
    (3, 2, 64, 300, 64, 0, 0, [300, 64, 65]),
    (4, 1, 128, 700, 1, 0, 0, [700, 0, 1, 2]),
    (2, 2, 128, 2500, 1000, 7, 993, [2500, 1001]),
    (2, 2, 128, 3001, 1500, 1, 64, [3001, -3]),
    (1, 1, 64, 70000, 5000, 4, 100, [69999]),
    (1, 2, 128, 50, 50, 3, 3, [50]),
]


@pytest.mark.parametrize("case", range(len(EVICT)))
@pytest.mark.parametrize("kind", ["plain", "ties", "special", "close"])
@pytest.mark.parametrize("inplace", [False, True])
def test_evict(device, case, kind, inplace):
    B, kv, D, cap, budget, sinks, recent, lens = EVICT[case]
    g = gen(900 + case)
    s = some_scores(g, B, kv, cap, kind)
    k, v = rnd(g, B, cap, kv, D), rnd(g, B, cap, kv, D)
    say("evict", case, kind, inplace)
    op = A.CacheEviction(B, kv, D, cap, budget, device, sinks=sinks, recent=recent)
    kd, vd, sd = k.to(device), v.to(device), s.to(device)
    ln = torch.tensor(lens, dtype=torch.int32, device=device)
    more = 3
    if inplace:
        keep, lens_out = torch.empty((B, kv, budget), dtype=torch.int32, device=device), ln
        op.run(kd, vd, sd, ln, keep, ln)
        ko, vo, so = kd.cpu(), vd.cpu(), sd.cpu()
    else:
        out = (torch.full((B, budget + more, kv, D), 9.0, dtype=BF, device=device),
               torch.full((B, kv, budget, D), 9.0, dtype=BF, device=device).transpose(1, 2),
               torch.full((B, kv, budget + more), 9.0, device=device))
        keep, lens_out = op(kd, vd, sd, ln, out=out)
        assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
        ko, vo, so = (t.cpu() for t in out)
    kept = R64.evict(s, lens, budget, sinks, recent)
    assert lens_out.cpu().tolist() == [max(0, min(n, cap, budget)) for n in lens]
    for b in range(B):
        for h in range(kv):
            want = kept[b][h]
            n = len(want)
            assert keep[b, h].cpu().tolist() == want + [-1] * (budget - n), (b, h)
            if n:
                assert torch.equal(ko[b, :n, h], k[b, want, h]) and torch.equal(vo[b, :n, h], v[b, want, h])
                assert torch.equal(so[b, h, :n].view(torch.int32), s[b, h, want].view(torch.int32))
            if inplace:
                assert torch.equal(ko[b, budget:, h], k[b, budget:, h]) and torch.equal(vo[b, budget:, h], v[b, budget:, h])
                if n < budget:
                    assert torch.equal(ko[b, :, h], k[b, :, h])
            else:
                assert (ko[b, n:, h] == 9).all() and (vo[b, n:, h] == 9).all() and (so[b, h, n:] == 9).all()


def test_scores_of_rows_that_see_none_of_the_new(device):
    """Tree masks without bits: the call's own keys get no weight, also where an
    earlier call on the same workspace gave them some."""
    g = gen(655)
    B, R, heads, kv, D, cap = 2, 4, 8, 2, 128, 400
    op = A.CacheAttention(B, R, heads, kv, D, cap, device, scored=True)
    q, k, v = rnd(g, B * R, heads * D).to(device), rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    lens = torch.tensor([400, 259], dtype=torch.int32, device=device)
    masks = torch.ones((B, R), dtype=torch.int64, device=device)
    for tree, new in ((masks * 15, True), (masks * 0, False)):
        s = torch.zeros((B, kv, cap), device=device)
        say("scores without bits", new)
        op(q, k, v, lens, tree=tree, scores=s)
        for b, n in enumerate((400, 259)):
            assert bool((s[b, :, n - R:n] > 0).all()) == new and bool((s[b, :, n - R:n] == 0).all()) != new
            assert ((s[b].sum(-1) - R * heads // kv).abs() < 1e-3).all()


# ------------------------------------------------- streams, graphs, devices
def test_on_another_stream_and_in_graphs(device):
    """Calls run on the current stream; two captured graphs of two objects,
    replayed in turn with eager calls between, give the eager results for the
    lengths of each replay."""
    g = gen(1000)
    B, heads, kv, D, cap = 4, 32, 8, 128, 3000
    k, v = rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    kp, vp = rnd(g, 500, kv, D).to(device), rnd(g, 500, kv, D).to(device)
    q = rnd(g, B, heads * D).to(device)
    lens = torch.tensor([3000, 1, 700, 0], dtype=torch.int32, device=device)
    one = A.CacheAttention(B, 1, heads, kv, D, cap, device, window=256, sinks=4, scored=True)
    two = A.CacheAttention(B, 1, heads, kv, D, cap, device, prefix=500)
    s0 = torch.zeros((B, kv, cap), device=device)
    s1 = torch.zeros_like(s0)
    ev = A.CacheEviction(B, kv, D, cap, 128, device, sinks=4, recent=16)
    ko, vo = (torch.zeros((B, 128, kv, D), dtype=BF, device=device) for _ in "kv")
    so = torch.zeros((B, kv, 128), device=device)

    def both():
        a = one(q, k, v, lens, scores=s0, scores_out=s1)
        keep, n = ev(k, v, s1, lens, out=(ko, vo, so))
        return a, s1, keep, n, ko, vo, so

    def other():
        return (two(q, k, v, lens, prefix=(kp, vp)),)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [t.clone() for t in both() + other()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, both() + other()):
        assert torch.equal(a, b)
    graphs = []
    for fn in (both, other):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = fn()
        graphs.append((gr, fn, out))
    for rep, ln in enumerate(([3000, 1, 700, 0], [5, 2999, 129, 128], [0, 0, 0, 0], [300, 300, 300, 300])):
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        for gr, fn, out in graphs:
            for t in (ko, vo, so, s1):
                t.zero_()
            want = [t.clone() for t in fn()]
            for t in (ko, vo, so, s1):
                t.zero_()
            gr.replay()
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(want, out)):
                assert torch.equal(a, b), (rep, i)


def test_same_call_twice_is_bit_equal(device):
    g = gen(1010)
    for R, kw in ((1, {}), (1, dict(prefix=700)), (16, {}), (300, dict(window=64, sinks=2))):
        B, heads, kv, D, cap = 3, 16, 4, 128, 900
        op = A.CacheAttention(B, R, heads, kv, D, cap, device, **kw)
        q = rnd(g, B * R, heads * D).to(device)
        k, v = rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
        shared = tuple(rnd(g, 700, kv, D).to(device) for _ in "kv") if kw.get("prefix") else None
        lens = torch.tensor([900, 500, 301], dtype=torch.int32, device=device)
        a = op(q, k, v, lens, prefix=shared)
        b = op(q, k, v, lens, prefix=shared)
        assert torch.equal(a, b)


def test_offsets_past_32_bits_for_many_rows(device):
    """The same distances for the tile kernel, the weights' second reading of K,
    and the cache write: rows of the last 200 slots."""
    slots, step, kv, D, heads, R = 36000, 65536, 2, 128, 8, 200
    base = torch.zeros((slots - 1) * step + kv * 2 * D, dtype=BF, device=device)
    view = lambda off: torch.as_strided(base, (1, slots, kv, D), (0, step, 2 * D, 1), off)
    k, v = view(0), view(D)
    g = gen(740)
    qkv = rnd(g, R, (heads + 2 * kv) * D).to(device)
    lens = torch.tensor([slots], dtype=torch.int32, device=device)
    table = A.rope_table(slots, D, 1e6, device)
    say("offsets past 32 bits, many rows")
    q = A.qk_norm_rope(qkv, None, None, 1e-6, table, lens, k, v)
    near = 2 * R
    kc, vc = torch.zeros((1, near, kv, D), dtype=BF), torch.zeros((1, near, kv, D), dtype=BF)
    kn, vn = kc.to(device), vc.to(device)
    again = A.qk_norm_rope(qkv, None, None, 1e-6, table, torch.tensor([near], dtype=torch.int32, device=device), kn, vn,
                           positions=torch.arange(slots - R, slots, dtype=torch.int32, device=device))
    assert torch.equal(q, again)
    assert torch.equal(k[:, -R:], kn[:, -R:]) and torch.equal(v[:, -R:], vn[:, -R:])
    say("attention")
    op = A.CacheAttention(1, R, heads, kv, D, slots, device, window=100, scored=True)
    small = A.CacheAttention(1, R, heads, kv, D, near, device, window=100, scored=True)
    s, t = torch.zeros((1, kv, slots), device=device), torch.zeros((1, kv, near), device=device)
    a = op(q, k, v, lens, scores=s)
    b = small(q, kn, vn, torch.tensor([near], dtype=torch.int32, device=device), scores=t)
    # Other steps and ranges.  Each side's weights are off by 2^-8, its outputs
    # by 2^-8 of at most the largest value; its scores by at most D * 2^-24 of
    # sum |q k| * scale, about 100 * 0.09 here, so a weight by less than 2^-13.
    assert ((a.double() - b.double()).abs() <= 2.0 ** -6 * vn.abs().max()).all()
    assert ((s[..., -near:] - t).abs() <= 2.0 ** -11 * t).all() and (s[..., :-near] == 0).all()


@pytest.mark.parametrize("what", ["decode", "scored", "tree", "prompt", "prompt_scored", "shared"])
def test_replays_follow_the_lengths(device, what):
    """A graph of the cache write and the attention behind it: every replay, at
    other lengths and rows, equals the eager calls bit by bit."""
    g = gen(1020)
    heads, kv, D, cap = 16, 4, 128, 1200
    B, R, kw = {"decode": (3, 1, {}), "scored": (3, 1, dict(scored=True)), "tree": (2, 8, {}), "prompt": (2, 100, {}),
                "prompt_scored": (2, 100, dict(scored=True)), "shared": (5, 1, dict(prefix=333))}[what]
    op = A.CacheAttention(B, R, heads, kv, D, cap, device, **kw)
    table = A.rope_table(4000, D, 1e6, device)
    k, v = rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    qkv = rnd(g, B * R, (heads + 2 * kv) * D).to(device)
    lens = torch.full((B,), R, dtype=torch.int32, device=device)
    more = {}
    if what == "tree":
        more["tree"] = tree_masks(g, B, R).to(device)
    if what == "shared":
        more["prefix"] = tuple(rnd(g, 333, kv, D).to(device) for _ in "kv")
    s = torch.zeros((B, kv, cap), device=device)
    if kw.get("scored"):
        more["scores"] = s
    q = torch.empty((B * R, heads * D), dtype=BF, device=device)
    out = torch.empty_like(q)

    def run():
        A.qk_norm_rope(qkv, None, None, 1e-6, table, lens, k, v, q_out=q)
        op.run(q, k, v, lens, out, **more)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    k0, v0 = k.clone(), v.clone()
    for n in range(4):
        lens.copy_(torch.randint(0, cap + 1, (B,), generator=g).int())
        qkv.copy_(rnd(g, *qkv.shape))
        got = []
        for call in (run, graph.replay):
            k.copy_(k0), v.copy_(v0), s.zero_(), q.zero_()
            call()
            torch.cuda.synchronize()
            got.append([t.clone() for t in (out, k, v, s)])
        for a, b in zip(*got):
            assert torch.equal(a, b), n


def test_two_objects_on_two_streams(device):
    """Objects have workspaces of their own, so their calls may run at once."""
    g = gen(1030)
    B, heads, kv, D, cap = 2, 32, 8, 128, 3000
    k, v = rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    q = [rnd(g, B, heads * D).to(device) for _ in range(2)]
    lens = torch.tensor([3000, 1700], dtype=torch.int32, device=device)
    ops = [A.CacheAttention(B, 1, heads, kv, D, cap, device) for _ in range(2)]
    want = [op(x, k, v, lens) for op, x in zip(ops, q)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [[torch.empty_like(w) for _ in range(20)] for w in want]
    torch.cuda.synchronize()
    for n in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                ops[i].run(q[i], k, v, lens, out[i][n])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in out[i])


def test_broadcast_caches(device):
    """Caches expanded over sequences and heads (strides of 0) are read as such."""
    g = gen(1040)
    for R in (1, 100):
        B, heads, kv, D, cap = 3, 8, 4, 64, 200
        k, v = rnd(g, 1, cap, 1, D).to(device), rnd(g, 1, cap, 1, D).to(device)
        q = rnd(g, B * R, heads * D).to(device)
        lens = torch.tensor([200, 130, 101], dtype=torch.int32, device=device)
        op = A.CacheAttention(B, R, heads, kv, D, cap, device)
        wide = [t.expand(B, cap, kv, D) for t in (k, v)]
        assert torch.equal(op(q, *wide, lens), op(q, *(t.contiguous() for t in wide), lens))
