"""Cache attention and eviction in the forms that the library chooses by shape,
each against the 64-bit oracle and named by its plan."""

from __future__ import annotations

import math

import pytest
import torch

from kernels import attention as A
from oracle import attn_ref as R64

from test_attn_gpu import BF, check_attention, close, gen, rnd, say, some_scores, weight_half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [1, 20, 150])
def test_the_largest_and_smallest_scales(device, R):
    """At the largest scale the highest score takes all the weight; at the
    smallest all visible keys weigh the same."""
    g = gen(1200 + R)
    heads, kv, D, cap = 4, 2, 128, 300
    q, k, v = rnd(g, R, heads * D), rnd(g, 1, cap, kv, D), rnd(g, 1, cap, kv, D)
    lens = torch.tensor([cap], dtype=torch.int32, device=device)
    run = lambda scale: A.CacheAttention(1, R, heads, kv, D, cap, device, scale=scale)(
        q.to(device), k.to(device), v.to(device), lens).cpu().view(R, heads, D)
    say("scales", R)
    dots = torch.einsum("rhd,thd->rht", q.view(R, heads, D).double(), k[0].double().repeat_interleave(heads // kv, dim=1))
    hidden = ~(torch.arange(cap)[None] <= torch.arange(cap - R, cap)[:, None])
    dots[hidden[:, None].expand(R, heads, cap)] = -math.inf
    two = dots.topk(2, dim=-1)
    clear = two.values[..., 0] - two.values[..., 1] > 1e-2  # fp32 sums of 128 products of up to 16: off by less than 2^-9
    want = v[0].repeat_interleave(heads // kv, dim=1)[two.indices[..., 0], torch.arange(heads)]
    assert clear.float().mean() > 0.9 and torch.equal(run(2.29e38)[clear], want[clear])
    mean = torch.stack([v[0, :cap - R + 1 + i].double().mean(dim=0) for i in range(R)]).repeat_interleave(heads // kv, dim=1)
    size = torch.stack([v[0, :cap - R + 1 + i].double().abs().mean(dim=0) for i in range(R)]).repeat_interleave(heads // kv, dim=1)
    # Weights are exactly 1; fp32 sums over the keys, one rounding to bf16.
    close(run(1e-44), mean, R64.BF16_HALF * mean.abs() * 1.01 + size * (2 * cap + 16) * R64.FP32_HALF, "mean")


@pytest.mark.parametrize("axis", [1, 2, 3])
def test_k_and_v_side_by_side_in_one_tensor(device, axis):
    """k and v as halves of one tensor, interleaved by sequence, slot or head:
    the cache write and the eviction in place equal those of separate caches."""
    g = gen(1210)
    B, cap, heads, kv, D = 2, 40, 8, 2, 128
    dims = [B, cap, kv, D]
    both = rnd(g, *dims[:axis], 2, *dims[axis:]).to(device)
    k, v = both.select(axis, 0), both.select(axis, 1)
    k2, v2 = k.contiguous(), v.contiguous()
    qkv = rnd(g, B * 3, (heads + 2 * kv) * D).to(device)
    lens = torch.tensor([40, 20], dtype=torch.int32, device=device)
    table = A.rope_table(50, D, 1e6, device)
    say("side by side", axis)
    q = [A.qk_norm_rope(qkv, None, None, 1e-6, table, lens, *c) for c in ((k, v), (k2, v2))]
    assert torch.equal(*q) and torch.equal(k, k2) and torch.equal(v, v2)
    s = torch.rand((B, kv, cap), generator=g).to(device)
    op = A.CacheEviction(B, kv, D, cap, 17, device, sinks=1, recent=3)
    keep = [op(*c, s.clone(), lens)[0] for c in ((k, v), (k2, v2))]
    assert torch.equal(*keep) and torch.equal(k, k2) and torch.equal(v, v2)


#: Own caches in several key ranges behind a shared prefix, by the rows of a
#: workgroup of the own caches' and of the prefix's.
BEHIND_A_PREFIX = {
    "16, 16": dict(B=1, R=1, heads=32, kv=8, D=128, cap=3000, lens=[2900], prefix=1000),
    "16, 16 of more": dict(B=3, R=1, heads=8, kv=2, D=64, cap=1500, lens=[1500, 0, 130], prefix=300),
    "16, 32": dict(B=8, R=1, heads=32, kv=8, D=128, cap=1000, lens=[1000, 1, 0, 129, 500, 257, 999, 64], prefix=500),
    "16, 32 window": dict(B=5, R=2, heads=16, kv=4, D=64, cap=700, lens=[700, 2, 131, 1, 600], prefix=260, window=300, sinks=5),
    "32, 32": dict(B=1, R=8, heads=32, kv=8, D=128, cap=1000, lens=[900], prefix=400),
    "32, 32 tree": dict(B=2, R=16, heads=8, kv=4, D=128, cap=800, lens=[800, 16], prefix=300, tree=True),
    "16, 128": dict(B=20, R=1, heads=32, kv=8, D=128, cap=2000, lens=[2000 - 97 * b for b in range(19)] + [0], prefix=300),
    "16, 128 tree": dict(B=10, R=3, heads=12, kv=4, D=64, cap=900, lens=[900 - 83 * b for b in range(10)], prefix=200, tree=True),
    "32, 128": dict(B=4, R=8, heads=32, kv=8, D=128, cap=1000, lens=[1000, 8, 500, 3], prefix=500),
    "32, 128 window": dict(B=4, R=9, heads=16, kv=4, D=128, cap=900, lens=[900, 9, 333, 700], prefix=300, window=400, sinks=7),
    "128, 128": dict(B=1, R=50, heads=8, kv=2, D=128, cap=2600, lens=[2500], prefix=700),
    "128, 128 window": dict(B=2, R=40, heads=8, kv=2, D=64, cap=3000, lens=[2900, 41], prefix=200, window=2600, sinks=9),
}


@pytest.mark.parametrize("form", BEHIND_A_PREFIX)
@pytest.mark.parametrize("layout", ["slots", "heads"])
def test_key_ranges_behind_a_prefix(device, form, layout):
    op = check_attention(device, 1300 + len(form), **BEHIND_A_PREFIX[form], layout=layout)
    own, prefix = (int(n.strip(",")) for n in form.split()[:2])
    assert (op.plan["rows"], op.plan["prefix_rows"]) == (own, prefix) and op.plan["splits"] > 1


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("B,R,window,sinks,rows", [(2, 1, 0, 0, 16), (2, 1, 60, 3, 16), (10, 1, 60, 0, 32), (30, 1, 0, 0, 128),
                                                    (30, 1, 60, 2, 128), (2, 40, 100, 2, 128)])
def test_nonfinite_values_in_a_shared_prefix(device, what, B, R, window, sinks, rows):
    """One of the first prefix keys and one of the last hold NaN or an infinity:
    with a window only some sequences' rows see them."""
    g = gen(1400 + B)
    heads, kv, D, cap, P = 8, 2, 128, 90, 150
    lens = [R + (b * 37) % (cap - R + 1) for b in range(B)]
    q, k, v = rnd(g, B * R, heads * D), rnd(g, B, cap, kv, D), rnd(g, B, cap, kv, D)
    kp, vp = rnd(g, P, kv, D), rnd(g, P, kv, D)
    vp[1, 0, 3::16] = what
    vp[P - 9, 1, 5::16] = what
    op = A.CacheAttention(B, R, heads, kv, D, cap, device, window=window, sinks=sinks, prefix=P)
    assert op.plan["prefix_rows"] == rows
    say("nonfinite prefix", what, B, R, window, sinks)
    ln = torch.tensor(lens, dtype=torch.int32, device=device)
    out = op(q.to(device), k.to(device), v.to(device), ln, prefix=(kp.to(device), vp.to(device))).cpu().view(B, R, heads, D).double()
    ref, _, _, size, top = R64.attention(q, k, v, lens, heads=heads, R=R, window=window, sinks=sinks, prefix=(kp, vp))
    fin = size.isfinite()
    tol = torch.where(fin, R64.attention_tolerance(torch.where(fin, ref, 0), torch.where(fin, size, 0), top, D, P + cap, weight_half(op)), 1.0)
    assert bool(ref.isfinite().all()) is False
    close(out, ref, tol, "out")


@pytest.mark.parametrize("cap,budget,lens", [(4096, 1000, [4096, 1001]), (4097, 700, [4097, 3000]), (5000, 4999, [5000, 10]),
                                             (12288, 4096, [12288, 5000]), (12289, 2000, [12289, 1999]), (36864, 5000, [36864, 20000]),
                                             (36865, 3000, [36865, 3001])])
@pytest.mark.parametrize("kind", ["plain", "ties", "special", "close"])
@pytest.mark.parametrize("inplace", [False, True])
def test_eviction_at_the_kernels_capacities(device, cap, budget, lens, kind, inplace):
    """Either side of the lengths at which a lane holds 4, 12, 36 keys, or none."""
    g = gen(1500 + cap)
    B, kv, D, sinks, recent = 2, 2, 64, 3, 100
    s = some_scores(g, B, kv, cap, kind)
    k, v = rnd(g, B, cap, kv, D), rnd(g, B, cap, kv, D)
    say("evict", cap, kind, inplace)
    op = A.CacheEviction(B, kv, D, cap, budget, device, sinks=sinks, recent=recent)
    kd, vd, sd = k.to(device), v.to(device), s.to(device)
    ln = torch.tensor(lens, dtype=torch.int32, device=device)
    out = None if inplace else (torch.zeros((B, budget, kv, D), dtype=BF, device=device),
                                torch.zeros((B, budget, kv, D), dtype=BF, device=device), torch.zeros((B, kv, budget), device=device))
    keep, after = op(kd, vd, sd, ln, out=out)
    ko, vo, so = (t.cpu() for t in (out or (kd, vd, sd)))
    assert after.cpu().tolist() == [min(n, budget) for n in lens]
    for b, heads in enumerate(R64.evict(s, lens, budget, sinks, recent)):
        for h, want in enumerate(heads):
            n = len(want)
            assert keep[b, h].cpu().tolist() == want + [-1] * (budget - n), (b, h)
            assert torch.equal(ko[b, :n, h], k[b, want, h]) and torch.equal(vo[b, :n, h], v[b, want, h])
            assert torch.equal(so[b, h, :n].view(torch.int32), s[b, h, want].view(torch.int32))
