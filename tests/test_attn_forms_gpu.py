"""Cache attention and eviction in the forms that the library chooses by shape,
each against the 64-bit oracle and named by its plan."""

from __future__ import annotations

import math

import pytest
import torch

from kernels import attention as A
from oracle import attn_ref as R64

from test_attn_gpu import BF, check_attention, close, gen, poison, rnd, say, some_scores, weight_half

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
