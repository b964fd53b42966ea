"""Low-rank adapters on the GPU against the 64-bit oracle."""

from __future__ import annotations

import math

import pytest
import torch

import kernels as K
from oracle import paged_ref as P64
from test_attn_gpu import close, gen, rnd, say

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32


def factors(g, n, widths, K_, rank):
    return rnd(g, n, len(widths) * rank, K_, scale=K_ ** -0.5), rnd(g, n, sum(widths), rank, scale=0.2)


def check(dev, seed, rows, widths, K_, rank, n, index, silu=False, scaled=True, strided=False, in_place=False):
    g = gen(seed)
    N = sum(widths)
    x, y = rnd(g, rows, K_), rnd(g, rows, N)
    a, b = factors(g, n, widths, K_, rank)
    scale = torch.rand(n, generator=g) * 3 - 1 if scaled else None
    if index == "random":
        index = torch.randint(-1, n, (rows,), generator=g)
    elif index == "runs":
        index = torch.randint(-1, n, (rows // 21 + 1,), generator=g).repeat_interleave(21)[:rows]
    else:
        index = torch.tensor([index[i % len(index)] for i in range(rows)])
    index = index.to(I32)
    say("adapters", seed, rows, widths, K_, rank, n, silu, strided, in_place)
    op = K.LowRankAdapters(rows, N, K_, rank, dev, slices=None if len(widths) == 1 else widths, silu=silu)
    xd, yd, ad, bd = x.to(dev), y.to(dev), a.to(dev), b.to(dev)
    if strided:
        xd = torch.cat([xd, xd], dim=1)[:, :K_]
        yd = torch.cat([yd, yd], dim=1)[:, N:]
        ad = torch.cat([ad, ad], dim=2)[:, :, :K_]
        bd = torch.cat([bd, bd], dim=1)[:, :N]
    kw = dict(scale=None if scale is None else scale.to(dev))
    first = op(xd, ad, bd, index.to(dev), yd, **kw)
    if in_place:
        yy = yd.clone()
        assert op.run(xd, ad, bd, index.to(dev), yy, yy, **kw) is yy
        assert torch.equal(yy.view(torch.int16), first.view(torch.int16))
    torch.cuda.synchronize()
    ref, tol = P64.adapters(x, a, b, index, y, scale, widths, rank, silu)
    close(first, ref, tol, "out")
    assert torch.equal(op(xd, ad, bd, index.to(dev), yd, **kw).view(torch.int16), first.view(torch.int16))
    return first


CASES = [
    # rows, widths, K, rank, adapters, index
    (1, [8], 8, 8, 1, [0]),
    (1, [2560], 2560, 16, 3, [2]),
    (1, [64], 512, 16, 3, [-1]),
    (5, [1024, 256, 256], 1024, 16, 4, "random"),
    (16, [640, 72], 520, 8, 2, [0, 1, -1, 5]),
    (17, [200], 136, 24, 40, "random"),
    (33, [2560], 9728, 64, 7, "random"),
    (64, [96, 96, 96, 96], 256, 128, 5, "random"),
    (100, [1536], 264, 40, 3, [0]),
    (257, [512, 128, 128], 384, 16, 6, "runs"),
    (300, [328], 1000, 32, 9, "random"),
    (1031, [264], 640, 48, 4, "runs"),
    (300, [264], 9728, 16, 4, "runs"),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("form", ["plain", "strided"])
def test_adapters(device, case, form):
    rows, widths, K_, rank, n, index = CASES[case]
    check(device, 900 + case, rows, widths, K_, rank, n, index, scaled=form == "plain", strided=form == "strided", in_place=True)


@pytest.mark.parametrize("rows,widths,K_,rank,n,index", [
    (1, [16], 64, 8, 1, [0]), (3, [1024, 1024], 256, 16, 2, [1, -1, 0]), (64, [200, 200], 520, 32, 8, "random"),
    (70, [400], 128, 8, 3, "runs"), (260, [136, 136], 256, 64, 2, "random"),
])
def test_silu(device, rows, widths, K_, rank, n, index):
    check(device, 950 + rows, rows, widths, K_, rank, n, index, silu=True, strided=rows == 64)


def test_rows_without_an_adapter_are_copied(device):
    """Bit for bit, -0 and what is not finite too; in place they stay."""
    g = gen(3)
    y = rnd(g, 40, 128)
    y[3, ::3], y[4, ::2], y[5, 1::2] = -0.0, math.inf, -math.inf
    index = torch.full((40,), -1, dtype=I32)
    index[10:20], index[30] = 7, -2147483648  # 7: behind the last
    a, b = factors(g, 7, [128], 256, 16)
    op = K.LowRankAdapters(40, 128, 256, 16, device)
    x = rnd(g, 40, 256).to(device)
    out = op(x, a.to(device), b.to(device), index.to(device), y.to(device))
    assert torch.equal(out.cpu().view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("rows", [20, 300])
def test_rows_do_not_reach_into_each_other(device, rows):
    g = gen(4)
    widths, K_, rank, n = [192], 264, 16, 3
    x, y = rnd(g, rows, K_), rnd(g, rows, 192)
    a, b = factors(g, n, widths, K_, rank)
    index = torch.randint(-1, n, (rows,), generator=g).to(I32)
    op = K.LowRankAdapters(rows, 192, K_, rank, device)
    args = [t.to(device) for t in (x, a, b, index, y)]
    clean = op(*args)
    bad = torch.arange(0, rows, 3)
    x[bad[::2], 7], x[bad[1::2], 5] = math.nan, math.inf
    args[0] = x.to(device)
    op.workspace.fill_(0xff)  # NaN: nothing is left of what a workspace held
    got = op(*args)
    keep = torch.ones(rows, dtype=torch.bool)
    keep[bad[index[bad] >= 0]] = False
    assert torch.equal(got[keep.to(device)], clean[keep.to(device)])
    a[1], b[1] = math.nan, math.inf  # another adapter
    got = op(x.to(device), a.to(device), b.to(device), index.to(device), y.to(device))
    keep &= index != 1
    assert torch.equal(got[keep.to(device)], clean[keep.to(device)])


def test_captured_with_other_adapters(device):
    g = gen(8)
    rows, widths, K_, rank, n = 24, [256, 64, 64], 512, 16, 5
    x, y, (a, b) = rnd(g, rows, K_), rnd(g, rows, 384), factors(g, n, widths, K_, rank)
    scale = torch.rand(n, generator=g)
    index = torch.randint(-1, n, (rows,), generator=g).to(I32).to(device)
    op = K.LowRankAdapters(rows, 384, K_, rank, device, slices=widths)
    xd, ad, bd, yd, sd = (t.to(device) for t in (x, a, b, y, scale))
    out = torch.empty_like(yd)
    op.run(xd, ad, bd, index, yd, out, scale=sd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run(xd, ad, bd, index, yd, out, scale=sd)
    for i in range(4):
        index.copy_(torch.randint(-1, n, (rows,), generator=g).to(I32).to(device))
        sd.copy_(torch.rand(n, generator=g).to(device))
        graph.replay()
        torch.cuda.synchronize()
        ref, tol = P64.adapters(x, a, b, index.cpu(), y, sd.cpu(), widths, rank)
        close(out, ref, tol, f"replay {i}")
        assert torch.equal(op(xd, ad, bd, index, yd, scale=sd), out)


def test_python_refusals(device):
    op = K.LowRankAdapters(4, 64, 128, 8, device)
    x, y = torch.zeros((4, 128), dtype=BF, device=device), torch.zeros((4, 64), dtype=BF, device=device)
    a, b = torch.zeros((2, 8, 128), dtype=BF, device=device), torch.zeros((2, 64, 8), dtype=BF, device=device)
    index = torch.zeros(4, dtype=I32, device=device)
    good = dict(x=x, a=a, b=b, index=index, y=y)
    op(**good)
    for name, bad in (("x", x[:3]), ("x", x.float()), ("a", a[0]), ("a", a[:, :4]), ("b", b[:1]), ("b", b[..., ::2]), ("index", index.long()),
                      ("index", index[:3]), ("y", y.cpu()), ("y", y[:, :32])):
        with pytest.raises(ValueError, match=name):
            op(**{**good, name: bad})
    with pytest.raises(ValueError, match="scale"):
        op(**good, scale=torch.ones(3, device=device))
