"""Forms of the paged attention and of the adapters that calls reach by their sizes
alone, against the 64-bit oracle: jobs of both kinds in turn, ranges cut anew where all
work is long, ranges joined in groups at head size 64, the largest rank over many rows;
and the norm and the projection that run by themselves where adapters follow them."""

from __future__ import annotations

import pytest
import torch

import kernels as K
from kernels import cache as C
from kernels import serve as V
from kernels import step as S
from oracle import gemm_ref as R

from test_adapters_gpu import check
from test_attn_gpu import close
from test_paged_gpu import check_step
from test_paged_step_gpu import CheckedStep, adapter_set, model, rows_of  # noqa: F401  (model: a fixture)

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32
STEP = 2.0 ** -8  # of a rounding to bf16, relative

#: new rows, keys, heads, kv, D, P, window, sinks, and what the cut has to come to (tests/test_paged_cut_cpu.py)
FORMS = {
    # 256 jobs and more of either kind, in turn, then what is left of one.
    "both kinds": ([1, 550] + [1 + 2 * (i % 3 == 0) for i in range(40)] + [2] * 20, [900, 700] + [(97 * i) % 600 + 20 for i in range(60)],
                   64, 4, 128, 16, 0, 0, dict(pairs=1)),
    "both kinds, window": ([550] + [1 + 2 * (i % 2) for i in range(63)], [1100] + [(61 * i) % 400 + 20 for i in range(63)],
                           64, 4, 64, 32, 200, 4, dict(pairs=1)),
    "both kinds, listed": ([1] * 40 + [550] + [2] * 40, [(97 * i) % 600 + 20 for i in range(40)] + [560] + [(31 * i) % 300 + 2 for i in range(40)],
                           64, 4, 128, 16, 0, 0, dict(pairs=1)),
    "both kinds, listed, window": ([1, 300] + [1] * 70 + [300], [90, 1300] + [(97 * i) % 900 + 20 for i in range(70)] + [300],
                                   64, 4, 64, 8, 150, 9, dict(pairs=1)),
    # A long share of work: short ranges, several a tile.
    "cut anew": ([1] * 60 + [2, 1, 16, 1], [(131 * i) % 700 + 300 for i in range(60)] + [6000, 9000, 5000, 7000], 32, 8, 128, 64, 0, 0,
                 dict(rounds=2, few_parts=9)),
    "cut anew, window": ([1] * 60 + [2, 1, 16, 1], [(131 * i) % 700 + 300 for i in range(60)] + [6000, 9000, 5000, 7000], 32, 8, 128, 64, 4000, 4,
                         dict(rounds=2, few_parts=5)),
    "cut anew, listed": ([1] * 90 + [2, 1, 16, 1], [(131 * i) % 700 + 300 for i in range(90)] + [6000, 9000, 5000, 7000], 8, 8, 64, 16, 0, 0,
                         dict(rounds=2, few_parts=9)),
    "cut anew beside many rows": ([1] * 40 + [16, 1, 70] + [1] * 30, [(131 * i) % 700 + 300 for i in range(40)] + [6000, 9000, 3000] + [2500] * 30,
                                  16, 16, 64, 16, 0, 0, dict(rounds=2, few_parts=4)),
    # Head size 64: more than 8 ranges of a tile, joined in groups.
    "groups of 32 rows": ([32], [9000], 8, 8, 64, 64, 0, 0, dict(few_parts=9)),
    "groups of 24 rows": ([24, 1], [7000, 30], 16, 16, 64, 16, 0, 0, dict(few_parts=9)),
    "groups of 16 rows of two heads": ([16], [6000], 4, 2, 64, 8, 0, 0, dict(few_parts=9)),
    "groups, listed": ([12] + [1] * 70, [9000] + [9] * 70, 8, 4, 64, 32, 0, 0, dict(few_parts=9)),
}


@pytest.mark.parametrize("name", list(FORMS))
def test_forms_of_a_call(device, name):
    new, keys, heads, kv, D, P, window, sinks, _ = FORMS[name]
    check_step(device, 800 + list(FORMS).index(name), new, keys, heads, kv, D, P, window=window, sinks=sinks, odd=name == "groups of 32 rows")


@pytest.mark.parametrize("rows,widths,K_,n,index,silu", [
    (300, [264], 640, 4, "random", False), (513, [128, 128, 136, 128], 392, 3, "runs", False), (270, [136, 136], 264, 5, "random", True),
    (1000, [272], 128, 2, "runs", True),
])
def test_the_largest_rank_of_many_rows(device, rows, widths, K_, n, index, silu):
    check(device, 970 + rows, rows, widths, K_, 128, n, index, silu=silu, in_place=not silu)


class NormedStep(CheckedStep):
    """Checks the norm and the projection in front of adapters, from the operands on."""

    normed = 0

    def _add(self, target, i, x, y, out=None):
        self.saw = (x.clone(), y.clone())
        return super()._add(target, i, x, y, out)

    def _normed(self, target, i, x, y, norm, xout, w):
        before = x.float() + y.float()
        self.saw = None
        got = super()._normed(target, i, x, y, norm, xout, w)
        if self._adapted(target):
            n, z = self.saw
            K = x.shape[1]
            assert torch.equal(xout, before.to(BF)), f"residual of {target}, layer {i}"
            s = xout.cpu().double()
            # Two roundings to bf16, and a sum of K squares, a root and two products in fp32.
            ref = s / (s.square().mean(dim=1, keepdim=True) + self.m.cfg.eps).sqrt() * norm.cpu().double()
            close(n, ref, ref.abs() * (2.01 * STEP + (K + 8) * 2.0 ** -24), f"norm of {target}, layer {i}")
            exact, size = R.linear_exact(n.cpu(), w.cpu())
            assert R.within_fp32_bound(z.cpu(), exact, size, K).all(), f"projection of {target}, layer {i}"
            NormedStep.normed += 1
        return got


@pytest.mark.parametrize("targets", [("qkv",), ("gu",), V.TARGETS])
@pytest.mark.parametrize("M", [6, 80])
def test_norms_and_projections_in_front_of_adapters(device, model, targets, M):  # noqa: F811
    adapters = adapter_set(model, 11, targets=targets)
    if M == 80:
        cache = V.PagedCache(model, 5, M, 40, 8)
        cache.labels.copy_(torch.tensor([2, -1, 0, 1, 2], dtype=I32))
        cache.schedule([40, 1, 8, 0, 31])
    else:
        cache = C.DecodeCache(model, 3, 50)
    for layer in model.layers:  # gains that are not all alike
        assert layer.in_norm.std() > 0.01 and layer.post_norm.std() > 0.01 and not torch.equal(layer.in_norm, layer.post_norm)
    step = NormedStep(model, M, cache=cache, adapters=adapters)
    if M != 80:
        step.index.copy_(torch.tensor([0, 0, -1, 1, 2, 2], dtype=I32))
    NormedStep.normed = 0
    step.run(rows_of(device, model, M, 12))
    assert NormedStep.normed == len(model.layers) * (("qkv" in targets) + ("gu" in targets))


@pytest.mark.parametrize("targets", [("qkv",), ("gu",), ("qkv", "gu")])
def test_zero_factors_in_front(device, model, targets):  # noqa: F811
    """A new AdapterSet holds zeros: the step is the plain one, but for where it rounds.
    Both round to bf16 about 10 times a layer (2^-9 of a value each, rms): over 2 layers
    and the head 2^-9 * sqrt(2 * 25) = 1.4% of the logits' norm, 4% are taken."""
    x = rows_of(device, model, 7, 4)
    plain = S.GemmStep(model, 7, cache=C.DecodeCache(model, 7, 20)).run(x)
    step = S.GemmStep(model, 7, cache=C.DecodeCache(model, 7, 20), adapters=V.AdapterSet(model, 2, 8, targets))
    step.index.fill_(1)
    got = step.run(x)
    assert float((got.double() - plain.double()).norm() / plain.double().norm()) < 0.04


@pytest.mark.parametrize("D,P,B,heads", [(128, 16, 33, 8), (64, 8, 70, 4)])
def test_weights_of_single_tokens_keep_32_bits(device, D, P, B, heads):
    """Two keys of weights 1 and w, and values that cancel but for what a bf16 leaves of w u:
    out = (w u + v0) / (1 + w), v0 = -bf16(w u).

    Scores are one exact product.  w is off by its exponent x's two roundings (|x| <= 2:
    2 ln 2 2^-23) and exp2's unit (2^-23): 2.4 * 2^-23.  Three products and their sums, the
    join of the waves and 1 / L: at most 8 half steps of fp32 of |w u| <= 2 |w u| / (1 + w)."""
    g = torch.Generator().manual_seed(B)
    x = -torch.rand((B, heads), generator=g) * 1.5 - 0.2  # scores: q x at key 1, 0 at key 0
    table = torch.randperm(B, generator=g).to(I32).view(B, 1)
    k, v, q = (torch.zeros(shape, dtype=BF) for shape in ((B, P, heads, D), (B, P, heads, D), (B, heads * D)))
    k[:, 1, :, 5] = x.to(BF)[torch.argsort(table[:, 0])]  # by page
    q.view(B, heads, D)[:, :, 5] = 1.0
    w = k[table[:, 0].long(), 1, :, 5].double().exp()[:, :, None]
    u = torch.randn((B, heads, D), generator=g).to(BF)
    v0 = (-w * u.double()).to(BF)
    v[table[:, 0].long(), 0], v[table[:, 0].long(), 1] = v0, u
    op = K.PagedAttention(B, B, heads, heads, D, P, 1, device, scale=1.0)
    starts, keys = torch.arange(B + 1, dtype=I32), torch.full((B,), 2, dtype=I32)
    out = op(*(t.to(device) for t in (q, k, v, table, starts, keys))).view(B, heads, D)
    ref, size = (w * u.double() + v0.double()) / (1 + w), w * u.double().abs() / (1 + w)
    assert (ref.abs() < 2.0 ** -7 * size + 1e-30).all()
    close(out, ref, STEP * ref.abs() * 1.01 + size * (2.4 * 2.0 ** -23 + 2 * 8 * 2.0 ** -24), "out")
