"""Whole steps over a PagedCache with an AdapterSet: prompts in chunks beside decoding
requests, drafts and their rollback, restarts; every layer's pages, attention and
adapters against the 64-bit oracle; eager against graph replay, and against a
DecodeCache of each request's own."""

from __future__ import annotations

import pytest
import torch

from kernels import cache as C
from kernels import serve as V
from kernels import step as S
from oracle import attn_ref as A64
from oracle import gemm_ref as R
from oracle import paged_ref as P64

from test_attn_gpu import close, gen, rnd, say

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def model(device):
    return S.synthetic_model(device, layers=2, seed=5, hidden=512, intermediate=1024, heads=8, kv_heads=2, vocab=1000)


def rows_of(device, model, M, seed):
    return R.randn_bf16((M, model.cfg.hidden), seed).to(device)


class Checked(V.PagedCache):
    """A PagedCache that checks every layer's pages and attention, and the tables
    against the host's count."""

    def attend(self, i, qkv, out):
        cfg, t = self.m.cfg, self.tables
        before, was = qkv.clone(), out.clone()
        old = [x.clone() for x in (self.k[i], self.v[i])]
        super().attend(i, qkv, out)
        new, starts = self._plan, t.starts.tolist()
        assert starts == [sum(new[:b]) for b in range(self.B + 1)]
        assert t.keys.tolist() == [have + n for have, n in zip(self.lens, new)] == t.lens.tolist()
        n = starts[-1]
        slots, pos, table = t.slots.tolist(), t.positions.tolist(), t.table.tolist()
        held = [p for b, L in enumerate(t.lens.tolist()) for p in table[b][:-(-L // self.page_size)]]
        assert len(set(held)) == len(held) == self.pages - int(t.count), "a page held twice, or lost"
        for b in range(self.B):
            for j in range(new[b]):
                p = self.lens[b] + j
                assert pos[starts[b] + j] == p
                assert slots[starts[b] + j] == table[b][p // self.page_size] * self.page_size + p % self.page_size
        assert slots[n:] == pos[n:] == [-1] * (self.rows - n)
        layer = self.m.layers[i]
        (rq, sq), (rk, sk), rv = A64.rope(before, layer.q_norm, layer.k_norm, cfg.eps, cfg.theta, torch.tensor(pos).clamp(min=0),
                                          cfg.heads, cfg.kv_heads, cfg.head_dim)
        rel = (cfg.head_dim + 16) * A64.FP32_HALF
        q = qkv[:, :cfg.heads * cfg.head_dim]
        close(q[:n].reshape(n, cfg.heads, -1), rq[:n], (A64.BF16_HALF * rq.abs() * 1.01 + sq * rel)[:n], "q")
        at = torch.tensor(slots[:n])
        k, v = (x.cpu().reshape(-1, cfg.kv_heads, cfg.head_dim) for x in (self.k[i], self.v[i]))
        close(k[at], rk[:n], (A64.BF16_HALF * rk.abs() * 1.01 + sk * rel)[:n], "k")
        assert torch.equal(v[at].double(), rv[:n])
        rest = torch.ones(len(k), dtype=torch.bool)
        rest[at] = False
        for x, o in zip((k, v), old):
            assert torch.equal(x[rest], o.cpu().reshape(x.shape)[rest]), "other slots were written"
        ref, _, tol, _ = P64.attention(q, self.k[i].cpu(), self.v[i].cpu(), table, starts, t.keys.tolist(), heads=cfg.heads,
                                       window=self.attention.window, sinks=self.attention.sinks)
        close(out[:n].view(n, cfg.heads, -1), ref[:n], tol[:n], f"attention, layer {i}")
        assert torch.equal(out[n:], was[n:]), "rows of no request were written"
        return out


class CheckedStep(S.GemmStep):
    """A GemmStep that checks every projection's adapters."""

    checked = 0

    def _add(self, target, i, x, y, out=None):
        before = y.clone()
        got = super()._add(target, i, x, y, out)
        if self._adapted(target):
            s = self.adapters
            ref, tol = P64.adapters(x, s.a[target][i], s.b[target][i], self.index.cpu(), before, s.scale.cpu(), s.widths[target], s.rank,
                                    target == "gu")
            close(got, ref, tol, f"adapters of {target}, layer {i}")
            CheckedStep.checked += 1
        return got


def adapter_set(model, seed, n=3, rank=16, targets=V.TARGETS):
    s = V.AdapterSet(model, n, rank, targets)
    g = gen(seed)
    for t in targets:
        for i in range(len(model.layers)):
            s.a[t][i].copy_(rnd(g, *s.a[t][i].shape, scale=s.depth[t] ** -0.5))
            s.b[t][i].copy_(rnd(g, *s.b[t][i].shape, scale=0.1))
    s.scale.copy_(torch.rand(n, generator=g) + 0.5)
    return s


#: Steps of 5 requests and 80 rows: new rows, then rows taken back and requests that end.
PLAN = [
    ([40, 0, 3, 0, 0], None, ()),
    ([37, 1, 1, 30, 0], None, ()),
    ([1, 1, 1, 70, 6], [0, 0, 0, 0, 4], ()),
    ([1, 1, 1, 1, 5], None, (3,)),
    ([1, 60, 0, 17, 1], None, (0, 1)),
    ([9, 1, 1, 1, 1], [3, 0, 0, 0, 0], ()),
]


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
@pytest.mark.parametrize("adapted", [False, True])
def test_steps_over_chunks_drafts_and_restarts(device, model, window, sinks, adapted):
    cache = Checked(model, 5, 80, 40, 8, window=window, sinks=sinks)
    cache.labels.copy_(torch.tensor([2, -1, 0, 1, 2], dtype=I32))
    step = CheckedStep(model, 80, cache=cache, adapters=adapter_set(model, 3) if adapted else None)
    CheckedStep.checked = 0
    for i, (new, back, ended) in enumerate(PLAN):
        say("step", i, new, cache.lens)
        assert cache.schedule(new) == [sum(new[:b]) for b in range(5)]
        logits = step.run(rows_of(device, model, 80, 50 + i))
        assert logits[:sum(new)].isfinite().all()
        if back:
            cache.rollback(back)
        for b in ended:
            cache.reset(b)
    assert CheckedStep.checked == (len(PLAN) * 8 if adapted else 0)


def test_refusals_leave_the_cache_as_it_was(device, model):
    cache = V.PagedCache(model, 3, 20, 6, 8, width=4, max_positions=30)
    step = S.GemmStep(model, 20, cache=cache)
    x = rows_of(device, model, 20, 1)
    with pytest.raises(RuntimeError, match="schedule"):
        step.run(x)
    cache.schedule([10, 9, 1])
    step.run(x)
    for new, msg in (([11, 10, 0], "21 rows"), ([0, 0], "each of 3"), ([0, -1, 0], "each of 3"), ([0, 0, 20], "7 of 6 pages"), ([20, 0, 0], "7 of 6 pages"),
                     ([7, 0, 13], "7 of 6 pages")):
        with pytest.raises(ValueError, match=msg):
            cache.schedule(new)
        assert cache.lens == [10, 9, 1]
    with pytest.raises(ValueError, match="positions"):
        V.PagedCache(model, 3, 40, 30, 8, max_positions=30).schedule([31, 0, 0])
    with pytest.raises(ValueError, match="rollback"):
        cache.rollback([0, 10, 0])
    for bad in (dict(cache=V.PagedCache(model, 2, 8, 4, 8)), dict(cache=cache, tree=torch.zeros((3, 1), dtype=torch.int64, device=device))):
        with pytest.raises(ValueError):
            S.GemmStep(model, 20, **bad)
    other = S.synthetic_model(device, layers=1, seed=5, hidden=512, intermediate=1024, heads=8, kv_heads=2, vocab=1000)
    with pytest.raises(ValueError, match="another model"):
        S.GemmStep(model, 20, adapters=V.AdapterSet(other, 1, 8))
    for kw in (dict(targets=()), dict(targets=("x",)), dict(rank=9), dict(adapters=0), dict(targets=("o", "o"))):
        with pytest.raises(ValueError):
            V.AdapterSet(model, **{**dict(adapters=1, rank=8), **kw})


def test_a_failed_step_gives_its_pages_back(device, model):
    cache = V.PagedCache(model, 2, 16, 6, 8)
    step = S.GemmStep(model, 16, cache=cache)
    x = rows_of(device, model, 16, 2)
    cache.schedule([9, 3])
    good = dict(step.mm)

    def broken(*a):
        raise RuntimeError("broken")

    step.mm["d"] = broken
    with pytest.raises(RuntimeError, match="broken"):
        step.run(x)
    step.mm.update(good)
    assert cache.lens == [0, 0]
    first = step.run(x).clone()
    assert cache.lens == [9, 3] and int(cache.tables.count) == 3
    fresh = V.PagedCache(model, 2, 16, 6, 8)
    fresh.schedule([9, 3])
    assert torch.equal(S.GemmStep(model, 16, cache=fresh).run(x)[:12], first[:12])


@pytest.mark.parametrize("adapted", [False, True])
def test_captured_steps_are_the_eager_ones(device, model, adapted):
    adapters = adapter_set(model, 4) if adapted else None
    caches = [V.PagedCache(model, 5, 80, 40, 8) for _ in range(2)]
    for c in caches:
        c.labels.copy_(torch.tensor([2, -1, 0, 1, 2], dtype=I32))
    eager, captured = (S.GemmStep(model, 80, cache=c, adapters=adapters) for c in caches)
    x = rows_of(device, model, 80, 9)
    captured.capture(x)
    with pytest.raises(RuntimeError, match="schedule"):
        captured.replay()
    for i, (new, back, ended) in enumerate(PLAN):
        x.copy_(rows_of(device, model, 80, 60 + i))
        for c in caches:
            c.schedule(new)
        want = eager.run(x).clone()
        got = captured.replay()
        torch.cuda.synchronize()
        n = sum(new)
        assert torch.equal(got[:n], want[:n]), i
        assert caches[0].lens == caches[1].lens
        for a, b in zip(caches[0].k + caches[0].v, caches[1].k + caches[1].v):
            assert torch.equal(a, b)
        for c in caches:
            if back:
                c.rollback(back)
            for b in ended:
                c.reset(b)


def test_each_request_as_if_alone(device, model):
    """A mixed step's rows against a DecodeCache of each request's own.  Both round to
    bf16 about 10 times a layer, at other places (2^-9 of a value each, rms): over 2 layers
    and the head, 2^-9 * sqrt(2 * 25) = 1.4% of the logits' norm, more where an error
    passes a norm; 4% are taken."""
    cache = V.PagedCache(model, 3, 40, 40, 8)
    step = S.GemmStep(model, 40, cache=cache)
    own = [C.DecodeCache(model, 1, 100) for _ in range(3)]
    for i, new in enumerate(([30, 1, 5], [1, 17, 1], [1, 1, 20])):
        x = rows_of(device, model, 40, 80 + i)
        starts = cache.schedule(new)
        logits = step.run(x).clone()
        for b, n in enumerate(new):
            want = S.GemmStep(model, n, cache=own[b]).run(x[starts[b]:starts[b] + n].contiguous())
            got = logits[starts[b]:starts[b] + n]
            err = float((got.double() - want.double()).norm() / want.double().norm())
            assert err < 0.04, (i, b, err)


def test_adapters_over_one_run_of_slots(device, model):
    """Adapters beside a DecodeCache, named by row."""
    step = CheckedStep(model, 6, cache=C.DecodeCache(model, 3, 50), adapters=adapter_set(model, 6, targets=("qkv", "gu")))
    CheckedStep.checked = 0
    step.index.copy_(torch.tensor([0, 0, -1, -1, 2, 2], dtype=I32))
    x = rows_of(device, model, 6, 3)
    with_them = step.run(x).clone()
    assert CheckedStep.checked == 4
    step.cache.reset()
    step.index.fill_(-1)
    without = step.run(x)
    assert not torch.equal(with_them[:2], without[:2]) and not torch.equal(with_them[4:], without[4:])


def test_zero_factors_change_nothing(device, model):
    """A new AdapterSet holds zeros: o and d give the plain step's outputs bit for bit."""
    x = rows_of(device, model, 7, 4)
    plain = S.GemmStep(model, 7, cache=C.DecodeCache(model, 7, 20)).run(x)
    step = S.GemmStep(model, 7, cache=C.DecodeCache(model, 7, 20), adapters=V.AdapterSet(model, 2, 8, ("o", "d")))
    step.index.fill_(1)
    assert torch.equal(step.run(x), plain)
