"""The whole decode step over a DecodeCache: a prompt, decode rows, an eviction
and more rows, each layer's cache rows and attention against the 64-bit oracle;
draft trees, windows and shared prefixes; eager against graph replay."""

from __future__ import annotations

import pytest
import torch

from kernels import cache as C
from kernels import step as S
from oracle import attn_ref as R64
from oracle import gemm_ref as R

from test_attn_gpu import close, gen, rnd, say, tree_masks, weight_half

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def model(device):
    return S.synthetic_model(device, layers=2, seed=5, hidden=512, intermediate=1024, heads=8, kv_heads=2, vocab=1000)


def x_rows(device, model, M, seed):
    return R.randn_bf16((M, model.cfg.hidden), seed).to(device)


class Checked(C.DecodeCache):
    """A DecodeCache that checks every layer's cache rows and attention."""

    def attend(self, i, qkv, out):
        cfg, Rr = self.m.cfg, self._rows
        before = qkv.clone()
        old = [t.clone() for t in (self.k[i], self.v[i])]
        was = self.scores[i].clone() if self.scored else None
        super().attend(i, qkv, out)
        lens = self.lens.tolist()
        layer = self.m.layers[i]
        pos = self._positions.cpu()
        (rq, sq), (rk, sk), rv = R64.rope(before, layer.q_norm, layer.k_norm, cfg.eps, cfg.theta, pos, cfg.heads,
                                          cfg.kv_heads, cfg.head_dim)
        rel = (cfg.head_dim + 16) * R64.FP32_HALF
        M = self.B * Rr
        q = qkv[:, :cfg.heads * cfg.head_dim]
        close(q.reshape(M, cfg.heads, -1), rq, R64.BF16_HALF * rq.abs() * 1.01 + sq * rel, "q")
        for b in range(self.B):
            at = slice(lens[b] - Rr, lens[b])
            rows = slice(b * Rr, (b + 1) * Rr)
            close(self.k[i][b, at], rk[rows], R64.BF16_HALF * rk[rows].abs() * 1.01 + sk[rows] * rel, "k")
            assert torch.equal(self.v[i][b, at].cpu().double(), rv[rows])
            for t, o in zip((self.k[i], self.v[i]), old):
                assert torch.equal(t[b, :lens[b] - Rr], o[b, :lens[b] - Rr]) and torch.equal(t[b, lens[b]:], o[b, lens[b]:])
        shared = None if self.prefix is None else self.prefix[i]
        ref, _, w, size, top = R64.attention(q.contiguous(), self.k[i], self.v[i], lens, heads=cfg.heads, R=Rr, window=self.window,
                                             sinks=self.sinks, prefix=shared,
                                             tree=None if self._tree is None else self._tree.tolist())
        keys = self.prefix_keys + self.capacity
        tol = R64.attention_tolerance(ref, size, top, cfg.head_dim, keys, weight_half(self._current))
        close(out.view(ref.shape), ref, tol, f"attention of layer {i}")
        if self.scored:
            rel = 2 * float(R64.score_error(top, cfg.head_dim).max()) + (keys + 64) * R64.FP32_HALF
            want = was.cpu().double() + w
            close(self.scores[i], want, w * rel + (Rr + 4) * R64.FP32_HALF * want.abs() + 1e-30, "scores")
        return out


def test_prompt_decode_evict_decode(device, model):
    B, cap = 3, 200
    cache = Checked(model, B, cap, scored=True)
    assert model.layers[0].q_norm.shape == (128,)
    say("prompt")
    S.GemmStep(model, B * 70, cache=cache).run(x_rows(device, model, B * 70, 1))
    one = S.GemmStep(model, B, cache=cache)
    for t in range(3):
        one.run(x_rows(device, model, B, 10 + t))
    assert cache.lens.tolist() == cache.seen.tolist() == [73] * B
    scores = [s.clone() for s in cache.scores]
    ks = [k.clone() for k in cache.k]
    lens = cache.lens.tolist()
    say("evict")
    kept = cache.evict(32, sinks=2, recent=8)
    for i, s in enumerate(scores):
        want = R64.evict(s, lens, 32, 2, 8)
        assert kept[i].tolist() == want
        for b in range(B):
            for h in range(2):
                assert torch.equal(cache.k[i][b, :32, h], ks[i][b, want[b][h], h])
                assert torch.equal(cache.scores[i][b, h, :32], s[b, h, want[b][h]])
        assert (cache.scores[i][:, :, 32:] == 0).all()
    assert cache.lens.tolist() == [32] * B and cache.seen.tolist() == [73] * B
    for t in range(2):
        one.run(x_rows(device, model, B, 20 + t))
    assert cache.lens.tolist() == [34] * B and cache.seen.tolist() == [75] * B
    cache.reset(1)
    assert cache.lens.tolist() == [34, 0, 34] and (cache.scores[0][1] == 0).all()
    one.run(x_rows(device, model, B, 30))
    assert cache.lens.tolist() == [35, 1, 35]


def test_window_prefix_and_tree(device, model):
    g = gen(7)
    B, R_, cap = 2, 6, 90
    prefix = [tuple(rnd(g, 50, 2, 128).to(device) for _ in "kv") for _ in model.layers]
    cache = Checked(model, B, cap, window=24, sinks=3, prefix=prefix)
    S.GemmStep(model, B * 30, cache=cache).run(x_rows(device, model, B * 30, 41))
    tree = tree_masks(g, B, R_).to(device)
    S.GemmStep(model, B * R_, cache=cache, tree=tree).run(x_rows(device, model, B * R_, 42))
    assert cache.lens.tolist() == [36, 36]
    cache.rollback([4, 0])
    assert cache.lens.tolist() == cache.seen.tolist() == [32, 36]
    S.GemmStep(model, B, cache=cache).run(x_rows(device, model, B, 43))
    assert cache.lens.tolist() == [33, 37]
    for bad in ([1], [34, 0], [0, -1]):
        with pytest.raises(ValueError, match="rollback"):
            cache.rollback(bad)


def test_rollback_forgets_scores(device, model):
    B = 2
    cache = Checked(model, B, 40, scored=True)
    S.GemmStep(model, B * 10, cache=cache).run(x_rows(device, model, B * 10, 44))
    cache.rollback([3, 10])
    assert cache.lens.tolist() == [7, 0]
    for s in cache.scores:
        assert (s[0, :, 7:] == 0).all() and (s[1] == 0).all() and (s[0, :, :7] > 0).all()
    S.GemmStep(model, B, cache=cache).run(x_rows(device, model, B, 45))


@pytest.mark.parametrize("kw", [dict(scored=True), dict(window=16, sinks=2), dict(tree=True)])
def test_replays_continue_like_eager_steps(device, model, kw):
    B, cap = 2, 64
    kw = dict(kw)
    tree = tree_masks(gen(3), B, 3).to(device) if kw.pop("tree", False) else None
    R_ = 3 if tree is not None else 1
    caches = [C.DecodeCache(model, B, cap, **kw) for _ in range(2)]
    steps = [S.GemmStep(model, B * R_, cache=c, tree=tree) for c in caches]
    xs = [x_rows(device, model, B * R_, 60 + t) for t in range(5)]
    prompt = x_rows(device, model, B * 20, 50)
    for c in caches:
        S.GemmStep(model, B * 20, cache=c).run(prompt)
    x = xs[0].clone()
    steps[1].capture(x)
    assert caches[1].lens.tolist() == [20] * B
    for t, row in enumerate(xs):
        want = steps[0].run(row).clone()
        x.copy_(row)
        got = steps[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), t
        assert torch.equal(caches[0].lens, caches[1].lens) and caches[0]._host == caches[1]._host
        for i in range(len(model.layers)):
            assert torch.equal(caches[0].k[i], caches[1].k[i])
            if kw.get("scored"):
                assert torch.equal(caches[0].scores[i], caches[1].scores[i])


def test_refusals(device, model):
    cache = C.DecodeCache(model, 2, 10, max_positions=12)
    with pytest.raises(ValueError, match="3 rows for a cache of 2"):
        S.GemmStep(model, 3, cache=cache)
    with pytest.raises(ValueError, match="tree masks need a cache"):
        S.GemmStep(model, 2, tree=torch.zeros((2, 1), dtype=torch.int64))
    st = S.GemmStep(model, 2 * 6, cache=cache)
    st.run(x_rows(device, model, 12, 1))
    with pytest.raises(ValueError, match="do not fit"):
        st.run(x_rows(device, model, 12, 2))
    with pytest.raises(ValueError, match="do not fit"):
        st.capture(x_rows(device, model, 12, 2))
    assert cache.lens.tolist() == [6, 6]
    with pytest.raises(ValueError, match="scored=True"):
        cache.evict(4)
    with pytest.raises(RuntimeError, match="begin"):
        C.DecodeCache(model, 2, 10).attend(0, None, None)
    scored = C.DecodeCache(model, 2, 10, scored=True)
    with pytest.raises(ValueError, match="draft tree"):
        scored.begin(2, tree=torch.ones((2, 2), dtype=torch.int64, device=device))
    with pytest.raises(ValueError, match="pairs for 2 layers"):
        C.DecodeCache(model, 2, 10, prefix=[])
