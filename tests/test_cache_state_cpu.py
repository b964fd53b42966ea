"""What a DecodeCache counts, without a GPU: refused and failed steps leave it
as it was."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from kernels import attention as A
from kernels import cache as C
from kernels import step as S

BF = torch.bfloat16


def model(layers=2, heads=4, kv_heads=2, hidden=16):
    cfg = S.QwenConfig(hidden=hidden, intermediate=32, layers=layers, heads=heads, kv_heads=kv_heads, head_dim=128, vocab=10)
    ones = torch.ones(128, dtype=BF)
    layer = SimpleNamespace(in_norm=None, post_norm=None, wqkv=None, wo=None, wgu=None, wd=None, q_norm=ones, k_norm=ones)
    return SimpleNamespace(cfg=cfg, device=torch.device("cpu"), layers=[layer] * layers, lm_head=None, final_norm=None)


def projections(m, M, fail=None):
    """Stand-ins for the five projections; the one named ``fail`` raises."""
    cols = {"qkv": (m.cfg.heads + 2 * m.cfg.kv_heads) * 128, "o": m.cfg.hidden, "gu": m.cfg.intermediate, "d": m.cfg.hidden,
            "lm": m.cfg.vocab}

    def make(name):
        def call(*_):
            if name == fail:
                raise ValueError(f"{name} refused")
            return torch.zeros((M, cols[name]), dtype=BF)
        return call

    return {name: make(name) for name in cols}


def counts(c):
    return c.lens.tolist(), c.seen.tolist(), [list(h) for h in c._host]


def masks(B, R, **kw):
    return torch.ones((B, R), **{"dtype": torch.int64, **kw})


@pytest.mark.parametrize("kw,R,tree,msg", [
    (dict(scored=True), 2, masks(2, 2), "draft tree"),
    ({}, 65, masks(2, 65), "64"),
    (dict(window=3), 4, masks(2, 4), "window"),
    ({}, 2, masks(2, 3), "tree"),
    ({}, 2, masks(1, 2), "tree"),
    ({}, 2, masks(2, 2, dtype=torch.int32), "tree"),
    ({}, 2, masks(2, 4)[:, ::2], "contiguous"),
    ({}, 2, [[1, 3], [1, 3]], "tree"),
    ({}, 70000, None, "too large"),
])
def test_refused_steps_leave_the_cache(kw, R, tree, msg):
    m = model()
    c = C.DecodeCache(m, 2, 100000 if R > 100 else 200, **kw)
    c.begin(5)
    before = counts(c)
    with pytest.raises(ValueError, match=msg):
        c.begin(R, tree=tree)
    assert counts(c) == before == ([5, 5], [5, 5], [[5, 5], [5, 5]])
    x = torch.zeros((2 * R, 16), dtype=BF)
    with pytest.raises(ValueError, match=msg):
        S.GemmStep(m, 2 * R, mm=projections(m, 2 * R), cache=c, tree=tree).run(x)
    step = S.GemmStep(m, 2 * R, mm=projections(m, 2 * R), cache=c) if R < 70000 else None
    for call in (step.run, step.capture) if step else ():
        step.tree = tree
        with pytest.raises(ValueError, match=msg):
            call(x)
        assert counts(c) == before


@pytest.mark.parametrize("fail", ["qkv", "attend"])
def test_failed_steps_leave_the_cache(fail):
    """A projection or an operator that raises behind begin() (here: CPU tensors
    are refused by every operator)."""
    m = model()
    c = C.DecodeCache(m, 2, 20)
    c.begin(5)
    before = counts(c)
    step = S.GemmStep(m, 6, mm=projections(m, 6, fail), cache=c)
    with pytest.raises(ValueError, match="refused" if fail == "qkv" else "GPU"):
        step.run(torch.zeros((6, 16), dtype=BF))
    assert counts(c) == before
    with pytest.raises(RuntimeError, match="begin"):
        c.attend(0, None, None)
    c.begin(15)  # all of the room is still there


def test_a_step_of_another_model_is_refused():
    c = C.DecodeCache(model(), 2, 20)
    for other in (model(layers=3), model(heads=8), model(kv_heads=4)):
        with pytest.raises(ValueError, match="another model"):
            S.GemmStep(other, 2, mm=projections(other, 2), cache=c)


@pytest.mark.parametrize("kw", [{}, dict(scored=True), dict(window=64, sinks=4)])
def test_many_row_counts_share_one_workspace(kw):
    """A thousand prompt lengths: the memory held stays below four times what the
    largest of them needs, and every shape's counters lie in the same place."""
    c = C.DecodeCache(model(), 3, 1500, **kw)
    for R in [1, 700, *range(2, 1000)]:
        c._op(R)
    need = max(A.workspace_bytes(3, R, 4, 2, 128, 1500, **kw) for R in range(1, 1000))
    held = {op.workspace.data_ptr(): op.workspace.numel() for op in c._ops.values() if op.workspace is not None}
    assert need <= max(held.values()) and sum(held.values()) <= 4 * need


def test_given_workspaces():
    need = A.workspace_bytes(2, 1, 8, 2, 128, 5000)
    assert need > 0 and A.workspace_bytes(2, 1, 8, 2, 128, 50) == 0
    make = lambda ws: A.CacheAttention(2, 1, 8, 2, 128, 5000, "cpu", workspace=ws)
    ws = torch.zeros(need + 5, dtype=torch.uint8)
    assert make(ws).workspace is ws
    for bad in (ws[:need - 1], ws.float(), torch.zeros(2 * need, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            make(bad)
    with pytest.raises(ValueError, match="64 and 128"):
        A.workspace_bytes(2, 1, 8, 2, 96, 50)


def test_building_waits_for_the_fill(monkeypatch):
    """Every object that owns memory waits for the stream that fills it."""
    waits = []
    monkeypatch.setattr(A, "filled", lambda device: waits.append(str(device)))
    A.CacheAttention(2, 1, 8, 2, 128, 5000, "cpu")
    assert waits == ["cpu"]
    c = C.DecodeCache(model(), 2, 5000)
    assert len(waits) == 2
    c.begin(1)
    assert len(waits) == 3


def pair(keys, kv=2, dim=128, dtype=BF):
    return tuple(torch.zeros((keys, kv, dim), dtype=dtype) for _ in "kv")


@pytest.mark.parametrize("kw,msg", [
    (dict(scored=True, prefix=[pair(5)] * 2), "shared prefix"),
    (dict(prefix=[pair(5), pair(6)]), "layer 1"),  # positions would differ from layer to layer
    (dict(prefix=[pair(5), pair(5, kv=1)]), "layer 1"),
    (dict(prefix=[pair(5, dim=64)] * 2), "layer 0"),
    (dict(prefix=[pair(5, dtype=torch.float32)] * 2), "layer 0"),
    (dict(prefix=[pair(5), (pair(5)[0], pair(4)[0])]), "layer 1"),
    (dict(prefix=[pair(5), pair(5)[:1]]), "layer 1"),
    (dict(prefix=[pair(5)]), "1 pairs for 2 layers"),
    (dict(sinks=3), "sinks need a window"), (dict(window=-1), "negative"), (dict(capacity=0), ">= 1"), (dict(B=0), ">= 1"),
])
def test_caches_that_no_step_could_use(kw, msg):
    with pytest.raises(ValueError, match=msg):
        C.DecodeCache(model(), **{**dict(B=2, capacity=20), **kw})


def test_accepted_paths_of_a_draft_tree():
    """Nodes that are not a tree's first move together in every layer; lengths and
    positions go on from the path, as behind a step of its rows alone."""
    c = C.DecodeCache(model(), 3, 30)
    c.begin(4)
    tree = torch.tensor([[1, 3, 5, 0b1001, 0b10101, 0b100101]] * 3)
    c.begin(6, tree=tree)
    assert c._positions.view(3, 6).tolist() == [[4, 5, 5, 5, 6, 6]] * 3
    for i, t in enumerate(c.k + c.v):
        t.copy_((torch.arange(30)[None, :] + 40 * torch.arange(3)[:, None] + i % 4)[:, :, None, None].expand(3, 30, 2, 128))
    before = [t.clone() for t in c.k + c.v]
    paths = [[0, 2, 5], [], [0, 1]]
    c.accept(6, paths)
    assert c.lens.tolist() == c.seen.tolist() == [7, 4, 6] and c._host == [[7, 7], [4, 4], [6, 6]]
    for t, was in zip(c.k + c.v, before):
        for b, p in enumerate(paths):
            assert torch.equal(t[b, :4], was[b, :4]) and torch.equal(t[b, 4:4 + len(p)], was[b, [4 + i for i in p]])
            assert torch.equal(t[b, 10:], was[b, 10:])
    c.begin(1)
    assert c._positions.tolist() == [7, 4, 6]


@pytest.mark.parametrize("R,paths", [(6, [[0]]), (6, [[0], [6]]), (6, [[0], [-1]]), (6, [[0], [1, 1]]), (6, [[2, 1], [0]]),
                                     (11, [[0], [0]]), (0, [[], []])])
def test_paths_refused(R, paths):
    c = C.DecodeCache(model(), 2, 30)
    c.begin(10)
    before = counts(c)
    with pytest.raises(ValueError, match="path"):
        c.accept(R, paths)
    assert counts(c) == before


def test_scored_caches_have_no_paths():
    c = C.DecodeCache(model(), 2, 30, scored=True)
    c.begin(3)
    with pytest.raises(ValueError, match="rollback"):
        c.accept(3, [[0], [0]])
    assert counts(c)[0] == [3, 3]
