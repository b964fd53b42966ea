"""A DecodeCache on the GPU across steps that fail, many sizes of step, and
streams."""

from __future__ import annotations

import pytest
import torch

from kernels import attention as A
from kernels import cache as C
from kernels import step as S
from oracle import gemm_ref as R

from test_attn_gpu import gen, rnd, say

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def model(device):
    return S.synthetic_model(device, layers=2, seed=5, hidden=512, intermediate=1024, heads=8, kv_heads=2, vocab=1000)


def x_rows(device, model, M, seed):
    return R.randn_bf16((M, model.cfg.hidden), seed).to(device)


@pytest.mark.parametrize("at", [1, 2, 3, 5, 6])
def test_failed_captures_leave_the_cache(device, model, at):
    """The at-th gate/up projection raises: in the warm-up (1 to 4) or while the
    graph is recorded.  Counts and scores are those from before, and the next
    capture replays like an eager step."""
    caches = [C.DecodeCache(model, 2, 40, scored=True) for _ in range(2)]
    for c in caches:
        S.GemmStep(model, 2 * 9, cache=c).run(x_rows(device, model, 18, 1))
    steps = [S.GemmStep(model, 2, cache=c) for c in caches]
    x = x_rows(device, model, 2, 2)
    broken = S.GemmStep(model, 2, mm=dict(steps[0].mm), cache=caches[0])
    calls, gu = [], broken.mm["gu"]

    def stops(*a):
        calls.append(0)
        if len(calls) == at:
            raise ValueError("stop")
        return gu(*a)

    broken.mm["gu"] = stops
    say("failed capture", at)
    with pytest.raises(ValueError, match="stop"):
        broken.capture(x)
    assert broken.graph is None and broken.out is None
    assert caches[0]._host == caches[1]._host
    for a, b in zip((caches[0].lens, caches[0].seen, *caches[0].scores), (caches[1].lens, caches[1].seen, *caches[1].scores)):
        assert torch.equal(a, b)
    steps[0].capture(x)
    got, want = steps[0].replay(), steps[1].run(x)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(caches[0].lens, caches[1].lens)


@pytest.mark.parametrize("kw", [{}, dict(scored=True), dict(window=40, sinks=3), "prefix"])
def test_steps_of_many_sizes_share_a_workspace(device, model, kw):
    """Steps whose attention joins its ranges in the kernel, in a launch of its
    own, or has one range, in turn on one workspace: each equals an object of its
    own bit by bit."""
    g = gen(1100)
    B, heads, kv, D, cap = 2, 8, 2, 128, 1500
    shared = None
    if kw == "prefix":
        shared, kw = tuple(rnd(g, 300, kv, D).to(device) for _ in "kv"), {}
    cache = C.DecodeCache(model, B, cap, prefix=None if shared is None else [shared] * 2, **kw)
    cache.k[0].copy_(rnd(g, B, cap, kv, D)), cache.v[0].copy_(rnd(g, B, cap, kv, D))
    scores = torch.zeros((B, kv, cap), device=device)
    for R_ in (1, 4, 100, 2, 16, 1, 33, 300, 5, 1, 100, 16, 2):
        q = rnd(g, B * R_, heads * D).to(device)
        own = A.CacheAttention(B, R_, heads, kv, D, cap, device, prefix=0 if shared is None else 300, **kw)
        say("one workspace", R_, own.plan)
        for n in (1500, 700, R_):
            lens = torch.tensor([n, n // 2 + 1], dtype=torch.int32, device=device)
            got, want = [], []
            for op, to in ((cache._op(R_), got), (own, want)):
                more = dict(scores=scores, scores_out=torch.zeros_like(scores)) if kw.get("scored") else {}
                to.append(op(q, cache.k[0], cache.v[0], lens, prefix=shared, **more))
                to.extend(t for name, t in more.items() if name == "scores_out")
            for a, b in zip(got, want):
                assert torch.equal(a, b), (R_, n)
    assert len({op.workspace.data_ptr() for op in cache._ops.values() if op.workspace is not None}) < len(cache._ops)


def test_first_calls_on_another_stream(device, model):
    """Objects built on a stream that is busy, over memory that held other values,
    and called at once on another: the counters are zero by then."""
    g = gen(1110)
    B, heads, kv, D, cap = 2, 32, 8, 128, 3000
    k, v = rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    q = rnd(g, B, heads * D).to(device)
    lens = torch.tensor([3000, 1700], dtype=torch.int32, device=device)
    want = A.CacheAttention(B, 1, heads, kv, D, cap, device)(q, k, v, lens)
    need = A.workspace_bytes(B, 1, heads, kv, D, cap)
    busy = torch.cuda.Stream()
    torch.cuda.synchronize()
    say("first call on another stream")
    for _ in range(3):
        with torch.cuda.stream(busy):
            junk = torch.full((need,), 255, dtype=torch.uint8, device=device)
            del junk
            torch.cuda._sleep(20_000_000)
            op = A.CacheAttention(B, 1, heads, kv, D, cap, device)
        assert torch.equal(op(q, k, v, lens), want)
        torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(20_000_000)
        cache = C.DecodeCache(model, 2, 40)
    cache.begin(3)
    assert cache.lens.tolist() == [3, 3] and cache._positions.tolist() == [0, 1, 2] * 2


def test_no_workspace_while_a_graph_is_captured(device):
    """Zeros that are only recorded would not be there for the next eager call."""
    t = torch.zeros(4, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.add_(1)
        with pytest.raises(RuntimeError, match="before the capture"):
            A.CacheAttention(2, 1, 32, 8, 128, 3000, device)
    graph.replay()
    assert t.tolist() == [1.0] * 4


def test_an_object_that_goes_before_its_call_has_run(device):
    """Its workspace is not given to another stream's tensors until then."""
    g = gen(1120)
    B, heads, kv, D, cap = 2, 32, 8, 128, 3000
    k, v = rnd(g, B, cap, kv, D).to(device), rnd(g, B, cap, kv, D).to(device)
    q = rnd(g, B, heads * D).to(device)
    lens = torch.tensor([3000, 1700], dtype=torch.int32, device=device)
    want = A.CacheAttention(B, 1, heads, kv, D, cap, device)(q, k, v, lens)
    need = A.workspace_bytes(B, 1, heads, kv, D, cap)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    say("object gone")
    for _ in range(3):
        op = A.CacheAttention(B, 1, heads, kv, D, cap, device)
        at = op.workspace.data_ptr()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            op.run(q, k, v, lens, out)
        del op
        other = torch.full((need,), 255, dtype=torch.uint8, device=device)
        assert other.data_ptr() != at
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del other


@pytest.mark.parametrize("captured", [False, True])
def test_decode_goes_on_from_an_accepted_path(device, model, captured):
    """A tree step of which nodes 0, 2 and 5 (and 0 and 1) are accepted, then a
    decode row: the cache holds the accepted nodes' rows in every layer, and that
    row's attention, checked against the oracle, sees them and no others."""
    from test_cache_step_gpu import Checked

    B = 2
    cache = (C.DecodeCache if captured else Checked)(model, B, 60)
    S.GemmStep(model, B * 20, cache=cache).run(x_rows(device, model, B * 20, 71))
    tree = torch.tensor([[1, 3, 5, 0b1001, 0b10101, 0b100101]] * B, device=device)
    step = S.GemmStep(model, B * 6, cache=cache, tree=tree)
    x = x_rows(device, model, B * 6, 72)
    if captured:
        step.capture(x)
        step.replay()
    else:
        step.run(x)
    before = [t.clone() for t in cache.k + cache.v]
    say("accept", captured)
    cache.accept(6, [[0, 2, 5], [0, 1]])
    assert cache.lens.tolist() == cache.seen.tolist() == [23, 22]
    for t, was in zip(cache.k + cache.v, before):
        assert torch.equal(t[0, :20], was[0, :20]) and torch.equal(t[0, 20:23], was[0, [20, 22, 25]])
        assert torch.equal(t[1, :22], was[1, :22])
    S.GemmStep(model, B, cache=cache).run(x_rows(device, model, B, 73))
    assert cache.lens.tolist() == [24, 23] and cache._positions.tolist() == [23, 22]
