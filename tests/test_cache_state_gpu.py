"""A DecodeCache on the GPU across steps that fail, many sizes of step, and
streams."""

from __future__ import annotations

import pytest
import torch

from kernels import cache as C
from kernels import step as S
from oracle import gemm_ref as R

from test_attn_gpu import say

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
