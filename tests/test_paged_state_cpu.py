"""PagedCache's host side: what a request leaves behind when it ends."""

from __future__ import annotations

import pytest
import torch

import kernels
from kernels import step


@pytest.fixture(scope="module")
def model():
    return step.synthetic_model("cpu", layers=1, hidden=64, intermediate=64, heads=2, kv_heads=1, head_dim=64, vocab=64)


def test_a_request_that_ends_takes_its_adapter_with_it(model):
    c = kernels.PagedCache(model, 4, 30, 8, 8)
    c.labels.copy_(torch.tensor([2, 0, 1, 3], dtype=torch.int32))
    c.schedule([3, 4, 5, 6])
    c.commit()
    c.rollback([1, 0, 0, 6])
    assert c.labels.tolist() == [2, 0, 1, 3]  # keys that are taken back end no request
    c.reset(1)
    assert c.labels.tolist() == [2, -1, 1, 3] and c.lens == [2, 0, 5, 0]
    c.labels[1] = 2
    c.schedule([0, 1, 0, 0])
    assert c.labels.tolist() == [2, 2, 1, 3]
    c.reset()
    assert c.labels.tolist() == [-1] * 4 and c.lens == [0] * 4
