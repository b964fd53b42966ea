"""Calls of the cache operators that could not give their results, refused
before anything is launched (fake, well-aligned addresses)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernels import _attn_lib as L
from kernels import attention as A

from test_attn_cpu import K, LENS, SC, SO, V, WS, args, cache, evict_args, rope_args, shape

BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    return L.load()


def refused(rc, code, msg):
    assert rc == code and msg in L.last_error(), (rc, L.last_error())


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scales_beyond_the_kernels_exponent(lib, scale):
    """scale * log2(e) would be infinite, and every output NaN."""
    s = shape()
    a = args(s, scale=scale)
    refused(lib.krk_attn_bf16(ctypes.byref(s), ctypes.byref(a), WS, 1 << 30, None), -1, "scale")
    with pytest.raises(ValueError, match="scale"):
        A.CacheAttention(2, 1, 8, 2, 128, 50, "cpu", scale=scale)


def test_scales_below_fp32():
    with pytest.raises(ValueError, match="scale"):
        A.CacheAttention(2, 1, 8, 2, 128, 50, "cpu", scale=1e-60)
