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


def strided(p, seq, slot, head):
    return L.Cache(p, seq, slot, head)


#: Strides (elements) of a [2, 50, 2, 128] cache whose rows share memory, though each is 128 or more.
SHARING = [(12800, 128, 128), (6400, 256, 128), (12800, 256, 192), (12800, 256, 256), (25600, 200, 128)]


@pytest.mark.parametrize("st", SHARING)
def test_written_caches_whose_rows_share_memory(lib, st):
    sharing = strided(K, *st)
    msg = "rows share memory"
    refused(lib.krk_qk_norm_rope_bf16(ctypes.byref(rope_args(k=sharing)), None), -3, msg)
    refused(lib.krk_qk_norm_rope_bf16(ctypes.byref(rope_args(v=sharing)), None), -3, msg)
    a = evict_args(True, k=sharing, k_out=sharing)
    refused(lib.krk_cache_evict_bf16(ctypes.byref(a), None), -3, msg)
    if st != (6400, 256, 128):  # of 20 slots these are apart
        a = evict_args(k_out=strided(1 << 41, *st))
        refused(lib.krk_cache_evict_bf16(ctypes.byref(a), None), -3, msg)


def test_written_scores_whose_rows_share_memory(lib):
    s = shape(scored=1)
    a = args(s, scores=SC, sc_seq=1000, sc_head=500, scores_out=SO, so_seq=500, so_head=500)
    refused(lib.krk_attn_bf16(ctypes.byref(s), ctypes.byref(a), WS, 1 << 30, None), -3, "rows share memory")
    refused(lib.krk_cache_evict_bf16(ctypes.byref(evict_args(so_seq=30, so_head=20)), None), -3, "rows share memory")


#: Where v may not begin, in elements behind a k of [2, 50, 2, 128] with these strides.
OVERLAPPING = [((12800, 256, 128), d) for d in (64, 128, 256, 12800, 12736, 25480, -64, -256 * 7)] + [
    ((25600, 512, 256), d) for d in (64, 120, 136, 256, 512, 25600, 512 * 3 + 64, -64, -25600)] + [
    ((25600, 256, 12800), d) for d in (64, 256, 192, -12800)]


@pytest.mark.parametrize("st,d", OVERLAPPING)
def test_k_and_v_that_share_memory(lib, st, d):
    k, v = strided(K, *st), strided(K + 2 * d, *st)
    refused(lib.krk_qk_norm_rope_bf16(ctypes.byref(rope_args(k=k, v=v)), None), -3, "share")
    refused(lib.krk_cache_evict_bf16(ctypes.byref(evict_args(True, k=k, v=v, k_out=k, v_out=v)), None), -3, "share")
    a = evict_args(k_out=strided(1 << 41, *st), v_out=strided((1 << 41) + 2 * d, *st), keep=LENS)
    msg = "with the inputs" if d == 25480 else "k_out and v_out"  # behind the 20 slots of a k_out
    refused(lib.krk_cache_evict_bf16(ctypes.byref(a), None), -3, msg)


def test_k_and_v_of_different_strides_in_one_tensor(lib):
    k, v = strided(K, 25600, 512, 256), strided(K + 256, 25600, 256, 128)
    refused(lib.krk_qk_norm_rope_bf16(ctypes.byref(rope_args(k=k, v=v)), None), -3, "share")


@pytest.mark.parametrize("st,d", [
    ((25600, 512, 256), 128), ((25600, 512, 256), -128), ((25600, 512, 128), 256), ((25600, 256, 128), 12800),
    ((25600, 256, 12800), 128), ((25600, 512, 256), 51200), ((12800, 256, 128), 25600), ((51200, 128, 6400), 12800),
])
def test_k_and_v_side_by_side_in_one_tensor(lib, st, d):
    """Interleaved by head, slot or sequence, or one behind the other: taken (the
    call is refused further on, as keep lies in lens)."""
    k, v = strided(K, *st), strided(K + 2 * d, *st)
    refused(lib.krk_cache_evict_bf16(ctypes.byref(evict_args(True, k=k, v=v, k_out=k, v_out=v, keep=LENS)), None), -3, "with the inputs")
