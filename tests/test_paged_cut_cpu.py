"""How calls of attention over pages are cut into jobs, replayed on the host with the
library's own arithmetic: every job comes up once, and all of them within the grid and
the workspace, up to the limits of what the library takes."""

from __future__ import annotations

import ctypes
import itertools
import random
import shutil
import subprocess
from pathlib import Path

import pytest

import kernels
from kernels import _paged_lib as PL
from test_paged_forms_gpu import FORMS

ROOT = Path(__file__).resolve().parent.parent
FIELDS = ("blocks", "rows", "counters", "jobs", "used", "pairs", "rounds", "few_parts", "many_parts", "wrong")


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    so = tmp_path_factory.mktemp("cut") / "cut.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-ffp-contract=off", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "kernel-rush-kawk_amd" / "csrc"), str(ROOT / "tests" / "paged_cut.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.replay.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float, ctypes.c_void_p]

    def run(new, keys, heads, kv, D, P, *, rows=None, width=None, window=0, sinks=0, nudge=1.0):
        """One call of requests of `new` rows and `keys` keys; refused shapes are a mistake of the test."""
        B = len(new)
        rows = rows or max(1, sum(new))
        width = width or max(1, max(-(-n // P) for n in keys))
        shape = PL.Shape(B, rows, heads, kv, D, P, width, window, sinks)
        PL.LIB.check(PL.LIB.load().krk_paged_check(ctypes.byref(shape)))
        starts = (ctypes.c_int32 * (B + 1))(0, *itertools.accumulate(new))
        out = (ctypes.c_int64 * len(FIELDS))()
        lib.replay(ctypes.byref(shape), starts, (ctypes.c_int32 * B)(*keys), nudge, out)
        r = dict(zip(FIELDS, out))
        assert r["jobs"] <= r["blocks"] and r["used"] <= r["rows"] and -(-r["used"] // 16) <= r["counters"] and r["wrong"] == 0, r
        return r

    return run


@pytest.mark.parametrize("rows,heads,kv,keys", [
    (1 << 18, 64, 1, 1 << 20),         # 2^17 tiles of 2^14 steps: 2^31
    (1 << 18, 64, 1, 1 << 21),         # 2^32
    (1 << 18, 64, 1, (1 << 27) - 64),  # the longest table
    (1 << 15, 4, 1, (1 << 27) - 64), (1 << 18, 127, 1, 3 << 20), (1 << 15, 1000, 8, 1 << 22),
])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_times_steps_beyond_31_bits(replay, rows, heads, kv, keys, D):
    """The work of one request: jobs stay within the grid where its tiles' steps pass 2^31."""
    r = replay([rows], [keys], heads, kv, D, 64)
    assert r["many_parts"] == 1  # far more tiles than workgroups
    replay([rows - 70] + [1] * 70, [keys] + [9] * 70, heads, kv, D, 64)


@pytest.mark.parametrize("kw", [
    dict(B=4096, rows=4096, heads=8191, kv_heads=8191, width=1), dict(B=4096, rows=4096, heads=8191, kv_heads=8191, width=100),
    dict(B=1, rows=1, heads=(1 << 25) - 1, kv_heads=(1 << 25) - 1, width=1),
])
def test_grids_beyond_32_bits_refused(kw):
    """A workgroup of 256 threads for every tile of a key/value head, and fewer than 2^32 threads in all."""
    lib, s = PL.LIB.load(), PL.Shape(head_dim=64, page_size=8, **kw)
    assert lib.krk_paged_check(ctypes.byref(s)) == -1 and "2^32 threads" in lib.krk_paged_last_error().decode()
    assert lib.krk_paged_workspace_bytes(ctypes.byref(s)) == 0
    with pytest.raises(ValueError, match="threads"):
        kernels.PagedAttention(**kw, head_dim=64, page_size=8, device="cpu")
    s.heads = s.kv_heads = s.heads // 4
    assert lib.krk_paged_check(ctypes.byref(s)) == 0


@pytest.mark.parametrize("name", list(FORMS))
def test_forms_that_the_gpu_tests_reach(replay, name):
    new, keys, heads, kv, D, P, window, sinks, want = FORMS[name]
    r = replay(new, keys, heads, kv, D, P, rows=sum(new) + 3, width=-(-max(keys) // P) + 1, window=window, sinks=sinks)
    assert all(r[k] >= n for k, n in want.items()), r


def spread(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


@pytest.mark.parametrize("seed", range(12))
def test_random_calls(replay, seed):
    """Requests of every kind, up to the limits; sums of the costs off by what their order may change."""
    rng = random.Random(seed)
    for _ in range(40):
        heads, kv = rng.choice([(32, 8), (8, 2), (4, 1), (16, 16), (24, 8), (40, 8), (64, 1), (7, 1), (1, 1)])
        B = spread(rng, 1, 4096 if rng.random() < 0.3 else 64)
        P = 1 << rng.randint(3, 12)
        most = min((1 << 27) - P, ((1 << 31) - 1) // B * P)
        longest = spread(rng, 1, most)
        budget = min(1 << 18, ((1 << 25) - 1) // heads)
        kinds = [rng.choice(["idle", "one", "one", "draft", "chunk"]) for _ in range(B)]
        new, left = [], budget
        for k in kinds:
            n = {"idle": 0, "one": 1, "draft": rng.randint(2, 40), "chunk": spread(rng, 40, 60000)}[k]
            n = min(n, left)
            left -= n
            new.append(n)
        keys = [rng.choice([longest, rng.randint(0, longest), spread(rng, 1, longest)]) for _ in range(B)]
        window = rng.choice([0, 0, spread(rng, 1, 1 << 20)])
        sinks = rng.choice([0, 4, 1000]) if window else 0
        rows = min(budget, max(1, sum(new)) + rng.choice([0, 0, 9, 5000]))
        for nudge in (1.0, 1 - 2.0 ** -18, 1 + 2.0 ** -18):
            replay(new, keys, heads, kv, rng.choice([64, 128]), P, rows=rows, width=-(-longest // P), window=window, sinks=sinks, nudge=nudge)
