"""The cache operators' library without a GPU: its surface, its layouts, its
plans, and the calls it refuses before anything is launched."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from kernels import _attn_lib as L
from kernels import attention as A

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "krk_attn.h"
BF = torch.bfloat16
# Fake, well-aligned device addresses far apart: validation never dereferences them.
Q, K, V, KP, VP, LENS, TREE, OUT, LSE, SC, SO, WS = (i << 36 for i in range(1, 13))


@pytest.fixture(scope="module")
def lib():
    return L.load()


def text():
    return re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)


def test_header_matches_binding(lib):
    names = sorted(set(re.findall(r"\b(krk_\w+)\s*\(", text())))
    assert names == sorted(L.SIGNATURES)
    for n in names:
        assert hasattr(lib, n)
    version = int(re.search(r"#define KRK_ATTN_ABI_VERSION (\d+)", HEADER.read_text()).group(1))
    assert version == lib.krk_attn_abi_version() == L.ABI_VERSION
    assert [lib.krk_attn_struct_size(i) for i in range(5)] == [ctypes.sizeof(s) for s in L.STRUCTS]
    assert lib.krk_attn_struct_size(5) == lib.krk_attn_struct_size(-1) == 0


@pytest.mark.parametrize("i,name", enumerate(["krk_attn_shape", "krk_attn_args", "krk_rope_args", "krk_evict_args",
                                              "krk_attn_plan_t"]))
def test_struct_fields_in_the_headers_order(i, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text(), re.S).group(1)
    fields = []
    for decl in body.split(";"):
        decl = re.sub(r"\b(const|void|float|int|int32_t|int64_t|krk_cache)\b", " ", decl).replace("*", " ")
        fields += [f.strip() for f in decl.split(",") if f.strip()]
    assert fields == [n for n, _ in L.STRUCTS[i]._fields_]


def test_binding_refuses_another_abi(monkeypatch):
    monkeypatch.setattr(L, "_lib", None)
    monkeypatch.setattr(L, "ABI_VERSION", 99)
    with pytest.raises(ImportError, match="ABI version"):
        L.load()


def shape(**kw):
    d = dict(B=2, R=1, heads=8, kv_heads=2, head_dim=128, capacity=500, window=0, sinks=0, prefix=0, scored=0)
    d.update(kw)
    return L.AttnShape(*[d[n] for n, _ in L.AttnShape._fields_])


@pytest.mark.parametrize("kw,msg", [
    (dict(B=0), ">= 1"), (dict(R=0), ">= 1"), (dict(R=-3), ">= 1"), (dict(kv_heads=0), ">= 1"), (dict(capacity=0), ">= 1"),
    (dict(heads=9), "multiple of kv_heads"), (dict(head_dim=96), "64 and 128"), (dict(head_dim=256), "64 and 128"),
    (dict(B=70000), "too large"), (dict(R=70000), "too large"), (dict(B=60000, R=60000), "2^25"),
    (dict(B=65535, heads=1024, kv_heads=1), "2^25"), (dict(B=65535, heads=256, kv_heads=256), "2^23"),
    (dict(capacity=1 << 27), "2^27"), (dict(capacity=1 << 26, prefix=1 << 26), "2^27"), (dict(window=-1), "negative"),
    (dict(window=4, sinks=-1), "negative"), (dict(prefix=-1), "negative"), (dict(sinks=4), "sinks need a window"),
    (dict(window=1 << 28), "2^28"), (dict(scored=2), "scored must be"), (dict(scored=1, prefix=5), "shared prefix"),
])
def test_shapes_refused(lib, kw, msg):
    s = shape(**kw)
    assert lib.krk_attn_check(ctypes.byref(s)) < 0 and msg in L.last_error()
    assert lib.krk_attn_workspace_bytes(ctypes.byref(s)) == 0
    d = dict(B=2, R=1, heads=8, kv_heads=2, head_dim=128, capacity=500)
    opts = {k: v for k, v in kw.items() if k in ("window", "sinks", "prefix")}
    d.update({k: v for k, v in kw.items() if k in d})
    if kw.get("scored") != 2:
        with pytest.raises(ValueError, match=re.escape(msg)):
            A.CacheAttention(*d.values(), "cpu", scored=bool(kw.get("scored")), **opts)


@pytest.mark.parametrize("kw,msg", [
    (dict(window=1 << 32), "window"), (dict(capacity=(1 << 32) + 500), "capacity"), (dict(R=1.0), "R must"),
    (dict(B=None), "B must"), (dict(prefix="3"), "prefix"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=1e300), "scale"),
    (dict(head_dim=0), "64 and 128"),
])
def test_sizes_that_do_not_fit(kw, msg):
    d = dict(B=2, R=1, heads=8, kv_heads=2, head_dim=128, capacity=500, device="cpu")
    with pytest.raises(ValueError, match=msg):
        A.CacheAttention(**{**d, **kw})


@pytest.mark.parametrize("kw", [dict(budget=1 << 32, capacity=1 << 33), dict(sinks=1.5), dict(B=None), dict(recent="2")])
def test_eviction_sizes_that_do_not_fit(kw):
    d = dict(B=2, kv_heads=2, head_dim=128, capacity=500, budget=100, device="cpu")
    with pytest.raises(ValueError, match="32 bits"):
        A.CacheEviction(**{**d, **kw})


def test_null_arguments(lib):
    assert lib.krk_attn_check(None) < 0 and lib.krk_attn_plan(None, None) < 0
    assert lib.krk_attn_bf16(None, None, None, 0, None) < 0
    assert lib.krk_qk_norm_rope_bf16(None, None) < 0 and lib.krk_cache_evict_bf16(None, None) < 0


def cache(p, slots, heads, dim=128, seqs=2):
    return L.Cache(p, slots * heads * dim, heads * dim, dim)


def args(s, **kw):
    a = L.AttnArgs()
    cols = s.heads * s.head_dim
    a.q, a.q_row, a.out, a.out_row, a.lens, a.scale = Q, cols, OUT, cols, LENS, 0.1
    a.k, a.v = cache(K, s.capacity, s.kv_heads), cache(V, s.capacity, s.kv_heads)
    for name, v in kw.items():
        field, _, sub = name.partition("__")
        if sub:
            setattr(getattr(a, field), sub, v)
        else:
            setattr(a, name, v)
    return a


@pytest.mark.parametrize("sk,kw,code,msg", [
    ({}, dict(q=0), -1, "q: null"), ({}, dict(out=0), -1, "out: null"), ({}, dict(lens=0), -1, "lens"),
    ({}, dict(k__p=0), -1, "k: null"), ({}, dict(v__p=0), -1, "v: null"),
    ({}, dict(q_row=512), -1, "row stride"), ({}, dict(q_row=1027), -2, "multiple of 8"), ({}, dict(q=Q + 8), -2, "16-byte"),
    ({}, dict(out_row=1000), -1, "row stride"), ({}, dict(k__slot=-8), -1, "out of range"), ({}, dict(v__head=4), -2, "multiples of 8"),
    ({}, dict(k__p=K + 2), -2, "16-byte"), ({}, dict(k__seq=1 << 41), -1, "out of range"),
    ({}, dict(scale=0.0), -1, "scale"), ({}, dict(scale=-1.0), -1, "scale"), ({}, dict(scale=math.nan), -1, "scale"),
    ({}, dict(scale=math.inf), -1, "scale"), ({}, dict(prefix=1), -1, "prefix"), ({}, dict(prefix=-1), -1, "prefix"),
    (dict(prefix=10), dict(prefix=10), -1, "prefix k: null"),
    (dict(R=65), dict(tree=TREE), -1, "R <= 64"), (dict(R=9, window=8), dict(tree=TREE), -1, "window of 0 or >= R"),
    ({}, dict(tree=TREE + 4), -2, "8-byte"), ({}, dict(lens=LENS + 2), -2, "4-byte"),
    ({}, dict(scores=SC), -1, "scored = 0"), (dict(scored=1), {}, -1, "scores: null"),
    (dict(scored=1), dict(scores=SC, sc_seq=1000, sc_head=500), -1, "scores_out: null"),
    (dict(scored=1), dict(scores=SC, sc_seq=1000, sc_head=500, scores_out=SO, so_seq=0, so_head=500), -1, "at least its"),
    (dict(scored=1), dict(scores=SC, sc_seq=1000, sc_head=500, scores_out=SC + 4, so_seq=1000, so_head=500), -3, "share memory"),
    ({}, dict(out=Q + 1024), -3, "share memory"), ({}, dict(out=K + 4096), -3, "share memory"),
    ({}, dict(lse=LENS), -3, "share memory"), ({}, dict(lse=OUT + 16), -3, "overlap"),
])
def test_calls_refused(lib, sk, kw, code, msg):
    s = shape(**sk)
    a = args(s, **kw)
    rc = lib.krk_attn_bf16(ctypes.byref(s), ctypes.byref(a), WS, 1 << 30, None)
    assert rc == code and msg in L.last_error(), L.last_error()


def test_workspace_refused(lib):
    s = shape(B=1, capacity=4000)
    need = lib.krk_attn_workspace_bytes(ctypes.byref(s))
    assert need > 0
    a = args(s)
    call = lambda ws, n: lib.krk_attn_bf16(ctypes.byref(s), ctypes.byref(a), ws, n, None)
    assert call(0, need) == -4 and call(WS, need - 1) == -4 and "workspace" in L.last_error()
    assert call(WS + 8, need) == -2
    assert call(OUT, need) == -3


@pytest.mark.parametrize("R", [1, 2, 4, 5, 8, 9, 16, 17, 64, 65, 2048])
def test_plans_cover_the_rows_and_fit_the_workspace(lib, R):
    for heads, kv, D in ((32, 8, 128), (4, 1, 128), (16, 16, 64), (40, 8, 128), (24, 1, 64)):
        for B in (1, 7, 64):
            for cap in (1, 33, 4000, 200000):
                for kw in ({}, dict(window=1), dict(window=4096, sinks=4), dict(prefix=1), dict(prefix=40000), dict(scored=1)):
                    s = shape(B=B, R=R, heads=heads, kv_heads=kv, head_dim=D, capacity=cap, **kw)
                    p = L.AttnPlan()
                    assert lib.krk_attn_plan(ctypes.byref(s), ctypes.byref(p)) == 0
                    assert p.splits >= 1 and p.rows >= 16 and (p.prefix_splits >= 1) == (s.prefix > 0)
                    rows = B * R * heads
                    n = p.splits + p.prefix_splits
                    need = (n * rows * (4 * D + 8) if n > 1 else 0) + (8 * rows if s.scored else 0)
                    if s.scored and p.rows == 16 and not s.window:
                        need += 4 * rows * (-(-cap // 32) * 32)  # kept q.k
                    got = lib.krk_attn_workspace_bytes(ctypes.byref(s))
                    assert need <= got <= need + 4 * B * kv + 8192


def _t(*s, dtype=BF):
    return torch.zeros(s, dtype=dtype)


def test_python_calls_refuse_cpu_tensors():
    op = A.CacheAttention(2, 1, 8, 2, 128, 50, "cpu")
    k = _t(2, 50, 2, 128)
    lens = _t(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        op(_t(2, 1024), k, k.clone(), lens)
    with pytest.raises(ValueError, match="GPU"):
        A.qk_norm_rope(_t(2, 1536), None, None, 1e-6, _t(50, 128, dtype=torch.float32), lens, k, k.clone())
    with pytest.raises(ValueError, match="GPU"):
        A.CacheEviction(2, 2, 128, 50, 20, "cpu")(k, k.clone(), _t(2, 2, 50, dtype=torch.float32), lens)
    with pytest.raises(ValueError, match="torch.Tensor"):
        op(None, k, k, lens)


@pytest.mark.parametrize("kw,msg", [
    (dict(budget=0), "budget"), (dict(budget=51), "budget"), (dict(sinks=-1), "sinks"), (dict(recent=-1), "recent"),
    (dict(sinks=11, recent=10), "together"), (dict(head_dim=80), "head_dim"), (dict(B=0), ">= 1"),
])
def test_eviction_constructor_refuses(kw, msg):
    d = dict(B=2, kv_heads=2, head_dim=128, capacity=50, budget=20, device="cpu", sinks=2, recent=3)
    d.update(kw)
    with pytest.raises(ValueError, match=msg):
        A.CacheEviction(d.pop("B"), d.pop("kv_heads"), d.pop("head_dim"), d.pop("capacity"), d.pop("budget"),
                        d.pop("device"), **d)


def rope_args(**kw):
    a = L.RopeArgs()
    a.B, a.R, a.heads, a.kv_heads, a.head_dim, a.capacity = 2, 3, 8, 2, 128, 50
    a.qkv, a.qkv_row, a.q_out, a.q_row = Q, 12 * 128, OUT, 1024
    a.q_norm, a.k_norm, a.eps, a.table, a.table_rows, a.lens = KP, VP, 1e-6, SC, 60, LENS
    a.k, a.v = cache(K, 50, 2), cache(V, 50, 2)
    for name, v in kw.items():
        field, _, sub = name.partition("__")
        setattr(getattr(a, field), sub, v) if sub else setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(R=0), -1, ">= 1"), (dict(heads=9), -1, "multiple"), (dict(head_dim=32), -6, "64 and 128"),
    (dict(qkv=0), -1, "qkv: null"), (dict(qkv_row=1024), -1, "row stride"), (dict(q_row=1028), -2, "multiple of 8"),
    (dict(q_norm=0), -1, "together"), (dict(lens=0), -1, "null"), (dict(table=0), -1, "null"), (dict(table_rows=0), -1, "table_rows"),
    (dict(eps=-1.0), -1, "eps"), (dict(eps=math.nan), -1, "eps"), (dict(table=SC + 4), -2, "16-byte"),
    (dict(positions=SO + 1), -2, "4-byte"), (dict(k__slot=64), -1, "at least head_dim"), (dict(v__p=K), -3, "share"),
    (dict(q_out=Q + 16), -3, "share"), (dict(q_out=Q), -3, "share"), (dict(k__p=Q), -3, "share"), (dict(lens=V + 64), -3, "share"),
])
def test_rope_refuses(lib, kw, code, msg):
    a = rope_args(**kw)
    assert lib.krk_qk_norm_rope_bf16(ctypes.byref(a), None) == code and msg in L.last_error(), L.last_error()


def evict_args(inplace=False, **kw):
    a = L.EvictArgs()
    a.B, a.kv_heads, a.head_dim, a.capacity, a.budget, a.sinks, a.recent = 2, 2, 128, 50, 20, 2, 3
    a.k, a.v = cache(K, 50, 2), cache(V, 50, 2)
    a.scores, a.sc_seq, a.sc_head = SC, 100, 50
    a.k_out, a.v_out = (a.k, a.v) if inplace else (cache(KP, 20, 2), cache(VP, 20, 2))
    a.scores_out, a.so_seq, a.so_head = (SC, 100, 50) if inplace else (SO, 40, 20)
    a.lens, a.lens_out, a.keep = LENS, LENS, WS
    for name, v in kw.items():
        field, _, sub = name.partition("__")
        setattr(getattr(a, field), sub, v) if sub else setattr(a, name, v)
    return a


@pytest.mark.parametrize("inplace,kw,code,msg", [
    (False, dict(budget=0), -1, "budget"), (False, dict(budget=60), -1, "budget"), (False, dict(sinks=18), -1, "together"),
    (False, dict(recent=-1), -1, ">= 0"), (False, dict(keep=0), -1, "null"), (False, dict(lens_out=0), -1, "null"),
    (False, dict(k_out__slot=64), -1, "at least head_dim"), (False, dict(v_out__p=KP), -3, "one tensor"),
    (False, dict(k_out__p=K + 512), -3, "share"), (False, dict(scores_out=SC + 4), -3, "share"), (False, dict(keep=SO), -3, "overlap"),
    (False, dict(keep=LENS), -3, "share"), (False, dict(so_head=10), -1, "at least its"),
    (True, dict(v_out__p=VP), -3, "in place"), (True, dict(scores_out=SO), -3, "in place"), (True, dict(k_out__head=256), -3, "in place"),
    (True, dict(k__slot=0, k_out__slot=0), -1, "at least head_dim"), (False, dict(lens=LENS + 1), -2, "4-byte"),
])
def test_evict_refuses(lib, inplace, kw, code, msg):
    a = evict_args(inplace, **kw)
    assert lib.krk_cache_evict_bf16(ctypes.byref(a), None) == code and msg in L.last_error(), L.last_error()


def test_rope_table():
    t = A.rope_table(40000, 128, 1e6, "cpu")
    pos = 39999
    want = [math.cos(pos * 1e6 ** (-2 * i / 128)) for i in range(64)]
    assert t.shape == (40000, 128) and t.dtype == torch.float32
    assert max(abs(a - b) for a, b in zip(t[pos, :64].tolist(), want)) <= 2.0 ** -24
    with pytest.raises(ValueError):
        A.rope_table(0, 128, 1e6, "cpu")
    with pytest.raises(ValueError):
        A.rope_table(5, 127, 1e6, "cpu")
