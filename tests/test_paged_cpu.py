"""The paged cache's and the adapters' libraries without a GPU: their surface, their
layouts, and the calls they refuse before anything is launched."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

import kernels
from kernels import _adapter_lib as AL
from kernels import _paged_lib as PL

ROOT = Path(__file__).resolve().parent.parent
BF = torch.bfloat16
# Fake, well-aligned device addresses far apart: validation never dereferences them.
(Q, K, V, TABLE, STARTS, KEYS, OUT, LSE, WS, LENS, KEEP, FRESH, LABELS, FREE, COUNT, SLOTS, POS, OWNER, COS, X, A, B_, SCALE, INDEX,
 Y) = (i << 36 for i in range(1, 26))

LIBS = [
    (PL, "krk_paged.h", "KRK_PAGED", ["krk_page_step_args", "krk_paged_rope_args", "krk_paged_shape", "krk_paged_attn_args"]),
    (AL, "krk_adapter.h", "KRK_ADAPTER", ["krk_adapter_shape", "krk_adapter_args"]),
]


def text(header):
    return re.sub(r"/\*.*?\*/", "", (ROOT / "include" / header).read_text(), flags=re.S)


@pytest.mark.parametrize("L,header,macro,structs", LIBS)
def test_header_matches_binding(L, header, macro, structs):
    lib = L.LIB.load()
    names = sorted(set(re.findall(r"\b(krk_\w+)\s*\(", text(header))))
    assert names == sorted(L.SIGNATURES)
    version = int(re.search(macro + r"_ABI_VERSION (\d+)", text(header)).group(1))
    assert version == getattr(lib, L.LIB.prefix + "abi_version")() == L.ABI_VERSION
    size = getattr(lib, L.LIB.prefix + "struct_size")
    assert [size(i) for i in range(len(structs))] == [ctypes.sizeof(s) for s in L.STRUCTS]
    assert size(len(structs)) == size(-1) == 0
    for cls, name in zip(L.STRUCTS, structs):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text(header), re.S).group(1)
        fields = []
        for decl in body.split(";"):
            decl = re.sub(r"\b(const|void|float|int|int32_t|int64_t|krk_pages)\b", " ", decl).replace("*", " ")
            decl = re.sub(r"\[\w+\]", "", decl)
            fields += [f.strip() for f in decl.split(",") if f.strip()]
        assert fields == [n for n, _ in cls._fields_]


@pytest.mark.parametrize("L", [PL, AL])
def test_binding_refuses_another_abi(L):
    other = type(L.LIB)(L.LIB_PATH, L.LIB.prefix, 99, L.STRUCTS, L.SIGNATURES)
    with pytest.raises(ImportError, match="ABI version"):
        other.load()
    gone = type(L.LIB)(Path("/nowhere.so"), L.LIB.prefix, 1, L.STRUCTS, L.SIGNATURES)
    with pytest.raises(ImportError, match="missing"):
        gone.load()


def refused(L, rc, code, msg):
    err = getattr(L.LIB.load(), L.LIB.prefix + "last_error")().decode()
    assert rc == code and msg in err, (rc, err)


# ------------------------------------------------------------- page tables
def step_args(**kw):
    a = PL.PageStepArgs(LENS, KEEP, FRESH, LABELS, TABLE, 10, FREE, COUNT, STARTS, KEYS, SLOTS, POS, OWNER, 4, 100, 50, 16, 10)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(B=0), -1, "B=0"), (dict(B=4097), -1, "4096"), (dict(rows=0), -1, "rows=0"), (dict(rows=(1 << 18) + 1), -1, "262144"),
    (dict(page_size=0), -1, "power of two"), (dict(page_size=4), -1, "power of two"), (dict(page_size=24), -1, "power of two"),
    (dict(page_size=8192), -1, "power of two"), (dict(pages=0), -1, "pages=0"), (dict(pages=1 << 27), -1, "2^31"),
    (dict(width=0), -1, "width=0"), (dict(width=1 << 23), -1, "2^27"), (dict(B=4096, width=1 << 19, table_row=1 << 19), -1, "2^31"),
    (dict(table_row=9), -1, "row stride 9"), (dict(free_count=0), -1, "come together"), (dict(free_pages=0), -1, "come together"),
    (dict(lens=0), -1, "lens"), (dict(fresh=0), -1, "fresh"), (dict(table=0), -1, "table"), (dict(starts=0), -1, "starts"),
    (dict(keys=0), -1, "keys"), (dict(slots=0), -1, "slots"), (dict(positions=0), -1, "positions"), (dict(owner=0), -1, "owner"),
    (dict(lens=LENS + 2), -2, "4-byte"), (dict(keep=KEEP + 1), -2, "4-byte"), (dict(labels=LABELS + 1), -2, "4-byte"),
    (dict(keep=LENS), -3, "share"), (dict(fresh=LENS + 12), -3, "share"), (dict(labels=SLOTS + 8), -3, "share"),
    (dict(keys=STARTS + 16), -3, "share"), (dict(positions=SLOTS), -3, "share"), (dict(free_count=FREE + 196), -3, "share"),
    (dict(owner=TABLE + 4 * 39), -3, "share"),
])
def test_page_steps_refused(kw, code, msg):
    refused(PL, PL.LIB.load().krk_page_step(ctypes.byref(step_args(**kw)), None), code, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(B=0), "B=0"), (dict(page_size=12), "power of two"), (dict(pages=0), "pages=0"), (dict(width=0), "width=0"),
    (dict(pages=1 << 28), "2^31"), (dict(rows=1.5), "rows must"), (dict(B="4"), "B must"), (dict(width=1 << 32), "32 bits"),
])
def test_tables_refused(kw, msg):
    d = dict(B=4, rows=10, pages=20, page_size=16, width=5, device="cpu")
    with pytest.raises(ValueError, match=re.escape(msg)):
        kernels.PageTables(**{**d, **kw})


def test_step_needs_the_gpu():
    t = kernels.PageTables(2, 4, 8, 8, 3, "cpu")
    assert t.free.tolist() == list(range(7, -1, -1)) and t.count.tolist() == [8] and t.slots.tolist() == [-1] * 4
    with pytest.raises(ValueError, match="GPU tensor"):
        t.step(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="Tensor"):
        t.step([1, 1])


# -------------------------------------------------------------------- rope
def pages(p, page, slot, head):
    return PL.Pages(p, page, slot, head)


def rope_args(**kw):
    a = PL.RopeArgs(Q, 12 * 128, 0, 0, 1e-6, COS, 100, SLOTS, POS, OUT, 1024, pages(K, 16 * 256, 256, 128), pages(V, 16 * 256, 256, 128),
                    5, 8, 2, 128, 50, 16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=0), -1, "rows=0"), (dict(heads=0), -1, "heads=0"), (dict(kv_heads=0), -1, "kv_heads=0"), (dict(heads=9), -1, "multiple"),
    (dict(head_dim=96), -6, "64 and 128"), (dict(page_size=10), -1, "power of two"), (dict(pages=0), -1, "pages=0"),
    (dict(qkv=0), -1, "qkv"), (dict(qkv_row=1000), -1, "row stride"), (dict(qkv_row=1540), -2, "multiple of 8"),
    (dict(qkv=Q + 8), -2, "16-byte"), (dict(q_norm=X), -1, "come together"), (dict(table_rows=0), -1, "table_rows"),
    (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"), (dict(table=0), -1, "table"), (dict(slots=0), -1, "slots"),
    (dict(positions=0), -1, "positions"), (dict(table=COS + 4), -2, "16-byte"), (dict(q_norm=X + 2, k_norm=Y), -2, "16-byte"),
    (dict(q_out=Q + 16), -3, "share"), (dict(q_out=Q, q_row=1024), -3, "share"), (dict(k=pages(V, 16 * 256, 256, 128)), -3, "share"),
    (dict(k=pages(K, 4096, 256, 64)), -3, "rows share"), (dict(k=pages(K, 2048, 256, 128)), -3, "rows share"),
    (dict(k=pages(K, 4096, 257, 128)), -2, "multiples of 8"), (dict(v=pages(V, -8, 256, 128)), -1, "out of range"),
    (dict(v=pages(V, (1 << 31) + 8, 256, 128)), -1, "out of range"), (dict(v=pages(V + 2, 4096, 256, 128)), -2, "16-byte"),
    (dict(v=pages(K + 128, 4096, 256, 128)), -3, "share"), (dict(slots=K + 64), -3, "share"), (dict(k=pages(0, 4096, 256, 128)), -1, "k: null"),
])
def test_paged_rope_refused(kw, code, msg):
    refused(PL, PL.LIB.load().krk_paged_rope_bf16(ctypes.byref(rope_args(**kw)), None), code, msg)


# --------------------------------------------------------------- attention
def shape(**kw):
    d = dict(B=4, rows=9, heads=8, kv_heads=2, head_dim=128, page_size=16, width=10, window=0, sinks=0)
    d.update(kw)
    return PL.Shape(*[d[n] for n, _ in PL.Shape._fields_])


@pytest.mark.parametrize("kw,msg", [
    (dict(B=0), "B=0"), (dict(B=5000), "4096"), (dict(rows=0), "rows=0"), (dict(rows=1 << 19), "262144"),
    (dict(rows=1 << 18, heads=128), "2^25"), (dict(heads=9), "multiple"), (dict(kv_heads=0), "multiple"), (dict(head_dim=256), "64 and 128"),
    (dict(page_size=20), "power of two"), (dict(width=0), "width=0"), (dict(width=1 << 23), "2^27"), (dict(window=-1), "window"),
    (dict(window=1 << 28), "2^28"), (dict(window=4, sinks=-1), "sinks"), (dict(sinks=4), "sinks need a window"),
])
def test_attention_shapes_refused(kw, msg):
    lib, s = PL.LIB.load(), shape(**kw)
    assert lib.krk_paged_check(ctypes.byref(s)) < 0 and msg in lib.krk_paged_last_error().decode()
    assert lib.krk_paged_workspace_bytes(ctypes.byref(s)) == 0
    d = dict(B=4, rows=9, heads=8, kv_heads=2, head_dim=128, page_size=16, width=10)
    with pytest.raises(ValueError, match=re.escape(msg)):
        kernels.PagedAttention(**{**d, **kw}, device="cpu")
    with pytest.raises(ValueError, match=re.escape(msg)):
        kernels.paged_workspace_bytes(**{**d, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=2.4e38), "scale"), (dict(scale=1e-60), "scale"),
    (dict(window=1 << 32), "window"), (dict(rows=2.0), "rows must"),
])
def test_attention_objects_refused(kw, msg):
    d = dict(B=4, rows=9, heads=8, kv_heads=2, head_dim=128, page_size=16, width=10, device="cpu")
    with pytest.raises(ValueError, match=msg):
        kernels.PagedAttention(**{**d, **kw})


def attn_args(**kw):
    a = PL.AttnArgs(Q, 1536, pages(K, 4096, 256, 128), pages(V, 4096, 256, 128), 50, 0.1, TABLE, 10, STARTS, KEYS, OUT, 1024, LSE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(pages=0), -1, "pages=0"), (dict(pages=1 << 27), -1, "2^31"), (dict(scale=0.0), -1, "scale"), (dict(scale=3.4e38), -1, "scale"),
    (dict(scale=float("nan")), -1, "scale"), (dict(q=0), -1, "q: null"), (dict(q_row=1000), -1, "row stride"), (dict(q=Q + 2), -2, "16-byte"),
    (dict(out_row=1028), -2, "multiple of 8"), (dict(out=0), -1, "out: null"), (dict(k=pages(0, 4096, 256, 128)), -1, "k: null"),
    (dict(v=pages(V, 4096, 252, 128)), -2, "multiples of 8"), (dict(k=pages(K, 1 << 32, 256, 128)), -1, "out of range"),
    (dict(k=pages(K, 4096, 1 << 31, 128)), -1, "out of range"), (dict(table=0), -1, "table"), (dict(table_row=9), -1, "row stride 9"),
    (dict(starts=0), -1, "starts"), (dict(keys=0), -1, "keys"), (dict(keys=KEYS + 1), -2, "4-byte"), (dict(lse=LSE + 2), -2, "4-byte"),
    (dict(out=Q), -3, "share"), (dict(lse=OUT + 64), -3, "overlap"), (dict(lse=KEYS), -3, "share"), (dict(out=K + 4096 * 20), -3, "share"),
])
def test_attention_calls_refused(kw, code, msg):
    s = shape()
    refused(PL, PL.LIB.load().krk_paged_attn_bf16(ctypes.byref(s), ctypes.byref(attn_args(**kw)), WS, 1 << 33, None), code, msg)


def test_attention_workspaces_refused():
    lib, s = PL.LIB.load(), shape()
    n = lib.krk_paged_workspace_bytes(ctypes.byref(s))
    if n:
        for ws, size, code in ((None, 0, -4), (WS, n - 1, -4), (WS + 8, n, -2), (K, n, -3)):
            rc = lib.krk_paged_attn_bf16(ctypes.byref(s), ctypes.byref(attn_args()), ws, size, None)
            assert rc == code, lib.krk_paged_last_error()


# ---------------------------------------------------------------- adapters
def adapter_shape(widths=(256,), **kw):
    d = dict(rows=5, N=256, K=512, rank=16, silu=0, slices=len(widths))
    d.update(kw)
    return AL.Shape(*[d[n] for n, _ in AL.Shape._fields_[:-1]], (ctypes.c_int * 4)(*widths))


@pytest.mark.parametrize("widths,kw,msg", [
    ((256,), dict(rows=0), "rows=0"), ((256,), dict(rows=(1 << 18) + 1), "262144"), ((256,), dict(K=12), "multiples of 8"),
    ((256,), dict(K=0), "multiples of 8"), ((260,), dict(N=260), "multiples of 8"), ((1 << 21,), dict(N=1 << 21), "1048576"),
    ((256,), dict(rank=0), "rank=0"), ((256,), dict(rank=12), "rank=12"), ((256,), dict(rank=136), "rank=136"), ((248,), {}, "248 columns"),
    ((128, 120, 12), {}, "slice 2"), ((256, 0), {}, "slice 1"), ((128, 64, 64), dict(silu=1), "silu"), ((192, 64), dict(silu=1), "silu"),
    ((264,), dict(N=264, silu=1), "silu"), ((256,), dict(silu=2), "silu must be"),
])
def test_adapter_shapes_refused(widths, kw, msg):
    lib, s = AL.LIB.load(), adapter_shape(widths, **kw)
    assert lib.krk_adapter_check(ctypes.byref(s)) < 0 and msg in lib.krk_adapter_last_error().decode(), lib.krk_adapter_last_error()
    assert lib.krk_adapter_workspace_bytes(ctypes.byref(s)) == 0
    d = dict(rows=5, N=256, K=512, rank=16)
    d.update({k: v for k, v in kw.items() if k in d})
    if kw.get("silu") != 2:
        with pytest.raises(ValueError, match=re.escape(msg)):
            kernels.LowRankAdapters(*d.values(), "cpu", slices=widths, silu=bool(kw.get("silu")))


@pytest.mark.parametrize("slices", [(), (8,) * 5])
def test_adapter_slices_refused(slices):
    with pytest.raises(ValueError, match="slices"):
        kernels.LowRankAdapters(5, 40, 64, 8, "cpu", slices=slices)


def adapter_args(**kw):
    a = AL.Args(X, 512, A, 16 * 512, 512, B_, 256 * 16, 16, SCALE, INDEX, Y, 256, OUT, 256, 7)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(adapters=0), -1, "adapters=0"), (dict(adapters=(1 << 20) + 1), -1, "1048576"), (dict(x=0), -1, "x: null"),
    (dict(ldx=504), -1, "row stride"), (dict(ldx=516), -2, "multiple of 8"), (dict(a=0), -1, "a: null"), (dict(a_row=504), -1, "a: strides"),
    (dict(a_adapter=-8), -1, "a: strides"), (dict(b_row=8), -1, "b: strides"), (dict(b_row=20), -2, "multiples of 8"),
    (dict(b=B_ + 8), -2, "16-byte"), (dict(scale=SCALE + 2), -2, "4-byte"), (dict(index=0), -1, "index"), (dict(y=0), -1, "y: null"),
    (dict(out=0), -1, "out: null"), (dict(ldo=248), -1, "row stride"), (dict(out=Y, ldo=264), -3, "share"), (dict(out=Y + 16), -3, "share"),
    (dict(out=X), -3, "share"), (dict(out=INDEX), -3, "share"), (dict(out=B_ + 1024), -3, "share"),
])
def test_adapter_calls_refused(kw, code, msg):
    s = adapter_shape()
    refused(AL, AL.LIB.load().krk_adapter_bf16(ctypes.byref(s), ctypes.byref(adapter_args(**kw)), WS, 1 << 30, None), code, msg)


def test_adapter_workspaces_and_silu_in_place_refused():
    lib, s = AL.LIB.load(), adapter_shape()
    n = lib.krk_adapter_workspace_bytes(ctypes.byref(s))
    for ws, size, code in ((None, 0, -4), (WS, n - 1, -4), (WS + 8, n, -2), (X, n, -3), (OUT, n, -3)):
        assert lib.krk_adapter_bf16(ctypes.byref(s), ctypes.byref(adapter_args()), ws, size, None) == code
    s = adapter_shape(silu=1)
    refused(AL, lib.krk_adapter_bf16(ctypes.byref(s), ctypes.byref(adapter_args(out=Y)), WS, 1 << 30, None), -3, "share")


def test_null_arguments():
    p, a = PL.LIB.load(), AL.LIB.load()
    assert p.krk_page_step(None, None) == -1 and p.krk_paged_rope_bf16(None, None) == -1
    assert p.krk_paged_attn_bf16(None, None, None, 0, None) == -1 and p.krk_paged_check(None) == -1
    assert a.krk_adapter_bf16(None, None, None, 0, None) == -1 and a.krk_adapter_check(None) == -1


def test_python_calls_need_the_gpu():
    q = torch.zeros((9, 1024), dtype=BF)
    pool = torch.zeros((5, 16, 2, 128), dtype=BF)
    i = torch.zeros(9, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        kernels.paged_qk_norm_rope(torch.zeros((9, 12 * 128), dtype=BF), None, None, 1e-6, torch.zeros((4, 128)), i, i, pool, pool)
    s = shape()
    if PL.LIB.load().krk_paged_workspace_bytes(ctypes.byref(s)) < 1 << 30:
        op = kernels.PagedAttention(4, 9, 8, 2, 128, 16, 10, "cpu")
        with pytest.raises(ValueError, match="GPU tensor"):
            op(q, pool, pool, torch.zeros((4, 10), dtype=torch.int32), i[:5], i[:4])
    ad = kernels.LowRankAdapters(9, 256, 1024, 16, "cpu")
    with pytest.raises(ValueError, match="GPU tensor"):
        ad(q, torch.zeros((2, 16, 1024), dtype=BF), torch.zeros((2, 256, 16), dtype=BF), i, torch.zeros((9, 256), dtype=BF))


# ------------------------------------------------- a model's cache, its host side
@pytest.fixture(scope="module")
def model():
    from kernels import step

    return step.synthetic_model("cpu", layers=1, hidden=64, intermediate=64, heads=2, kv_heads=1, head_dim=64, vocab=64)


def test_schedules(model):
    c = kernels.PagedCache(model, 3, 30, 8, 8, width=5)
    with pytest.raises(RuntimeError, match="schedule"):
        c.planned()
    assert c.schedule([17, 0, 9]) == [0, 17, 17]
    c.planned()
    assert c.new.tolist() == [17, 0, 9] and c.keep.tolist() == [0, 0, 0] and c.lens == [0, 0, 0]
    c.commit()
    assert c.lens == [17, 0, 9]
    for new, msg in (([1, 0], "each of 3"), ([1, -1, 0], "each of 3"), ([10, 10, 11], "31 rows"), ([24, 0, 0], "pass its 5 pages"),
                     ([8, 14, 8], "9 of 8 pages")):
        with pytest.raises(ValueError, match=msg):
            c.schedule(new)
        assert c.lens == [17, 0, 9] and c.new.tolist() == [17, 0, 9]
    c.rollback([2, 0, 9])
    with pytest.raises(RuntimeError, match="schedule"):
        c.planned()
    with pytest.raises(ValueError, match="rollback"):
        c.rollback([16, 0, 0])
    c.schedule([1, 24, 0])  # 2 + 3 pages
    assert c.keep.tolist() == [15, 0, 0]
    c.commit()
    c.reset(1)
    assert c.lens == [16, 0, 0]
    c.reset()
    assert c.lens == [0, 0, 0]
    c.check(30)
    with pytest.raises(ValueError, match="M=29"):
        c.check(29)


def test_adapter_sets(model):
    s = kernels.AdapterSet(model, 2, 8)
    assert [tuple(s.a[t][0].shape) for t in s.targets] == [(2, 24, 64), (2, 8, 128), (2, 16, 64), (2, 8, 64)]
    assert [tuple(s.b[t][0].shape) for t in s.targets] == [(2, 256, 8), (2, 64, 8), (2, 128, 8), (2, 64, 8)]
    for kw in (dict(targets=()), dict(targets=("lm",)), dict(targets=("o", "o")), dict(rank=9), dict(adapters=0)):
        with pytest.raises(ValueError):
            kernels.AdapterSet(model, **{**dict(adapters=1, rank=8), **kw})
