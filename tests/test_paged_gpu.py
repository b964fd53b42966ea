"""The paged cache on the GPU against the oracle: page tables, rotary embedding into
pages, attention of mixed steps, and calls captured in graphs."""

from __future__ import annotations

import math
import random

import pytest
import torch

import kernels as K
from kernels.step import synthetic_model
from oracle import attn_ref as A64
from oracle import paged_ref as P64
from test_attn_gpu import close, gen, rnd, say

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32


def i32(dev, values):
    return torch.tensor(values, dtype=I32, device=dev)


# ------------------------------------------------------------- page tables
NAMES = ("starts", "keys", "slots", "positions", "owner", "lens", "table", "free")


def same(op, ref, step):
    torch.cuda.synchronize()
    for name in NAMES:
        if name == "free" and not ref.managed:
            continue
        assert getattr(op, name).tolist() == getattr(ref, name), (step, name)
    if ref.managed:
        assert int(op.count) == ref.count, step


@pytest.mark.parametrize("B,rows,pages,P,width", [
    (1, 1, 1, 8, 1), (1, 7, 5, 8, 3), (3, 16, 20, 16, 4), (5, 64, 30, 8, 9), (70, 200, 100, 16, 12), (64, 64, 40, 32, 3),
    (300, 500, 700, 8, 6), (1025, 1500, 900, 8, 3), (4096, 5000, 3000, 64, 2), (9, 20000, 3000, 8, 1000), (4, 17000, 600, 32, 140),
])
def test_random_steps(device, B, rows, pages, P, width):
    """Random cuts and rows, more of both than fit now and then, negative ones among them."""
    rng = random.Random(B * 31 + pages)
    op, ref = K.PageTables(B, rows, pages, P, width, device), P64.Tables(B, rows, pages, P, width)
    for step in range(8):
        mean = max(1, 2 * rows // B)
        new = [rng.choice([0, 1, 1, rng.randint(-2, mean), rng.randint(0, 2 * mean) if rng.random() < 0.2 else 1]) for _ in range(B)]
        keep = None if step % 3 == 0 else [rng.choice([n, n, 0, -5, rng.randint(0, n + 1), 1 << 30]) for n in ref.lens]
        labels = None if step % 2 else [rng.randint(-3, 9) for _ in range(B)]
        say("step", step, B, rows)
        op.step(i32(device, new), keep=None if keep is None else i32(device, keep), labels=None if labels is None else i32(device, labels))
        ref.step(new, keep, labels)
        same(op, ref, step)


def test_rows_that_do_not_fit(device):
    op, ref = K.PageTables(4, 10, 3, 8, 2, device), P64.Tables(4, 10, 3, 8, 2)
    for new in ([4, 4, 4, 0], [4, 2, 3, 1], [17, 2, 0, 9], [0, 0, 0, 0], [1, 1, 1, 1]):
        op.step(i32(device, new))
        ref.step(new)
        same(op, ref, new)
    new, keep = [2000000000] * 4, [0] * 4  # sums beyond 31 bits
    op.step(i32(device, new), keep=i32(device, keep))
    ref.step(new, keep)
    same(op, ref, new)


def test_pages_come_back_in_order(device):
    """A request that restarts gets its own pages again; one that ends feeds the next in the same step."""
    op = K.PageTables(3, 64, 8, 8, 8, device)
    op.step(i32(device, [17, 9, 8]))
    assert op.table[0, :3].tolist() == [0, 1, 2] and op.table[1, :2].tolist() == [3, 4] and op.table[2, 0].item() == 5
    op.step(i32(device, [17, 0, 30]), keep=i32(device, [0, 0, 8]))
    assert op.table[0, :3].tolist() == [0, 1, 2] and op.table[2, :5].tolist() == [5, 3, 4, 6, 7] and op.count.item() == 0
    assert op.lens.tolist() == [17, 0, 38] and op.keys.tolist() == [17, 0, 38]


def test_tables_of_the_caller(device):
    op = K.PageTables(3, 12, 6, 8, 4, device, managed=False)
    ref = P64.Tables(3, 12, 6, 8, 4, managed=False)
    ref.table = [[5, 0, -1, 3], [2, 6, 1, 1], [4, 4, 4, 4]]
    op.table.copy_(i32(device, ref.table))
    for new, keep in (([5, 3, 0], None), ([4, 8, 0], None), ([2, 1, 9], None), ([3, 3, 3], [30, 2, 0]), ([2, 0, 40], [31, 1, 3])):
        op.step(i32(device, new), keep=None if keep is None else i32(device, keep))
        ref.step(new, keep)
        same(op, ref, new)


def test_states_that_no_step_leaves(device):
    """Lengths and counts that a caller wrote: taken into their ranges."""
    op = K.PageTables(2, 8, 4, 8, 2, device)
    op.lens.copy_(i32(device, [-3, 100]))
    op.count.fill_(99)
    op.step(i32(device, [1, 0]))
    torch.cuda.synchronize()
    assert op.lens.tolist() == [1, 16] and op.slots.tolist()[:2] == [0, -1] and int(op.count) == 3


def test_lengths_of_more_pages_than_there_are(device):
    """Pages given back that were never taken, with the count close to 2^31 together: the stack holds what it can."""
    B, width = 4096, 500000
    op = K.PageTables(B, 8, 1 << 27, 8, width, device)
    op.lens.fill_(8 * width)
    op.step(i32(device, [1] + [0] * (B - 1)), keep=torch.zeros(B, dtype=I32, device=device))
    torch.cuda.synchronize()
    assert int(op.count) == (1 << 27) - 1 and op.lens.tolist() == [1] + [0] * (B - 1) and op.slots.tolist() == [0] + [-1] * 7


def test_step_captured_and_on_other_streams(device):
    B, rows = 40, 90
    op, ref = K.PageTables(B, rows, 200, 8, 30, device), P64.Tables(B, rows, 200, 8, 30)
    new, keep = torch.zeros(B, dtype=I32, device=device), torch.zeros(B, dtype=I32, device=device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        op.step(new, keep=keep)
    torch.cuda.synchronize()
    ref.step([0] * B, [0] * B)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.step(new, keep=keep)
    rng = random.Random(5)
    for i in range(6):
        n, k = [rng.randint(0, 3) for _ in range(B)], [rng.randint(0, x) if rng.random() < 0.3 else x for x in ref.lens]
        new.copy_(i32(device, n))
        keep.copy_(i32(device, k))
        if i % 3 == 2:
            op.step(new, keep=keep)
        else:
            g.replay()
        ref.step(n, k)
        same(op, ref, i)


# -------------------------------------------------------------------- rope
def pool(g, dev, pages, P, kv, D, layout, fill=None, shift=0.0):
    """A pool and its copy on the CPU; layouts of the same [pages, P, kv, D] view."""
    cpu = torch.full((pages, P, kv, D), fill, dtype=BF) if fill is not None else rnd(g, pages, P, kv, D, shift=shift)
    if layout == "heads":  # [pages, kv, P, D]
        return cpu.transpose(1, 2).contiguous().to(dev).transpose(1, 2), cpu
    if layout == "wide":  # every other row of a wider tensor, heads farther apart
        big = torch.zeros((pages, 2 * P, kv, D + 24), dtype=BF, device=dev)
        view = big[:, ::2, :, 8:8 + D]
        view.copy_(cpu.to(dev))
        return view, cpu
    return cpu.to(dev), cpu


@pytest.mark.parametrize("M,heads,kv,D,P,layout,norm", [
    (1, 32, 8, 128, 16, "slots", True), (33, 8, 2, 128, 8, "heads", True), (70, 16, 16, 64, 64, "wide", True), (5, 24, 8, 64, 32, "slots", False),
    (9, 7, 1, 128, 16, "heads", False), (300, 4, 1, 128, 128, "slots", True),
])
def test_paged_rope(device, M, heads, kv, D, P, layout, norm):
    g = gen(M)
    pages, n = M // P + 9, 900
    qkv = rnd(g, M, (heads + 2 * kv) * D)
    qn, kn = (rnd(g, D, scale=0.1, shift=1.0) for _ in "qk")
    (kd, k), (vd, v) = (pool(g, device, pages, P, kv, D, layout, fill=7.0) for _ in "kv")
    slots = torch.randperm(pages * P, generator=g)[:M].to(I32)
    pos = torch.randint(0, n, (M,), generator=g).to(I32)
    off = {2: (0, -1), 3: (-1, None), 4: (pages * P, None)}  # no position; no slot; a slot behind the pool
    for r, (s, p) in off.items():
        if r < M:
            if s:
                slots[r] = s
            if p is not None:
                pos[r] = p
    if M > 6:
        pos[6] = n
    say("paged rope", M, heads, kv, D, P, layout)
    table = K.rope_table(n, D, 1e6, device)
    q = torch.full((M, heads * D), 5.0, dtype=BF, device=device)
    gains = (qn.to(device), kn.to(device)) if norm else (None, None)
    K.paged_qk_norm_rope(qkv.to(device), *gains, 1e-6, table, slots.to(device), pos.to(device), kd, vd, q_out=q)
    (rq, sq), (rk, sk), rv = A64.rope(qkv, qn if norm else None, kn if norm else None, 1e-6, 1e6, pos.clamp(0, n - 1), heads, kv, D)
    live = (slots >= 0) & (slots < pages * P) & (pos >= 0) & (pos < n)
    # fp32 throughout (24 roundings and the table's) and one rounding to bf16.
    for got, want, size, was in ((q.cpu().view(M, heads, D), rq, sq, 5.0), (kd.cpu().reshape(-1, kv, D), rk, sk, 7.0)):
        if got.shape[0] != M or was == 7.0:
            full, tol = torch.full(got.shape, 7.0, dtype=torch.float64), torch.zeros(got.shape, dtype=torch.float64)
            full[slots[live].long()] = want[live]
            tol[slots[live].long()] = (A64.BF16_HALF * want.abs() + 40 * A64.FP32_HALF * size)[live]
        else:
            full = torch.where(live[:, None, None], want, torch.full_like(want, was))
            tol = torch.where(live[:, None, None], A64.BF16_HALF * want.abs() + 40 * A64.FP32_HALF * size, torch.zeros_like(want))
        close(got, full, tol, "rope")
    full = torch.full((pages * P, kv, D), 7.0, dtype=torch.float64)
    full[slots[live].long()] = rv[live]
    assert torch.equal(vd.cpu().reshape(-1, kv, D).double(), full)
    # In place, and bit for bit what the contiguous cache's operator gives for one sequence.
    inp = qkv.to(device)
    K.paged_qk_norm_rope(inp, *gains, 1e-6, table, slots.to(device), pos.to(device), kd, vd, q_out=inp[:, :heads * D])
    assert torch.equal(inp[:, :heads * D][live.to(device)], q[live.to(device)])
    k1, v1 = (torch.zeros((1, M, kv, D), dtype=BF, device=device) for _ in "kv")
    q1 = K.qk_norm_rope(qkv.to(device), *gains, 1e-6, table, i32(device, [M]), k1, v1, positions=pos.clamp(0, n - 1).to(device))
    assert torch.equal(q1[live.to(device)], q[live.to(device)])
    assert torch.equal(k1[0][live.to(device)], kd.reshape(-1, kv, D)[slots[live].long().to(device)])


# --------------------------------------------------------------- attention
def check_step(dev, seed, new, keys, heads, kv, D, P, window=0, sinks=0, layout="slots", pad=3, scale=None, spread=1.0, width=None,
               bad=False, odd=False):
    """Requests of `new` rows and `keys` keys in shuffled pages; slots that no row sees hold NaN and infinities."""
    g = gen(seed)
    B = len(new)
    width = width or max(1, max(-(-max(n, 0) // P) for n in keys)) + 1
    need = [min(width, -(-max(n, 0) // P)) for n in keys]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g)
    table, at = torch.full((B, width), 1 << 30 if bad else 0, dtype=torch.int64), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    rows = sum(new) + pad
    starts = [sum(new[:b]) for b in range(B + 1)]
    (kd, k), (vd, v) = pool(g, dev, pages, P, kv, D, layout), pool(g, dev, pages, P, kv, D, layout, shift=0.05)
    used = torch.zeros((pages, P), dtype=torch.bool)
    for b, n in enumerate(keys):
        for t in range(max(0, min(n, width * P))):
            first = min(n, width * P) - new[b]
            if new[b] and (window == 0 or t > first - window or t < sinks):
                used[table[b, t // P], t % P] = True
            elif bad and new[b] == 0:
                table[b, t // P] = -7
    for cpu, gpu in ((k, kd), (v, vd)):
        cpu[~used] = math.nan
        if cpu is v:
            cpu[~used] = torch.where(torch.arange(D) % 2 == 0, math.inf, -math.inf).to(BF)
        if odd and cpu is v:  # seen by some rows of a tile and not by others
            for b, n in enumerate(keys):
                if new[b] > 2:
                    t = n - new[b] // 2
                    cpu[table[b, t // P], t % P, 0, 3] = math.inf
                    cpu[table[b, (t + 1) // P if t + 1 < n else t // P], (t + 1) % P if t + 1 < n else t % P, kv - 1, 5] = math.nan
        gpu.copy_(cpu.to(dev))
    qkv = rnd(g, rows, (heads + 2 * kv) * D, scale=spread)
    say("paged attention", seed, new, keys, heads, kv, D, P, window, sinks, layout)
    op = K.PagedAttention(B, rows, heads, kv, D, P, width, dev, window=window, sinks=sinks, scale=scale)
    out = torch.full((rows, heads * D), 3.0, dtype=BF, device=dev)
    lse = torch.full((rows, heads), 3.0, device=dev)
    args = (qkv.to(dev)[:, :heads * D], kd, vd, table.to(I32).to(dev), i32(dev, starts), i32(dev, keys))
    op.run(*args, out, lse=lse)
    torch.cuda.synchronize()
    ref, rlse, tol, ltol = P64.attention(qkv[:, :heads * D], k, v, table.tolist(), starts, keys, heads=heads, window=window, sinks=sinks,
                                         scale=scale)
    n = starts[-1]
    close(out[:n].view(n, heads, D), ref[:n], tol[:n], "out")
    close(lse[:n], rlse[:n], ltol[:n], "lse")
    assert torch.all(out[n:] == 3.0) and torch.all(lse[n:] == 3.0), "rows of no request were written"
    again = op(*args)
    assert torch.equal(again[:n].view(torch.int16), out[:n].view(torch.int16)) and not again[n:].any(), "another result, or rows of no request"
    return op, args, out


STEPS = [
    # new rows, keys, heads, kv, D, P
    ([1], [1], 32, 8, 128, 16),
    ([1], [2], 4, 1, 128, 8),
    ([1, 1, 1], [300, 33, 64], 32, 8, 128, 16),
    ([1, 0, 1, 0], [40, 77, 513, 0], 8, 2, 128, 32),
    ([0, 0], [5, 9], 8, 2, 64, 8),
    ([1] * 70, [(37 * i) % 211 + 1 for i in range(70)], 8, 2, 128, 8),
    ([2, 1, 5, 1], [2, 90, 5, 31], 16, 16, 64, 64),
    ([7, 16, 3], [700, 1987, 4], 12, 4, 64, 16),
    ([1, 1], [333, 129], 24, 1, 128, 16),
    ([1, 3], [4100, 2500], 40, 8, 128, 128),
    ([16, 16], [500, 16], 32, 8, 128, 64),
    ([17, 33, 1], [17, 300, 1000], 8, 4, 128, 256),
    ([65, 1, 130], [65, 900, 400], 8, 8, 64, 16),
    ([200, 1, 1, 40], [200, 64, 65, 999], 32, 8, 128, 16),
    ([33], [2048], 32, 8, 128, 32),
    ([300, 7], [1200, 3000], 8, 2, 64, 8),
    ([1, 600], [50, 601], 4, 1, 128, 16),
]


@pytest.mark.parametrize("case", range(len(STEPS)))
@pytest.mark.parametrize("layout", ["slots", "heads", "wide"])
def test_steps(device, case, layout):
    check_step(device, 500 + case, *STEPS[case], layout=layout)


#: More requests than a wave has lanes: planned by a launch in front.
CROWDS = [
    ([1] * 65, [(53 * i) % 97 + 1 for i in range(65)], 8, 2, 128, 16),
    ([(0, 1, 1, 7, 1)[i % 5] for i in range(300)], [(37 * i) % 150 + 7 for i in range(300)], 4, 1, 128, 8),
    ([130 if i == 40 else 40 if i == 41 else i % 2 for i in range(120)], [900 if i in (40, 99) else (29 * i) % 300 + 41 for i in range(120)],
     8, 2, 64, 32),
    ([1] * 1030, [i % 40 + 1 for i in range(1030)], 2, 2, 64, 8),
    ([300 if i == 3 else 1 for i in range(70)], [2500 if i == 3 else 1500 if i == 60 else 30 + i for i in range(70)], 32, 8, 128, 16),
    ([0] * 80, [5] * 80, 8, 2, 128, 16),
]


@pytest.mark.parametrize("case", range(len(CROWDS)))
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 2)])
def test_many_requests(device, case, window, sinks):
    check_step(device, 550 + case, *CROWDS[case], window=window, sinks=sinks)


@pytest.mark.parametrize("new,keys,heads,kv,D,P", [
    ([20], [5244], 4, 1, 128, 16), ([32], [9000], 32, 8, 128, 64), ([17, 1], [3300, 40], 8, 2, 64, 16), ([12], [5000], 8, 2, 128, 16),
    ([70, 9], [2900, 4000], 4, 1, 128, 8), ([24] + [1] * 70, [7000] + [9] * 70, 4, 1, 128, 16),
])
def test_many_ranges(device, new, keys, heads, kv, D, P):
    """Few tiles over many keys: ranges that are joined in groups, and the groups then."""
    check_step(device, 760 + sum(new), new, keys, heads, kv, D, P, odd=len(new) == 2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 0), (33, 40), (100, 4), (5000, 9)])
@pytest.mark.parametrize("P", [8, 64])
def test_window_and_sinks(device, window, sinks, P):
    check_step(device, 600 + window + sinks, [1, 5, 0, 90, 1], [400, 211, 50, 333, 3], 8, 2, 128, P, window=window, sinks=sinks, bad=True)


@pytest.mark.parametrize("new,keys", [([5, 3], [3, 0]), ([100, 1], [40, -4]), ([1, 2], [0, 1]), ([20, 300], [19, 299])])
def test_rows_without_a_key(device, new, keys):
    """More rows than keys: the first rows' positions are negative, and they give zeros."""
    _, _, out = check_step(device, 650, new, keys, 8, 2, 128, 16)
    for b, (n, L) in enumerate(zip(new, keys)):
        s = sum(new[:b])
        assert not out[s:s + n - max(L, 0)].any()


def test_keys_beyond_the_table(device):
    check_step(device, 660, [1, 2], [1000, 90], 8, 2, 128, 16, width=6)


@pytest.mark.parametrize("new,keys", [([16, 1], [100, 50]), ([90, 1], [300, 50]), ([4], [4])])
def test_infinities_and_nans_that_some_rows_see(device, new, keys):
    check_step(device, 670, new, keys, 8, 2, 128, 16, odd=True)


@pytest.mark.parametrize("spread,scale", [(1e4, None), (1.0, 1e-3), (1e-3, None), (1.0, 50.0)])
def test_scores_of_any_size(device, spread, scale):
    check_step(device, 680, [1, 3, 80], [200, 77, 300], 8, 2, 64, 16, spread=spread, scale=scale)


def test_page_numbers_outside_the_pool_read_another_page(device):
    """Seen entries that name no page: the results are of another page's keys, in bounds."""
    g = gen(5)
    k, v = rnd(g, 4, 8, 2, 128).to(device), rnd(g, 4, 8, 2, 128).to(device)
    q = rnd(g, 3, 1024)
    table = torch.tensor([[0, -1, 2], [2147483647, 3, -2147483648]], dtype=I32)
    op = K.PagedAttention(2, 3, 8, 2, 128, 8, 3, device)
    out = op(q.to(device), k, v, table.to(device), i32(device, [0, 1, 3]), i32(device, [24, 20]))
    ref, _, tol, _ = P64.attention(q, k.cpu(), v.cpu(), table.tolist(), [0, 1, 3], [24, 20], heads=8)
    close(out.view(3, 8, 128), ref, tol, "out")


@pytest.mark.parametrize("starts", [[0, 5, 2, 9], [-4, 3, 700, 2], [9, 9, 9, 9], [3, 1, 0, -8]])
@pytest.mark.parametrize("more", [0, 80])
def test_starts_that_do_not_ascend(device, starts, more):
    """In bounds, whatever they hold; rows behind the call's are untouched, and the
    workspace serves the next call."""
    g = gen(6)
    k, v = rnd(g, 20, 8, 2, 128).to(device), rnd(g, 20, 8, 2, 128).to(device)
    big = torch.full((30, 1024), 3.0, dtype=BF, device=device)
    table = torch.randint(0, 20, (3 + more, 6), generator=g).to(I32).to(device)
    op = K.PagedAttention(3 + more, 9, 8, 2, 128, 8, 6, device)
    q, keys = rnd(g, 9, 1024).to(device), i32(device, [48, 20, 33] + [30] * more)
    op.run(q, k, v, table, i32(device, starts + [9, 0] * (more // 2)), keys, big[10:19])
    torch.cuda.synchronize()
    assert torch.all(big[:10] == 3.0) and torch.all(big[19:] == 3.0) and big[10:19].isfinite().all()
    good = i32(device, [0, 3, 5, 9] + [9] * more)
    other = K.PagedAttention(3 + more, 9, 8, 2, 128, 8, 6, device)
    assert torch.equal(op(q, k, v, table, good, keys), other(q, k, v, table, good, keys))


def test_pool_offsets_beyond_32_bits(device):
    """Pages whose elements lie behind 2^32 (a pool of 9 GB, views of one k and v)."""
    P, kv, D = 16, 8, 128
    pages = 140000
    kv_pool = torch.zeros((pages, 2, P, kv, D), dtype=BF, device=device)
    k, v = kv_pool[:, 0], kv_pool[:, 1]
    g = gen(9)
    table = torch.tensor([[139999, 5, 131072, 139998], [131073, 7, 139997, 0]], dtype=I32)
    keys, new, heads = [60, 33], [1, 20], 32
    for b in range(2):
        for i in range(4):
            for t in (k, v):
                t[int(table[b, i])] = rnd(g, P, kv, D).to(device)
    q = rnd(g, 21, heads * D)
    op = K.PagedAttention(2, 21, heads, kv, D, P, 4, device)
    out = op(q.to(device), k, v, table.to(device), i32(device, [0, 1, 21]), i32(device, keys))
    ids = sorted(set(table.flatten().tolist()))
    small = torch.tensor([[ids.index(int(x)) for x in row] for row in table])
    ref, _, tol, _ = P64.attention(q, k[ids].cpu(), v[ids].cpu(), small.tolist(), [0, 1, 21], keys, heads=heads)
    close(out.view(21, heads, D), ref, tol, "out")
    slots = i32(device, [139999 * P + 3, 5 * P])
    qkv = rnd(g, 2, (heads + 2 * kv) * D).to(device)
    K.paged_qk_norm_rope(qkv, None, None, 1e-6, K.rope_table(4, D, 1e6, device), slots, i32(device, [0, 0]), k, v)
    assert torch.equal(v[139999, 3].flatten(), qkv[0, (heads + kv) * D:]) and torch.equal(v[5, 0].flatten(), qkv[1, (heads + kv) * D:])


def test_attention_captured_with_other_lengths(device):
    """One graph, replayed for steps of other lengths, pages and row counts, eager work between."""
    op, args, _ = check_step(device, 700, [1, 120, 0, 1], [3000, 400, 10, 64], 8, 2, 128, 16, pad=60, width=200)
    q, k, v, table, starts, keys = args
    k.nan_to_num_(0.0, 0.0, 0.0), v.nan_to_num_(0.0, 0.0, 0.0)
    table.random_(0, k.shape[0])
    out = torch.zeros((q.shape[0], 1024), dtype=BF, device=device)
    op.run(q, k, v, table, starts, keys, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.run(q, k, v, table, starts, keys, out)
    other = K.PagedAttention(op.B, op.rows, 8, 2, 128, 16, 200, device)
    for i, (st, ks) in enumerate([([0, 1, 2, 3, 4], [3200, 1, 900, 70]), ([0, 0, 0, 0, 0], [5, 5, 5, 5]), ([0, 150, 151, 151, 180], [150, 2000, 0, 31]),
                                  ([0, 1, 121, 121, 122], [3000, 400, 10, 64]), ([0, 40, 80, 120, 160], [3000, 3001, 3002, 3003])]):
        starts.copy_(i32(device, st))
        keys.copy_(i32(device, ks))
        table.random_(0, k.shape[0])
        out.fill_(2.0)
        g.replay()
        eager = torch.full_like(out, 2.0)
        other.run(q, k, v, table, starts, keys, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        ref, _, tol, _ = P64.attention(q.cpu(), k.cpu(), v.cpu(), table.tolist(), st, ks, heads=8)
        n = st[-1]
        close(out[:n].view(n, 8, 128), ref[:n], tol[:n], f"replay {i}")


def test_objects_on_two_streams_and_a_shared_workspace(device):
    op, args, out = check_step(device, 710, [1, 30, 1], [2000, 500, 64], 8, 2, 128, 16)
    n = 32
    need = K.paged_workspace_bytes(3, op.rows, 8, 2, 128, 16, op.width)
    ws = torch.zeros(max(need, 16) + 64, dtype=torch.uint8, device=device)
    shared = K.PagedAttention(3, op.rows, 8, 2, 128, 16, op.width, device, workspace=ws)
    assert torch.equal(shared(*args)[:n], out[:n])
    other = K.PagedAttention(3, op.rows, 8, 2, 128, 16, op.width, device)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    res = []
    for _ in range(4):
        with torch.cuda.stream(a):
            res.append(op(*args))
        with torch.cuda.stream(b):
            res.append(other(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(r[:n], out[:n]) for r in res)
    if need:
        with pytest.raises(ValueError, match="workspace"):
            K.PagedAttention(3, op.rows, 8, 2, 128, 16, op.width, device, workspace=ws[:need - 1])


def test_shapes_that_share_a_workspace(device):
    """Of other sizes, head sizes and planning, one after the other in one workspace."""
    made = [check_step(device, 720 + i, *c) for i, c in enumerate([
        ([1, 1], [3000, 900], 8, 2, 128, 16), ([200, 1, 1], [3000, 2000, 64], 8, 2, 64, 8), ([1] * 70, [700] * 70, 4, 1, 128, 16),
        ([30], [5000], 8, 8, 128, 64)])]
    need = max(K.paged_workspace_bytes(o.B, o.rows, o.heads, o.kv_heads, o.head_dim, o.page_size, o.width) for o, _, _ in made)
    ws = torch.zeros(need, dtype=torch.uint8, device=device)
    shared = [K.PagedAttention(o.B, o.rows, o.heads, o.kv_heads, o.head_dim, o.page_size, o.width, device, workspace=ws) for o, _, _ in made]
    for i in (0, 1, 2, 3, 2, 0, 3, 1, 0, 2):
        _, args, out = made[i]
        n = int(args[4][-1])
        assert torch.equal(shared[i](*args)[:n], out[:n]), i


@pytest.mark.parametrize("B,P,width", [(70, 8, 16), (300, 64, 2), (70, 16, 1)])
def test_a_workspace_shared_with_requests_of_one_range(device, B, P, width):
    """Many requests of a few keys, which are listed in the workspace and never cut, leave the counters at its front zero."""
    cut, args, out = check_step(device, 730, [1, 1], [3000, 900], 8, 2, 128, 16)
    short, sargs, sout = check_step(device, 731, [1] * B, [width * P] * B, 8, 2, 128, P, width=width)
    need = [K.paged_workspace_bytes(o.B, o.rows, o.heads, o.kv_heads, o.head_dim, o.page_size, o.width) for o in (cut, short)]
    ws = torch.zeros(max(need), dtype=torch.uint8, device=device)
    shared = [K.PagedAttention(o.B, o.rows, o.heads, o.kv_heads, o.head_dim, o.page_size, o.width, device, workspace=ws) for o in (cut, short)]
    for i in range(3):
        assert torch.equal(shared[1](*sargs)[:B], sout[:B]), i
        assert int(ws[:256].sum()) == 0
        assert torch.equal(shared[0](*args)[:2], out[:2]), i


def test_python_refusals(device):
    op = K.PagedAttention(2, 4, 8, 2, 128, 16, 3, device)
    q = torch.zeros((4, 1024), dtype=BF, device=device)
    k = torch.zeros((5, 16, 2, 128), dtype=BF, device=device)
    table, starts, keys = torch.zeros((2, 3), dtype=I32, device=device), i32(device, [0, 1, 2]), i32(device, [3, 4])
    good = dict(q=q, k=k, v=k.clone(), table=table, starts=starts, keys=keys)
    op(**good)
    for name, bad in (("q", q[:3]), ("q", q.float()), ("k", k[:, :8]), ("k", k[..., ::2]), ("v", k[:4]), ("table", table.long()),
                      ("table", table[:, :2]), ("starts", starts[:2]), ("keys", keys.cpu()), ("keys", keys.float()), ("k", k[0])):
        with pytest.raises(ValueError, match=name):
            op(**{**good, name: bad})
    t = K.PageTables(2, 4, 5, 16, 3, device)
    for kw in (dict(new=keys.long()), dict(new=keys[:1]), dict(new=keys, keep=keys.cpu()), dict(new=keys, labels=starts)):
        with pytest.raises(ValueError):
            t.step(**kw)
    model = synthetic_model(device, layers=1, hidden=64, intermediate=64, heads=8, kv_heads=2, vocab=64)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q.zero_()
        for build in (lambda: K.PageTables(2, 4, 5, 16, 3, device), lambda: K.PagedAttention(2, 4, 8, 2, 128, 16, 3, device),
                      lambda: K.PagedAttention(2, 4, 8, 2, 128, 16, 3, device, workspace=op.workspace),
                      lambda: K.LowRankAdapters(4, 64, 128, 8, device), lambda: K.PagedCache(model, 2, 4, 8, 16),
                      lambda: K.AdapterSet(model, 2, 8)):
            with pytest.raises(RuntimeError, match="before the capture"):
                build()
