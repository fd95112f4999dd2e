"""The paged KV cache (write, read, attention over pages) and the attention over packed
prompts against a 64-bit evaluation (paged_ref.py)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16, Q8 = torch.float32, torch.float16, torch.bfloat16, torch.int8


def rows_of(gen, n, heads, d, dtype):
    x = torch.randn((n, heads, d), generator=gen)
    x[..., 5::29] *= 4.0
    return x.to(dtype)


def pool_of(gen, b, g, d, kv, layout="rows"):
    """Pages with something in every row: (k, v, k_scale, v_scale), page views on the GPU."""
    out = []
    for _ in range(2):
        x = rows_of(gen, b.n_pages * b.page, g, d, F32 if kv == Q8 else kv).view(b.n_pages, b.page, g, d)
        out.append(ref.quantise(x) if kv == Q8 else (x, None))
    pages = [p.cuda() for p, _ in out]
    if layout == "heads":
        pages = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pages]
    return pages + [s.cuda() if s is not None else None for _, s in out]


def stored(b, pages, scale, s):
    """The cached rows of sequence s, float64 on the CPU."""
    pg, ro = (torch.from_numpy(x) for x in b.places(s))
    r = pages.cpu()[pg, ro].double()
    return r * scale.cpu()[pg, ro].double().unsqueeze(-1) if scale is not None else r


def check(got, want, tol, what=""):
    got = got.double().cpu()
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(off / tol).max():.3g} of the bound"


def check_attention(b, out, q, pool, window, scale, dtype, untouched, absent=None):
    for s in range(len(b.rows)):
        n, lo = b.rows[s], int(b.start[s])
        if n == 0:
            continue
        k, v = (stored(b, pool[i], pool[2 + i], s) for i in (0, 1))
        want, bound = ref.attention(q[lo:lo + n].double(), k, v, b.lens[s] - n, window, scale,
                                    absent[s] if absent is not None else None)
        check(out[lo:lo + n], want, bound(dtype), f"sequence {s}: {n} rows, {b.lens[s]} keys")
    for r in list(range(b.start[0])) + list(range(b.start[-1], b.n_rows)):
        assert torch.equal(out[r].cpu(), untouched[r].cpu()), f"padding row {r} written"


def run_attention(pkg, b, h, g, d, dtype, kv, window=0, layout="rows", seed=1, change=None, absent=None, scale=None):
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(seed)
    pool = pool_of(gen, b, g, d, kv, layout)
    q = torch.randn((b.n_rows, h, d), generator=gen).to(dtype)
    if change:
        change(pool)
    out = torch.full((b.n_rows, h, d), 7.0, dtype=dtype).cuda()
    before = out.clone()
    ops.PagedAttentionCall(ops.PagedCache(*pool), b.device(ops), q.cuda(), out, window=window, score_scale=scale)()
    torch.cuda.synchronize()
    check_attention(b, out, q, pool, window, scale or 1 / math.sqrt(d), dtype, before, absent)
    return out


HEADS = [(16, 8, 128), (14, 2, 64), (8, 4, 256), (32, 4, 128), (3, 3, 64), (40, 1, 128)]


@pytest.mark.parametrize("h,g,d", HEADS)
@pytest.mark.parametrize("dtype,kv", [(F16, F16), (BF16, BF16), (F16, Q8), (BF16, Q8)])
def test_tokens_over_pages(pkg, h, g, d, dtype, kv):
    """One row per sequence; lengths of one, of a page, past it, and long ones."""
    b = ref.Batch([1] * 8, [1, 16, 17, 15, 333, 64, 700, 129], 16, 3)
    run_attention(pkg, b, h, g, d, dtype, kv)


@pytest.mark.parametrize("h,g,d", HEADS)
@pytest.mark.parametrize("dtype,kv", [(F16, F16), (BF16, BF16), (F16, Q8), (BF16, Q8)])
def test_mixed_rows_over_pages(pkg, h, g, d, dtype, kv):
    """Chunks, single tokens, whole prompts, a sequence without rows, one without keys, one
    with more rows than keys, padding in front and behind."""
    b = ref.Batch([7, 1, 0, 130, 33, 2, 5, 64], [300, 1, 90, 130, 95, 0, 3, 513], 32, 4, lead=3, tail=5)
    run_attention(pkg, b, h, g, d, dtype, kv)


@pytest.mark.parametrize("h,g,d", [(8, 4, 256), (14, 2, 64), (16, 8, 128)])
@pytest.mark.parametrize("window", [1, 5, 64, 100])
@pytest.mark.parametrize("dtype,kv", [(F16, F16), (BF16, BF16), (F16, Q8)])
def test_window_over_pages(pkg, h, g, d, window, dtype, kv):
    b = ref.Batch([1, 70, 200, 9], [301, 400, 200, 77], 64, 5)
    run_attention(pkg, b, h, g, d, dtype, kv, window=window)


@pytest.mark.parametrize("rows,lens", [([1], [5003]), ([1], [70001]), ([1, 1, 1], [4100, 31, 2500]), ([5] * 3, [3001, 6, 1700]),
                                       ([61], [2900]), ([300], [1903]), ([1] * 70, list(range(1, 71)))])
@pytest.mark.parametrize("dtype,kv,h,g,d", [(F16, F16, 32, 8, 128), (BF16, BF16, 8, 4, 256), (F16, Q8, 32, 8, 128),
                                            (BF16, Q8, 14, 2, 64), (F16, Q8, 8, 4, 256)])
def test_long_keys_over_pages(pkg, rows, lens, dtype, kv, h, g, d):
    """Few rows over long caches: work divided along the keys and joined."""
    run_attention(pkg, ref.Batch(rows, lens, 16, 6), h, g, d, dtype, kv)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("layout", ["rows", "heads"])
def test_pages_and_layouts(pkg, page, layout):
    b = ref.Batch([1, 40, 77], [500, 40, 300], page, 7)
    for kv in (F16, Q8):
        run_attention(pkg, b, 16, 8, 128, F16, kv, layout=layout)


@pytest.mark.parametrize("scale", [1.0, 0.01])
def test_score_scale(pkg, scale):
    b = ref.Batch([1, 40], [500, 300], 16, 8)
    for kv in (F16, Q8):
        run_attention(pkg, b, 16, 8, 128, F16, kv, scale=scale)


@pytest.mark.parametrize("kv", [F16, BF16, Q8])
def test_pages_that_are_not_there(pkg, kv):
    """Page ids outside the pool: their keys do not exist; a sequence of none gets zeros."""
    b = ref.Batch([1, 40, 3, 200], [500, 300, 20, 200], 16, 9)
    for s, at, bad in ((0, 3, -1), (0, 31, b.n_pages), (1, 0, 2 ** 31 - 1), (1, 18, -5), (2, 0, -1), (2, 1, -1), (3, 5, -1)):
        b.table[s, at] = bad
    absent = [torch.zeros(n, dtype=torch.bool) for n in b.lens]
    for s in range(4):
        pos = np.arange(b.lens[s])
        ids = b.table[s][pos // 16]
        absent[s] = torch.from_numpy((ids < 0) | (ids >= b.n_pages))
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(2)
    pool = pool_of(gen, b, 8, 128, kv)
    dtype = F16 if kv == Q8 else kv
    q = torch.randn((b.n_rows, 16, 128), generator=gen).to(dtype)
    out = torch.full((b.n_rows, 16, 128), 7.0, dtype=dtype).cuda()
    before = out.clone()
    ops.PagedAttentionCall(ops.PagedCache(*pool), b.device(ops), q.cuda(), out)()
    torch.cuda.synchronize()
    b.table = np.where((b.table < 0) | (b.table >= b.n_pages), 0, b.table)
    check_attention(b, out, q, pool, 0, 1 / math.sqrt(128), dtype, before, absent)
    assert not out[int(b.start[2]):int(b.start[3])].any(), "a sequence without pages gets zeros"


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("rows,window", [([1, 1, 1], 0), ([90, 200, 5], 0), ([90, 200, 5], 40)])
def test_hidden_rows_may_hold_anything(pkg, kv, rows, window):
    """inf and NaN in rows no sequence owns, in the rest of a last page, and in rows that a
    row does not see (its own future, keys out of its window)."""
    b = ref.Batch(rows, [100, 250, 37], 32, 10)
    marks = {}

    def change(pool):
        for i in (0, 1):
            own = torch.zeros(b.n_pages, b.page, dtype=torch.bool)
            for s in range(3):
                own[tuple(torch.from_numpy(x) for x in b.places(s))] = True
            hole = (~own).nonzero(as_tuple=True)
            x = pool[i].cpu()
            x[hole] = torch.tensor([math.inf, math.nan, -math.inf]).repeat(hole[0].numel())[:hole[0].numel()].view(-1, 1, 1).to(x.dtype)
            # one visible-to-some key of sequence 1: NaN in K and V from position 203 on
            if rows[1] > 1 and i == 1:
                pg, ro = b.places(1)
                x[int(pg[203]), int(ro[203])] = math.nan
                x[int(pg[230]), int(ro[230])] = math.inf
                marks["bad"] = 203
            pool[i].copy_(x)

    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(3)
    pool = pool_of(gen, b, 8, 128, kv)
    change(pool)
    q = torch.randn((b.n_rows, 16, 128), generator=gen).to(kv)
    out = torch.zeros((b.n_rows, 16, 128), dtype=kv).cuda()
    ops.PagedAttentionCall(ops.PagedCache(*pool), b.device(ops), q.cuda(), out, window=window)()
    torch.cuda.synchronize()
    out = out.cpu()
    for s in range(3):
        n, lo = b.rows[s], int(b.start[s])
        k, v = (stored(b, pool[i], None, s) for i in (0, 1))
        p0 = b.lens[s] - n
        bad = torch.zeros(n, dtype=torch.bool)
        if "bad" in marks and s == 1:
            pos = torch.arange(p0, p0 + n)
            for at in (203, 230):
                bad |= (pos >= at) & ((pos < at + window) if window else True)
            assert not out[lo:lo + n][bad].isfinite().all(-1).all(-1).any(), "rows that see a NaN show it"
            v = v.clone()
            v[[203, 230]] = 0.0
        want, bound = ref.attention(q[lo:lo + n].double(), k, v, p0, window, 1 / math.sqrt(128))
        check(out[lo:lo + n][~bad], want[~bad], bound(kv)[~bad], f"sequence {s}")


def test_future_infinity_reaches_the_rows_that_see_it(pkg):
    """An infinite V element: rows in front of it are finite, rows that see it get that infinity
    in that element and their ordinary values in the others."""
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(4)
    for dtype in (F16, BF16):
        q, k, v = (torch.randn((150, x, 64), generator=gen).to(dtype) for x in (4, 2, 2))
        v[77, 1, 9] = math.inf
        v[90, 0, 3] = -math.inf
        out = ops.packed_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, 150], dtype=torch.int32).cuda(),
                                   max_rows=150).cpu()
        clean = v.clone()
        clean[77, 1, 9] = 0
        clean[90, 0, 3] = 0
        want, bound = ref.attention(q.double(), k.double(), clean.double(), 0, 0, 1 / 8)
        tol = bound(dtype)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[77:, 2:, 9] = True
        hit[90:, :2, 3] = True
        assert torch.all(out[77:, 2:, 9] == math.inf) and torch.all(out[90:, :2, 3] == -math.inf)
        check(out[~hit], want[~hit], tol[~hit])


@pytest.mark.parametrize("h,g,d", HEADS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[1], [2, 1, 1, 3], [129, 31, 0, 64, 1, 255], [700], [16] * 70, [1] * 130])
def test_packed_prompts(pkg, h, g, d, dtype, lens):
    run_packed(pkg, lens, h, g, d, dtype)


def run_packed(pkg, lens, h, g, d, dtype, window=0, lead=2, tail=3, seed=5):
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(seed)
    start = np.concatenate([[lead], lead + np.cumsum(lens)]).astype(np.int32)
    n = int(start[-1]) + tail
    # slices of one projection's output: strides larger than the rows
    qkv = torch.randn((n, h + 2 * g, d), generator=gen).to(dtype).cuda()
    q, k, v = qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]
    out = torch.full((n, h, d), 7.0, dtype=dtype).cuda()
    ops.PackedAttentionCall(q, k, v, torch.from_numpy(start).cuda(), out, max_rows=max(lens), window=window)()
    torch.cuda.synchronize()
    q, k, v, out = (x.cpu() for x in (q, k, v, out))
    for s, m in enumerate(lens):
        at = slice(int(start[s]), int(start[s]) + m)
        if m:
            want, bound = ref.attention(q[at].double(), k[at].double(), v[at].double(), 0, window, 1 / math.sqrt(d))
            check(out[at], want, bound(dtype), f"prompt {s} of {m}")
    assert (out[:lead] == 7).all() and (out[n - tail:] == 7).all(), "padding rows written"
    return out


@pytest.mark.parametrize("window", [1, 33, 128, 1024])
@pytest.mark.parametrize("h,g,d", [(8, 4, 256), (14, 2, 64), (16, 8, 128)])
def test_packed_window(pkg, h, g, d, window):
    run_packed(pkg, [300, 65, 513], h, g, d, BF16, window=window)
    run_packed(pkg, [300, 65, 513], h, g, d, F16, window=window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("h,g,d", [(32, 8, 128), (8, 4, 256), (14, 2, 64)])
def test_packed_many_rows(pkg, h, g, d, dtype):
    """Enough rows for the kernels of large launches."""
    run_packed(pkg, [1100, 37, 800, 2049, 1, 500], h, g, d, dtype)


@pytest.mark.parametrize("rows_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kv", [F16, BF16, Q8])
@pytest.mark.parametrize("g,d", [(8, 128), (2, 64), (1, 64), (4, 256), (3, 128)])
def test_write_and_read(pkg, rows_dtype, kv, g, d):
    """Every row lands in its place, rounded or quantised exactly; nothing else changes; read
    gives it back; rows without a place are dropped and read as zeros."""
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(6)
    b = ref.Batch([1, 5, 0, 40, 3, 17, 2], [1, 21, 9, 40, 100, 17, 1], 16, 11, lead=2, tail=4)
    b.table[4, 6] = -1          # the last page of sequence 4: positions 96 ..
    pool = pool_of(gen, b, g, d, kv)
    want = [p.cpu().clone() if p is not None else None for p in pool]
    k, v = (rows_of(gen, b.n_rows, g, d, rows_dtype) for _ in "kv")
    k[4, 0] = 0.0               # an all-zero head row
    v[5, g - 1] *= 1e-4
    if rows_dtype != F16:       # head rows whose scale would be denormal, and the smallest that is kept
        k[6] = 2.0 ** -126
        k[7] = 2.0 ** -100
    back = [torch.full_like(k, 9.0).cuda() for _ in "kv"]
    expect = [x.cpu().clone() for x in back]
    for i, x in enumerate((k, v)):
        for s in range(len(b.rows)):
            for j in range(b.rows[s]):
                r, pos = int(b.start[s]) + j, b.lens[s] - b.rows[s] + j
                pg = int(b.table[s, pos // 16]) if pos >= 0 else -1
                if pg < 0:
                    expect[i][r] = 0.0
                    continue
                if kv == Q8:
                    want[i][pg, pos % 16], want[2 + i][pg, pos % 16] = ref.quantise(x[r])
                    expect[i][r] = (want[i][pg, pos % 16].float() * want[2 + i][pg, pos % 16].unsqueeze(-1)).to(rows_dtype)
                else:
                    want[i][pg, pos % 16] = x[r].to(kv)
                    expect[i][r] = want[i][pg, pos % 16].to(rows_dtype)
    cache, batch = ops.PagedCache(*pool), b.device(ops)
    ops.PagedWriteCall(cache, batch, k.cuda(), v.cuda())()
    ops.PagedReadCall(cache, batch, *back)()
    torch.cuda.synchronize()
    for got, w in zip(pool, want):
        if w is not None:
            assert torch.equal(got.cpu(), w)
    for got, w in zip(back, expect):
        assert torch.equal(got.cpu(), w)


def test_write_of_many_sequences_and_strides(pkg):
    """More sequences than one level of the row search takes, empty ones among them; rows from
    a projection's slices, pages [head][row][dim]."""
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(7)
    rng = np.random.default_rng(3)
    rows = [int(x) for x in rng.integers(0, 3, 5000)]
    lens = [n + int(x) for n, x in zip(rows, rng.integers(0, 20, 5000))]
    b = ref.Batch(rows, lens, 16, 12)
    for kv in (F16, Q8):
        pool = pool_of(gen, b, 2, 64, kv, "heads")
        kvrows = rows_of(gen, b.n_rows, 8, 64, BF16).cuda()
        k, v = kvrows[:, 2:4], kvrows[:, 6:8]
        cache, batch = ops.PagedCache(*pool), b.device(ops)
        back = [torch.empty((b.n_rows, 2, 64), dtype=F32).cuda() for _ in "kv"]
        ops.PagedWriteCall(cache, batch, k, v)()
        ops.PagedReadCall(cache, batch, *back)()
        torch.cuda.synchronize()
        for x, y in zip((k, v), back):
            if kv == Q8:
                c, s = ref.quantise(x)
                assert torch.equal(y.cpu(), c.float() * s.unsqueeze(-1))
            else:
                assert torch.equal(y.cpu(), x.cpu().to(F16).float())


@pytest.mark.parametrize("kv", [F16, Q8])
def test_steps_of_a_served_batch(pkg, kv):
    """As a serving loop uses them: prompts packed (attention over their own rows, rows stored),
    then a chunk and single tokens stored and attended, a sequence that shares another's
    first pages, all against one 64-bit history per sequence."""
    from gguf_runner_amd import ops
    h, g, d, page = 16, 8, 128, 16
    gen = torch.Generator().manual_seed(8)
    prompts = [50, 7, 129]
    history = {s: [[], []] for s in range(3)}
    n_pages = 64
    codes = Q8 if kv == Q8 else F16
    pool = [torch.zeros((n_pages, page, g, d), dtype=codes).cuda() for _ in "kv"]
    if kv == Q8:
        pool += [torch.ones((n_pages, page, g), dtype=F32).cuda() for _ in "kv"]
    cache = ops.PagedCache(*pool)
    table = np.full((3, 12), -1, np.int32)
    table[0], table[1], table[2] = np.arange(12), np.arange(20, 32), np.arange(40, 52)
    lens = [0, 0, 0]

    def step(rows):
        nonlocal lens
        lens = [a + b for a, b in zip(lens, rows)]
        start = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()
        n = sum(rows)
        q, k, v = (torch.randn((n, x, d), generator=gen).to(F16) for x in (h, g, g))
        batch = ops.PagedBatch(start, torch.tensor(lens, dtype=torch.int32).cuda(), torch.from_numpy(table).cuda(),
                               n_rows=n, max_rows=max(rows), max_len=max(lens))
        ops.PagedWriteCall(cache, batch, k.cuda(), v.cuda())()
        out = ops.paged_attention(cache, batch, q.cuda())
        at = 0
        for s, m in enumerate(rows):
            for i, x in enumerate((k, v)):
                r = x[at:at + m]
                if kv == Q8:
                    c, sc = ref.quantise(r)
                    r = c.double() * sc.double().unsqueeze(-1)
                history[s][i].append(r.double())
            if m:
                ks, vs = (torch.cat(history[s][i]) for i in (0, 1))
                want, bound = ref.attention(q[at:at + m].double(), ks, vs, lens[s] - m, 0, 1 / math.sqrt(d))
                check(out[at:at + m], want, bound(F16), f"sequence {s}, {m} rows of {lens[s]}")
            at += m
        return q, k, v, start, out

    q, k, v, start, out = step(prompts)
    packed = ops.packed_attention(q.cuda(), k.cuda(), v.cuda(), start, max_rows=max(prompts)).cpu()
    if kv == F16:  # the same attention, over the rows themselves and over the pages
        at = 0
        for s, m in enumerate(prompts):
            want, bound = ref.attention(*(x[at:at + m].double() for x in (q, k, v)), 0, 0, 1 / math.sqrt(d))
            check(packed[at:at + m], want, bound(F16))
            at += m
    step([1, 1, 1])
    step([1, 30, 0])
    # sequence 1 goes on as a copy of sequence 0's first two pages
    table[1][:2] = table[0][:2]
    lens[1] = 32
    history[1] = [[torch.cat(history[0][i])[:32]] for i in (0, 1)]
    step([2, 5, 40])
    step([1, 1, 1])


def test_replayed_graphs(pkg):
    """Captured once and replayed: lengths, tables and rows are read as they are at replay time;
    two graphs of two prepared calls on two streams at once; eager calls in between."""
    from gguf_runner_amd import ops
    h, g, d = 32, 8, 128
    gen = torch.Generator().manual_seed(9)
    b = ref.Batch([1, 1, 1, 1], [900, 30, 2000, 517], 16, 13)
    pool = pool_of(gen, b, g, d, F16)
    cache, batch = ops.PagedCache(*pool), b.device(ops)
    q = torch.randn((4, h, d), generator=gen).to(F16).cuda()
    outs = [torch.zeros_like(q) for _ in range(3)]
    calls = [ops.PagedAttentionCall(cache, batch, q, o) for o in outs]
    for c in calls:
        c()
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=streams[i]):
            calls[i]()
        graphs.append(gr)
    kv_len = batch._keep[1]
    for turn in range(4):
        lens = [900 - 100 * turn, 30, 2000 - 611 * turn, 517 + turn]
        lens[3] = min(lens[3], 517)
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn((4, h, d), generator=gen).to(F16))
        torch.cuda.synchronize()
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        calls[2]()
        torch.cuda.synchronize()
        b.lens = lens
        check_attention(b, outs[2], q.cpu(), pool, 0, 1 / math.sqrt(d), F16, outs[2])
        for i in range(2):
            assert torch.equal(outs[i], outs[2]), f"graph {i}, turn {turn}"


def test_two_streams_and_repeats(pkg):
    """Calls on two streams at once, each with its own workspace, repeat bit for bit."""
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(10)
    b = ref.Batch([1, 64, 9], [3000, 2000, 700], 32, 14)
    pool = pool_of(gen, b, 8, 128, Q8)
    cache, batch = ops.PagedCache(*pool), b.device(ops)
    q = torch.randn((b.n_rows, 32, 128), generator=gen).to(F16).cuda()
    first = ops.paged_attention(cache, batch, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in streams]
    calls = [ops.PagedAttentionCall(cache, batch, q, o) for o in outs]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(calls, streams):
            c(s)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)


@pytest.mark.parametrize("kv", [F16, Q8])
def test_offsets_past_32_bits(pkg, kv):
    """A pool of more than 2^32 bytes per tensor, its used pages at both ends."""
    from gguf_runner_amd import ops
    h, g, d, page = 8, 8, 128, 256
    n_pages = (2 ** 32 // (page * g * d * (1 if kv == Q8 else 2))) + 40
    gen = torch.Generator().manual_seed(11)
    b = ref.Batch([3, 70], [700, 1000], page, 15)
    used = np.unique(b.table[b.table >= 0])
    where = np.concatenate([np.arange(len(used) // 2), n_pages - 1 - np.arange(len(used) - len(used) // 2)])
    move = {int(u): int(w) for u, w in zip(used, where)}
    pool = [torch.zeros((n_pages, page, g, d), dtype=kv, device="cuda") for _ in "kv"]
    if kv == Q8:
        pool += [torch.ones((n_pages, page, g), dtype=F32, device="cuda") for _ in "kv"]
    for s in range(2):
        b.table[s] = [move.get(int(x), -1) for x in b.table[s]]
    b.n_pages = n_pages
    cache, batch = ops.PagedCache(*pool), b.device(ops)
    # store both histories whole, then attend and read the last rows
    whole = ref.Batch(b.lens, b.lens, page, 1)
    whole.table, whole.n_pages = b.table, n_pages
    k, v = (rows_of(gen, whole.n_rows, g, d, F16) for _ in "kv")
    ops.PagedWriteCall(cache, whole.device(ops), k.cuda(), v.cuda())()
    q = torch.randn((b.n_rows, h, d), generator=gen).to(F16)
    out = ops.paged_attention(cache, batch, q.cuda())
    back = [torch.empty((whole.n_rows, g, d), dtype=F32).cuda() for _ in "kv"]
    ops.PagedReadCall(cache, whole.device(ops), *back)()
    torch.cuda.synchronize()
    rows = []
    for x, y in zip((k, v), back):
        r = x.float()
        if kv == Q8:
            c, s = ref.quantise(x)
            r = c.float() * s.unsqueeze(-1)
        assert torch.equal(y.cpu(), r)
        rows.append(r.double())
    for s in range(2):
        n, lo, at = b.rows[s], int(b.start[s]), int(whole.start[s])
        want, bound = ref.attention(q[lo:lo + n].double(), rows[0][at:at + b.lens[s]], rows[1][at:at + b.lens[s]],
                                    b.lens[s] - n, 0, 1 / math.sqrt(d))
        check(out[lo:lo + n], want, bound(F16), f"sequence {s}")


def test_empty_batches(pkg):
    """No sequences, no rows: nothing happens."""
    from gguf_runner_amd import ops
    pool = [torch.zeros((2, 16, 8, 128), dtype=F16).cuda() for _ in "kv"]
    cache = ops.PagedCache(*pool)
    zero = torch.zeros(1, dtype=torch.int32).cuda()
    none = ops.PagedBatch(zero, zero[:0], torch.zeros((0, 1), dtype=torch.int32).cuda(), n_rows=4, max_rows=1, max_len=1)
    rows = torch.ones((4, 8, 128), dtype=F16).cuda()
    out = ops.paged_attention(cache, none, rows)
    ops.PagedWriteCall(cache, none, rows, rows.clone())()
    empty = ops.PagedBatch(torch.zeros(2, dtype=torch.int32).cuda(), zero + 5, zero.view(1, 1), n_rows=0, max_rows=1, max_len=5)
    ops.PagedAttentionCall(cache, empty, rows[:0], out[:0])()
    ops.packed_attention(rows[:0], rows[:0], rows[:0], torch.zeros(2, dtype=torch.int32).cuda(), max_rows=1)
    torch.cuda.synchronize()
    assert not out.any() and not pool[0].any()


def test_offsets_out_of_range_are_clamped(pkg):
    """Row offsets and lengths that do not fit what they index never reach outside it: rows past
    n_rows belong to nobody, lengths end with the table."""
    from gguf_runner_amd import ops
    gen = torch.Generator().manual_seed(12)
    b = ref.Batch([4, 6], [40, 32], 16, 16, table_extra=0)
    pool = pool_of(gen, b, 8, 128, F16)
    cache = ops.PagedCache(*pool)
    q = torch.randn((8, 16, 128), generator=gen).to(F16)
    table = torch.from_numpy(b.table).cuda()
    batch = ops.PagedBatch(torch.tensor([0, 4, 2 ** 31 - 1], dtype=torch.int32).cuda(),
                           torch.tensor([-7, 2 ** 31 - 1], dtype=torch.int32).cuda(), table,
                           n_rows=8, max_rows=6, max_len=48)
    out = ops.paged_attention(cache, batch, q.cuda())
    torch.cuda.synchronize()
    assert not out[:4].any()
    # sequence 1: rows 4 .. 7 are the last of its table's positions; its third page is not there
    k, v = (stored(b, pool[i], None, 1) for i in (0, 1))
    k, v = (torch.cat([x, torch.zeros(16, 8, 128, dtype=torch.float64)]) for x in (k, v))
    absent = torch.arange(48) >= 32
    want, bound = ref.attention(q[4:].double(), k, v, 44, 0, 1 / math.sqrt(128), absent)
    check(out[4:], want, bound(F16))


# bounds that lead to each of a head_dim's kernels whatever the batch is (they "choose kernels;
# a wrong value costs time, not results"): few rows, whole blocks, blocks cut along the keys
HINTS = [(1, 1), (1, 1 << 20), (500, 1), (300, 1 << 20), (4096, 1 << 20)]


def hinted(ops, b, hint):
    return ops.PagedBatch(torch.from_numpy(b.start).cuda(), torch.tensor(b.lens, dtype=torch.int32).cuda(),
                          torch.from_numpy(b.table).cuda(), n_rows=b.n_rows, max_rows=hint[0], max_len=hint[1])


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("h,g,d", [(14, 2, 64), (16, 8, 128), (8, 4, 256)])
@pytest.mark.parametrize("dtype,kv", [(F16, F16), (BF16, BF16), (F16, Q8), (BF16, Q8)])
@pytest.mark.parametrize("many,window", [(False, 0), (False, 70), (True, 0)])
def test_bounds_choose_kernels_not_results(pkg, hint, h, g, d, dtype, kv, many, window):
    """Every kernel of a head_dim and type over one mixed batch, and over more sequences than a
    wave has lanes."""
    from gguf_runner_amd import ops
    if many:
        b = ref.Batch([3, 17, 0, 1, 40] * 20, [i % 90 + 40 for i in range(100)], 16, 21, tail=2, table_extra=2000)
    else:
        b = ref.Batch([7, 1, 0, 130, 33, 300], [300, 1, 90, 130, 20, 1000], 16, 22, lead=1, tail=3, table_extra=2000)
    gen = torch.Generator().manual_seed(13)
    pool = pool_of(gen, b, g, d, kv)
    q = torch.randn((b.n_rows, h, d), generator=gen).to(dtype)
    out = torch.full((b.n_rows, h, d), 7.0, dtype=dtype).cuda()
    before = out.clone()
    ops.PagedAttentionCall(ops.PagedCache(*pool), hinted(ops, b, hint), q.cuda(), out, window=window)()
    torch.cuda.synchronize()
    check_attention(b, out, q, pool, window, 1 / math.sqrt(d), dtype, before)


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("h,g,d", [(14, 2, 64), (16, 8, 128), (8, 4, 256)])
@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("window", [0, 40])
def test_infinities_reach_only_the_rows_that_see_them(pkg, hint, h, g, d, kv, window):
    """Infinite V elements of visible keys, NaN and inf everywhere no sequence has a row, in
    every kernel of a head_dim."""
    from gguf_runner_amd import ops
    b = ref.Batch([1, 90, 200, 5], [100, 90, 250, 37], 16, 23, table_extra=2000)
    gen = torch.Generator().manual_seed(14)
    pool = pool_of(gen, b, g, d, kv)
    marks = {0: [(70, g - 1, 3, math.inf)], 2: [(203, 0, 9, math.inf), (230, g - 1, 40, -math.inf), (60, 0, 11, math.inf)]}
    own = torch.zeros(b.n_pages, b.page, dtype=torch.bool)
    for s in range(4):
        own[tuple(torch.from_numpy(x) for x in b.places(s))] = True
    hole = (~own).nonzero(as_tuple=True)
    for i in (0, 1):
        x = pool[i].cpu()
        x[hole] = torch.tensor([math.inf, math.nan, -math.inf]).repeat(hole[0].numel())[:hole[0].numel()].view(-1, 1, 1).to(x.dtype)
        for s, at in marks.items() if i == 1 else ():
            pg, ro = b.places(s)
            for pos, head, e, value in at:
                x[int(pg[pos]), int(ro[pos]), head, e] = value
        pool[i].copy_(x)
    q = torch.randn((b.n_rows, h, d), generator=gen).to(kv)
    out = torch.zeros((b.n_rows, h, d), dtype=kv).cuda()
    ops.PagedAttentionCall(ops.PagedCache(*pool), hinted(ops, b, hint), q.cuda(), out, window=window)()
    torch.cuda.synchronize()
    out = out.cpu()
    for s in range(4):
        n, lo = b.rows[s], int(b.start[s])
        k, v = (stored(b, pool[i], None, s) for i in (0, 1))
        p0 = b.lens[s] - n
        pos = torch.arange(p0, p0 + n)
        hit = torch.zeros(n, h, d, dtype=torch.bool)
        for at, head, e, value in marks.get(s, []):
            sees = (pos >= at) & ((pos < at + window) if window else True)
            hit[sees, head * (h // g):(head + 1) * (h // g), e] = True
            assert (out[lo:lo + n][sees, head * (h // g):(head + 1) * (h // g), e] == value).all()
            v[at, head, e] = 0.0
        want, bound = ref.attention(q[lo:lo + n].double(), k, v, p0, window, 1 / math.sqrt(d))
        check(out[lo:lo + n][~hit], want[~hit], bound(kv)[~hit], f"sequence {s}")


@pytest.mark.parametrize("log_page", [20, 28, 29, 30])
@pytest.mark.parametrize("kv", [F16, Q8])
@pytest.mark.parametrize("rows", [1, 100])
def test_pages_of_any_size(pkg, log_page, kv, rows):
    """One page per sequence, far larger than the rows that are in it (the memory behind them is
    never touched): pages of up to 2^30 rows."""
    from gguf_runner_amd import ops
    b = ref.Batch([rows], [200], 256, 24, spare=0, table_extra=0)
    gen = torch.Generator().manual_seed(15)
    pool = pool_of(gen, b, 2, 64, kv)
    cache, batch = ops.PagedCache(*pool), b.device(ops)
    cache.desc.page_size = 1 << log_page
    q = torch.randn((b.n_rows, 14, 64), generator=gen).to(F16)
    out = torch.full((b.n_rows, 14, 64), 7.0, dtype=F16).cuda()
    ops.PagedAttentionCall(cache, batch, q.cuda(), out)()
    back = [torch.empty((b.n_rows, 2, 64), dtype=F32).cuda() for _ in "kv"]
    ops.PagedReadCall(cache, batch, *back)()
    torch.cuda.synchronize()
    check_attention(b, out, q, pool, 0, 1 / 8, F16, out)
    for i in (0, 1):
        assert torch.equal(back[i].cpu().double(), stored(b, pool[i], pool[2 + i], 0)[200 - rows:].float().double())
