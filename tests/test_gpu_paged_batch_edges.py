"""A ragged batch's step at its edges, against plain implementations in 64 bits: which kind of value
an infinity of a token gives, rows that a step leaves out, what a reservation leaves alone, segments of 64 queries."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_paged_batch import BF, DEV, FP, HF, _cache, _check, _i32, _near, _tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("HD", [16, 64, 96, 128, 256])
@pytest.mark.parametrize("scale", [1, 8])
@pytest.mark.parametrize("lens,new,share", [([50], [32], ()), ([2550, 3], [32, 1], ()), ([633, 650], [8, 8], [([0, 1], 624)]), ([0], [30], ())])
def test_infinities_of_values_keep_their_kind(dt, HD, scale, lens, new, share):
    """An infinity of v is the sum's for every token that sees it, two of both signs are NaN,
    wherever the cut of the work puts the token; the others' sums are finite.  With q and k of 8
    the weights of whole parts vanish in 32 bits, which changes nothing."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(31)
    QH, KVH, PS = 8, 2, 16
    MP = -(-max(n + m for n, m in zip(lens, new)) // PS)
    kp, vp, table = _cache(g, lens, new, share, MP, KVH, PS, HD, dt)
    kp *= scale                                           # (powers of two: exact)
    N, qd = sum(new), QH * HD
    qkv = torch.randn(N, (QH + 2 * KVH) * HD, generator=g)
    qkv[:, :qd + KVH * HD] *= scale
    v0 = qd + KVH * HD
    for t, d, value in ((2, 3, math.inf), (3, 4, -math.inf), (4, 6, math.nan), (6, 5, math.inf), (7, 5, -math.inf), (1, HD, math.inf)):
        qkv[t, v0 + d] = value
    qkv = qkv.to(DEV, dt)
    cos, sin = _tables(HD, MP * PS)
    plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), N, QH)
    c, kx, q = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin)
    torch.cuda.synchronize()
    starts, _, _, _, ok = ref.maps(table.cpu(), torch.tensor(lens), torch.tensor(new), N, kp.shape[0], PS)
    o = ref.batch_attention(q, kp, vp, table.cpu(), lens, starts, ok)
    assert all(o["c"].eq(x).any() for x in (math.inf, -math.inf)) and o["c"].isnan().any() and o["kctx"].isfinite().all()
    for got, want in ((c.cpu(), o["c"]), (kx.cpu(), o["kctx"])):
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(got), kind(want)), kind.__name__


# ------------------------------------------------------------------ rows that a step leaves out

def _at_work(dt, rows, max_len, n_pages=None, L=1, KVH=2, HD=64, PS=16):
    from loom_amd.paged import PagedKVCache
    cache = PagedKVCache(L, rows, max_len, KVH, HD, dt, page_size=PS, n_pages=n_pages)
    cache.k_pages.normal_()                               # what former holders of the pages left there
    cache.v_pages.normal_()
    cache.start(torch.ones(rows, dtype=torch.bool, device=DEV))
    return cache


def _step(cache, streams, new, places, QH, tables):
    """reserve, plan, attend, advance; the outputs (c, kctx, q) of the tokens by row."""
    lens, counts = cache.lens.tolist(), _i32(new)
    cache.reserve(counts)
    plan = cache.plan(counts, places, QH)
    flat = torch.cat([streams[r, lens[r]:lens[r] + m] for r, m in enumerate(new)] + [streams[0, :places]])[:places].contiguous()
    got = cache.attend_batch(0, plan, flat, *tables)
    cache.advance(counts)
    at = plan.starts.tolist()
    return [[y[at[r]:at[r + 1]] for y in got] for r in range(len(new))]


def _right(cache, r, got, first, dt):
    """Outputs of row r's tokens from `first` on against the cache's own rows in 64 bits."""
    c, kx, q = (y.cpu() for y in got)
    T = first + q.shape[0]
    o = ref.batch_attention(q, cache.k_pages[0], cache.v_pages[0], cache.table[r:r + 1].cpu(), [first], [0, q.shape[0]], [True])
    _near(c, o["c"], o["c_abs"], o, dt, q.shape[2], "c")
    _near(kx, o["kctx"], o["kctx_abs"], o, dt, q.shape[2], "kctx")
    assert int(cache.lens[r]) >= T


@pytest.mark.parametrize("dt", [BF, FP])
def test_a_row_that_does_not_fit_into_the_batch_does_not_advance(dt):
    """A step whose last row finds no places, and the same row again in the next one: its lens stays, check
    raises, and what it then reads is what was written."""
    g = torch.Generator().manual_seed(41)
    QH, KVH, HD = 8, 2, 64
    streams = torch.randn(3, 60, (QH + 2 * KVH) * HD, generator=g).to(DEV, dt)
    cache, tables = _at_work(dt, 3, 60), _tables(HD, 64)
    out = _step(cache, streams, [4, 3, 0], 7, QH, tables)
    cache.check()
    out = _step(cache, streams, [2, 0, 20], 9, QH, tables)   # 22 tokens for 9 places
    assert cache.lens.tolist() == [6, 3, 0]
    _right(cache, 0, out[0], 4, dt)
    with pytest.raises(RuntimeError, match="1 row.* no place"):
        cache.check()
    out = _step(cache, streams, [1, 1, 20], 30, QH, tables)
    assert cache.lens.tolist() == [7, 4, 20]
    _right(cache, 2, out[2], 0, dt)
    out = _step(cache, streams, [1, 1, 1], 3, QH, tables)
    assert cache.lens.tolist() == [8, 5, 21]
    for r, first in ((0, 7), (1, 4), (2, 20)):
        _right(cache, r, out[r], first, dt)
    for r in range(3):                                    # the cache holds the rows' tokens and no others
        n = int(cache.lens[r])
        held = ref.rows_of(cache.v_pages[0].cpu(), cache.table[r].cpu(), n)
        assert torch.equal(held, streams[r, :n].view(n, -1, HD)[:, QH + KVH:].transpose(0, 1).cpu().to(held.dtype))
    cache.reset()
    cache.check()


def test_rows_without_pages_or_behind_the_table_do_not_advance():
    g = torch.Generator().manual_seed(42)
    QH, KVH, HD = 8, 2, 64
    streams = torch.randn(2, 100, (QH + 2 * KVH) * HD, generator=g).to(DEV, BF)
    tables = _tables(HD, 128)
    cache = _at_work(BF, 2, 64, n_pages=4)
    _step(cache, streams, [33, 40], 73, QH, tables)       # three pages each of four
    assert cache.lens.tolist() == [33, 0]
    with pytest.raises(RuntimeError, match="2 pages could not be had.*1 row"):
        cache.check()
    cache = _at_work(BF, 2, 64)
    _step(cache, streams, [60, 3], 63, QH, tables)
    _step(cache, streams, [5, 1], 6, QH, tables)          # 65 of 64
    assert cache.lens.tolist() == [60, 4]
    out = _step(cache, streams, [4, 1], 5, QH, tables)
    assert cache.lens.tolist() == [64, 5]
    _right(cache, 0, out[0], 60, BF)


def test_two_plans_of_one_step_advance_their_own_rows():
    """Prompts and single tokens planned apart, of which one prompt finds no places; and rows whose step
    was planned by the operator itself."""
    from loom_amd import ops
    cache = _at_work(BF, 4, 64)
    a, b = _i32([5, 0, 30, 0]), _i32([0, 2, 0, -1])
    cache.reserve(_i32([5, 2, 30, 0]))
    cache.plan(a, 20, 8)
    cache.plan(b, 2, 8)
    cache.advance(a)
    cache.advance(b)
    assert cache.lens.tolist() == [5, 2, 0, 0]
    other, new = _at_work(BF, 4, 64), _i32([1, 2, 3, 0])
    other.reserve(new)
    ops.paged_plan(other.k_pages, other.table, other.lens, new, 6, 8)
    other.advance(new)
    assert other.lens.tolist() == [1, 2, 3, 0]
    other.check()


def test_a_captured_step_leaves_out_what_does_not_fit():
    g = torch.Generator().manual_seed(43)
    QH, KVH, HD = 8, 2, 64
    streams = torch.randn(3, 200, (QH + 2 * KVH) * HD, generator=g).to(DEV, BF)
    tables = _tables(HD, 208)
    cache, new, flat = _at_work(BF, 3, 200), _i32([0, 0, 0]), torch.zeros(12, (QH + 2 * KVH) * HD, dtype=BF, device=DEV)

    def step():
        cache.reserve(new)
        plan = cache.plan(new, 12, QH)
        out = cache.attend_batch(0, plan, flat, *tables)
        cache.advance(new)
        return [plan.starts] + out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    lens = [0, 0, 0]
    for counts in ([4, 3, 5], [1, 1, 11], [1, 1, 10], [12, 1, 1], [13, 1, 1], [1, 1, 1], [2, 9, 2]):
        rows = [streams[r, lens[r]:lens[r] + m] for r, m in enumerate(counts)]
        flat.copy_(torch.cat(rows + [flat])[:12])
        new.copy_(_i32(counts))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        at = outs[0].tolist()
        for r, m in enumerate(counts):
            if at[r] + m <= 12:
                _right(cache, r, [y[at[r]:at[r] + m] for y in outs[1:]], lens[r], BF)
                lens[r] += m
        assert cache.lens.tolist() == lens, counts
    with pytest.raises(RuntimeError, match="no place"):
        cache.check()


def test_a_reservation_leaves_lens_as_they_are():
    """Whatever stands there for rows that hold no sequence."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(51)
    k, v = (torch.randn(1, 20, 2, 16, 32, generator=g).to(DEV, BF) for _ in range(2))
    held = [-2, 5, -1, -2 ** 31, 0, 100]
    lens, refs, status = _i32(held), torch.zeros(20, dtype=torch.int32, device=DEV), _i32([0])
    table = torch.full((6, 4), -1, dtype=torch.int32, device=DEV)
    table[1, 0] = 3
    refs[3] = 1
    ops.paged_reserve(k, v, table, lens, refs, status, _i32([9, 30, 1, 2, 0, 1]))
    assert lens.tolist() == held
    assert table.tolist() == [[-1] * 4, [3, 0, 1, -1]] + [[-1] * 4] * 4 and int(status) == 1


# ------------------------------------------------------------------ segments of 64 queries

@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("HD", [16, 64, 96, 128])
@pytest.mark.parametrize("kind", ["alone", "beside rows that share", "G of 4"])
def test_own_segments_of_64_queries(dt, HD, kind):
    """Own segments are halved where halves fill the device and whole ones do not."""
    slots_of = lambda KVH: 2 * torch.cuda.get_device_properties(0).multi_processor_count // KVH  # noqa: E731
    QH, KVH = (64, 16) if kind == "G of 4" else (32, 32)
    slots, G = slots_of(KVH), QH // KVH
    # rows of more than 64 queries and up to 128, as many as take more than half the places
    n = slots // 2 + 1
    new = [(65 + (29 * i) % 64 + G - 1) // G for i in range(n)]
    lens = [(83 * i) % 200 for i in range(n)]
    share = []
    if kind != "alone":                                   # single tokens behind one prompt, fewer than whole segments leave room for
        more = slots - n - 1
        share = [(range(n, n + more), 96)]
        lens, new = lens + [96 + (7 * i) % 40 for i in range(more)], new + [1] * more
    halves, wholes = (sum(-(-m * G // q) for m in new) for q in (64, 128))
    assert wholes < slots <= halves
    _check(dt, lens, new, QH, KVH, HD, 16, 24, 61, share=share, pad=2)
