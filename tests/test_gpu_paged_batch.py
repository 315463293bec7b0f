"""GPU parity of a ragged batch's step over the paged cache (reservation per row, slot
maps, attention that reads common pages once) with plain implementations in 64 bits."""
import math

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(HD, n):
    inv = 10000.0 ** (-torch.arange(0, HD, 2, dtype=torch.float64) / HD)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * torch.cat([inv, inv])[None]
    return ang.cos().float().to(DEV), ang.sin().float().to(DEV)


def _bits(t):
    return t.view(torch.int32 if t.dtype == FP else torch.int16)


def _cache(g, lens, new, share, MP, KVH, PS, HD, dt, spare=2, layout="head"):
    """Pools and a table of pages in random order that hold lens + new tokens of each row.
    share: (rows, tokens) groups whose rows hold the same pages of their first tokens (whole
    pages).  What no token may read is NaN: free pages, and places behind lens (the new
    tokens' own included)."""
    R = len(lens)
    need = [-(-(n + max(m, 0)) // PS) if n >= 0 else 0 for n, m in zip(lens, new)]
    rows, used = [[-1] * MP for _ in range(R)], 0
    for group, tokens in share:
        for s in range(tokens // PS):
            for r in group:
                rows[r][s] = used
            used += 1
    for r in range(R):
        for s in range(need[r]):
            if rows[r][s] < 0:
                rows[r][s] = used
                used += 1
    NP = used + spare
    order = torch.randperm(NP, generator=g).tolist()
    rows = [[order[p] if p >= 0 else -1 for p in row] for row in rows]
    shape = (NP, KVH, PS, HD) if layout == "head" else (NP, PS, KVH, HD)
    kp, vp = torch.randn(*shape, generator=g).to(dt), torch.randn(*shape, generator=g).to(dt)
    if layout != "head":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    for pool in (kp, vp):
        for r, n in enumerate(lens):
            for s in range(max(n, 0) // PS, need[r]):
                pool[rows[r][s], :, max(n - s * PS, 0):] = math.nan
        for p in order[used:]:
            pool[p] = math.nan
    if layout != "head":
        return (kp.transpose(1, 2).contiguous().to(DEV).transpose(1, 2),
                vp.transpose(1, 2).contiguous().to(DEV).transpose(1, 2), torch.tensor(rows, dtype=torch.int32).to(DEV))
    return kp.to(DEV), vp.to(DEV), torch.tensor(rows, dtype=torch.int32).view(R, MP).to(DEV)


def _near(got, want, spread, o, dt, HD, what):
    """|got - want| within: the output's rounding; the weights' rounding to a 16-bit type
    before the products (half a step of the weights, on the sum of absolute values); the
    fp32 score's error (a product and an addition per dimension, HD of them, on sum |q k|,
    plus its scaling) and that of 2^s (its argument's rounding on |s| log2 e and the
    instruction's), in numerator and denominator; and n fp32 additions."""
    half, u = torch.finfo(dt).eps / 2, 2.0 ** -24
    ds = o["qk_abs"] * (HD + 4) * u + 4 * (o["s_max"] + 1) * u
    rel = (0 if dt == FP else half) + 2 * ds + (o["n"][:, None] + 64) * u
    bound = half * want.abs() + rel[..., None] * spread + torch.finfo(dt).tiny
    if dt == HF:
        bound = bound + 2.0 ** -24          # half's subnormal step
    over = (got.cpu().double() - want).abs() / bound
    assert float(over.max()) <= 1, f"{what}: {float(over.max())} of the bound"


def _check(dt, lens, new, QH, KVH, HD, PS, MP, seed, share=(), pad=0, layout="head", kctx=True, shared=None, extra=0):
    from loom_amd import ops
    g = torch.Generator().manual_seed(seed)
    kp, vp, table = _cache(g, lens, new, share, MP, KVH, PS, HD, dt, layout=layout)
    if extra:                                           # a table and projection rows that are views of wider ones
        wide = torch.full((len(lens), MP + extra), 7, dtype=torch.int32, device=DEV)
        wide[:, :MP] = table
        table = wide[:, :MP]
    N = sum(max(m, 0) for n, m in zip(lens, new) if n >= 0) + pad
    width = (QH + 2 * KVH) * HD
    qkv = torch.randn(N, width + 16 * extra, generator=g).to(DEV, dt)[:, :width]
    cos, sin = _tables(HD, MP * PS)
    k0, v0 = kp.clone(), vp.clone()
    plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), N, QH)
    starts, rows, pos, slots, ok = ref.maps(table.cpu(), torch.tensor(lens), torch.tensor(new), N, kp.shape[0], PS)
    assert plan.starts.tolist() == starts and plan.rows.tolist() == rows
    assert plan.positions.tolist() == pos and plan.slots.tolist() == slots
    if shared is not None:
        assert plan.shared.tolist() == shared
    c, kx, q = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin, want_kctx=kctx)
    torch.cuda.synchronize()
    half = torch.finfo(dt).eps / 2
    x = qkv.cpu().view(N, QH + 2 * KVH, HD)
    k0, v0, kc, vc = k0.cpu(), v0.cpu(), kp.cpu(), vp.cpu()
    qc, cc = q.cpu(), c.cpu()
    for t in range(N):
        if slots[t] < 0:
            for y in (qc, cc) + ((kx.cpu(),) if kctx else ()):
                assert y[t].float().isnan().all() if rows[t] >= 0 else not y[t].float().any(), t
    at = torch.tensor([t for t in range(N) if slots[t] >= 0], dtype=torch.int64)
    if len(at) == 0:
        assert torch.equal(_bits(kc), _bits(k0)) and torch.equal(_bits(vc), _bits(v0))
        return
    p, sl = torch.tensor(pos)[at], torch.tensor(slots)[at]
    co, si = cos.cpu()[p][:, None], sin.cpu()[p][:, None]
    xs = x[at]
    want = ref.rope(xs[:, :QH + KVH], co, si)
    size = (xs[:, :QH + KVH].double() * co.double()).abs() + torch.cat(
        [t.abs() for t in (xs[:, :QH + KVH, HD // 2:], xs[:, :QH + KVH, :HD // 2])], -1).double() * si.double().abs()
    bound = half * want.abs() + 2.0 ** -22 * size + torch.finfo(dt).tiny + (2.0 ** -24 if dt == HF else 0)
    got = torch.cat([qc[at], kc[sl // PS, :, sl % PS]], 1).double()
    assert ((got - want).abs() <= bound).all(), "rope"
    # the tokens' places hold them, and nothing else of the pools was written
    v0[sl // PS, :, sl % PS] = xs[:, QH + KVH:]
    k0[sl // PS, :, sl % PS] = kc[sl // PS, :, sl % PS]
    assert torch.equal(_bits(kc), _bits(k0)) and torch.equal(_bits(vc), _bits(v0))
    o = ref.batch_attention(q, kp, vp, table.cpu(), lens, starts, ok)
    here = {k: v[at] for k, v in o.items()}
    _near(cc[at], here["c"], here["c_abs"], here, dt, HD, "c")
    if kctx:
        _near(kx.cpu()[at], here["kctx"], here["kctx_abs"], here, dt, HD, "kctx")
    else:
        assert kx is None


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("lens,new", [([0], [1]), ([0], [17]), ([1, 0, -1, 15], [1, 3, 4, 0]), ([16, 17, 31, 64], [1, 15, 64, 65]),
                                      ([127, 128, -1, 0], [1, 130, 1, 2]), ([300, 0, 5, 511], [1, 0, 200, 1]), ([0, 0], [0, 0])])
def test_lengths(dt, lens, new):
    _check(dt, lens, new, 8, 2, 96, 16, 40, 1, pad=3)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("QH,KVH", [(1, 1), (3, 1), (5, 5), (8, 2), (16, 2), (16, 1), (24, 1), (32, 8), (6, 2), (70, 1)])
def test_heads(dt, QH, KVH):
    _check(dt, [70, 3, -1, 200, 128, 128], [1, 40, 0, 9, 1, 2], QH, KVH, 64, 32, 9, 2, share=[([4, 5, 0], 64)])


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("HD", [8, 16, 32, 64, 96, 128, 256])
@pytest.mark.parametrize("PS", [16, 64, 1024])
def test_head_sizes_and_pages(dt, HD, PS):
    _check(dt, [150, 0, 333, 150], [1, 80, 20, 1], 8, 2, HD, PS, 1024 // PS, 3, share=[([0, 3], 128)])


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("HD", [96, 128, 16])
def test_token_major_pages_no_kctx_views(dt, HD):
    _check(dt, [150, 0, 333, -1, 150], [1, 30, 5, -2, 2], 8, 2, HD, 16, 40, 4, layout="token", kctx=False, extra=3,
           share=[([0, 4], 144)])


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("W,P,QH,KVH", [(2, 64, 8, 2), (4, 333, 8, 2), (5, 1000, 8, 2), (8, 320, 8, 2), (17, 640, 16, 2), (33, 256, 8, 8),
                                        (3, 500, 24, 1), (64, 128, 8, 2)])
def test_groups_of_one_prompt(dt, W, P, QH, KVH):
    """Continuations of one prompt, each with tokens of its own: queries of one, two and
    more blocks of 16, 32, 64."""
    lens = [P + (11 * i) % 70 for i in range(W)]
    whole = P // 16 * 16
    _check(dt, lens, [1] * W, QH, KVH, 64, 16, -(-max(lens) // 16) + 1, 5, share=[(range(W), P)],
           shared=[whole] * W)


@pytest.mark.parametrize("dt", [BF, FP])
def test_groups_apart_and_between_each_other(dt):
    """Rows of two prompts in turn, one row alone, an idle one, one that brings nothing, a prompt that
    shares pages but fills a block by itself, and one whose pages part early."""
    lens = [200, 150, 210, 155, 90, -1, 400, 200, 131, 260]
    new = [1, 2, 1, 1, 1, 1, 0, 100, 1, 1]
    share = [([0, 2, 6, 7], 192), ([1, 3], 144), ([8, 9], 128)]
    _check(dt, lens, new, 8, 2, 96, 16, 30, 6, share=share, pad=1, shared=[192, 144, 192, 144, 0, 0, 0, 0, 128, 128])


@pytest.mark.parametrize("dt", [BF, FP])
def test_what_rows_share_ends_with_their_least_common_page(dt):
    """All pages shared, more than the shortest row has whole tokens of; and less than pays."""
    _check(dt, [100, 128, 130, 129], [1, 1, 1, 1], 8, 2, 96, 16, 10, 7, share=[([1, 2, 3], 128), ([0, 1, 2, 3], 96)],
           shared=[96, 96, 96, 96])
    _check(dt, [50, 49], [1, 1], 8, 2, 96, 16, 10, 7, share=[([0, 1], 48)], shared=[0, 0])


@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_several_tokens_of_rows_that_share(dt):
    """Up to 32 queries a row, tokens of the group in one list that crosses its blocks."""
    _check(dt, [130, 140, 133, 128, 129, 300], [8, 1, 7, 3, 5, 8], 8, 2, 64, 16, 24, 8, share=[(range(6), 128)], shared=[128] * 6)


@pytest.mark.parametrize("dt", [BF, FP])
def test_long_rows_split_and_joined(dt):
    _check(dt, [5000, 3, 1, 4097, -1, 900], [1, 2, 1, 70, 0, 1], 8, 2, 96, 64, 79, 9)
    _check(dt, [5000, 4900, 4990, 4864], [1, 1, 1, 1], 8, 2, 128, 64, 79, 9, share=[(range(4), 4864)])


@pytest.mark.parametrize("dt", [BF, FP])
def test_many_rows(dt):
    lens = [(37 * i) % 190 - 1 for i in range(300)]
    _check(dt, lens, [i % 3 for i in range(300)], 4, 2, 32, 16, 13, 10,
           share=[([i for i in range(300) if lens[i] >= 100], 96), ([i for i in range(300) if 80 <= lens[i] < 100], 64)])


def test_most_rows():
    _check(BF, [16 * (i % 5) + 64 for i in range(1024)], [1] * 1024, 2, 1, 32, 16, 9, 11, share=[(range(0, 1024, 2), 64)])


@pytest.mark.parametrize("dt", [BF, FP])
def test_prompts_into_an_empty_cache(dt):
    _check(dt, [0] * 5, [1, 257, 64, 700, 63], 8, 2, 96, 16, 44, 12, pad=7)


# ------------------------------------------------------------------ what has no influence, what is refused

@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("HD", [16, 96, 128])
def test_later_tokens_that_are_not_finite(dt, HD):
    """An infinity or NaN in a token's k or v reaches that token and those behind it only."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(13)
    QH, KVH, PS, lens, new = 8, 2, 16, [37, 0, 5], [60, 20, 1]
    kp, vp, table = _cache(g, lens, new, (), 8, KVH, PS, HD, dt)
    N, qd = sum(new), QH * HD
    clean = torch.randn(N, (QH + 2 * KVH) * HD, generator=g).to(DEV, dt)
    cos, sin = _tables(HD, 128)
    plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), N, QH)
    k0, v0 = kp.clone(), vp.clone()
    base = ops.paged_batch_step(plan, clean, k0, v0, table, cos, sin)
    for t, at, value in ((33, qd + KVH * HD + 3, math.inf), (33, qd + 5, math.nan), (70, qd + 1, -math.inf), (79, qd + 2 * HD + 1, math.nan)):
        qkv = clean.clone()
        qkv[t, at] = value
        k1, v1 = kp.clone(), vp.clone()
        got = ops.paged_batch_step(plan, qkv, k1, v1, table, cos, sin)
        last = 60 if t < 60 else 80                       # the end of the token's row
        for y, b in zip(got, base):
            yc, bc = y.cpu().float(), b.cpu().float()
            # tokens in front of it: the same sums, in another order where their tile holds it
            keep = [i for i in range(N) if not t <= i < last]
            torch.testing.assert_close(yc[keep], bc[keep], rtol=2.0 ** -6 if dt != FP else 1e-5, atol=2.0 ** -6 if dt != FP else 1e-5)
        heads = range(QH // KVH)                          # the kv head that holds it, or its q heads
        assert not got[0].cpu().float()[t:last, list(heads)].isfinite().all()
        for i in range(t, last):
            assert not (got[0][i].float().isfinite().all() and got[1][i].float().isfinite().all()), i


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("HD", [16, 64, 96, 128])
@pytest.mark.parametrize("kctx", [True, False])
def test_tokens_that_are_not_finite_where_rows_share_and_split(dt, HD, kctx):
    """The same in rows whose sums come from several parts (a common one, chunks of a long row), of
    1 to 64 queries that share and of 128 that do not: what is finite in 64 bits is right, the rest
    is not finite."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(27)
    QH, KVH, PS = 8, 2, 16
    lens, new = [640, 650, 645, 641, 2500, 700], [16, 8, 4, 1, 40, 1]
    kp, vp, table = _cache(g, lens, new, [([0, 1, 2, 3], 640)], 170, KVH, PS, HD, dt)
    N, qd = sum(new), QH * HD
    qkv = torch.randn(N, (QH + 2 * KVH) * HD, generator=g).to(dt)
    v0 = qd + KVH * HD
    for t, at, value in ((5, v0 + 3, math.inf), (11, v0 + HD, math.nan), (17, v0 + 1, -math.inf), (26, qd + 2, math.nan),
                         (45, v0 + 5, math.inf), (50, v0 + 5, -math.inf), (60, qd + HD, math.nan)):
        qkv[t, at] = value
    qkv = qkv.to(DEV)
    cos, sin = _tables(HD, 2720)
    plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), N, QH)
    assert plan.shared.tolist() == [640] * 4 + [0] * 2
    c, kx, q = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin, want_kctx=kctx)
    torch.cuda.synchronize()
    starts, _, _, _, ok = ref.maps(table.cpu(), torch.tensor(lens), torch.tensor(new), N, kp.shape[0], PS)
    o = ref.batch_attention(q, kp, vp, table.cpu(), lens, starts, ok)
    here = {k: torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0) for k, v in o.items()}
    for got, what in ((c, "c"), (kx, "kctx"))[:1 + kctx]:
        want, y = o[what], got.cpu().double()
        fine = want.isfinite()
        assert 0 < int((~fine).sum()) < fine.numel() // 2
        assert not y[~fine].isfinite().any()
        _near(torch.where(fine, y, 0), torch.where(fine, want, 0), here[what + "_abs"], here, dt, HD, what)


@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_rows_without_their_pages_or_their_places(dt):
    """A row that lacks a page (of the past or to come), whose tokens pass its table, or do not fit
    into the batch: NaN, and nothing written."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(14)
    QH, KVH, PS, HD = 8, 2, 16, 96
    lens, new = [20, 40, 30, 10, 60, 12], [2, 3, 4, 1, 5, 2]
    kp, vp, table = _cache(g, lens, [2, 3, 4, 1, 4, 2], (), 4, KVH, PS, HD, dt)
    table[1, 0] = -1
    table[2, 2] = kp.shape[0]
    N = 14                                                # the last row brings two tokens for one place left
    _, rows, _, slots, ok = ref.maps(table.cpu(), torch.tensor(lens), torch.tensor(new), N, kp.shape[0], PS)
    assert ok == [True, False, False, True, False, False]
    plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), N, QH)
    assert plan.slots.tolist() == slots and plan.rows.tolist() == rows
    qkv = torch.randn(N, (QH + 2 * KVH) * HD, generator=g).to(DEV, dt)
    cos, sin = _tables(HD, 64)
    k0, v0 = kp.clone(), vp.clone()
    out = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin)
    bad = torch.tensor([s < 0 for s in slots])
    for y in out:
        assert y.cpu().float()[bad].isnan().all() and y.cpu().float()[~bad].isfinite().all()
    for pool, was in ((kp, k0), (vp, v0)):
        changed = (_bits(pool) != _bits(was)).flatten(3).any(3).any(1).cpu()
        assert {(int(p) * PS + int(i)) for p, i in changed.nonzero()} <= {s for s in slots if s >= 0}


@pytest.mark.parametrize("dt", [BF, FP])
def test_positions_past_the_rotary_tables(dt):
    from loom_amd import ops
    g = torch.Generator().manual_seed(15)
    kp, vp, table = _cache(g, [30, 10], [6, 1], (), 4, 2, 16, 64, dt)
    qkv = torch.randn(7, 12 * 64, generator=g).to(DEV, dt)
    cos, sin = _tables(64, 33)
    v0 = vp.clone()
    plan = ops.paged_plan(kp, table, _i32([30, 10]), _i32([6, 1]), 7, 8)
    out = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin)
    for y in out:
        y = y.cpu().float()
        assert y[3:6].isnan().all() and y[:3].isfinite().all() and y[6].isfinite().all()
    changed = (_bits(vp) != _bits(v0)).flatten(3).any(3).any(1).cpu().nonzero()
    assert len(changed) == 4


def test_refusals():
    from loom_amd import ops
    g = torch.Generator().manual_seed(16)
    kp, vp, table = _cache(g, [30, 10], [1, 1], (), 4, 2, 16, 64, BF)
    lens, new = _i32([30, 10]), _i32([1, 1])
    cos, sin = _tables(64, 64)
    qkv = torch.randn(2, 12 * 64, generator=g).to(DEV, BF)
    plan = ops.paged_plan(kp, table, lens, new, 2, 8)
    step = lambda **k: ops.paged_batch_step(*dict(dict(plan=plan, qkv=qkv, k_pages=kp, v_pages=vp, table=table, cos=cos, sin=sin), **k).values())  # noqa: E731
    for args, message in [((kp, table, lens[:1], new, 2, 8), "lens must be"), ((kp, table, lens, new.long(), 2, 8), "new must be"),
                          ((kp, table, lens, new, -1, 8), "n_tokens"), ((kp, table, lens, new, 1 << 21, 8), "n_tokens"),
                          ((kp, table, lens, new, 2, 7), "7 query heads"), ((kp[0], table, lens, new, 2, 8), "k_pages must be"),
                          ((kp, table.cpu(), lens, new, 2, 8), "CUDA"), ((kp[:, :, :8], table, lens, new, 2, 8), "power of two")]:
        with pytest.raises(RuntimeError, match=message):
            ops.paged_plan(*args)
    for change, message in [(dict(qkv=qkv[:1]), "plan.rows must be"), (dict(qkv=qkv.float()), "pools' dtype"), (dict(qkv=qkv[:, :64]), "qkv must be"),
                            (dict(k_pages=kp[:-1], v_pages=vp[:-1]), "other sizes"), (dict(table=table[:, :3]), "other sizes"),
                            (dict(table=table[:1]), "other sizes"), (dict(cos=cos[:, :32]), "cos and sin"), (dict(v_pages=vp[:-1]), "same layout"),
                            (dict(plan=plan._replace(work=plan.work[:64])), "plan of"), (dict(plan=plan._replace(sizes=())), "not one of paged_plan"),
                            (dict(plan=plan._replace(slots=plan.positions)), "not one of paged_plan"),
                            (dict(qkv=qkv[:, :4 * 64 + 5 * 64]), "query heads over")]:
        with pytest.raises(RuntimeError, match=message):
            step(**change)
    assert len(step()) == 3


def test_no_rows_and_no_tokens():
    from loom_amd import ops
    g = torch.Generator().manual_seed(17)
    kp, vp, table = _cache(g, [30, 10], [1, 1], (), 4, 2, 16, 64, BF)
    cos, sin = _tables(64, 64)
    plan = ops.paged_plan(kp, table[:0], _i32([]), _i32([]), 0, 8)
    assert plan.starts.tolist() == [0] and plan.rows.numel() == 0
    out = ops.paged_batch_step(plan, torch.empty(0, 768, dtype=BF, device=DEV), kp, vp, table[:0], cos, sin)
    assert [tuple(y.shape) for y in out] == [(0, 8, 64)] * 3
    plan = ops.paged_plan(kp, table[:0], _i32([]), _i32([]), 5, 8)
    out = ops.paged_batch_step(plan, torch.ones(5, 768, dtype=BF, device=DEV), kp, vp, table[:0], cos, sin)
    assert not any(y.float().any() for y in out)
    plan = ops.paged_plan(kp, table, _i32([30, 10]), _i32([0, -5]), 0, 8)
    assert plan.starts.tolist() == [0, 0, 0] and plan.shared.tolist() == [0, 0]


# ------------------------------------------------------------------ reservation

def _pools(g, L, NP, KVH, PS, HD, dt):
    return [torch.randn(L, NP, KVH, PS, HD, generator=g).to(DEV, dt) for _ in range(2)]


@pytest.mark.parametrize("seed", range(8))
def test_reserve(seed):
    """Counts per row: forks with a partly filled page, rows that bring nothing, whose tables end,
    pages ahead, and a pool that runs out."""
    from loom_amd import ops
    import random
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    R, MP, PS, NP, L = rng.choice([3, 20, 70]), 9, 16, 400, 2
    if seed % 4 == 3:
        NP = 3 * R                                        # too few
    free = list(range(NP))
    rng.shuffle(free)
    lens, rows = [], []
    for r in range(R):
        if r and rows[-1][0] >= 0 and rng.random() < 0.5:   # a fork of the row before
            lens.append(lens[-1])
            rows.append(list(rows[-1][:-(-lens[-1] // PS)]) + [-1] * (MP - -(-lens[-1] // PS)))
            continue
        n = rng.choice([-1, 0, rng.randrange(1, 40)])
        have = min(-(-max(n, 0) // PS) + (rng.random() < 0.2), len(free))
        lens.append(n if n <= have * PS else -1)
        if lens[-1] < 0:
            have = 0
        rows.append([free.pop() for _ in range(have)] + [-1] * (MP - have))
    refs = [0] * NP
    for row in rows:
        for p in row:
            if p >= 0:
                refs[p] += 1
    new = [rng.choice([0, 1, 1, 5, 40, 200, -3, 2 ** 31 - 1]) for _ in range(R)]
    k, v = _pools(g, L, NP, 2, PS, 32, BF)
    table, ln, rf = _i32(rows), _i32(lens), _i32(refs)
    want = ref.reserve(k.cpu(), v.cpu(), table.cpu(), ln.cpu(), rf.cpu(), torch.tensor(new))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_reserve(k, v, table, ln, rf, status, _i32(new))
    assert ln.tolist() == lens and int(status) == want[4]
    assert torch.equal(table.cpu(), want[2]) and torch.equal(rf.cpu(), want[3])
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


@pytest.mark.parametrize("n", [0, 1, 17])
def test_reserve_the_same_for_all_is_update(n):
    from loom_amd import ops
    g = torch.Generator().manual_seed(3)
    lens = [5, 16, -1, 0, 31]
    k, v = _pools(g, 1, 30, 2, 16, 32, BF)
    outs = []
    for each in (True, False):
        table = _i32([[7, -1, -1, -1], [3, -1, -1, -1], [-1] * 4, [-1] * 4, [7, 9, -1, -1]])
        refs = torch.zeros(30, dtype=torch.int32, device=DEV)
        refs[[3, 9]] = 1
        refs[7] = 2
        status, kk, vv, ln = _i32([0]), k.clone(), v.clone(), _i32(lens)
        if each:
            ops.paged_reserve(kk, vv, table, ln, refs, status, _i32([n] * 5))
        else:
            ops.paged_update(kk, vv, table, ln, refs, status, n_new=n)
        outs.append((table, ln, refs, status, kk, vv))
    for x, y in zip(*outs):
        assert torch.equal(x, y)


# ------------------------------------------------------------------ together

def _serve(dt, graph=False):
    """Requests of different lengths behind one instruction through a cache: the instruction once,
    forks of it, their prompts in two pieces, then single tokens; every token's outputs."""
    from loom_amd import ops  # noqa: F401
    from loom_amd.paged import PagedKVCache
    g = torch.Generator().manual_seed(21)
    QH, KVH, HD, L, R = 8, 2, 64, 2, 5
    cache = PagedKVCache(L, R, 400, KVH, HD, dt, page_size=16, n_pages=120)
    cos, sin = _tables(HD, 400)
    every = lambda *v: _i32(list(v))  # noqa: E731
    streams = torch.randn(R, 400, L, (QH + 2 * KVH) * HD, generator=g).to(DEV, dt)
    streams[:, :150] = streams[:1, :150]                  # the instruction
    outs = [[] for _ in range(R)]

    def step(new, pad):
        lens = [max(n, 0) for n in cache.lens.tolist()]
        N = sum(new) + pad
        cache.reserve(every(*new))
        plan = cache.plan(every(*new), N, QH)
        rows = torch.cat([streams[r, lens[r]:lens[r] + m] for r, m in enumerate(new)] + [streams[0, :pad]])
        got = [cache.attend_batch(layer, plan, rows[:, layer].contiguous(), cos, sin) for layer in range(L)]
        a = plan.starts.tolist()
        for r in range(R):
            for i in range(a[r], a[r + 1]):
                outs[r].append([y[i].cpu() for layer in got for y in layer])
        cache.advance(every(*new))
        return plan

    cache.start(torch.tensor([True] + [False] * (R - 1), device=DEV))
    step([150, 0, 0, 0, 0], 2)
    cache.update(parent=torch.zeros(R, dtype=torch.int32, device=DEV))
    first = list(outs[0])
    for r in range(1, R):
        outs[r] += first
    step([20, 1, 0, 33, 64], 0)
    step([1, 40, 3, 2, 1], 5)
    shared = []
    for _ in range(12):
        shared.append(step([1] * R, 1).shared.tolist())
    cache.check()
    return cache, streams, outs, shared, (cos, sin)


@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_serving_steps_together(dt):
    cache, streams, outs, shared, (cos, sin) = _serve(dt)
    assert shared[-1] == [144] * 5
    QH, KVH, HD = 8, 2, 64
    half = torch.finfo(dt).eps / 2
    for r in range(5):
        T = int(cache.lens[r])
        assert len(outs[r]) == T
        for layer in range(2):
            x = streams[r, :T, layer].cpu().view(T, QH + 2 * KVH, HD)
            qk = ref.rope(x[:, :QH + KVH], cos.cpu()[:T][:, None], sin.cpu()[:T][:, None])
            c, kx, q = (torch.stack([o[3 * layer + i] for o in outs[r]]) for i in range(3))
            tol = half * qk[:, :QH].abs() + 2.0 ** -20 * x.double().abs().amax() + (2.0 ** -24 if dt == HF else 0)
            assert ((q.double() - qk[:, :QH]).abs() <= tol).all()
            pages = cache.k_pages[layer], cache.v_pages[layer]
            o = ref.batch_attention(q, *pages, cache.table[r:r + 1].cpu(), [0], [0, T], [True])
            _near(c, o["c"], o["c_abs"], o, dt, HD, "c")
            _near(kx, o["kctx"], o["kctx_abs"], o, dt, HD, "kctx")


def test_a_captured_step_serves_other_lengths():
    """One graph of reservation, plan and step, replayed as the rows grow, against the eager calls;
    eager work and synchronisations lie between the replays."""
    from loom_amd.paged import PagedKVCache
    g = torch.Generator().manual_seed(22)
    QH, KVH, HD, R = 8, 2, 96, 6
    cos, sin = _tables(HD, 600)
    caches = [PagedKVCache(1, R, 600, KVH, HD, BF, page_size=16, n_pages=200) for _ in range(2)]
    prompt = torch.randn(130, 12 * HD, generator=g).to(DEV, BF)
    for c in caches:
        c.start(torch.tensor([True] + [False] * (R - 1), device=DEV))
        first = _i32([130] + [0] * (R - 1))
        c.reserve(first)
        c.attend_batch(0, c.plan(first, 130, QH), prompt, cos, sin)
        c.advance(first)
        c.update(parent=torch.zeros(R, dtype=torch.int32, device=DEV))
    new, qkv = _i32([1] * R), torch.randn(20, 12 * HD, generator=g).to(DEV, BF)

    def step(c):
        c.reserve(new)
        plan = c.plan(new, 20, QH)
        out = c.attend_batch(0, plan, qkv, cos, sin)
        c.advance(new)
        return [plan.starts, plan.rows, plan.slots, plan.shared] + out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[1])                                   # warm up, on another cache
    torch.cuda.current_stream().wait_stream(side)
    eager, captured = caches[1], caches[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(captured)
    graph.replay()                                        # what the warm-up did on the other one
    torch.cuda.synchronize()
    for i, counts in enumerate([[1] * R, [3, 1, 1, 0, 2, 1], [1, 0, 0, 0, 0, 0], [0] * R, [4, 3, 3, 4, 3, 3], [1, 1, 1, 1, 1, 1]]):
        new.copy_(_i32(counts))
        qkv.copy_(torch.randn(20, 12 * HD, generator=g))
        want = [t.clone() for t in step(eager)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i
        assert torch.equal(captured.table, eager.table) and torch.equal(captured.lens, eager.lens)
    captured.check()


def test_two_steps_at_once_on_two_streams():
    from loom_amd import ops
    g = torch.Generator().manual_seed(23)
    lens, new = [400, 410, 390, 3], [1, 1, 1, 50]
    kp, vp, table = _cache(g, lens, new, [([0, 1, 2], 384)], 30, 2, 16, 96, BF)
    cos, sin = _tables(96, 480)
    N = sum(new)
    qkv = [torch.randn(N, 12 * 96, generator=g).to(DEV, BF) for _ in range(2)]
    plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), N, 8)
    pools = [(kp.clone(), vp.clone()) for _ in range(4)]
    want = [ops.paged_batch_step(plan, x, k, v, table, cos, sin) for x, (k, v) in zip(qkv, pools)]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for x, (k, v), s in zip(qkv, pools[2:], streams):
        with torch.cuda.stream(s):
            p = ops.paged_plan(k, table, _i32(lens), _i32(new), N, 8)
            got.append(ops.paged_batch_step(p, x, k, v, table, cos, sin))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_the_same_call_gives_the_same_bits():
    from loom_amd import ops
    g = torch.Generator().manual_seed(24)
    lens, new = [3000 + 7 * i for i in range(20)], [1] * 20
    kp, vp, table = _cache(g, lens, new, [(range(20), 2992)], 200, 2, 16, 96, BF)
    cos, sin = _tables(96, 3200)
    qkv = torch.randn(20, 12 * 96, generator=g).to(DEV, BF)
    runs = []
    for _ in range(3):
        plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), 20, 8)
        runs.append(ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [BF, FP])
def test_pages_past_2_to_the_32_elements(dt):
    """The same pages at the end of a pool whose elements pass 2^32 bytes and 2^31 elements."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(25)
    lens, new, PS, HD, NP = [2100, 2090, 2048, 0], [1, 9, 1, 30], 1024, 128, 17000
    kp, vp, table = _cache(g, lens, new, [([0, 1, 2], 2048)], 4, 1, PS, HD, dt, spare=1)
    n, N = kp.shape[0], sum(new)
    qkv = torch.randn(N, 6 * HD, generator=g).to(DEV, dt)
    cos, sin = _tables(HD, 4 * PS)
    big = [torch.empty(NP, 1, PS, HD, dtype=dt, device=DEV) for _ in range(2)]
    for b, small in zip(big, (kp, vp)):
        b[NP - n:] = small
    far = torch.where(table >= 0, table + (NP - n), table).to(torch.int32)
    want = ops.paged_batch_step(ops.paged_plan(kp, table, _i32(lens), _i32(new), N, 4), qkv, kp, vp, table, cos, sin)
    plan = ops.paged_plan(big[0], far, _i32(lens), _i32(new), N, 4)
    got = ops.paged_batch_step(plan, qkv, *big, far, cos, sin)
    torch.cuda.synchronize()
    assert not want[0].float().isnan().any()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for b, small in zip(big, (kp, vp)):
        assert torch.equal(_bits(b[NP - n:]), _bits(small))


def test_a_plan_of_the_most_tokens():
    """2^20 flat places, rows of up to half a million new tokens."""
    from loom_amd import ops
    PS, N, lens = 1024, 1 << 20, [5, -1, 70000, 0, 1]
    new = [300000, 9, 0, 500000, N - 800000 - 11]
    MP = 512
    table = torch.arange(5 * MP, dtype=torch.int32).view(5, MP)
    k = torch.empty(5 * MP, 2, PS, 8, dtype=BF, device=DEV)
    plan = ops.paged_plan(k, table.to(DEV), _i32(lens), _i32(new), N, 8)
    n = torch.tensor([m if at >= 0 else 0 for m, at in zip(new, lens)])
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
    rows = torch.repeat_interleave(torch.arange(5), n)
    pos = torch.arange(int(n.sum())) - starts[rows] + torch.tensor(lens)[rows]
    slots = table[rows, pos // PS].long() * PS + pos % PS
    end = torch.full((11,), -1)
    assert plan.starts.tolist() == starts.tolist()
    assert torch.equal(plan.rows.cpu().long(), torch.cat([rows, end]))
    assert torch.equal(plan.positions.cpu().long(), torch.cat([pos, end]))
    assert torch.equal(plan.slots.cpu(), torch.cat([slots, end]))
    assert plan.shared.tolist() == [0] * 5


def test_a_plan_made_before_its_tables_changed_reads_and_writes_in_range():
    """Table entries that are no pages any more: no place outside the pool is touched, and rows
    that the change does not concern come out as before."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(26)
    lens, new = [300, 310, 200, 90], [1, 2, 1, 40]
    for dt, HD in ((BF, 96), (FP, 16)):
        kp, vp, table = _cache(g, lens, new, [([0, 1], 256)], 24, 2, 16, HD, dt)
        cos, sin = _tables(HD, 24 * 16)
        qkv = torch.randn(44, 12 * HD, generator=g).to(DEV, dt)
        plan = ops.paged_plan(kp, table, _i32(lens), _i32(new), 44, 8)
        want = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin)
        k1, v1 = kp.clone(), vp.clone()
        table[2, 3:] = -1
        table[3, 0] = 1 << 30
        got = ops.paged_batch_step(plan, qkv, kp, vp, table, cos, sin)
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a[:3], b[:3])
        assert torch.equal(_bits(kp), _bits(k1)) and torch.equal(_bits(vp), _bits(v1))
