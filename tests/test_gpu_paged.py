"""GPU parity of the paged cache's operators, the beam selection and the row
reordering with plain implementations in 64 bits (oracle.paged)."""
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


def _cache(g, lens, MP, KVH, PS, HD, dt, spare=2, layout="head"):
    """Pools, a table of pages in random order and lens; what no row reads is NaN:
    free pages, and in every page the tokens behind lens."""
    need = [-(-(n + 1) // PS) if n >= 0 else 0 for n in lens]
    NP = sum(need) + spare
    order = torch.randperm(NP, generator=g).tolist()
    shape = (NP, KVH, PS, HD) if layout == "head" else (NP, PS, KVH, HD)
    kp = torch.randn(*shape, generator=g).to(dt)
    vp = torch.randn(*shape, generator=g).to(dt)
    if layout != "head":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    table = torch.full((len(lens), MP), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for s in range(need[b]):
            table[b, s] = order.pop()
        if n >= 0:
            p = int(table[b, n // PS])
            kp[p, :, n % PS:] = math.nan
            vp[p, :, n % PS:] = math.nan
    for p in order:
        kp[p] = math.nan
        vp[p] = math.nan
    if layout == "head":
        return kp.to(DEV), vp.to(DEV), table.to(DEV), _i32(lens)
    return (kp.transpose(1, 2).contiguous().to(DEV).transpose(1, 2),
            vp.transpose(1, 2).contiguous().to(DEV).transpose(1, 2), table.to(DEV), _i32(lens))


def _near(got, want, spread, o, dt, n, HD, what):
    """|got - want| within: the output's rounding; the weights' rounding to a
    16-bit type before the products (half a step of the weights, on the sum of
    absolute values); the fp32 score's error (a product and an addition per
    dimension, HD of them, on sum |q k|, plus its scaling) and that of 2^s (its
    argument's rounding on |s| log2 e and the instruction's), in numerator and
    denominator; and n fp32 additions."""
    half = torch.finfo(dt).eps / 2
    u = 2.0 ** -24
    ds = o["qk_abs"] * (HD + 4) * u + 4 * (o["s_max"] + 1) * u
    rel = (0 if dt == FP else half) + 2 * ds + (n + 64) * u
    bound = half * want.abs() + rel[..., None] * spread + torch.finfo(dt).tiny
    if dt == HF:
        bound = bound + 2.0 ** -24          # half's subnormal step
    over = (got.cpu().double() - want).abs() / bound
    assert float(over.max()) <= 1, f"{what}: {float(over.max())} of the bound"


def _check_step(dt, lens, QH, KVH, HD, PS, MP, seed, layout="head", kctx=True, ld_extra=0):
    from loom_amd import ops
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    kp, vp, table, ln = _cache(g, lens, MP, KVH, PS, HD, dt, layout=layout)
    if ld_extra:                                        # a table that is a view of a wider one
        wide = torch.full((B, MP + ld_extra), 7, dtype=torch.int32, device=DEV)
        wide[:, :MP] = table
        table = wide[:, :MP]
    qkv = torch.randn(B, (QH + 2 * KVH) * HD, generator=g).to(DEV, dt)
    cos, sin = _tables(HD, MP * PS)
    k0, v0 = kp.clone(), vp.clone()
    c, kx, q = ops.paged_decode_step(qkv, kp, vp, table, ln, cos, sin, want_kctx=kctx)
    torch.cuda.synchronize()
    half = torch.finfo(dt).eps / 2
    x = qkv.cpu().view(B, QH + 2 * KVH, HD)
    tab = table.cpu()
    k0, v0 = k0.cpu(), v0.cpu()
    for b, n in enumerate(lens):
        if n < 0:
            assert not q[b].float().any() and not c[b].float().any()
            continue
        co, si = cos[n].cpu(), sin[n].cpu()
        want = ref.rope(x[b, :QH + KVH], co, si)
        size = (x[b, :QH + KVH].double() * co.double()).abs() + torch.cat(
            [t.abs() for t in (x[b, :QH + KVH, HD // 2:], x[b, :QH + KVH, :HD // 2])], -1).double() * si.double().abs()
        bound = half * want.abs() + 2.0 ** -22 * size + torch.finfo(dt).tiny + (2.0 ** -24 if dt == HF else 0)
        page = int(tab[b, n // PS])
        got = torch.cat([q[b].cpu(), kp[page, :, n % PS].cpu()]).double()
        assert ((got - want).abs() <= bound).all(), ("rope", b)
        assert torch.equal(vp[page, :, n % PS].cpu(), x[b, QH + KVH:]), ("v", b)
        k0[page, :, n % PS] = kp[page, :, n % PS].cpu()
        v0[page, :, n % PS] = x[b, QH + KVH:]
    # nothing else of the pools was written
    assert torch.equal(kp.cpu().view(torch.int32 if dt == FP else torch.int16), k0.view(torch.int32 if dt == FP else torch.int16))
    assert torch.equal(vp.cpu().view(torch.int32 if dt == FP else torch.int16), v0.view(torch.int32 if dt == FP else torch.int16))
    o = ref.attention(q, kp, vp, tab, [n + 1 for n in lens])
    n = max(lens) + 1
    _near(c, o["c"], o["c_abs"], o, dt, n, HD, "c")
    if kctx:
        _near(kx, o["kctx"], o["kctx_abs"], o, dt, n, HD, "kctx")
    else:
        assert kx is None
    c2, kx2 = ops.paged_decode_attention(q, kp, vp, table, ln + (ln >= 0).int(), want_kctx=kctx)
    _near(c2, o["c"], o["c_abs"], o, dt, n, HD, "c of the attention alone")
    if kctx:
        _near(kx2, o["kctx"], o["kctx_abs"], o, dt, n, HD, "kctx of the attention alone")


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("lens", [[0], [1, 0, -1, 15], [16, 17, 31, 32, 33], [127, 128, 129, -1], [300, -1, 5, 511]])
def test_step_lengths(dt, lens):
    _check_step(dt, lens, 8, 2, 96, 16, 33, 1)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("QH,KVH", [(1, 1), (3, 1), (5, 5), (8, 2), (16, 2), (16, 1), (24, 1), (32, 8), (6, 2)])
def test_step_heads(dt, QH, KVH):
    _check_step(dt, [70, 3, -1, 200], QH, KVH, 64, 32, 9, 2)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("HD", [8, 16, 32, 64, 96, 128, 256])
@pytest.mark.parametrize("PS", [16, 64, 1024])
def test_step_head_sizes_and_pages(dt, HD, PS):
    _check_step(dt, [150, 0, 333], 8, 2, HD, PS, 1024 // PS, 3)


@pytest.mark.parametrize("dt", [BF, FP])
def test_step_token_major_pages_no_kctx_table_view(dt):
    _check_step(dt, [150, 0, 333, -1, -1], 8, 2, 96, 16, 40, 4, layout="token", kctx=False, ld_extra=3)


@pytest.mark.parametrize("dt", [BF, FP])
def test_step_long_rows_split_and_joined(dt):
    _check_step(dt, [5000, 3, 1, 4097, -1, 900], 8, 2, 96, 64, 79, 5)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("lens", [[5000, 3, -1, 4000, 0, 900, 77], [0, -1, 1, 8191, -1, -1], [511] * 17, [8200]])
def test_step_rows_laid_end_to_end(dt, lens):
    """32 kv heads leave 16 blocks to each: enough tiles per block that the blocks take
    equal stretches of all rows laid end to end (from 256 tiles of 32 tokens)."""
    assert sum(-(-(n + 1) // 32) if n >= 0 else 1 for n in lens) >= 256
    _check_step(dt, lens, 32, 32, 32, 64, 130, 15)
    if dt == BF:
        _check_step(dt, lens, 32, 32, 96, 16, 520, 16, kctx=False)


def test_step_many_rows():
    _check_step(BF, [(37 * i) % 90 - 1 for i in range(1, 301)], 4, 2, 32, 16, 8, 6)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("B", [3, 140])
@pytest.mark.parametrize("cap", [112, 128, 144, 256, 272, 512, 528])
def test_step_around_the_capacities_that_split(dt, B, cap):
    """Whether a row is split, and by how many waves it is done, goes by the capacity
    and the number of rows: both sides of each bound."""
    lens = [cap - 1, 0, cap // 2] + [(29 * i) % cap - 1 for i in range(B - 3)]
    _check_step(dt, lens, 4, 2, 96, 16, cap // 16, 17, kctx=cap % 32 == 0)
    if B == 3:
        for HD in (8, 16, 256):                     # the vector form's steps are 128, 64 and 16 tokens
            _check_step(dt, lens, 2, 2, HD, 16, cap // 16, 18)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("HD", [96, 16])
def test_step_ropes_to_the_exact_values_rounding(dt, HD):
    """The products of a 16-bit and a 32-bit value are exact in 64 bits."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(19)
    lens = [(31 * i) % 96 for i in range(256)]
    kp, vp, table, ln = _cache(g, lens, 6, 2, 16, HD, dt)
    qkv = torch.randn(256, 12 * HD, generator=g).to(DEV, dt)
    cos, sin = _tables(HD, 96)
    q = ops.paged_decode_step(qkv, kp, vp, table, ln, cos, sin)[2]
    x = qkv.view(256, 12, HD)[:, :8].double()
    co, si = cos[ln.long()][:, None].double(), sin[ln.long()][:, None].double()
    turned = torch.cat([-x[..., HD // 2:], x[..., :HD // 2]], -1)
    assert torch.equal(q, (x * co + turned * si).float().to(dt))


def test_step_equals_dense_step():
    """Rows of one length: loom_gqa_decode_step over the dense cache with the same rows."""
    from loom_amd import _lib, ops
    lib = _lib.load()
    g = torch.Generator().manual_seed(7)
    B, QH, KVH, HD, PS, n = 4, 8, 2, 96, 16, 777
    MP = 50
    kp, vp, table, ln = _cache(g, [n] * B, MP, KVH, PS, HD, BF)
    qkv = torch.randn(B, (QH + 2 * KVH) * HD, generator=g).to(DEV, BF)
    cos, sin = _tables(HD, MP * PS)
    at = table.clamp(min=0).long()
    # (zeros where the pools hold NaN: the dense kernel multiplies rows it masks by a weight of 0)
    kc = kp[at].transpose(1, 2).reshape(B, KVH, MP * PS, HD).nan_to_num(0).contiguous()
    vc = vp[at].transpose(1, 2).reshape(B, KVH, MP * PS, HD).nan_to_num(0).contiguous()
    q, c, kx = (torch.empty(B, QH, HD, dtype=BF, device=DEV) for _ in range(3))
    nb = lib.loom_gqa_workspace_bytes(B, n + 1, QH, KVH, HD)
    ws = torch.empty(nb // 4 + 64, device=DEV)
    P = _lib.ptr
    _lib.call("loom_gqa_decode_step", 1, P(qkv), P(kc), P(vc), KVH * MP * PS * HD, HD, MP * PS * HD, P(cos), P(sin),
              P(q), P(c), P(kx), QH * HD, P(ws), nb, B, n + 1, None, QH, KVH, HD, _lib.stream_of(qkv))
    c2, kx2, q2 = ops.paged_decode_step(qkv, kp, vp, table, ln, cos, sin)
    assert torch.equal(q, q2)
    # both round the weights and the outputs to bf16: two halves of a step each
    for a, b, src in ((c, c2, vc), (kx, kx2, kc)):
        most = src[:, :, :n].float().abs().amax(2).repeat_interleave(QH // KVH, 1)
        assert ((a.float() - b.float()).abs() <= 4 * 2.0 ** -8 * most).all()


@pytest.mark.parametrize("dt", [BF, FP])
def test_step_broken_rows_give_nan_and_write_nothing(dt):
    """A missing page, a page id that is none, a position past the table or past
    the rotary tables: NaN for that row, the others as without it."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(8)
    QH, KVH, HD, PS, MP = 8, 2, 96, 16, 20
    lens = [100, 40, 200, 319, 17]
    kp, vp, table, ln = _cache(g, lens, MP, KVH, PS, HD, dt)
    qkv = torch.randn(5, (QH + 2 * KVH) * HD, generator=g).to(DEV, dt)
    cos, sin = _tables(HD, MP * PS)
    good = [t.clone() for t in ops.paged_decode_step(qkv, kp.clone(), vp.clone(), table, ln, cos, sin)]
    for what in ("hole", "high", "past", "tables", "last"):
        t2, l2, co, si = table.clone(), ln.clone(), cos, sin
        bad = [1]
        if what == "hole":
            t2[1, 1] = -1
        elif what == "high":
            t2[1, 0] = kp.shape[0]
        elif what == "past":
            l2[1] = MP * PS
        elif what == "last":
            t2[1, 2] = -5
        else:
            co, si = cos[:300], sin[:300]
            bad = [3]
        k2, v2 = kp.clone(), vp.clone()
        got = ops.paged_decode_step(qkv, k2, v2, t2, l2, co, si)
        for r in range(5):
            for a, b in zip(got[:2], good[:2]):
                if r in bad:
                    assert torch.isnan(a[r].float()).all(), (what, r)
                else:
                    assert torch.equal(a[r], b[r]), (what, r)
        # pages that no good row appends to are as they were (a hole's row still appends to its own last page)
        own = set(int(table[r, lens[r] // PS]) for r in range(5) if r not in bad or what in ("hole", "high"))
        rest = [p for p in range(kp.shape[0]) if p not in own]
        bits = torch.int32 if dt == FP else torch.int16
        assert torch.equal(k2[rest].view(bits), kp[rest].view(bits)), what
        assert torch.equal(v2[rest].view(bits), vp[rest].view(bits)), what


def test_attention_of_nothing_is_zero_and_values_that_are_not_finite_stay():
    from loom_amd import ops
    g = torch.Generator().manual_seed(9)
    for dt, HD in ((BF, 64), (FP, 64), (HF, 8)):
        kp, vp, table, _ = _cache(g, [40, 40, 40, 40], 4, 2, 16, HD, dt)
        q = torch.randn(4, 4, HD, generator=g).to(DEV, dt)
        c, kx = ops.paged_decode_attention(q, kp, vp, table, _i32([0, -1, -7, 33]))
        assert not c[:3].float().any() and not kx[:3].float().any()
        assert torch.isfinite(c[3].float()).all()
        vp[int(table[3, 1]), :, 3] = math.inf
        kp[int(table[2, 0]), :, 5] = math.nan
        c, kx = ops.paged_decode_attention(q, kp, vp, table, _i32([33, 33, 33, 33]))
        assert torch.isfinite(c[:2].float()).all()
        assert torch.isnan(c[2].float()).all() and torch.isnan(kx[2].float()).all()
        assert (c[3].float() == math.inf).all() and torch.isfinite(kx[3].float()).all()
        kp[int(table[1, 2])] = math.nan                 # all of a row's last page: behind 32 tokens, not read
        c2, _ = ops.paged_decode_attention(q, kp, vp, table, _i32([33, 32, 33, 33]))
        assert torch.isfinite(c2[1].float()).all()


# ------------------------------------------------------------------ pages

def _state(g, L, R, MP, KVH, PS, HD, dt, lens, NP, share):
    """Rows that share the pages of row 0's first `share` slots where they hold them."""
    order = torch.randperm(NP, generator=g).tolist()
    table = torch.full((R, MP), -1, dtype=torch.int32)
    refs = torch.zeros(NP, dtype=torch.int32)
    common = [order.pop() for _ in range(share)]
    for r in range(R):
        for s in range(-(-max(lens[r], 0) // PS)):
            p = common[s] if s < share else order.pop()
            table[r, s] = p
            refs[p] += 1
    kp, vp = (torch.randn(L, NP, KVH, PS, HD, generator=g).to(dt) for _ in range(2))
    return [t.to(DEV) for t in (kp, vp, table, _i32(lens), refs)]


def _compare_update(s, **kw):
    from loom_amd import ops
    status = _i32([5])
    cpu = [t.cpu() for t in s]
    par = kw.get("parent")
    want = ref.update(*cpu, **dict(kw, parent=None if par is None else par.cpu()))
    ops.paged_update(*s, status, **kw)
    for name, a, b in zip(("k", "v", "table", "lens", "refs"), s, want):
        assert torch.equal(a.cpu(), b), (name, kw)
    assert int(status) == 5 + want[5]
    t = s[2].cpu()
    assert torch.equal(torch.bincount(t[t >= 0].long(), minlength=s[4].numel()).int(), s[4].cpu())
    return want[5]


@pytest.mark.parametrize("seed", range(6))
def test_update_random_walk(seed):
    """Forks, advances, reservations, freed and restarted rows in a row, each against the oracle."""
    g = torch.Generator().manual_seed(seed)
    R, MP, PS, NP = 7, 9, 16, 7 * 9
    dt = [BF, FP, HF][seed % 3]
    s = _state(g, 2, R, MP, 2, PS, 32, dt, [40, 40, 33, 16, -1, 0, 48], NP, 2)
    _compare_update(s, n_new=1)
    for step in range(12):
        par = torch.randint(-1, R + 1, (R,), generator=g).int()
        keep = torch.rand(R, generator=g) < 0.4
        par[keep] = torch.arange(R).int()[keep]
        kw = dict(n_new=int(torch.randint(0, 20, (1,), generator=g)), advance=0)
        if step % 3:
            kw["parent"] = par.to(DEV)
        if step % 2:
            kw["advance"] = 1
        _compare_update(s, **kw)
        if step % 4 == 3:                               # idle rows start again
            s[3][s[3] < 0] = 0


def test_update_beam_step_keeps_the_written_token():
    """lens tokens, one written since at a page's first place: fork with advance = 1 passes its page on."""
    g = torch.Generator().manual_seed(3)
    s = _state(g, 1, 4, 6, 2, 16, 32, BF, [32] * 4, 30, 1)
    _compare_update(s, n_new=1)
    written = [s[0][0, int(p), :, 0].clone() for p in s[2][:, 2]]
    _compare_update(s, parent=_i32([1, 1, 0, 1]), advance=1, n_new=1)
    assert s[3].tolist() == [33] * 4
    for r, p in enumerate([1, 1, 0, 1]):
        assert torch.equal(s[0][0, int(s[2][r, 2]), :, 0], written[p]), r
    assert len(set(s[2][:, 2].tolist())) == 4           # a page of its own for each row


def test_update_out_of_pages_and_past_the_table():
    g = torch.Generator().manual_seed(4)
    # 4 rows share a partly filled page; two free pages: the third copy finds none
    s = _state(g, 1, 4, 2, 2, 16, 32, BF, [20] * 4, 4, 2)
    assert _compare_update(s, n_new=1) == 1
    assert (s[2][:, 1] < 0).sum() == 1
    s = _state(g, 1, 3, 3, 2, 16, 32, BF, [47, 48, 20], 9, 0)
    assert _compare_update(s, n_new=5) == 2             # 47 has one place left, 48 none
    s = _state(g, 1, 3, 8, 2, 16, 32, BF, [0, 0, 0], 5, 0)
    assert _compare_update(s, n_new=60) == 7            # 12 pages wanted, 5 there


def test_update_large_pool_and_many_rows():
    """More pages than one scan round holds (16384), the free ones behind and among
    them; 1024 rows that all copy."""
    g = torch.Generator().manual_seed(5)
    NP, R = 40000, 1024
    s = _state(g, 1, R, 3, 1, 16, 8, FP, [20] * R, NP, 2)
    refs = s[4]
    # every page below 38000 that is free gets a holder outside the table
    blocked = (torch.arange(NP, device=DEV) < 38000) & (refs == 0) & (torch.arange(NP, device=DEV) % 1000 != 7)
    refs[blocked] = 1
    cpu = [t.cpu() for t in s]
    from loom_amd import ops
    status = _i32([0])
    ops.paged_update(*s, status, n_new=1)
    want = ref.update(*cpu, n_new=1)
    for a, b in zip(s, want):
        assert torch.equal(a.cpu(), b)
    assert int(status) == 0


@pytest.mark.parametrize("seed", range(4))
def test_compact(seed):
    from loom_amd import ops
    g = torch.Generator().manual_seed(seed)
    NP = [1, 50, 5000, 300][seed]
    if seed == 0:
        s = _state(g, 2, 1, 1, 2, 16, 32, BF, [5], 1, 0)
    else:
        s = _state(g, 2, 6, 9, 2, 16, 32, [BF, HF, FP, BF][seed], [100, -1, 17, 140, 0, 100], NP, 3)
    used = _i32([-1])
    want = ref.compact(*[s[i].cpu() for i in (0, 1, 2, 4)])
    for _ in range(2):                                   # the second call has nothing to move
        ops.paged_compact(s[0], s[1], s[2], s[4], used)
        for a, b in zip([s[i] for i in (0, 1, 2, 4)], want):
            assert torch.equal(a.cpu(), b)
        assert int(used) == want[4]


@pytest.mark.parametrize("dt", [BF, FP])
def test_write_dense_rows(dt):
    from loom_amd import ops
    g = torch.Generator().manual_seed(6)
    L, R, KVH, PS, HD, T = 2, 4, 2, 16, 96, 150
    s = _state(g, L, R, 10, KVH, PS, HD, dt, [150, 150, 40, -1], 40, 0)
    dense = [torch.randn(L, R, KVH, T, HD, generator=g).to(DEV, dt) for _ in range(2)]
    first, last = [0, 37, 5, 0], [150, 90, 150, 150]    # rows 2, 3: pages for 48 and no tokens
    want = [s[0].clone(), s[1].clone()]
    for r in range(R):
        for t in range(first[r], last[r]):
            p = int(s[2][r, t // PS])
            if p >= 0:
                for w, d in zip(want, dense):
                    w[:, p, :, t % PS] = d[:, r, :, t]
    ops.paged_write(s[0], s[1], s[2], dense[0], dense[1], _i32(first), _i32(last))
    assert torch.equal(s[0], want[0]) and torch.equal(s[1], want[1])


# ------------------------------------------------------------------ selection, reordering

def _check_select(x, sc, K, finished=None, eos=-1, pad=0):
    from loom_amd import ops
    ws, wp, wt, wf = ref.beam_select(x, sc, K, finished, eos, pad)
    s, p, t, f = ops.beam_select(x, sc, K, finished=finished, eos_id=eos, pad_id=pad)
    assert torch.equal(p.cpu(), wp) and torch.equal(t.cpu(), wt) and torch.equal(f.cpu(), wf)
    s = s.cpu().double()
    fin = torch.isfinite(ws)
    assert torch.equal(torch.isfinite(s), fin) and torch.equal(s[~fin], ws[~fin])
    # a value's rounding to fp32; the exponential sum: 32 fp32 additions and the
    # exponentials' own (two units), and their arguments' rounding on sum p |x - max|
    xd = x.cpu().double()
    pr = torch.softmax(xd, 1)
    far = torch.nan_to_num(pr * (xd - xd.amax(1, keepdim=True)).abs(), 0, 0, 0).sum(1)
    tol = 2.0 ** -24 * ws.abs() + 40 * 2.0 ** -24 + 2.0 ** -22 * torch.nan_to_num(far, 0, 0, 0).max()
    assert ((s - ws).abs()[fin] <= tol[fin]).all()


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("S,W,V,K", [(1, 1, 1, 1), (1, 4, 4096, 4), (3, 5, 777, 10), (2, 8, 8193, 16), (1, 32, 501, 64),
                                     (2, 3, 20000, 3), (1, 1, 70, 64), (1, 2, 9, 18),
                                     # one block per group: its largest sizes, and one more
                                     (2, 1, 32768, 32), (2, 1, 32769, 32), (1, 16, 2048, 32), (1, 9, 2047, 7), (1, 16, 2049, 5),
                                     (2, 2, 16383, 31), (1, 17, 300, 4), (1, 5, 4095, 33)])
def test_select(dt, S, W, V, K):
    g = torch.Generator().manual_seed(V + K)
    x = (torch.randn(S * W, V, generator=g) * 3).to(DEV, dt)
    sc = (-20 - 5 * torch.rand(S, W, generator=g)).to(DEV)
    _check_select(x, sc, K)


def test_select_many_rows_steps_through_long_slices():
    g = torch.Generator().manual_seed(11)
    x = (torch.randn(1536, 30011, generator=g)).to(DEV, BF)
    sc = (-5 * torch.rand(512, 3, generator=g)).to(DEV)
    from loom_amd import ops
    s, p, t, f = ops.beam_select(x, sc, 5)
    v = torch.log_softmax(x.double(), 1) + sc.view(-1, 1).double()
    best, at = torch.sort(v.view(512, -1), dim=1, descending=True, stable=True)
    rows = torch.arange(512, device=DEV)[:, None] * 3 + at[:, :5] // 30011
    assert torch.equal(p, rows.int()) and torch.equal(t, at[:, :5] % 30011)
    assert ((s.double() - best[:, :5]).abs() <= 2e-5).all()


@pytest.mark.parametrize("kind", ["ascending", "descending", "constant", "steps", "blocks"])
@pytest.mark.parametrize("V", [24001, 24000, 8185])
def test_select_ties_and_orders(kind, V):
    """Logits whose largest values lie together, rise towards the end or are all
    the same; ties inside a row and between rows go to the lowest (beam, token)."""
    W = 4
    i = torch.arange(V, dtype=torch.float64)
    x = {"ascending": i / 1000, "descending": -i / 1000, "constant": 0 * i, "steps": (i // 300) / 8,
         "blocks": torch.where((i >= 7000) & (i < 7128), 5.0, 0.0)}[kind]
    x = x.float().expand(512, V).contiguous().to(DEV)   # 512 rows: several steps per slice
    sc = torch.zeros(128, W, device=DEV)
    from loom_amd import ops
    s, p, t, f = ops.beam_select(x, sc, 8)
    order = torch.sort(x[0].cpu(), descending=True, stable=True)
    v, n = order.values[0], int((order.values == order.values[0]).sum())
    want = []                                            # (beam, token): rows are equal, so ties run through the beams
    for k in range(8):
        want.append((k // n, int(order.indices[k % n])) if n < 8 and k < n * W else (0, int(order.indices[k])) if n >= 8 else None)
    for k, w in enumerate(want):
        if w is None:
            continue
        assert (p[:, k].cpu() == torch.arange(128) * W + w[0]).all(), (kind, k)
        assert (t[:, k].cpu() == w[1]).all(), (kind, k)


def test_select_finished_dead_and_ruled_out():
    g = torch.Generator().manual_seed(12)
    for dt, V in ((BF, 3000), (FP, 3000), (BF, 30000)):
        S, W = 7, 4
        x = (torch.randn(S * W, V, generator=g) * 2).to(DEV, dt)
        sc = (-2 * torch.rand(S, W, generator=g)).to(DEV)
        fin = torch.zeros(S * W, dtype=torch.bool, device=DEV)
        fin[[0, 5, 6, 12, 13, 14, 15]] = True            # group 3: all at their end
        sc[1, 2:] = -math.inf                             # dead beams
        sc[2] = torch.tensor([0, -math.inf, -math.inf, -math.inf])
        sc[4, 1] = math.nan
        sc[4, 2] = math.inf
        x[16, 5] = math.nan                               # group 4: nothing but beam 3
        x[20] = -math.inf                                 # group 5: a row without a token
        x[21, 7:] = -math.inf
        x[22, 100] = math.inf
        x[23, :] = -math.inf
        x[23, [9, 2500]] = 1.0
        sc[6] = -math.inf                                 # group 6: no candidate at all
        _check_select(x, sc, 8, fin, eos=7, pad=3)
        _check_select(x, sc, 8, None, eos=-1, pad=0)


def test_select_views_and_alignment():
    g = torch.Generator().manual_seed(13)
    wide = (torch.randn(12, 1500, generator=g) * 3).to(DEV, BF)
    sc = (-5 * torch.rand(3, 4, generator=g)).to(DEV)
    for a in (0, 1, 3, 8):
        _check_select(wide[:, a:a + 1111], sc, 4)
        _check_select(wide[:, a:a + 7], sc, 4)
    _check_select(wide.t().contiguous().t(), sc, 4)
    _check_select(wide, sc.t().contiguous().t(), 4)


@pytest.mark.parametrize("R", [1, 2, 5, 16, 33, 130, 256, 300, 1024])
def test_reorder_rows(R):
    from loom_amd import ops
    g = torch.Generator().manual_seed(R)
    ts = [torch.randn(3, R, 40, generator=g).to(DEV, BF), torch.randn(R, 13, 3, 3, generator=g).to(DEV, BF),
          torch.randint(0, 255, (R, 19), generator=g, dtype=torch.uint8).to(DEV),
          torch.randint(0, 9, (R, 70), generator=g).to(DEV), torch.randn(R, generator=g).to(DEV),
          torch.randn(R, 515, generator=g).to(DEV, HF)[:, 1:], torch.randn(R, 0, generator=g).to(DEV),
          torch.randn(2, 3, R, 64, generator=g).to(DEV), torch.randint(0, 2, (R,), generator=g).bool().to(DEV)]
    dims = [1, 0, 0, 0, 0, 0, 0, 2, 0]
    for par in (torch.randint(0, R, (R,), generator=g), torch.randperm(R, generator=g), torch.arange(R),
                torch.randint(-2, R + 2, (R,), generator=g)):
        want = [ref.reorder_rows(t, par, d).clone() for t, d in zip(ts, dims)]
        ops.reorder_rows(ts, par.int().to(DEV), dims)
        for k, (a, b) in enumerate(zip(ts, want)):
            assert torch.equal(a, b), k


def test_reorder_more_than_sixteen_tensors():
    from loom_amd import ops
    ts = [torch.arange(5, device=DEV) * 10 + k for k in range(35)]
    want = [t[[4, 0, 0, 3, 1]].clone() for t in ts]
    ops.reorder_rows(ts, _i32([4, 0, 0, 3, 1]))
    assert all(torch.equal(a, b) for a, b in zip(ts, want))


def test_empty_calls_and_refusals():
    from loom_amd import ops
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)  # noqa: E731
    kp, vp, pool = z(10, 2, 16, 96), z(10, 2, 16, 96), z(2, 10, 2, 16, 96)
    co = z(80, 96, dt=FP)
    c, kx, q = ops.paged_decode_step(z(0, 1152), kp, vp, i(0, 5), i(0), co, co)
    assert c.shape == kx.shape == q.shape == (0, 8, 96)
    ops.paged_update(pool, pool, i(0, 5), i(0), i(10), i(1), n_new=1)
    ops.reorder_rows([], i(4))
    ops.reorder_rows([z(0, 3)], i(0))
    step = lambda **k: ops.paged_decode_step(*{**dict(q=z(3, 1152), k=kp, v=vp, t=i(3, 5), n=i(3), c=co, s=co), **k}.values())  # noqa: E731
    upd = lambda **k: ops.paged_update(*{**dict(k=pool, v=pool, t=i(3, 5), n=i(3), r=i(10), s=i(1)), **k}.values())  # noqa: E731
    x, sc = z(8, 100), z(2, 4, dt=FP)
    bad = [(lambda: step(q=z(3, 1150)), "qkv must be"), (lambda: step(q=z(3, 1152, dt=FP)), "dtype"), (lambda: step(q=z(4, 1152)), "rows of"),
           (lambda: step(q=z(3, 384)), "qkv must be"), (lambda: step(q=z(3, 1248)), "9 query heads"),
           (lambda: step(k=z(10, 2, 16, 96, dt=HF)), "one dtype"), (lambda: step(v=z(9, 2, 16, 96)), "same layout"),
           (lambda: step(v=z(10, 16, 2, 96).transpose(1, 2)), "same layout"), (lambda: step(k=pool, v=pool), "pages, kv_heads"),
           (lambda: step(t=i(3, 5).long()), "table must be"), (lambda: step(n=i(4)), "lens must be"), (lambda: step(n=i(3).long()), "lens must be"),
           (lambda: step(c=z(80, 96)), "cos and sin"), (lambda: step(s=z(81, 96, dt=FP)), "cos and sin"), (lambda: step(t=i(3, 5).t()), "table must be"),
           (lambda: step(q=z(3, 80 * 12), k=z(10, 2, 16, 80), v=z(10, 2, 16, 80), c=z(80, 80, dt=FP), s=z(80, 80, dt=FP)), "head_dim 80"),
           (lambda: step(k=z(10, 2, 24, 96), v=z(10, 2, 24, 96)), "power of two"), (lambda: step(q=torch.zeros(3, 1152)), "CUDA"),
           (lambda: step(t=i(1, 5).expand(3, 5)), "row stride 0"),
           (lambda: upd(k=kp, v=kp), "layers, pages"), (lambda: upd(r=i(9)), "refs must be"), (lambda: upd(s=i(2)), "status must be"),
           (lambda: ops.paged_update(pool, pool, i(3, 5), i(3), i(10), i(1), parent=i(2)), "parent must be"),
           (lambda: ops.paged_update(pool, pool, i(3, 5), i(3), i(10), i(1), n_new=81), "n_new=81"),
           (lambda: ops.paged_write(pool, pool, i(3, 5), z(2, 3, 2, 40, 64), z(2, 3, 2, 40, 64), i(3), i(3)), "k_rows and v_rows"),
           (lambda: ops.paged_compact(pool, pool, i(3, 5), i(10), i(2)), "used must be"),
           (lambda: ops.beam_select(x, sc.double()), "float32"), (lambda: ops.beam_select(x, sc[:1]), "each row"), (lambda: ops.beam_select(x, sc, 0), "n_out"),
           (lambda: ops.beam_select(x, sc, 65), "n_out"), (lambda: ops.beam_select(x, sc, finished=z(8)), "bool"), (lambda: ops.beam_select(x.long(), sc), "logits must be"),
           (lambda: ops.beam_select(x, sc, pad_id=100), "pad_id"), (lambda: ops.beam_select(z(33, 50), z(1, 33, dt=FP)), "beams"),
           (lambda: ops.beam_select(z(0, 50), z(0, 4, dt=FP)), "a group"),
           (lambda: ops.reorder_rows([x], i(7)), "7 rows"), (lambda: ops.reorder_rows([x.t()], i(100)), "dense"),
           (lambda: ops.reorder_rows([x, x], i(8)), "twice"), (lambda: ops.reorder_rows([x], i(8), [0, 1]), "one dimension"),
           (lambda: ops.reorder_rows([x[:1].expand(8, 100)], i(8)), "overlap"), (lambda: ops.reorder_rows([x], i(8).long()), "int32"),
           (lambda: ops.reorder_rows([z(1100, 4)], i(1100)), "0 to 1024 rows"), (lambda: ops.reorder_rows([5], i(8)), "tensors")]
    p = i(8)
    bad.append((lambda: ops.reorder_rows([p], p), "parent must not"))
    for n, (f, msg) in enumerate(bad):
        with pytest.raises(RuntimeError, match=msg):
            f()
            print("not refused:", n, msg)
    with pytest.raises(TypeError):
        ops.paged_update(pool, pool, i(3, 5), i(3), i(10), i(1), n_new=1.5)
    with pytest.raises(TypeError):
        ops.reorder_rows(7, i(8))


# ------------------------------------------------------------------ together

class _Loop:
    """A few beam steps of one layer with stand-in logits: select, reorder, update, step."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.S, self.W, self.PS, self.MP, V = 2, 3, 16, 6, 500
        R = 6
        r = lambda *s, dt=BF: torch.randn(*s, generator=g).to(DEV, dt)  # noqa: E731
        self.kp, self.vp = r(1, 36, 2, 16, 96), r(1, 36, 2, 16, 96)
        self.table = torch.full((R, self.MP), -1, dtype=torch.int32, device=DEV)
        self.lens, self.refs, self.status = _i32([-1] * R), _i32([0] * 36), _i32([0])
        self.lens[0] = self.lens[3] = 0
        self.emb, self.w = r(V, 12 * 96), r(8 * 96, V, dt=FP) * 0.2
        self.scores = torch.full((2, 3), -math.inf, device=DEV)
        self.scores[:, 0] = 0
        self.fin = torch.zeros(R, dtype=torch.bool, device=DEV)
        self.ids = torch.zeros(R, 40, dtype=torch.int64, device=DEV)
        self.n = torch.zeros(1, dtype=torch.int64, device=DEV)
        self.logits = r(R, V, dt=FP)
        self.cos, self.sin = _tables(96, 96)

    def step(self):
        from loom_amd import ops
        s, par, tok, fin = ops.beam_select(self.logits, self.scores, finished=self.fin, eos_id=3, pad_id=1)
        self.scores.copy_(s)
        self.fin.copy_(fin.view(-1))
        ops.reorder_rows([self.ids], par.view(-1))
        self.ids.scatter_(1, self.n.expand(6, 1), tok.view(-1, 1))
        ops.paged_update(self.kp, self.vp, self.table, self.lens, self.refs, self.status, parent=par.view(-1),
                         n_new=1, advance=0)
        qkv = self.emb[tok.view(-1)]
        c, kx, q = ops.paged_decode_step(qkv, self.kp[0], self.vp[0], self.table, self.lens, self.cos, self.sin)
        self.lens.add_((self.lens >= 0).int())
        self.logits.copy_((c.float() + kx.float()).view(6, -1) @ self.w)
        self.n.add_(1)

    def state(self):
        return [t.clone() for t in (self.scores, self.fin, self.ids, self.table, self.lens, self.refs, self.status, self.logits)]


def _same(a, b):
    return all(torch.equal(x.nan_to_num(7), y.nan_to_num(7)) if x.is_floating_point() else torch.equal(x, y) for x, y in zip(a, b))


def test_loop_keeps_each_beams_own_history():
    """After every step each beam's pages hold the rows of exactly its own tokens."""
    a = _Loop(1)
    half = a.emb.view(500, 12, 96)
    for n in range(1, 30):
        a.step()
        for r in range(6):
            assert int(a.lens[r]) == n
            got = ref.rows_of(a.vp[0].cpu(), a.table[r].tolist(), n)
            want = half[a.ids[r, :n], 10:].cpu().double().transpose(0, 1)
            assert torch.equal(got, want), (n, r)
    assert int(a.status) == 0
    assert int(a.refs.sum()) == int((a.table >= 0).sum())


def test_loop_captured_and_replayed_beside_another_graph():
    """Two loops captured into graphs and replayed in turn, with eager work and
    synchronizations between, equal two eager loops after every step."""
    eager, loops, graphs = [_Loop(2), _Loop(3)], [_Loop(2), _Loop(3)], []
    for lp in loops:
        lp.step()                                        # warm up: also the first step
    for lp in loops:
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            lp.step()
        graphs.append(gr)
    for e in eager:
        e.step()
    for n in range(12):
        for e, lp, gr in zip(eager, loops, graphs):
            e.step()
            gr.replay()
            assert _same(e.state(), lp.state()), n
        torch.cuda.synchronize()
        torch.randn(1000, device=DEV).sum().item()


def test_loop_on_another_stream():
    a, b = _Loop(4), _Loop(4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        a.step()
    with torch.cuda.stream(st):
        for _ in range(5):
            b.step()
    torch.cuda.current_stream().wait_stream(st)
    assert _same(a.state(), b.state())


def test_step_offsets_past_32_bits():
    """Pools of more than 2^32 bytes: pages whose element offsets pass 31 and 32 bits."""
    from loom_amd import ops
    KVH, PS, HD = 8, 64, 128
    NP = (1 << 32) // (KVH * PS * HD) + 200
    kp = torch.zeros(NP, KVH, PS, HD, dtype=BF, device=DEV)
    vp = torch.zeros_like(kp)
    g = torch.Generator().manual_seed(5)
    high, low = [NP - 1, NP - 7, NP // 2 + 3, 40], [0, 1, 2, 3]
    for a, b in zip(high, low):
        kp[a] = torch.randn(KVH, PS, HD, generator=g).to(DEV, BF)
        vp[a] = torch.randn(KVH, PS, HD, generator=g).to(DEV, BF)
        kp[b], vp[b] = kp[a], vp[a]
    qkv = torch.randn(1, 48 * HD, generator=g).to(DEV, BF).expand(2, -1)
    cos, sin = _tables(HD, 256)
    c, kx, q = ops.paged_decode_step(qkv, kp, vp, _i32([high, low]), _i32([230, 230]), cos, sin)
    assert torch.equal(c[0], c[1]) and torch.equal(kx[0], kx[1]) and torch.isfinite(c.float()).all()
    assert torch.equal(kp[40], kp[3]) and torch.equal(vp[40], vp[3])
