"""Edges of the paged cache's operators, the beam selection and the row reordering:
values, sizes and layouts at which they could go wrong, against plain
implementations in 64 bits (oracle.paged)."""
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


# ------------------------------------------------------------------ selection

def _mixed_zeros(n, seed):
    """Zeros of both signs in random order, the first one negative."""
    z = torch.zeros(n)
    z[torch.rand(n, generator=torch.Generator().manual_seed(seed)) < 0.5] = -0.0
    z[0] = -0.0
    z[-1] = 0.0
    return z


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("S,W,V,K", [(1, 1, 2, 1), (1, 1, 2, 2), (1, 1, 9, 3), (2, 4, 700, 4), (1, 4, 8192, 8), (1, 16, 2048, 32),
                                     (1, 1, 40000, 1), (1, 3, 20011, 64)])
def test_select_zeros_of_both_signs_are_one_value(dt, S, W, V, K):
    """A row of nothing but zeros, zeros as the largest values, and zeros on the last
    place that is chosen: -0.0 and +0.0 tie, the lowest place goes first."""
    from loom_amd import ops
    zero = torch.stack([_mixed_zeros(V, 7 * r + V) for r in range(S * W)])
    below = torch.where(torch.rand(S * W, V, generator=torch.Generator().manual_seed(K)) < 0.9, -2.0, zero)
    some = below.clone()
    some[:, V // 2:V // 2 + (K + 1) // 2] = 1.5
    apart = -torch.arange(S * W, device=DEV).float().view(S, W) / 8
    for x, sc in ((zero, torch.zeros_like(apart)), (zero, apart), (below, apart), (some, apart)):
        x = x.to(DEV, dt)
        s, p, t, f = ops.beam_select(x, sc, K)
        ws, wp, wt, _ = ref.beam_select(x, sc, K)
        assert torch.equal(p.cpu(), wp) and torch.equal(t.cpu(), wt)
        # the value's rounding, and the sum of V exponentials of arguments of at most
        # 3.5: 32 additions and the exponentials' own two units
        tol = 2.0 ** -24 * ws.abs() + 40 * 2.0 ** -24 + 2.0 ** -22 * 3.5
        assert ((s.cpu().double() - ws).abs() <= tol).all()


@pytest.mark.parametrize("dt", [BF, FP])
def test_select_zeros_of_both_signs_over_many_steps(dt):
    """512 rows: a slice takes several steps, whose bounds are zeros."""
    from loom_amd import ops
    V, K = 30011, 6
    g = torch.Generator().manual_seed(3)
    x = torch.where(torch.rand(512, V, generator=g) < 0.5, 0.0, -0.0)
    x[torch.rand(512, V, generator=g) < 0.3] = -1.0
    x = x.to(DEV, dt)
    sc = torch.zeros(128, 4, device=DEV)
    sc[:, 1:] = -3.0                                  # only the first beam's tokens are chosen
    s, p, t, f = ops.beam_select(x, sc, K)
    want = torch.sort(x[::4].cpu().double() + 0.0, dim=1, descending=True, stable=True)     # (-0.0 + 0.0 is +0.0)
    assert torch.equal(t.cpu(), want.indices[:, :K])
    assert torch.equal(p, (4 * torch.arange(128, device=DEV)).int()[:, None].expand(128, K))


@pytest.mark.parametrize("dt,snan", [(BF, 0x7F81), (HF, 0x7D01), (FP, 0x7F800001)])
@pytest.mark.parametrize("V,K", [(16000, 1), (8192, 4), (30000, 1), (100000, 3)])
def test_select_rows_with_signalling_nans(dt, snan, V, K):
    """A NaN that is not quiet, with larger logits before it and a tie behind it in
    every eight: the row has no candidate, and the rows beside it keep theirs."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(V)
    W = 2 if V <= 16384 else 3
    x = (torch.randn(2 * W, V, generator=g) * 3).to(DEV, dt)
    bits = torch.int32 if dt == FP else torch.int16
    for row in (0, W + 1):                           # the first of a group, and one in the middle or at the end
        x[row] = 5.0
        x[row, :V // 8 * 8].view(-1, 8)[:, :5] = 7.0
        x[row, :V // 8 * 8].view(-1, 8)[:, 5].copy_(torch.tensor(snan, dtype=bits, device=DEV).view(dt))
    assert int(torch.isnan(x[0].float()).sum()) == V // 8
    sc = torch.zeros(2, W, device=DEV)
    s, p, t, f = ops.beam_select(x, sc, K)
    dead = sc.clone()
    dead[0, 0] = dead[1, 1] = -math.inf
    y = torch.where(torch.isnan(x.float()), 0.0, x.float()).to(dt)
    s2, p2, t2, f2 = ops.beam_select(y, dead, K)     # the same with those rows ruled out
    ws, wp, wt, _ = ref.beam_select(y, dead, K)
    assert torch.equal(p.cpu(), wp) and torch.equal(t.cpu(), wt)
    assert torch.equal(s, s2) and torch.equal(p, p2) and torch.equal(t, t2)


@pytest.mark.parametrize("kind", ["ascending", "descending", "constant", "steps", "blocks"])
@pytest.mark.parametrize("V,K", [(24001, 8), (24000, 9), (8185, 16), (4096, 8)])
def test_select_every_place_of_ties_and_orders(kind, V, K):
    """Equal rows of one group: the K places are the first of all candidates by (value,
    beam, token), scores too."""
    from loom_amd import ops
    W, S = 4, 128
    i = torch.arange(V, dtype=torch.float64)
    x = {"ascending": i / 1000, "descending": -i / 1000, "constant": 0 * i, "steps": (i // 300) / 8,
         "blocks": torch.where((i >= 3000) & (i < 3003), 5.0, 0.0)}[kind].float()
    s, p, t, f = ops.beam_select(x.expand(S * W, V).contiguous().to(DEV), torch.zeros(S, W, device=DEV), K)
    top = torch.sort(x, descending=True, stable=True)
    each = [(-float(top.values[k]), w, int(top.indices[k])) for k in range(K) for w in range(W)]
    want = sorted(each)[:K]
    xd = x.double()
    lse = float(torch.logsumexp(xd, 0))
    ws = torch.tensor([-v - lse for v, _, _ in want], dtype=torch.float64)
    assert torch.equal(p.cpu(), torch.tensor([w for _, w, _ in want]).int()[None] + 4 * torch.arange(S).int()[:, None])
    assert torch.equal(t.cpu(), torch.tensor([k for _, _, k in want])[None].expand(S, K))
    # the value's rounding, the sum's 40 units, and its arguments' on sum p |x - max|
    far = float((torch.softmax(xd, 0) * (xd - xd.max()).abs()).sum())
    tol = 2.0 ** -24 * ws.abs() + 40 * 2.0 ** -24 + 2.0 ** -22 * far
    assert ((s.cpu().double() - ws).abs() <= tol).all()


def test_select_refuses_more_places_before_it_makes_outputs():
    from loom_amd import ops
    x, sc = torch.zeros(8, 100, device=DEV), torch.zeros(2, 4, device=DEV)
    for n in (65, 1 << 40, 1 << 62, -1):
        with pytest.raises(RuntimeError, match="n_out must be 1 to 64"):
            ops.beam_select(x, sc, n)


# ------------------------------------------------------------------ attention

def test_rows_end_to_end_of_more_units_than_32_bits_name():
    """1024 rows of 131072 tokens (two pages shared by all) over 512 kv heads: one
    block of each head has all the work, and the numbers of those behind it, times its
    units, pass 2^32.  Half of the values are ones, so a part of a row's sum shows."""
    from loom_amd import ops
    KVH, HD, PS, MP, B = 512, 32, 1024, 128, 1024
    kp = torch.zeros(2, KVH, PS, HD, dtype=BF, device=DEV)
    vp = torch.zeros_like(kp)
    vp[0] = 1.0
    table = (torch.arange(MP, device=DEV) >= MP // 2).int().expand(B, MP).contiguous()
    q = torch.ones(B, KVH, HD, dtype=BF, device=DEV)
    c, _ = ops.paged_decode_attention(q, kp, vp, table, _i32([MP * PS] * B), want_kctx=False)
    assert (c == 0.5).all()


@pytest.mark.parametrize("dt,HD", [(BF, 64), (HF, 96), (FP, 64), (HF, 8), (BF, 256)])
@pytest.mark.parametrize("n", [1, 45, 3000])
def test_scores_of_minus_infinity(dt, HD, n):
    """Row 0: every score is -inf, the softmax of which is NaN; row 1: all but the last;
    row 2: none; row 3 holds no token, row 4 no sequence: zeros."""
    from loom_amd import ops
    PS, MP = 16, -(-n // 16)
    g = torch.Generator().manual_seed(n)
    kp, vp = torch.randn(3 * MP, 1, PS, HD, generator=g), torch.randn(3 * MP, 1, PS, HD, generator=g)
    q = torch.randn(5, 2, HD, generator=g)
    q[:2] = 0.0
    q[:2, :, 1] = 1.0
    kp[:2 * MP, :, :, 1] = -math.inf
    kp[MP + (n - 1) // PS, :, (n - 1) % PS, 1] = 0.5
    table = torch.cat([torch.arange(3 * MP).view(3, MP), torch.zeros(2, MP).long()]).int()
    kp, vp, q = kp.to(DEV, dt), vp.to(DEV, dt), q.to(DEV, dt)
    c, kx = ops.paged_decode_attention(q, kp, vp, table.to(DEV), _i32([n, n, n, 0, -1]))
    assert torch.isnan(c[0].float()).all() and torch.isnan(kx[0].float()).all()
    last = vp[MP + (n - 1) // PS, 0, (n - 1) % PS]
    assert torch.equal(c[1], last.expand(2, HD))
    assert torch.isfinite(c[2].float()).all() and torch.isfinite(kx[2].float()).all()
    assert not c[3:].float().any() and not kx[3:].float().any()


@pytest.mark.parametrize("dt", [BF, HF])
def test_step_ropes_to_the_nearest_value_but_for_ties_of_fp32(dt):
    """The rotation is computed in 64 bits, rounded to fp32 and then to the type: it is
    the nearest value of the type, or beside it where fp32's rounding falls on the
    middle of two (one in some 16000 values of half, one in 150000 of bf16)."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(20)
    HD, B = 128, 256
    kp, vp = (torch.zeros(B, 2, 16, HD, dtype=dt, device=DEV) for _ in range(2))
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None].contiguous()
    ang = torch.rand(16, HD, generator=g, dtype=torch.float64) * 6
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    lens = torch.arange(B, dtype=torch.int32, device=DEV) % 16
    x = torch.randn(B, 20, HD, generator=g).to(DEV, dt)
    q = ops.paged_decode_step(x.view(B, -1), kp, vp, table, lens, cos, sin)[2]
    xd = x[:, :16].double()
    turned = torch.cat([-xd[..., HD // 2:], xd[..., :HD // 2]], -1)
    d = xd * cos[lens.long()][:, None].double() + turned * sin[lens.long()][:, None].double()
    err, bits = (q.double() - d).abs(), q.view(torch.int16).int()
    beside = torch.minimum(*[((bits + k).to(torch.int16).view(dt).double() - d).abs() for k in (-1, 1)])
    off = beside < err
    assert float(off.double().mean()) <= 2.0 ** -12
    assert (err[off] <= beside[off] + 2 * 2.0 ** -24 * d.abs()[off]).all()


# ------------------------------------------------------------------ pages

def test_compact_a_page_of_almost_two_gib():
    """A page of 2^31 - 32768 bytes, the largest that this shape allows."""
    from loom_amd import ops
    KVH, PS, HD = 771, 1024, 680
    assert KVH * PS * HD * 4 == 2 ** 31 - 32768
    pools = [torch.randint(-2 ** 31, 2 ** 31 - 1, (1, 2, KVH, PS, HD), dtype=torch.int32, device=DEV) for _ in range(2)]
    want = [p[:, 1].clone() for p in pools]
    table, refs, used = _i32([[1]]), _i32([0, 1]), _i32([0])
    ops.paged_compact(pools[0].view(FP), pools[1].view(FP), table, refs, used)
    assert table.tolist() == [[0]] and refs.tolist() == [1, 0] and int(used) == 1
    for p, w in zip(pools, want):
        assert torch.equal(p[:, 0], w) and torch.equal(p[:, 1], w)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("n", [700, 131072, 1 << 20])
@pytest.mark.parametrize("down", [14.3, 20.3, 24.6, 25.1, 28.7])
def test_one_dominant_token_and_a_long_tail(dt, n, down):
    """All tokens but one have a weight 2^-down of the largest, of value one: their sum
    is what a long row keeps of them, however small each of them is."""
    from loom_amd import ops
    HD, PS = 64, 64
    MP = n // PS + 1
    kp, vp = torch.zeros(3, 1, PS, HD), torch.ones(3, 1, PS, HD)
    q = torch.zeros(3, 2, HD)
    q[..., 0] = torch.tensor([8.0, 7.75])            # the score is k / sqrt(64) times this
    kp[1, 0, 5, 0] = kp[2, 0, 50, 0] = down * math.log(2)
    vp[1, 0, 5] = vp[2, 0, 50] = 0.0
    table = torch.zeros(3, MP, dtype=torch.int32)
    table[0, 0], table[1, (n - 1) // PS - 1], table[2, MP // 2] = 1, 2, 1     # early, at the end, in the middle
    kp, vp, q = kp.to(DEV, dt), vp.to(DEV, dt), q.to(DEV, dt)
    c, kx = ops.paged_decode_attention(q, kp, vp, table.to(DEV), _i32([n] * 3))
    top = kp[1, 0, 5, 0].double()
    s = q[:, :, 0].double() * top / 8
    rest = (n - 1) * torch.exp(-s)
    want_c, want_k = (rest / (1 + rest)).cpu(), (top / (1 + rest)).cpu()
    # roundings: of the output and of each weight (half a step each; of half's small ones
    # 2^-38 of the largest), of the score (a product, 64 additions, the scaling; its
    # exponential's argument and result), and one per tile of 32 tokens and per chunk of
    # the sums, in the numerator and the denominator
    half, u = torch.finfo(dt).eps / 2, 2.0 ** -24
    rel = half + (0 if dt == FP else half) + 2 * (72 * float(s.max()) + 8) * u + 2 * (n / 32 + 512) * u
    least = n * 2.0 ** -38 + 2.0 ** -24 if dt == HF else 2.0 ** -126
    over_c = ((c.cpu().double() - want_c[..., None]).abs() / (rel * want_c + least)[..., None]).max()
    over_k = ((kx[..., 0].cpu().double() - want_k).abs() / (rel * want_k)).max()
    assert float(over_c) <= 1 and float(over_k) <= 1
    assert not kx[..., 1:].float().any()


def _shared_rows(g, R, MP, PS, tokens, NP, KVH=1, HD=8, dt=FP):
    """R rows that hold the same pages of `tokens` tokens."""
    n = -(-tokens // PS)
    order = torch.randperm(NP, generator=g)[:n].int()
    table = torch.full((R, MP), -1, dtype=torch.int32)
    table[:, :n] = order
    refs = torch.zeros(NP, dtype=torch.int32)
    refs[order.long()] = R
    pools = [torch.randn(2, NP, KVH, PS, HD, generator=g).to(dt) for _ in range(2)]
    return [t.to(DEV) for t in (*pools, table, torch.full((R,), tokens, dtype=torch.int32), refs)]


def _update_as_the_oracle(s, **kw):
    """paged_update against the plain restatement; every page of the tokens made
    writable is its row's alone."""
    from loom_amd import ops
    status, PS = _i32([0]), s[0].shape[3]
    par = kw.get("parent")
    want = ref.update(*[t.cpu() for t in s], **dict(kw, parent=None if par is None else par.cpu()))
    ops.paged_update(*s, status, **kw)
    for name, a, b in zip(("k", "v", "table", "lens", "refs"), s, want):
        assert torch.equal(a.cpu(), b), (name, kw)
    assert int(status) == want[5]
    t, refs, lens = s[2].tolist(), s[4].tolist(), s[3].tolist()
    assert refs == torch.bincount(s[2].cpu()[s[2].cpu() >= 0].long(), minlength=len(refs)).tolist()
    for r, n in enumerate(lens):
        if n >= 0 and kw.get("n_new", 0) > 0:
            for at in range(n // PS, min((n + kw["n_new"] - 1) // PS + 1, len(t[r]))):
                assert t[r][at] < 0 or refs[t[r][at]] == 1, (r, at, kw)


@pytest.mark.parametrize("lens", [[64, 32], [64, 40], [32, 33], [0, 64], [1, 0], [48, 16], [64, -1]])
@pytest.mark.parametrize("n_new", [1, 20, 48])
@pytest.mark.parametrize("forked", [False, True])
def test_update_behind_lowered_lengths(lens, n_new, forked):
    """Two rows of the same four pages, whose last tokens are dropped: what is made
    writable is no page that the other holds."""
    s = _shared_rows(torch.Generator().manual_seed(1), 2, 8, 16, 64, 40)
    s[3].copy_(_i32(lens))
    _update_as_the_oracle(s, n_new=n_new, **({"parent": _i32([0, 1])} if forked else {}))
    _update_as_the_oracle(s, n_new=1, advance=n_new, parent=_i32([1, 0]))


@pytest.mark.parametrize("R,MP,pool", [(6, 9, 200), (6, 9, 25), (300, 30, 20000), (300, 30, 3000)])
@pytest.mark.parametrize("seed", [1, 2])
def test_update_random_walk_with_lowered_lengths(R, MP, pool, seed):
    """Forks, advances, reservations and dropped tokens in a row, in pools that suffice
    and that do not; the table's fork in its own launch and not."""
    g = torch.Generator().manual_seed(seed)
    s = _shared_rows(g, R, MP, 16, 50, pool)
    for step in range(10):
        kw = dict(n_new=int(torch.randint(0, 60, (1,), generator=g)), advance=0)
        if step % 2:
            par = torch.randint(-1, R + 1, (R,), generator=g).int()
            keep = torch.rand(R, generator=g) < 0.4
            par[keep] = torch.arange(R).int()[keep]
            kw["parent"] = par.to(DEV)
        _update_as_the_oracle(s, **kw)
        # some of the reserved tokens are written, and some rows drop tokens again
        add = torch.randint(0, kw["n_new"] + 1, (R,), generator=g).to(DEV)
        down = (torch.randint(0, 40, (R,), generator=g) * (torch.rand(R, generator=g) < 0.5)).to(DEV)
        grown = torch.minimum(s[3] + add, torch.tensor(MP * 16, device=DEV))
        s[3].copy_(torch.where(s[3] >= 0, (grown - down).clamp(min=0), s[3]))


def test_compact_a_cache_of_no_rows():
    """Pages that refs count but no table holds move too."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(2)
    pools = [torch.randn(2, 7, 2, 16, 32, generator=g).to(DEV, BF) for _ in range(2)]
    want = [p.clone() for p in pools]
    refs, used = _i32([0, 2, 0, 0, 1, 0, 1]), _i32([0])
    for p in want:
        p[:, 0], p[:, 2] = p[:, 4].clone(), p[:, 6].clone()
    table = torch.empty(0, 5, dtype=torch.int32, device=DEV)
    ops.paged_compact(*pools, table, refs, used)
    assert refs.tolist() == [1, 2, 1, 0, 0, 0, 0] and int(used) == 3
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])


# ------------------------------------------------------------------ layouts

def _odd(t, d):
    """The same tensor with another stride in its dimension d of one entry."""
    assert t.shape[d] == 1
    return t.as_strided(t.shape, [s + 3 if k == d else s for k, s in enumerate(t.stride())], t.storage_offset())


def test_strides_of_dimensions_of_one_entry_say_nothing():
    from loom_amd import ops
    g = torch.Generator().manual_seed(4)
    for L, NP, KVH in ((1, 6, 2), (2, 1, 2), (2, 6, 1)):
        k, v = (torch.randn(L, NP, KVH, 16, 32, generator=g).to(DEV, BF) for _ in range(2))
        k2, v2 = k.clone(), v.clone()
        for d in range(3):
            if k2.shape[d] == 1:
                v2 = _odd(v2, d)
        n = 10 if NP == 1 else 30
        start = lambda: [torch.full((1, 3), -1, dtype=torch.int32, device=DEV), _i32([0]), _i32([0] * NP), _i32([0])]  # noqa: E731
        rows = [torch.randn(L, 1, KVH, 40, 32, generator=g).to(DEV, BF) for _ in range(2)]
        q = torch.randn(1, 4, 32, generator=g).to(DEV, BF)
        out = []
        for kp, vp, kr, vr in ((k, v, *rows), (k2, v2, rows[0], _odd(rows[1], 1))):
            table, lens, refs, status = start()
            ops.paged_update(kp, vp, table, lens, refs, status, n_new=n)
            ops.paged_write(kp, vp, table, kr, vr, _i32([0]), _i32([n]))
            used = _i32([0])
            ops.paged_compact(kp, vp, table, refs, used)
            out.append([kp, vp, table, used, *ops.paged_decode_attention(q, kp[-1], vp[-1], table, _i32([n]))])
        assert int(out[0][3]) == -(-n // 16)
        for a, b in zip(*out):
            assert torch.equal(a, b)
        one = [r[:, :, :, 4:5].contiguous() for r in rows]      # a source of one position
        for kp, vp, kr, vr in ((k, v, *one), (k2, v2, _odd(one[0], 3), one[1])):
            ops.paged_write(kp, vp, out[0][2], kr, vr, _i32([0]), _i32([1]))
        assert torch.equal(k, k2) and torch.equal(v, v2)


def _laid_out(t, how):
    """The values of a pool [L, NP, KVH, PS, HD] in another layout, and in memory behind it."""
    L, NP, KVH, PS, HD = t.shape
    if how == "token":
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    if how == "page":                                # a page of all layers together
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((L, NP, KVH + 1, PS, HD + 8), 3.0, dtype=t.dtype, device=t.device)      # rows and pages apart
    wide[:, :, :KVH, :, :HD] = t
    return wide[:, :, :KVH, :, :HD]


@pytest.mark.parametrize("how", ["token", "page", "wide"])
@pytest.mark.parametrize("R,MP", [(5, 9), (300, 28)])
def test_bookkeeping_of_other_layouts_and_table_views(how, R, MP):
    """Update, dense rows and compaction over pools of other strides and a table that is
    a view of a wider one: as over dense ones, and nothing between the rows changes."""
    from loom_amd import ops
    g = torch.Generator().manual_seed(R)
    a = _shared_rows(g, R, MP, 16, 40, 12 + 3 * R, KVH=2, HD=24, dt=BF)
    b = [t.clone() for t in a]
    b[0], b[1] = _laid_out(a[0], how), _laid_out(a[1], how)
    table = torch.full((R, MP + 5), 77, dtype=torch.int32, device=DEV)
    table[:, :MP] = a[2]
    b[2] = table[:, :MP]
    par = torch.randint(-1, R, (R,), generator=g).int().to(DEV)
    rows = [torch.randn(2, R, 40, 2, 24, generator=g).to(DEV, BF).transpose(2, 3) for _ in range(2)]
    first, last = torch.full((R,), 35, device=DEV).int(), torch.full((R,), 38, device=DEV).int()
    for s in (a, b):
        status, used = _i32([0]), _i32([0])
        ops.paged_update(*s, status, n_new=1)
        ops.paged_write(s[0], s[1], s[2], *rows, first, last)
        ops.paged_update(*s, status, parent=par, n_new=10)
        ops.paged_compact(s[0], s[1], s[2], s[4], used)
        s += [status, used]
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert (table[:, MP:] == 77).all()
    if how == "wide":
        for t in b[:2]:
            whole = t.as_strided((2, t.shape[1], 3, 16, 32), t.stride())
            assert (whole[:, :, 2] == 3.0).all() and (whole[..., 24:] == 3.0).all()


@pytest.mark.parametrize("dt,V,W,K", [(BF, 1 << 24, 2, 64), (FP, (1 << 24) - 3, 1, 1), (HF, 1 << 24, 1, 5)])
def test_select_over_the_largest_vocabularies(dt, V, W, K):
    from loom_amd import ops
    g = torch.Generator(device=DEV).manual_seed(K)
    x = torch.empty(W, V, dtype=dt, device=DEV)
    for r in range(W):
        x[r] = torch.randn(V, generator=g, device=DEV).clamp(max=3).to(dt)
    at = torch.randperm(V, generator=g, device=DEV)[:40 * W].view(W, 40)
    at[:, 0], at[:, 1] = V - 1, 0
    x.scatter_(1, at, (4 + torch.arange(40, device=DEV) % 7).to(dt).expand(W, 40).contiguous())       # with ties
    sc = torch.zeros(1, W, device=DEV)
    s, p, t, f = ops.beam_select(x, sc, K)
    each = []
    for r in range(W):
        xr = x[r].double()
        lse = float(torch.logsumexp(xr, 0))
        least = float(torch.topk(x[r].float(), K).values[-1])
        tok = (x[r].float() >= least).nonzero().view(-1)
        each += [(lse - float(v), r, int(k)) for v, k in zip(xr[tok].tolist(), tok.tolist())]
    want = sorted(each)[:K]
    assert p.tolist() == [[r for _, r, _ in want]] and t.tolist() == [[k for _, _, k in want]]
    # the value's rounding, 40 units of the sums, and the arguments' (at most 16) two units
    ws = torch.tensor([-v for v, _, _ in want], dtype=torch.float64)
    assert ((s[0].cpu().double() - ws).abs() <= 2.0 ** -24 * ws.abs() + 40 * 2.0 ** -24 + 2.0 ** -22 * 16).all()
