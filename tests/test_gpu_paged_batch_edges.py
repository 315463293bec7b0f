"""A ragged batch's step at its edges, against plain implementations in 64 bits: which kind of value
an infinity of a token gives."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_paged_batch import BF, DEV, FP, HF, _cache, _i32, _tables

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
