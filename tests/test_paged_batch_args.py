"""CPU checks of what a ragged batch's operators refuse (before any device work, with a
message), of what they accept without rows or tokens, and of the oracle's plain forms."""
import ctypes
import math

import pytest
import torch

from oracle import paged as ref

P = ctypes.c_void_p(256)


def _refuses(name, base, changes):
    from loom_amd import _lib
    for change, message in changes:
        with pytest.raises(RuntimeError, match=message):
            _lib.call(name, *dict(base, **change).values())


SIZES = [(dict(rows=1025), "0 to 1024 rows"), (dict(rows=-1), "0 to 1024 rows"), (dict(n_tokens=-1), "tokens, got -1"),
         (dict(n_tokens=(1 << 20) + 1), "tokens, got 1048577"), (dict(KVH=3), "bad heads"), (dict(KVH=0), "bad heads"),
         (dict(QH=1), "bad heads"), (dict(QH=2048), "bad heads"), (dict(page_size=24), "power of two"), (dict(page_size=8), "power of two"),
         (dict(page_size=2048), "power of two"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 30), "n_pages"),
         (dict(max_pages=0), "1 page to 2\\^24"), (dict(max_pages=(1 << 20) + 1, table_ld=1 << 21), "1 page to 2\\^24"),
         (dict(max_pages=1 << 60, table_ld=1 << 60), "1 page to 2\\^24"), (dict(table_ld=4), "row stride 4")]


def test_plan_refuses():
    base = dict(table=P, table_ld=5, max_pages=5, n_pages=10, page_size=16, lens=P, new=P, rows=3, n_tokens=7, QH=8, KVH=2,
                starts=P, rows_of=P, positions=P, slots=P, shared=P, plan=P, plan_bytes=1 << 30, stream=None)
    _refuses("loom_paged_plan", base, SIZES + [(dict({k: None}), "required pointer") for k in
                                               ("table", "lens", "new", "starts", "rows_of", "positions", "slots", "shared")])
    _refuses("loom_paged_plan", base, [(dict(plan=None), "plan of"), (dict(plan=ctypes.c_void_p(272)), "64-byte aligned plan"),
                                       (dict(plan_bytes=64), "plan of")])


STEP = dict(dtype=1, qkv=P, qkv_ld=1152, k=P, v=P, page=2 * 16 * 96, tok=96, head=16 * 96, n_pages=10, page_size=16, table=P,
            table_ld=5, max_pages=5, rows=3, rows_of=P, positions=P, slots=P, plan=P, plan_bytes=1 << 30, cos=P, sin=P, n_pos=80,
            q_out=P, c=P, kctx=P, out_ld=768, ws=P, ws_bytes=1 << 34, n_tokens=7, QH=8, KVH=2, HD=96, stream=None)


def test_step_refuses():
    _refuses("loom_paged_batch_step", STEP, SIZES + [(dict({k: None}), "required pointer") for k in
                                                     ("qkv", "k", "v", "table", "rows_of", "positions", "slots", "plan", "cos", "sin", "q_out", "c")])
    _refuses("loom_paged_batch_step", STEP, [
        (dict(dtype=5), "unsupported dtype"), (dict(HD=80), "head_dim 80"), (dict(HD=512, tok=512), "head_dim 512"),
        (dict(tok=88), "page strides"), (dict(tok=1 << 27), "page strides"), (dict(page=-96), "page strides"), (dict(head=-8), "page strides"),
        (dict(tok=97), "multiples of 16 bytes"), (dict(k=ctypes.c_void_p(264)), "multiples of 16 bytes"),
        (dict(qkv_ld=1144), "hold 1152"), (dict(qkv_ld=1153), "qkv must be 16-byte"), (dict(qkv=ctypes.c_void_p(258)), "qkv must be 16-byte"),
        (dict(out_ld=760), "output rows"), (dict(out_ld=769), "output rows"), (dict(q_out=ctypes.c_void_p(264)), "16-byte aligned"),
        (dict(kctx=ctypes.c_void_p(264)), "16-byte aligned"), (dict(sin=ctypes.c_void_p(260)), "16-byte aligned"), (dict(n_pos=0), "rotary tables"),
        (dict(plan_bytes=64), "plan of"), (dict(plan=ctypes.c_void_p(272)), "64-byte aligned plan"), (dict(ws=None), "workspace"),
        (dict(ws_bytes=16), "workspace"), (dict(ws=ctypes.c_void_p(260)), "workspace")])


def test_step_refuses_more_blocks_than_a_launch_has():
    n = 1 << 20
    for QH, KVH in ((1024, 1), (1024, 2)):
        width = (QH + 2 * KVH) * 96
        _refuses("loom_paged_batch_step", dict(STEP, n_tokens=n, QH=QH, KVH=KVH, qkv_ld=width, out_ld=QH * 96, plan_bytes=1 << 40,
                                               ws_bytes=1 << 50), [(dict(), "too many for one call")])


def test_no_tokens_is_no_error():
    from loom_amd import _lib
    none = {k: None for k in ("qkv", "k", "v", "table", "rows_of", "positions", "slots", "plan", "cos", "sin", "q_out", "c", "kctx", "ws")}
    _lib.call("loom_paged_batch_step", *dict(STEP, n_tokens=0, plan_bytes=0, ws_bytes=0, **none).values())


def test_reserve_refuses():
    base = dict(dtype=1, k=P, v=P, layers=2, layer=10 * 2 * 16 * 96, page=2 * 16 * 96, tok=96, head=16 * 96, n_pages=10, page_size=16,
                KVH=2, HD=96, table=P, table_ld=5, max_pages=5, lens=P, refs=P, status=P, new=P, ws=P, ws_bytes=1 << 20, rows=3, stream=None)
    _refuses("loom_paged_reserve", base, [(dict({k: None}), "required pointer") for k in ("table", "lens", "refs", "status", "new")] + [
        (dict(dtype=3), "unsupported dtype"), (dict(k=None), "pools must be given"), (dict(tok=64), "bad pool strides"),
        (dict(rows=1025), "0 to 1024 rows"), (dict(max_pages=0), "1 page to 2\\^24"), (dict(page_size=100), "power of two"),
        (dict(ws_bytes=47), "48 bytes"), (dict(ws=None), "48 bytes"), (dict(ws=ctypes.c_void_p(8)), "16-byte aligned workspace")])
    from loom_amd import _lib
    _lib.call("loom_paged_reserve", *dict(base, rows=0, table=None, lens=None, refs=None, status=None, new=None, ws=None, ws_bytes=0).values())


@pytest.mark.parametrize("rows,n,QH,KVH", [(0, 0, 8, 2), (1, 1, 8, 2), (1024, 1 << 20, 8, 2), (1024, 1 << 20, 1024, 1), (1024, 1 << 20, 1024, 1024)])
def test_sizes_of_plan_and_workspace(rows, n, QH, KVH):
    """Everything that is counted in 32 bits on the device stays within them."""
    from loom_amd import _lib
    lib = _lib.load()
    p = lib.loom_paged_plan_bytes(rows, n, QH, KVH)
    assert 0 < p < 1 << 34
    assert (lib.loom_paged_batch_workspace_bytes(rows, n, QH, KVH, 96) > 0) == (n > 0)
    for bad in ((-1, n, QH, KVH), (1025, n, QH, KVH), (rows, -1, QH, KVH), (rows, n, QH, 0), (rows, n, KVH - 1, KVH), (rows, n, 2048, 1)):
        assert lib.loom_paged_plan_bytes(*bad) == 0


def test_the_oracle_sees_no_later_token():
    """batch_attention of whole rows, against a softmax written out, with a NaN further on."""
    g = torch.Generator().manual_seed(0)
    kp, vp = (torch.randn(3, 2, 16, 8, generator=g) for _ in range(2))
    vp[1, 0, 4] = math.nan                                # position 20 of the row
    q = torch.randn(22, 4, 8, generator=g)
    o = ref.batch_attention(q, kp, vp, torch.tensor([[2, 1, 0]], dtype=torch.int32), [5], [0, 22], [True])
    k, v = (torch.cat([x[2, 0], x[1, 0]]).double() for x in (kp, vp))
    for i in (0, 14):
        n = 6 + i
        w = torch.softmax(k[:n] @ q[i, 1].double() / math.sqrt(8), 0)
        torch.testing.assert_close(o["c"][i, 1], w @ v[:n])
        torch.testing.assert_close(o["kctx"][i, 1], w @ k[:n])
    assert o["c"][15:, :2].isnan().all() and o["c"][:15].isfinite().all() and o["c"][:, 2:].isfinite().all()


def test_the_oracle_of_maps_and_reservation():
    table = torch.tensor([[0, -1], [0, 2], [-1, -1]], dtype=torch.int32)
    lens, new = torch.tensor([5, 20, -1]), torch.tensor([12, 2, 9])
    k = torch.randn(1, 4, 1, 16, 8)
    refs = torch.tensor([2, 0, 1, 0])
    kp, _, tab, rf, status = ref.reserve(k, k, table, lens, refs, new)
    # the first row copies the page it shares and takes another; the second row has room in its own
    assert tab.tolist() == [[1, 3], [0, 2], [-1, -1]] and rf.tolist() == [1, 1, 1, 1] and status == 0
    assert torch.equal(kp[0, 1, :, :5], k[0, 0, :, :5])
    starts, rows, pos, slots, ok = ref.maps(tab, lens, new, 15, 4, 16)
    assert starts == [0, 12, 14, 14] and rows == [0] * 12 + [1] * 2 + [-1] and ok == [True, True, False]
    assert pos == list(range(5, 17)) + [20, 21, -1] and slots == list(range(21, 32)) + [48, 2 * 16 + 4, 2 * 16 + 5, -1]
