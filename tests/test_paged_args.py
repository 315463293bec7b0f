"""CPU checks of what the paged cache's operators, the beam selection and the row
reordering refuse: before any device work (no GPU here), with a message."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)


def _refuses(name, base, changes):
    """Each change of one named argument is refused with its message."""
    from loom_amd import _lib
    for change, message in changes:
        args = dict(base, **change)
        with pytest.raises(RuntimeError, match=message):
            _lib.call(name, *args.values())


STEP = dict(dtype=1, qkv=P, qkv_ld=1152, k=P, v=P, page=2 * 16 * 96, tok=96, head=16 * 96, n_pages=10, page_size=16,
            table=P, table_ld=5, max_pages=5, lens=P, cos=P, sin=P, n_pos=80, q_out=P, c=P, kctx=P, out_ld=768, ws=P,
            ws_bytes=1 << 30, B=3, QH=8, KVH=2, HD=96, stream=None)
PAGED = [(dict(dtype=5), "unsupported dtype"), (dict(B=1025), "0 to 1024 rows"), (dict(B=-1), "0 to 1024 rows"),
         (dict(KVH=3), "bad heads"), (dict(KVH=0), "bad heads"), (dict(QH=1), "bad heads"), (dict(HD=80), "head_dim 80"),
         (dict(page_size=24), "power of two"), (dict(page_size=8), "power of two"), (dict(page_size=2048), "power of two"),
         (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 31), "n_pages"), (dict(max_pages=0), "1 page to 2\\^24"),
         (dict(max_pages=(1 << 20) + 1, table_ld=1 << 21), "1 page to 2\\^24"), (dict(table_ld=4), "row stride 4"),
         (dict(tok=88), "page strides"), (dict(tok=1 << 27), "page strides"), (dict(page=-96), "page strides"),
         (dict(tok=97), "multiples of 16 bytes"), (dict(k=ctypes.c_void_p(264)), "multiples of 16 bytes"),
         (dict(c=None), "required pointer"), (dict(lens=None), "required pointer"), (dict(table=None), "required pointer"),
         (dict(out_ld=760), "output rows"), (dict(ws_bytes=16), "workspace"), (dict(ws=None), "workspace"),
         (dict(ws=ctypes.c_void_p(260)), "workspace")]


def test_paged_decode_refuses():
    # rows of 80 tokens are not split and need no workspace; rows of 256 pages do
    base = dict(STEP, max_pages=256, table_ld=256, n_pos=4096)
    _refuses("loom_paged_decode_step", base, PAGED + [
        (dict(qkv_ld=1144), "qkv must be 16-byte aligned and hold 1152"), (dict(qkv_ld=1153), "qkv must be 16-byte"),
        (dict(qkv=ctypes.c_void_p(258)), "qkv must be 16-byte"), (dict(cos=None), "rotary tables"),
        (dict(n_pos=0), "rotary tables"), (dict(sin=ctypes.c_void_p(260)), "16-byte aligned"),
        (dict(q_out=ctypes.c_void_p(264)), "16-byte aligned")])
    att = {k: v for k, v in base.items() if k not in ("cos", "sin", "n_pos", "q_out")}
    _refuses("loom_paged_decode_attention", dict(att, qkv_ld=768), PAGED + [(dict(qkv_ld=760), "q must be 16-byte")])


def test_no_rows_is_no_error():
    from loom_amd import _lib
    _lib.call("loom_paged_decode_step", *dict(STEP, B=0).values())
    _lib.call("loom_reorder_rows", 0, None, None, None, None, None, None, 5, None)
    _lib.call("loom_reorder_rows", 3, None, None, None, None, None, None, 0, None)


POOL = dict(dtype=1, k=P, v=P, layers=2, layer=10 * 2 * 16 * 96, page=2 * 16 * 96, tok=96, head=16 * 96, n_pages=10,
            page_size=16, KVH=2, HD=96)
POOLS = [(dict(dtype=3), "unsupported dtype"), (dict(k=None), "pools must be given"), (dict(v=ctypes.c_void_p(8)), "multiples of 16 bytes"),
         (dict(tok=100), "multiples of 16 bytes"), (dict(tok=64), "bad pool strides"), (dict(layer=-8), "bad pool strides"),
         (dict(layers=0), "bad pool shape"), (dict(HD=4, tok=8), "bad pool shape"), (dict(HD=2048, tok=2048), "bad pool shape"),
         (dict(KVH=0), "bad pool shape"), (dict(layers=4096, KVH=4096, HD=1024, tok=1024), "more than a copy takes"), (dict(n_pages=0), "n_pages"), (dict(page_size=100), "power of two"),
         (dict(table=None), "required pointer"), (dict(rows=1025), "0 to 1024 rows"), (dict(max_pages=0), "1 page to 2\\^24"),
         (dict(table_ld=3), "row stride 3")]


def test_paged_update_write_compact_refuse():
    update = dict(POOL, table=P, table_ld=5, max_pages=5, lens=P, refs=P, status=P, parent=P, n_new=1, advance=0, ws=P,
                  ws_bytes=1 << 20, rows=3, stream=None)
    _refuses("loom_paged_update", update, POOLS + [
        (dict(lens=None), "required pointer"), (dict(refs=None), "required pointer"), (dict(status=None), "required pointer"),
        (dict(n_new=-1), "n_new=-1"), (dict(n_new=81), "n_new=81"), (dict(advance=-1), "advance=-1"),
        (dict(ws_bytes=47), "48 bytes"), (dict(ws=None), "48 bytes"), (dict(ws=ctypes.c_void_p(8)), "16-byte aligned workspace")])
    write = dict(POOL, table=P, table_ld=5, max_pages=5, kr=P, vr=P, sl=3 * 2 * 40 * 96, sr=2 * 40 * 96, sh=40 * 96, st=96,
                 tokens=40, first=P, last=P, rows=3, stream=None)
    _refuses("loom_paged_write", write, POOLS + [
        (dict(kr=None), "required pointer"), (dict(last=None), "required pointer"), (dict(st=64), "bad source shape"),
        (dict(tokens=-1), "bad source shape"), (dict(sr=-96), "bad source shape"), (dict(st=97), "source rows"),
        (dict(vr=ctypes.c_void_p(24)), "source rows")])
    compact = dict(POOL, table=P, table_ld=5, max_pages=5, refs=P, used=P, ws=P, ws_bytes=1 << 20, rows=3, stream=None)
    _refuses("loom_paged_compact", compact, POOLS + [
        (dict(refs=None), "required pointer"), (dict(used=None), "required pointer"), (dict(ws_bytes=135), "136 bytes"),
        (dict(ws=None), "136 bytes")])


def test_beam_select_and_reorder_refuse():
    sel = dict(dtype=1, logits=P, ld=20000, scores=P, finished=None, os=P, op=P, ot=P, of=None, groups=2, beams=4,
               V=20000, n_out=4, eos=-1, pad=0, ws=P, ws_bytes=1 << 24, stream=None)
    _refuses("loom_beam_select", sel, [
        (dict(dtype=9), "unsupported dtype"), (dict(beams=33), "1 to 32 beams"), (dict(beams=0), "1 to 32 beams"),
        (dict(groups=-1), "1 to 32 beams"), (dict(groups=65535), "at most 65535 rows"), (dict(V=0, n_out=0), "vocabulary"),
        (dict(V=(1 << 24) + 1, ld=1 << 25), "vocabulary"), (dict(ld=19999), "row stride 19999"), (dict(n_out=0), "n_out"),
        (dict(n_out=65), "n_out"), (dict(V=10, n_out=41), "n_out"), (dict(pad=20000), "pad_id"), (dict(pad=-1), "pad_id"),
        (dict(logits=None), "required pointer"), (dict(ot=None), "required pointer"), (dict(ws_bytes=10), "workspace"),
        (dict(ws=ctypes.c_void_p(260)), "workspace")])
    one = lambda v: (ctypes.c_int64 * 1)(v)  # noqa: E731
    p1, p0 = (ctypes.c_void_p * 1)(256), (ctypes.c_void_p * 1)(None)
    re = dict(n=1, t=p1, outer=one(1), os=one(0), rs=one(64), rb=one(64), parent=P, rows=4, stream=None)
    _refuses("loom_reorder_rows", re, [
        (dict(n=17), "at most 16"), (dict(n=-1), "at most 16"), (dict(rows=1025), "0 to 1024 rows"), (dict(t=None), "required pointer"),
        (dict(parent=None), "required pointer"), (dict(t=p0), "tensor 0 is NULL"), (dict(rs=one(60)), "bad shape of tensor 0"),
        (dict(outer=one(-1)), "bad shape"), (dict(rb=one(1 << 50), rs=one(1 << 50)), "too much data")])


def test_workspace_queries():
    from loom_amd import _lib
    lib = _lib.load()
    # 256 CUs assumed without a device: two blocks per CU over 2 kv heads = 256 blocks, a record for
    # each row that one of them works on
    assert lib.loom_paged_decode_workspace_bytes(32, 4096, 8, 2, 96) == (32 + 256) * 8 * 2 * 97 * 4
    assert lib.loom_paged_decode_workspace_bytes(2, 528, 8, 2, 96) == (2 + 256) * 8 * 2 * 97 * 4
    assert lib.loom_paged_decode_workspace_bytes(200, 256, 8, 2, 96) == 0      # one chunk per row: no join
    assert lib.loom_paged_update_workspace_bytes(7) == 7 * 16
    assert lib.loom_paged_compact_workspace_bytes(10) == 136
    assert lib.loom_beam_select_workspace_bytes(0, 4, 100, 4) == 0
    assert lib.loom_beam_select_workspace_bytes(2, 4, 100, 4) == 0              # one block per group
    assert lib.loom_beam_select_workspace_bytes(2, 4, 100000, 4) >= 8 * (12 + 8 * 4)


def test_mirror_refuses_cpu_tensors():
    from loom_amd import ops
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    pool, layer = torch.zeros(2, 10, 2, 16, 96), torch.zeros(10, 2, 16, 96)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_decode_step(torch.zeros(3, 1152), layer, layer, i32(3, 5), i32(3), torch.zeros(80, 96), torch.zeros(80, 96))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_decode_attention(torch.zeros(3, 8, 96), layer, layer, i32(3, 5), i32(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_update(pool, pool, i32(3, 5), i32(3), i32(10), i32(1), n_new=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_write(pool, pool, i32(3, 5), torch.zeros(2, 3, 2, 40, 96), torch.zeros(2, 3, 2, 40, 96), i32(3), i32(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_compact(pool, pool, i32(3, 5), i32(10), i32(1))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.beam_select(torch.zeros(4, 10), torch.zeros(1, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.reorder_rows([torch.zeros(4, 10)], i32(4))
