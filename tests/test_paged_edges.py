"""CPU checks of what the entry points of the paged cache, the beam selection and the
row reordering accept and refuse at the edges of their arguments."""
import ctypes

import pytest

P = ctypes.c_void_p(256)


def test_a_batch_of_no_rows_needs_no_pointers():
    from loom_amd import _lib
    pool = (1, P, P, 2, 10 * 2 * 16 * 96, 2 * 16 * 96, 96, 16 * 96, 10, 16, 2, 96)
    _lib.call("loom_paged_update", *pool, None, 5, 5, None, None, None, None, 1, 0, None, 0, 0, None)
    _lib.call("loom_paged_write", *pool, None, 5, 5, None, None, 0, 0, 0, 96, 40, None, None, 0, None)
    with pytest.raises(RuntimeError, match="required pointer"):
        _lib.call("loom_paged_compact", *pool, None, 5, 5, None, P, P, 136, 0, None)


def _refused(name, args, message):
    from loom_amd import _lib
    with pytest.raises(RuntimeError, match=message):
        _lib.call(name, *args.values())


def test_sizes_whose_products_pass_64_bits_are_refused():
    step = dict(dtype=1, qkv=P, qkv_ld=1152, k=P, v=P, page=2 * 16 * 96, tok=96, head=16 * 96, n_pages=10, page_size=16, table=P,
                table_ld=5, max_pages=5, lens=P, cos=P, sin=P, n_pos=80, q_out=P, c=P, kctx=P, out_ld=768, ws=P,
                ws_bytes=1 << 30, B=3, QH=8, KVH=2, HD=96, stream=None)
    for n in (1 << 60, (1 << 60) + 1, 1 << 59):
        _refused("loom_paged_decode_step", dict(step, max_pages=n, table_ld=n), "1 page to 2\\^24")
    for n in (1 << 59, 1 << 60, (1 << 59) + 96):
        _refused("loom_paged_decode_step", dict(step, tok=n), "page strides")
    pool = dict(dtype=1, k=P, v=P, layers=2, layer=10 * 2 * 16 * 96, page=2 * 16 * 96, tok=96, head=16 * 96, n_pages=10,
                page_size=16, KVH=2, HD=96, table=P, table_ld=1 << 60, max_pages=1 << 60)
    _refused("loom_paged_update", dict(pool, lens=P, refs=P, status=P, parent=P, n_new=0, advance=0, ws=P, ws_bytes=1 << 20,
                                       rows=3, stream=None), "1 page to 2\\^24")
    _refused("loom_paged_compact", dict(pool, refs=P, used=P, ws=P, ws_bytes=1 << 20, rows=3, stream=None), "1 page to 2\\^24")


def test_reorder_of_slices_whose_number_passes_64_bits_is_refused():
    one = lambda v: (ctypes.c_int64 * 1)(v)  # noqa: E731
    p1 = (ctypes.c_void_p * 1)(256)
    for outer, rb in ((1 << 62, 1 << 10), (1 << 31, 16), (1 << 62, 1 << 40), (4, 1 << 50)):
        _refused("loom_reorder_rows", dict(n=1, t=p1, outer=one(outer), os=one(0), rs=one(rb), rb=one(rb), parent=P, rows=4, stream=None),
                 "too much data")
