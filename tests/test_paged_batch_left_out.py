"""CPU checks of what a cache makes of rows that a step leaves out, and of the C call that tells it."""
import pytest
import torch

from test_paged_batch_args import P, SIZES, _refuses


def test_plan_checked_refuses_as_plan_does():
    base = dict(table=P, table_ld=5, max_pages=5, n_pages=10, page_size=16, lens=P, new=P, rows=3, n_tokens=7, QH=8, KVH=2,
                starts=P, rows_of=P, positions=P, slots=P, shared=P, plan=P, plan_bytes=1 << 30, limit=P, left_out=P, stream=None)
    _refuses("loom_paged_plan_checked", base, SIZES + [(dict(lens=None), "required pointer"), (dict(slots=None), "required pointer"),
                                                       (dict(plan=None), "plan of"), (dict(plan_bytes=64), "plan of")])


def test_rows_left_out_stay_and_are_reported():
    from loom_amd.paged import PagedKVCache
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    c = PagedKVCache(1, 4, 64, 2, 32, torch.float32, device="cpu", page_size=16)
    c.lens.copy_(i32(5, 6, -1, 0))
    c._limit[1] = 0                                       # as a plan leaves it for a row without slots
    c.advance(i32(3, 4, 5, -1))
    assert c.lens.tolist() == [8, 6, -1, 0]
    c.check()
    c.left_out += 2
    with pytest.raises(RuntimeError, match="2 rows' tokens had no place"):
        c.check()
    c.status += 3
    with pytest.raises(RuntimeError, match="3 pages could not be had.*2 rows"):
        c.check()
    c.reset()
    c.check()
    c.lens.zero_()
    c.advance(i32(1, 1, 1, 1))
    assert c.lens.tolist() == [1, 1, 1, 1]
