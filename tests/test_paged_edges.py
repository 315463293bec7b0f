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
