"""CPU: sizes that the cache operators refuse before anything is launched."""

from __future__ import annotations

import ctypes
import os

import pytest

from imba_chess_b200 import _native

AT, BIG = 1 << 20, 1 << 40


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.LIB_PATH):
        from imba_chess_b200.build import build

        build()
    return _native.load()


@pytest.mark.parametrize("rows", [(1 << 28) + 1, (1 << 30) + 1, 2**31 - 1])
def test_append_refuses_more_rows_than_a_plan_takes(lib, rows):
    """A step of more than 2^28 rows has no plan (its bytes are 0), so no
    plan's size is large enough for it."""
    assert lib.imba_append_plan_bytes(rows) == 0
    cache, pool = _native.CacheDesc(2, 4, 64, 64, _native.DTYPE_E4M3), _native.PoolDesc(AT, 16)
    d = _native.AppendDesc(rows, 0, _native.DTYPE_BF16, 0, AT, AT, AT)
    byref = ctypes.byref
    assert lib.imba_kv_append(byref(cache), byref(pool), byref(d), AT, BIG, None) == _native.IMBA_ERR_ARG
    assert lib.imba_append_plan(byref(pool), rows, AT, AT, BIG, None, None) == _native.IMBA_ERR_ARG


def test_attention_refuses_more_extra_keys_than_a_warp_counts(lib):
    """The extra keys of a warp's rows, up to 24 times all of a step's, are
    counted in 32 bits: at most 2^26."""
    cache, byref = _native.CacheDesc(2, 4, 64, 64, _native.DTYPE_E4M3), ctypes.byref
    pool = _native.PoolDesc(AT, 16)

    def rows(extra):
        r = _native.AttendDesc(4, 2, 2, 8, extra, 4)
        for name in ("seg_row_off", "row_vis", "group_page_off", "group_pages", "row_extra_off", "extra_slot", "extra_pos"):
            setattr(r, name, AT)
        return r

    assert lib.imba_attend_plan_bytes(byref(cache), byref(rows(1 << 26))) > 0
    for extra in ((1 << 26) + 1, 2**31 - 1):
        r = rows(extra)
        assert lib.imba_attend_plan_bytes(byref(cache), byref(r)) == 0
        args = _native.AttendArgs(0, _native.DTYPE_BF16, AT, AT)
        assert lib.imba_attend(byref(cache), byref(pool), byref(r), byref(args), AT, BIG, None) == _native.IMBA_ERR_RANGE
        assert lib.imba_attend_plan(byref(cache), byref(pool), byref(r), AT, BIG, None) == _native.IMBA_ERR_RANGE
