"""The plan query of paged attention (no GPU: nothing is launched)."""

import ctypes as C

import pytest

from logkv_amd import _lib, _paged
from test_paged_capi import paged_args


def plan(**over):
    out = (C.c_int32 * 8)(*[-7] * 8)
    rc = _paged.paged_lib().logkv_paged_plan(C.byref(paged_args(**over)), out)
    return rc, list(out)


def test_a_plan_follows_the_sizes():
    rc, p = plan()      # 3 queries, 6 of a prefix
    assert rc == _lib.LOGKV_OK and p == [0, 1, 1, 1, 0, 1, 1, 1]
    rc, p = plan(n_prefixes=0)
    assert rc == _lib.LOGKV_OK and p[4:] == [0] * 4
    rc, p = plan(n_batch=48, n_heads=32, n_groups=8, tq=2, table_len=20, n_prefixes=2, prefix_len=94)
    assert rc == _lib.LOGKV_OK and p == [0, 2, 1, 1, 8, 0, 4, 8]


@pytest.mark.parametrize("over", [dict(tq=0), dict(n_prefixes=3), dict(dk=60), dict(tq=1 << 18)])
def test_refused_sizes(over):
    rc, p = plan(**over)
    assert rc == _lib.LOGKV_EINVAL and p == [-7] * 8


def test_a_place_for_it_is_needed():
    assert _paged.paged_lib().logkv_paged_plan(C.byref(paged_args()), None) == _lib.LOGKV_EINVAL
    assert _paged.paged_lib().logkv_paged_plan(None, (C.c_int32 * 8)()) == _lib.LOGKV_EINVAL
