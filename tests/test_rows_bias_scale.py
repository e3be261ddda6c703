"""The factor of a tree attention's bias at the C ABI (no GPU: only refused calls)."""

import ctypes as C
import math

import pytest

from logkv_amd import _lib, _rows
from test_rows_capi import FAKE, no_device, rows_args


@no_device
@pytest.mark.parametrize("value", [-1.0, math.nan, math.inf])
def test_the_factor_is_positive(value):
    lib, a = _rows.rows_lib(), rows_args(bias=FAKE, bias_scale=value)
    assert lib.logkv_tree_attention(C.byref(a), FAKE, 1 << 40, None) == _lib.LOGKV_EINVAL
    assert "bias_scale" in lib.logkv_last_error().decode()
