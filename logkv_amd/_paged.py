"""ctypes binding of the rotary, append and paged attention entry points (the C ABI in include/logkv_paged.h)."""

from __future__ import annotations

import ctypes as C
from functools import lru_cache
from struct import Struct

from ._lib import _i32, _i64, _p, lib
from ._rows import _CODES, _packer

F32 = 2


class RotaryArgs(C.Structure):
    _fields_ = [
        ("q", _p), ("q_sb", _i64), ("q_sh", _i64), ("q_st", _i64),
        ("q_out", _p), ("qo_sb", _i64), ("qo_sh", _i64), ("qo_st", _i64),
        ("k", _p), ("k_sb", _i64), ("k_sh", _i64), ("k_st", _i64),
        ("k_out", _p), ("ko_sb", _i64), ("ko_sh", _i64), ("ko_st", _i64),
        ("v", _p), ("v_sb", _i64), ("v_sh", _i64), ("v_st", _i64),
        ("k_pages", _p), ("kp_sp", _i64), ("kp_sg", _i64), ("kp_st", _i64),
        ("v_pages", _p), ("vp_sp", _i64), ("vp_sg", _i64), ("vp_st", _i64),
        ("table", _p), ("table_sb", _i64), ("lengths", _p), ("counts", _p), ("frequencies", _p),
        ("positions", _p), ("pos_sb", _i64), ("pos_st", _i64), ("first_dev", _p), ("first", _i64),
        ("n_batch", _i32), ("n_heads", _i32), ("n_groups", _i32), ("tokens", _i32), ("dim", _i32), ("dim_v", _i32),
        ("rotated", _i32), ("dtype", _i32), ("cache_dtype", _i32), ("interleaved", _i32),
        ("freq_float", _i32), ("pos_int", _i32), ("len_add", _i32), ("page", _i32), ("table_len", _i32),
        ("n_pages", _i32), ("amplitude", C.c_float), ("sign", C.c_float),
    ]


class PagedArgs(C.Structure):
    _fields_ = [
        ("q", _p), ("q_sb", _i64), ("q_sh", _i64), ("q_st", _i64),
        ("k", _p), ("k_sb", _i64), ("k_sg", _i64), ("k_st", _i64),
        ("v", _p), ("v_sb", _i64), ("v_sg", _i64), ("v_st", _i64),
        ("k_pages", _p), ("kp_sp", _i64), ("kp_sg", _i64), ("kp_st", _i64),
        ("v_pages", _p), ("vp_sp", _i64), ("vp_sg", _i64), ("vp_st", _i64),
        ("table", _p), ("table_sb", _i64), ("lengths", _p), ("counts", _p),
        ("visible", _p), ("vis_sb", _i64), ("vis_st", _i64),
        ("prefix_table", _p), ("prefix_sb", _i64),
        ("prefix_k", _p), ("pk_sb", _i64), ("pk_sg", _i64), ("pk_st", _i64),
        ("prefix_v", _p), ("pv_sb", _i64), ("pv_sg", _i64), ("pv_st", _i64),
        ("bias", _p), ("b_sb", _i64), ("b_sg", _i64), ("b_st", _i64),
        ("prefix_lengths", _p), ("prefix_lengths2", _p),
        ("out", _p), ("o_sb", _i64), ("o_sh", _i64), ("o_st", _i64),
        ("n_batch", _i32), ("n_heads", _i32), ("n_groups", _i32), ("tq", _i32), ("dk", _i32), ("dv", _i32),
        ("dtype", _i32), ("page", _i32), ("table_len", _i32), ("n_pages", _i32), ("n_prefixes", _i32),
        ("prefix_len", _i32), ("len_stride", _i32), ("len_add", _i32), ("prefix_stride", _i32),
        ("prefix_add", _i32), ("bias_half", _i32), ("scale", C.c_float), ("bias_scale", C.c_float),
    ]


pack_rotary = _packer(RotaryArgs).pack
# The rotation's rows (q, q_out, k, k_out) and the rest, whose last field is the sign.
_ROWS = 16
pack_rotary_rows = Struct("=" + "Qqqq" * 4).pack
pack_rotary_rest = Struct("=" + "".join(_CODES[t] for _, t in RotaryArgs._fields_[_ROWS:-1])).pack
ROTARY_SIGNS = {sign: Struct("=f").pack(sign) for sign in (1.0, -1.0)}
pack_paged = _packer(PagedArgs).pack

# Exported symbol -> (restype, argtypes); the tests check this table against the header. The structs are passed as
# their bytes or by reference.
SIGNATURES = {
    "logkv_rotary": (_i32, [_p, _p]),
    "logkv_paged_append": (_i32, [_p, _p]),
    "logkv_paged_workspace_bytes": (_i64, [_p]),
    "logkv_paged_plan": (_i32, [_p, _p]),
    "logkv_paged_attention": (_i32, [_p, _p, _i64, _p]),
}


@lru_cache(maxsize=1)
def paged_lib() -> C.CDLL:
    handle = lib()
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.restype, fn.argtypes = res, args
    return handle
