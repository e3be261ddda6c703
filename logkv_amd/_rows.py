"""ctypes binding of the row attention and eviction entry points (the C ABI in include/logkv_rows.h)."""

from __future__ import annotations

import ctypes as C
from functools import lru_cache
from struct import Struct

from ._lib import _i32, _i64, _p, lib

BF16, F16 = 0, 1


class RowsArgs(C.Structure):
    _fields_ = [
        ("q", _p), ("q_sb", _i64), ("q_sh", _i64), ("q_st", _i64),
        ("k", _p), ("k_sb", _i64), ("k_sg", _i64), ("k_st", _i64),
        ("v", _p), ("v_sb", _i64), ("v_sg", _i64), ("v_st", _i64),
        ("cache_k", _p), ("ck_sb", _i64), ("ck_sg", _i64), ("ck_st", _i64),
        ("cache_v", _p), ("cv_sb", _i64), ("cv_sg", _i64), ("cv_st", _i64),
        ("bias", _p), ("b_sb", _i64), ("b_sg", _i64), ("b_st", _i64),
        ("lengths", _p), ("lengths2", _p),
        ("visible", _p), ("vis_sb", _i64), ("vis_st", _i64),
        ("counts", _p), ("weights", _p), ("w_sb", _i64), ("w_sg", _i64),
        ("out", _p), ("o_sb", _i64), ("o_sh", _i64), ("o_st", _i64),
        ("n_batch", _i32), ("n_heads", _i32), ("n_groups", _i32), ("tq", _i32), ("cap", _i32), ("dk", _i32),
        ("dv", _i32), ("dtype", _i32), ("len_stride", _i32), ("len_add", _i32), ("bias_half", _i32),
        ("scale", C.c_float), ("bias_scale", C.c_float),
    ]


class EvictArgs(C.Structure):
    _fields_ = [
        ("cache_k", _p), ("ck_sb", _i64), ("ck_sg", _i64), ("ck_st", _i64),
        ("cache_v", _p), ("cv_sb", _i64), ("cv_sg", _i64), ("cv_st", _i64),
        ("weights", _p), ("w_sb", _i64), ("w_sg", _i64),
        ("positions", _p), ("p_sb", _i64), ("p_sg", _i64), ("lengths", _p),
        ("out_k", _p), ("ok_sb", _i64), ("ok_sg", _i64), ("ok_st", _i64),
        ("out_v", _p), ("ov_sb", _i64), ("ov_sg", _i64), ("ov_st", _i64),
        ("out_weights", _p), ("ow_sb", _i64), ("ow_sg", _i64),
        ("out_positions", _p), ("op_sb", _i64), ("op_sg", _i64), ("kept", _p), ("out_lengths", _p),
        ("n_batch", _i32), ("n_groups", _i32), ("cap", _i32), ("dk", _i32), ("dv", _i32), ("size", _i32),
        ("len_add", _i32), ("keep", _i32), ("recent", _i32),
    ]


# The structs as packed bytes, a third of a ctypes structure's cost to fill on a call's path (the layouts above
# have no padding but the last field's, which the tests check against the header).
_CODES = {_p: "Q", _i64: "q", _i32: "i", C.c_float: "f"}


def _packer(struct) -> Struct:
    fmt = Struct("=" + "".join(_CODES[t] for _, t in struct._fields_))
    return Struct(f"{fmt.format}{C.sizeof(struct) - fmt.size}x")


pack_rows = _packer(RowsArgs).pack
pack_evict = _packer(EvictArgs).pack

# Exported symbol -> (restype, argtypes); the tests check this table against the header. The structs are passed as
# their bytes or by reference.
SIGNATURES = {
    "logkv_rows_workspace_bytes": (_i64, [_p]),
    "logkv_tree_attention": (_i32, [_p, _p, _i64, _p]),
    "logkv_weight_attention": (_i32, [_p, _p, _i64, _p]),
    "logkv_evict_rows": (_i32, [_p, _p]),
}


@lru_cache(maxsize=1)
def rows_lib() -> C.CDLL:
    handle = lib()
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.restype, fn.argtypes = res, args
    return handle
