"""The C ABI of the rotation, the paged append and paged attention without a GPU: the ctypes table and structs against
include/logkv_paged.h, and the argument checks that precede every launch (fake addresses, so only where no HIP device is
visible)."""

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from logkv_amd import _lib, _paged

HEADER = Path(__file__).resolve().parents[1] / "include" / "logkv_paged.h"
FAKE = 0x10000
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses are only passed where no HIP device is visible")


def header_text():
    return re.sub(r"/\*.*?\*/", " ", HEADER.read_text(), flags=re.S)


def test_library_exports_the_header():
    names = set(re.findall(r"\b(logkv_[a-z0-9_]+)\s*\(", header_text()))
    assert names == set(_paged.SIGNATURES)
    handle = C.CDLL(str(_lib.LIB_PATH))
    for name in sorted(names):
        assert hasattr(handle, name), name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc")
def test_ctypes_structs_match_the_header(tmp_path):
    structs = {"logkv_rotary_args": _paged.RotaryArgs, "logkv_paged_args": _paged.PagedArgs}
    declared = {name: [f.strip().lstrip("*").strip() for decl in body.split(";") if decl.strip()
                       for f in re.sub(r"^\s*(const\s+)?\w+", "", decl).split(",")]
                for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", header_text(), flags=re.S)}
    assert {n: [f for f, _ in c._fields_] for n, c in structs.items()} == declared
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, fields in declared.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f in fields]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    want = [x for n, c in structs.items() for x in [C.sizeof(c)] + [getattr(c, f).offset for f, _ in c._fields_]]
    assert got == want
    for cls, pack in ((_paged.RotaryArgs, _paged.pack_rotary), (_paged.PagedArgs, _paged.pack_paged)):
        values = [3 * i + 1 for i in range(len(cls._fields_))]
        a = cls.from_buffer_copy(pack(*values))
        assert [getattr(a, f) for f, _ in cls._fields_] == values
    # The rotation's struct in its three parts.
    values = [3 * i + 1 for i in range(len(_paged.RotaryArgs._fields_) - 1)] + [1.0]
    assert _paged.pack_rotary_rows(*values[:16]) + _paged.pack_rotary_rest(*values[16:-1]) + _paged.ROTARY_SIGNS[1.0] \
        == _paged.pack_rotary(*values)


def rotary_args(**over):
    a = _paged.RotaryArgs()
    for name in ("q", "q_out", "k", "k_out", "v", "k_pages", "v_pages", "table", "lengths", "frequencies"):
        setattr(a, name, FAKE)
    a.n_batch, a.n_heads, a.n_groups, a.tokens, a.dim, a.dim_v, a.rotated = 2, 4, 2, 3, 64, 64, 64
    a.page, a.table_len, a.n_pages, a.amplitude, a.sign = 16, 4, 8, 1.0, 1.0
    for k, x in over.items():
        setattr(a, k, x)
    return a


@no_device
@pytest.mark.parametrize("over,message", [
    ({"n_batch": 0}, "shape"), ({"tokens": 0}, "shape"), ({"n_heads": 0}, "shape"), ({"n_groups": 0}, "shape"),
    ({"dim": 0}, "widths"), ({"dim": 513}, "widths"), ({"rotated": 3}, "widths"), ({"rotated": 66}, "widths"),
    ({"rotated": -2}, "widths"), ({"dtype": 3}, "float32"), ({"q_out": 0}, "NULL"), ({"frequencies": 0}, "NULL"),
    ({"amplitude": float("nan")}, "amplitude"), ({"sign": 0.5}, "sign")])
def test_rotation_arguments(over, message):
    lib = _paged.paged_lib()
    for entry, rest in ((lib.logkv_rotary, {"v": 0}), (lib.logkv_paged_append, {})):
        a = rotary_args(**{**rest, **over})
        assert entry(C.byref(a), None) == _lib.LOGKV_EINVAL
        assert message in lib.logkv_last_error().decode()


@no_device
@pytest.mark.parametrize("over,message", [
    ({"page": 8}, "power of two"), ({"page": 48}, "power of two"), ({"table_len": -1}, "power of two"),
    ({"n_pages": -1}, "power of two"), ({"dim_v": 0}, "power of two"), ({"dim_v": 600}, "power of two"),
    ({"table_len": 1 << 28}, "power of two"), ({"cache_dtype": 2}, "bf16 or fp16"), ({"v": 0}, "NULL"), ({"k": 0}, "NULL"),
    ({"table": 0}, "NULL"), ({"v_pages": 0}, "NULL")])
def test_append_arguments(over, message):
    lib = _paged.paged_lib()
    a = rotary_args(**over)
    assert lib.logkv_paged_append(C.byref(a), None) == _lib.LOGKV_EINVAL
    assert message in lib.logkv_last_error().decode()


@no_device
def test_a_rotation_takes_no_values_and_some_rows():
    lib = _paged.paged_lib()
    for over, message in (({}, "values"), ({"v": 0, "q": 0, "k": 0}, "shape"), ({"v": 0, "k_out": 0}, "NULL")):
        assert lib.logkv_rotary(C.byref(rotary_args(**over)), None) == _lib.LOGKV_EINVAL
        assert message in lib.logkv_last_error().decode()
    assert lib.logkv_rotary(None, None) == lib.logkv_paged_append(None, None) == _lib.LOGKV_EINVAL


def paged_args(**over):
    a = _paged.PagedArgs()
    for name in ("q", "k", "v", "k_pages", "v_pages", "table", "prefix_table", "out", "lengths", "prefix_lengths"):
        setattr(a, name, FAKE)
    a.n_batch, a.n_heads, a.n_groups, a.tq, a.dk, a.dv, a.scale = 4, 4, 2, 3, 64, 64, 0.125
    a.page, a.table_len, a.n_pages, a.n_prefixes, a.prefix_len = 16, 4, 8, 2, 5
    for s in ("q", "o"):
        setattr(a, s + "_sb", 4 * 3 * 64), setattr(a, s + "_sh", 3 * 64), setattr(a, s + "_st", 64)
    for s in ("k", "v"):
        setattr(a, s + "_sb", 2 * 3 * 64), setattr(a, s + "_sg", 3 * 64), setattr(a, s + "_st", 64)
    for s in ("kp", "vp"):
        setattr(a, s + "_sp", 2 * 16 * 64), setattr(a, s + "_sg", 16 * 64), setattr(a, s + "_st", 64)
    for k, x in over.items():
        setattr(a, k, x)
    return a


@no_device
@pytest.mark.parametrize("over,message", [
    ({"n_heads": 3}, "shape"), ({"tq": 0}, "shape"), ({"n_batch": 0}, "shape"), ({"n_prefixes": 3}, "divide"),
    ({"n_prefixes": -1}, "divide"), ({"n_batch": 40000}, "65535"), ({"tq": 1 << 18}, "2^19"), ({"dk": 60}, "multiples of 8"),
    ({"dv": 264}, "multiples of 8"), ({"page": 24}, "power of two"), ({"table_len": 1 << 27}, "power of two"),
    ({"prefix_len": 1 << 27}, "power of two"), ({"dtype": 2}, "bf16 or fp16"), ({"q": 0}, "NULL"), ({"table": 0}, "NULL"),
    ({"k_pages": 0}, "NULL"), ({"prefix_table": 0}, "prefix is NULL"), ({"bias": FAKE}, "contiguous rows"),
    ({"q": FAKE + 8}, "16-byte aligned"), ({"kp_st": 68}, "16-byte aligned"), ({"vp_sp": 4}, "16-byte aligned"),
    ({"o_st": 66}, "8-byte aligned"), ({"scale": 0.0}, "scale"), ({"bias_scale": float("inf")}, "bias_scale"),
    ({"visible": FAKE, "counts": FAKE}, "mask")])
def test_paged_attention_arguments(over, message):
    lib, a = _paged.paged_lib(), paged_args(**over)
    assert lib.logkv_paged_attention(C.byref(a), FAKE, 1 << 40, None) == _lib.LOGKV_EINVAL
    assert message in lib.logkv_last_error().decode()


@no_device
def test_workspace_is_checked():
    lib, a = _paged.paged_lib(), paged_args()
    need = lib.logkv_paged_workspace_bytes(C.byref(a))
    assert need > lib.logkv_paged_workspace_bytes(C.byref(paged_args(n_prefixes=0))) > 0
    for ws, size in ((FAKE, need - 1), (None, need), (FAKE + 8, need)):
        assert lib.logkv_paged_attention(C.byref(a), ws, size, None) == _lib.LOGKV_EINVAL
        assert "workspace" in lib.logkv_last_error().decode()
    assert lib.logkv_paged_workspace_bytes(C.byref(paged_args(dk=4))) == -1
    assert lib.logkv_paged_workspace_bytes(None) == -1
    assert lib.logkv_paged_attention(None, FAKE, need, None) == _lib.LOGKV_EINVAL


def test_every_size_has_a_plan():
    """Workspaces of calls of any size that the entry point takes, in bounded time."""
    import random

    lib, r, planned = _paged.paged_lib(), random.Random(5), 0
    for _ in range(2000):
        n = r.choice((1, 1, 2, 3, 8))
        groups = r.choice((1, 2, 8, 16))
        a = _paged.PagedArgs(
            n_batch=n * r.choice((1, 1, 2, 7, 64, 500)), n_groups=groups, n_heads=groups * r.choice((1, 1, 2, 3, 8, 64)),
            tq=r.choice((1, 1, 2, 7, 33, 300, 4000)), dk=8 * r.randint(1, 32), dv=8 * r.randint(1, 32), dtype=r.choice((0, 1)),
            page=r.choice((16, 64, 1 << 20)), table_len=r.choice((0, 1, 5, 100, 1024)), n_prefixes=n,
            prefix_len=r.choice((0, 1, 3, 50, 1000)), prefix_table=r.choice((0, 1)))
        need = lib.logkv_paged_workspace_bytes(C.byref(a))
        planned += need > 0
        assert need > 0 or any(x in lib.logkv_last_error().decode() for x in ("2^19", "65535", "too many"))
    assert planned > 1500
