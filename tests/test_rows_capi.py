"""The C ABI of the row attention operators without a GPU: the ctypes table and structs against
include/logkv_rows.h, and the argument checks that precede every launch (fake addresses, so only
where no HIP device is visible)."""

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from logkv_amd import _lib, _rows

HEADER = Path(__file__).resolve().parents[1] / "include" / "logkv_rows.h"
FAKE = 0x10000
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device addresses are only passed where no HIP device is visible")


def header_text():
    return re.sub(r"/\*.*?\*/", " ", HEADER.read_text(), flags=re.S)


def test_library_exports_the_header():
    names = set(re.findall(r"\b(logkv_[a-z0-9_]+)\s*\(", header_text()))
    assert names == set(_rows.SIGNATURES)
    handle = C.CDLL(str(_lib.LIB_PATH))
    for name in sorted(names):
        assert hasattr(handle, name), name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc")
def test_ctypes_structs_match_the_header(tmp_path):
    structs = {"logkv_rows_args": _rows.RowsArgs, "logkv_evict_args": _rows.EvictArgs}
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
    # The packed form of the structs.
    for cls, pack in ((_rows.RowsArgs, _rows.pack_rows), (_rows.EvictArgs, _rows.pack_evict)):
        values = [3 * i + 1 for i in range(len(cls._fields_))]
        a = cls.from_buffer_copy(pack(*values))
        assert [getattr(a, f) for f, _ in cls._fields_] == values


def rows_args(**over):
    a = _rows.RowsArgs()
    for name in ("q", "k", "v", "cache_k", "cache_v", "out", "visible", "lengths"):
        setattr(a, name, FAKE)
    a.n_batch, a.n_heads, a.n_groups, a.tq, a.cap, a.dk, a.dv, a.scale = 2, 4, 2, 3, 64, 64, 64, 0.125
    for s in ("q", "o"):
        setattr(a, s + "_sb", 4 * 3 * 64), setattr(a, s + "_sh", 3 * 64), setattr(a, s + "_st", 64)
    for s in ("k", "v"):
        setattr(a, s + "_sb", 2 * 3 * 64), setattr(a, s + "_sg", 3 * 64), setattr(a, s + "_st", 64)
    for s in ("ck", "cv"):
        setattr(a, s + "_sb", 2 * 64 * 64), setattr(a, s + "_sg", 64 * 64), setattr(a, s + "_st", 64)
    a.vis_sb, a.vis_st, a.w_sb, a.w_sg = 0, 3, 128, 64
    for k, x in over.items():
        setattr(a, k, x)
    return a


@no_device
@pytest.mark.parametrize("over,message", [
    ({"n_heads": 3}, "shape"), ({"tq": 0}, "shape"), ({"n_batch": 0}, "shape"), ({"n_batch": 40000}, "65535"),
    ({"tq": 1 << 19}, "2^19"), ({"dk": 60}, "multiples of 8"), ({"dv": 264}, "multiples of 8"), ({"cap": -1}, "capacity"),
    ({"dtype": 2}, "bf16 or fp16"), ({"q": 0}, "NULL"), ({"cache_v": 0}, "NULL"), ({"q": FAKE + 8}, "16-byte aligned"),
    ({"ck_st": 68}, "16-byte aligned"), ({"k_sg": 4}, "16-byte aligned"), ({"o_st": 66}, "8-byte aligned"),
    ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"visible": 0}, "mask"), ({"weights": FAKE}, "mask"),
    ({"counts": FAKE}, "mask")])
def test_tree_attention_arguments(over, message):
    lib, a = _rows.rows_lib(), rows_args(**over)
    assert lib.logkv_tree_attention(C.byref(a), FAKE, 1 << 40, None) == _lib.LOGKV_EINVAL
    assert message in lib.logkv_last_error().decode()


@no_device
def test_weight_attention_arguments():
    lib = _rows.rows_lib()
    for over, message in (({}, "takes weights"), ({"weights": FAKE}, "no mask"),
                          ({"weights": FAKE, "visible": 0, "bias": FAKE}, "no bias")):
        a = rows_args(**over)
        assert lib.logkv_weight_attention(C.byref(a), FAKE, 1 << 40, None) == _lib.LOGKV_EINVAL
        assert message in lib.logkv_last_error().decode()


@no_device
def test_workspace_is_checked():
    lib = _rows.rows_lib()
    a = rows_args()
    need = lib.logkv_rows_workspace_bytes(C.byref(a))
    assert need > 0
    for ws, size in ((FAKE, need - 1), (None, need), (FAKE + 8, need)):
        assert lib.logkv_tree_attention(C.byref(a), ws, size, None) == _lib.LOGKV_EINVAL
        assert "workspace" in lib.logkv_last_error().decode()
    assert lib.logkv_rows_workspace_bytes(C.byref(rows_args(dk=4))) == -1
    # The weights' scratch comes on top.
    more = lib.logkv_rows_workspace_bytes(C.byref(rows_args(weights=FAKE, visible=0)))
    assert more > need


def evict_args(**over):
    a = _rows.EvictArgs()
    for name in ("cache_k", "cache_v", "weights", "out_k", "out_v", "out_weights", "kept", "out_lengths", "lengths"):
        setattr(a, name, FAKE)
    a.n_batch, a.n_groups, a.cap, a.dk, a.dv, a.size, a.keep, a.recent = 1, 2, 64, 64, 64, 2, 32, 8
    for s in ("ck", "cv", "ok", "ov"):
        setattr(a, s + "_sb", 128 * 64), setattr(a, s + "_sg", 64 * 64), setattr(a, s + "_st", 64)
    for k, x in over.items():
        setattr(a, k, x)
    return a


@no_device
@pytest.mark.parametrize("over,message", [
    ({"n_groups": 0}, "shape"), ({"cap": 0}, "shape"), ({"keep": 0}, "keeps"), ({"recent": 33}, "keeps"),
    ({"recent": -1}, "keeps"), ({"size": 3}, "bytes"), ({"dk": 12}, "multiples of 16"), ({"kept": 0}, "NULL"),
    ({"positions": FAKE}, "NULL"), ({"cache_k": FAKE + 2}, "aligned"), ({"ov_st": 60}, "aligned")])
def test_eviction_arguments(over, message):
    lib, a = _rows.rows_lib(), evict_args(**over)
    assert lib.logkv_evict_rows(C.byref(a), None) == _lib.LOGKV_EINVAL
    assert message in lib.logkv_last_error().decode()


def test_python_refusals_on_the_host():
    """The Python layer's checks that need no device; a CPU tensor is refused, never computed."""
    from logkv_amd import log_kv_evict, log_kv_tree_attention, log_kv_weight_attention

    bf = torch.bfloat16
    q, k, ck = torch.zeros(1, 4, 3, 64, dtype=bf), torch.zeros(1, 2, 3, 64, dtype=bf), torch.zeros(1, 2, 10, 64, dtype=bf)
    eye, w = torch.eye(3, dtype=torch.bool), torch.zeros(1, 2, 10)
    with pytest.raises(ValueError, match="ROCm device"):
        log_kv_tree_attention(q, k, k, ck, ck, 5, eye, 0.1)
    with pytest.raises(ValueError, match="ROCm device"):
        log_kv_weight_attention(q, k, k, ck, ck, w, 5, 0.1)
    with pytest.raises(ValueError, match="ROCm device"):
        log_kv_evict(ck, ck, w, 5, 3)
    for bad in (eye[:2], eye.float(), torch.ones(2, 3, 3, dtype=torch.bool)):
        with pytest.raises(ValueError, match="visible"):
            log_kv_tree_attention(q, k, k, ck, ck, 5, bad, 0.1)
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        log_kv_tree_attention(q, k, k, ck.float(), ck.float(), 5, eye, 0.1)
    with pytest.raises(ValueError, match="dividing"):
        log_kv_tree_attention(q[:, :3], k, k, ck, ck, 5, eye, 0.1)
    with pytest.raises(ValueError, match="one per query"):
        log_kv_tree_attention(q, k[:, :, :2], k, ck, ck, 5, eye, 0.1)
    with pytest.raises(ValueError, match="weights must be float32"):
        log_kv_weight_attention(q, k, k, ck, ck, w.double(), 5, 0.1)
    with pytest.raises(ValueError, match="counts"):
        log_kv_weight_attention(q, k, k, ck, ck, w, 5, 0.1, counts=torch.zeros(3, dtype=torch.int32))
    for keep, recent in ((0, 0), (3, 4), (3, -1)):
        with pytest.raises(ValueError, match="keep"):
            log_kv_evict(ck, ck, w, 5, keep, recent=recent)


@no_device
def test_weight_attention_needs_a_cache():
    lib, a = _rows.rows_lib(), rows_args(weights=FAKE, visible=0, cap=0)
    assert lib.logkv_weight_attention(C.byref(a), FAKE, 1 << 40, None) == _lib.LOGKV_EINVAL
    assert "at least one row" in lib.logkv_last_error().decode()


def test_rows_written_must_not_share_memory():
    """Expanded tensors where a call writes."""
    from logkv_amd import EvictedRows, log_kv_weight_attention
    from logkv_amd.row_attention import _check_evict_out, _repeats

    bf = torch.bfloat16
    q, k, ck = torch.zeros(2, 4, 3, 64, dtype=bf), torch.zeros(2, 2, 3, 64, dtype=bf), torch.zeros(2, 2, 10, 64, dtype=bf)
    w = torch.zeros(2, 2, 10)
    for cache, weights in ((ck, w[:1].expand(2, -1, -1)), (ck[:, :1].expand(-1, 2, -1, -1), w)):
        with pytest.raises(ValueError, match="share memory"):
            log_kv_weight_attention(q, k, k, cache, ck, weights, 5, 0.1)
    with pytest.raises(NotImplementedError, match="gradient"):
        log_kv_weight_attention(q, k, k, ck, ck, w.clone().requires_grad_(), 5, 0.1)
    assert not _repeats(ck[:1].expand(1, -1, -1, -1)) and _repeats(ck[:1].expand(2, -1, -1, -1))

    def out(**over):
        fields = {"k": ck.clone(), "v": ck.clone(), "weights": w.clone(), "positions": None,
                  "kept": torch.zeros(2, 2, 4, dtype=torch.int32), "lengths": torch.zeros(2, dtype=torch.int32), **over}
        return EvictedRows(**fields)

    _check_evict_out(out(), ck, ck.clone(), w, None, None, 4)
    for over in ({"k": ck[:1].clone().expand(2, -1, -1, -1)}, {"weights": w[:, :1].clone().expand(-1, 2, -1)}):
        with pytest.raises(ValueError, match="out must be"):
            _check_evict_out(out(**over), ck, ck.clone(), w, None, None, 4)
