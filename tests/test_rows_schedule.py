"""The order of the tiled row attention kernel's LDS accesses, walked on the CPU from the functions that the kernel takes
its buffers from: between two barriers no buffer is written that is read, and every read finds the rows it is for."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "logkv_amd" / "csrc" / "rows_schedule.hpp"

PROGRAM = """
#include <cstdio>
#include "{header}"
template <int RB> void one() {{
  typedef logkv::RowsSchedule<RB> S;
  printf("%d %d %d %d", RB, S::kAhead, S::kKBuffers, S::kVBuffers);
  for (int i = 0; i < S::kKBuffers; ++i) printf(" %d", S::next_k(i));
  for (int i = 0; i < S::kVBuffers; ++i) printf(" %d", S::next_v(i));
  printf("\\n");
}}
int main() {{ one<1>(); one<2>(); return 0; }}
"""


def walk(tiles, blocks, ahead, next_k, next_v):
    """Faults of a share of ``tiles`` tiles: (iteration, buffer) pairs written where they are read, reads of other rows."""
    k_holds, v_holds = {0: 0, next_k[0]: min(1, tiles - 1)}, {0: 0}     # stored before the first barrier
    faults, k, v = [], 0, 0
    for t in range(tiles):
        reads, writes = [], []
        far = next_k[k]
        for _ in range(ahead - 1):
            far = next_k[far]
        for kb in range(blocks):
            reads.append(("v", v, t))
            # Scores of the block to come; with more than one a tile, then the first operands of the one after it.
            for to_come in (kb + 1,) if blocks == 1 else (kb + 1, kb + 2):
                tile = t + to_come // blocks
                if tile < tiles:
                    assert tile - t <= 1
                    reads.append(("k", next_k[k] if tile > t else k, tile))
        if t + 1 < tiles:
            writes.append(("v", next_v[v], t + 1))
        if t + ahead < tiles:
            writes.append(("k", far, t + ahead))
        for kind, buffer, tile in reads:
            if (k_holds if kind == "k" else v_holds).get(buffer) != tile:
                faults.append((t, kind, buffer, "holds another tile"))
            if any(w[:2] == (kind, buffer) for w in writes):
                faults.append((t, kind, buffer, "read and written"))
        for kind, buffer, tile in writes:
            (k_holds if kind == "k" else v_holds)[buffer] = tile
        k, v = next_k[k], next_v[v]
    return faults


@pytest.fixture(scope="module")
def schedules(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++")
    d = tmp_path_factory.mktemp("schedule")
    (d / "s.cpp").write_text(PROGRAM.format(header=HEADER))
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", str(d / "s.cpp"), "-o", str(d / "s")], check=True)
    out = {}
    for line in subprocess.run([str(d / "s")], check=True, capture_output=True, text=True).stdout.splitlines():
        blocks, ahead, nk, nv, *rest = map(int, line.split())
        out[blocks] = (ahead, rest[:nk], rest[nk:nk + nv])
    return out


@pytest.mark.parametrize("blocks", [1, 2])
def test_no_buffer_is_written_where_it_is_read(schedules, blocks):
    ahead, next_k, next_v = schedules[blocks]
    for tiles in (1, 2, 3, 4, 5, 17, 30):
        assert walk(tiles, blocks, ahead, next_k, next_v) == []


def test_two_blocks_a_tile_do_not_fit_two_buffers(schedules):
    """The walk finds the overlap that a third buffer is there for, and none for one block."""
    assert walk(5, 1, 2, [1, 0], [1, 0]) == []
    faults = walk(5, 2, 2, [1, 0], [1, 0])
    assert (0, "k", 0, "read and written") in faults
    assert len(schedules[2][1]) == 3
