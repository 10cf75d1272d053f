"""Which rows the packed scan's CTAs take (csrc/mms_units.h, compiled for the host): every row of a
list that is as it should be once, and none outside the arrays or the workspace whatever the list holds."""
from __future__ import annotations

import ctypes
import itertools
import subprocess

import pytest
import torch

from conftest import REPO

SOURCE = """
#include "mms_units.h"
extern "C" int unit_rows(int unit, int fulls, int seg, int s, int first, int end, int *out) {
    mms::Unit u{};
    const int ok = mms::unit_rows(unit, fulls, seg, s, first, end, u);
    const int v[] = {u.s, u.i, u.segs, u.t0, u.t1, u.row};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
    return ok;
}
"""


@pytest.fixture(scope="module")
def unit_rows(tmp_path_factory):
    where = tmp_path_factory.mktemp("units")
    (where / "units.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-I", str(REPO / "mamba-metal-scan_b200/csrc"),
                    str(where / "units.cpp"), "-o", str(where / "units.so")], check=True)
    lib, out = ctypes.CDLL(str(where / "units.so")), (ctypes.c_int * 6)()

    def call(unit, fulls, seg, s, first, end):
        """(s, i, segs, t0, t1, row), or None where the unit has no rows."""
        return tuple(out) if lib.unit_rows(unit, fulls, seg, s, first, end, out) else None

    return call


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 64, 65, 96, 130])
def test_any_sequence_for_any_unit_stays_inside(unit_rows, rows):
    """Every pair of starts within the rows, for every unit: also those that a search among starts that do not
    ascend comes to, such as a sequence behind the unit (starts 32, 0, 32 of 32 rows)."""
    seg, fulls = 32, rows // 32
    edges = sorted({e for k in range(0, rows + 1, 32) for e in (k - 1, k, k + 1, k + 7) if 0 <= e <= rows} | {rows})
    for first, end in itertools.product(edges, edges):
        for unit in range(fulls + 2):
            u = unit_rows(unit, fulls, seg, 0, first, end)
            if u is None:
                continue
            _, i, segs, t0, t1, row = u
            assert 0 <= i < segs and first <= t0 <= t1 <= max(first, end) <= rows
            if i < segs - 1:                               # leaves its end in the workspace
                assert row + i < fulls
            if segs > 1:                                   # so does its sequence what it goes on from
                assert rows > seg and row < fulls


def test_every_row_once(unit_rows):
    g = torch.Generator().manual_seed(0)
    for _ in range(300):
        count = int(torch.randint(1, 9, (1,), generator=g))
        lens = [int(v) for v in torch.randint(0, 120, (count,), generator=g)]
        lens = [v // 32 * 32 if v % 3 == 0 else v % 5 if v % 3 == 1 else v for v in lens]
        starts = [int(torch.randint(0, 40, (1,), generator=g))]
        for n in lens:
            starts.append(starts[-1] + n)
        rows, seg = starts[-1] + int(torch.randint(0, 40, (1,), generator=g)), 32
        fulls, taken, ends = rows // seg, [0] * rows, set()
        for unit in range(fulls + count):
            s = unit - fulls
            if unit < fulls:
                s = max([i for i in range(count) if starts[i] // seg <= unit], default=-1)
            u = unit_rows(unit, fulls, seg, s, starts[s], starts[s + 1]) if s >= 0 else None
            if u is None:
                continue
            for t in range(u[3], u[4]):
                taken[t] += 1
            if u[1] < u[2] - 1:
                assert u[5] + u[1] not in ends
                ends.add(u[5] + u[1])
        assert taken == [int(starts[0] <= t < starts[-1]) for t in range(rows)]
