"""The division of an expert's rows in expert_mm_units.h, compiled for the host: every row in one unit and in one step, also where a tensor has
as many rows as there may be, 2^31 - 1."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include "expert_mm_units.h"
extern "C" {
int steps(int length, int each) { return esmoe::mm_steps(length, each); }
uint32_t units(int rows) { return esmoe::mm_units(rows); }
int unit_rows(int rows) { return esmoe::mm_unit_rows(rows); }
}
"""

MOST = (1 << 31) - 1
# from the largest multiples of 256, 64 and 32 on, and where the sum of rows and units passes 31 bits
LONG = [MOST - i for i in range(600)] + [MOST - (1 << 23) + i for i in range(-300, 300)] + [1 << 30, (1 << 30) + 1]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("host")
    (d / "host.cpp").write_text(SOURCE)
    csrc = os.path.join(ROOT, "expert_specialization_moe_amd", "csrc")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{csrc}", str(d / "host.cpp"), "-o", str(d / "host.so")], check=True)
    lib = ctypes.CDLL(str(d / "host.so"))
    lib.units.restype = ctypes.c_uint32
    return lib


@pytest.mark.parametrize("lengths", [range(0, 2000), LONG], ids=["short", "long"])
def test_units_hold_every_row_once(host, lengths):
    for rows in lengths:
        units, high = host.units(rows), host.unit_rows(rows)
        assert units == -(-rows // 256)
        if rows == 0:
            assert high == 0
            continue
        assert 0 < high <= 256 and high % 16 == 0
        assert (units - 1) * high <= MOST            # where a unit begins is an int
        assert units * high >= rows                  # ... and together they hold all rows,
        assert high - 16 < -(-rows // units)         # none higher than equal ones by a sixteen


@pytest.mark.parametrize("each", [32, 64])
@pytest.mark.parametrize("lengths", [range(0, 2000), LONG], ids=["short", "long"])
def test_steps_hold_every_row_once(host, lengths, each):
    for rows in lengths:
        assert host.steps(rows, each) == -(-rows // each)


# The walk of the weights' gradient for few tiles: a step's copies begin at row 32 * step, and the last step is the one that the next would be
# behind all rows of.  `step * 32 >= rows` instead, in 31 bits, never says so of the longest experts.
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 64, 65, (1 << 30) - 31, MOST - 32, MOST - 31, MOST - 30, MOST - 1, MOST])
def test_a_step_of_32_rows_begins_at_an_int(host, rows):
    last = host.steps(rows, 32) - 1
    assert 0 <= last * 32 < rows <= MOST and rows - last * 32 <= 32
    wraps = ctypes.c_int32((last + 1) * 32).value < rows
    assert wraps == (rows > MOST - 31)
