"""The units of mxfp4_units.h, compiled for the host: every tile of every expert once, and never a row outside the tensor, also where
the counts on the device add up to more than 32 bits."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The kernels' walk: 64 experts at a time, a lane each, prefix sums by steps of 1, 2, 4, ... lanes; a unit is looked up in the first
# expert whose sum lies above it.  `wrap` plants plain 32-bit sums in their place.
SOURCE = r"""
#include "mxfp4_units.h"
using namespace esmoe;
static uint32_t add(uint32_t a, uint32_t b, int wrap) { return wrap ? a + b : sum_or_most(a, b); }
struct Some {
  int m[64], off[64];
  uint32_t end[64];
  void read(int e0, const int* rows, const int* offsets, int experts, int total, int wrap) {
    for (int l = 0; l < 64; l++) {
      const int e = e0 + l;
      off[l] = e < experts ? offsets[e] : 0;
      m[l] = e < experts ? fp4_rows(rows[e], off[l], total) : 0;
      end[l] = fp4_tiles(m[l]);
    }
    for (int d = 1; d < 64; d *= 2)
      for (int l = 63; l >= d; l--) end[l] = add(end[l], end[l - d], wrap);
  }
};
extern "C" {
long most_units(int experts, int total) { return fp4_most_units(experts, total); }
// all units together, as the sums have it
uint32_t units(const int* rows, const int* offsets, int experts, int total, int wrap) {
  uint32_t n = 0;
  Some s;
  for (int e0 = 0; e0 < experts; e0 += 64) s.read(e0, rows, offsets, experts, total, wrap), n = add(n, s.end[63], wrap);
  return n;
}
int unit(const int* rows, const int* offsets, int experts, int total, uint32_t u, int wrap, int* out) {
  uint32_t before = 0;
  Some s;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    s.read(e0, rows, offsets, experts, total, wrap);
    if (u >= add(before, s.end[63], wrap)) {
      before = add(before, s.end[63], wrap);
      continue;
    }
    for (int l = 0; l < 64; l++)
      if (s.end[l] > u - before) {
        const Fp4Unit g = fp4_unit(e0 + l, s.off[l], s.m[l], u - before, l ? s.end[l - 1] : 0);
        out[0] = g.expert, out[1] = g.row0, out[2] = g.rows;
        return 1;
      }
    return 0;
  }
  return 0;
}
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("host")
    (d / "host.cpp").write_text(SOURCE)
    csrc = os.path.join(ROOT, "expert_specialization_moe_amd", "csrc")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{csrc}", str(d / "host.cpp"), "-o", str(d / "host.so")], check=True)
    lib = ctypes.CDLL(str(d / "host.so"))
    lib.most_units.restype, lib.units.restype = ctypes.c_long, ctypes.c_uint32
    return lib


def _int32(x):
    return np.ascontiguousarray(x, np.int32)


def _units(host, rows, offsets, total, wrap=0):
    r, o = _int32(rows), _int32(offsets)
    return host.units(r.ctypes.data_as(ctypes.c_void_p), o.ctypes.data_as(ctypes.c_void_p), len(r), total, wrap)


def _unit(host, rows, offsets, total, u, wrap=0):
    r, o, out = _int32(rows), _int32(offsets), np.zeros(3, np.int32)
    found = host.unit(r.ctypes.data_as(ctypes.c_void_p), o.ctypes.data_as(ctypes.c_void_p), len(r), total, ctypes.c_uint32(u), wrap,
                      out.ctypes.data_as(ctypes.c_void_p))
    return tuple(int(v) for v in out) if found else None


@pytest.mark.parametrize("experts", [1, 3, 64, 65, 200, 1024])
def test_every_tile_once(host, experts):
    rng = np.random.default_rng(experts)
    rows = rng.integers(0, 50, experts) * (rng.random(experts) < 0.6)
    rows[-1] = 17
    offsets = np.concatenate([[0], np.cumsum(rows)[:-1]])
    total = int(rows.sum())
    want = [(e, int(o) + t, min(16, int(m) - t)) for e, (m, o) in enumerate(zip(rows, offsets)) for t in range(0, int(m), 16)]
    n = _units(host, rows, offsets, total)
    assert n == len(want) <= host.most_units(experts, total)
    assert [_unit(host, rows, offsets, total, u) for u in range(n)] == want
    assert _unit(host, rows, offsets, total, n) is None


# (experts, rows of the tensor): all of them say that they own every row
@pytest.mark.parametrize("experts,total", [(1024, 1 << 25), (1000, (1 << 25) + 37), (64, 1 << 30), (1024, (1 << 31) - 1), (130, 2 ** 29 + 5)])
def test_counts_that_add_up_to_more_than_32_bits(host, experts, total):
    rows, offsets = [total] * experts, [0] * experts
    each = (total + 15) // 16
    n, limit = _units(host, rows, offsets, total), host.most_units(experts, total)
    assert n == min(experts * each, 2 ** 32 - 1) and limit < 2 ** 31
    for u in sorted({0, 1, each - 1, each, limit // 3, limit // 2, limit - 1, 2 ** 31 - 1, min(n, 2 ** 32 - 1) - 1}):
        if u < n:
            assert _unit(host, rows, offsets, total, u) == (u // each, u % each * 16, min(16, total - u % each * 16))


def test_plain_sums_would_leave_the_rows(host):
    """What saturation is for: with sums that wrap, a unit below the limit is looked up in an expert that it does not belong to."""
    experts, total = 64, 1 << 30
    rows, offsets = [total] * experts, [0] * experts
    limit = host.most_units(experts, total)
    outside = 0
    for u in np.linspace(0, limit - 1, 1000).astype(np.int64):
        good, bad = _unit(host, rows, offsets, total, int(u)), _unit(host, rows, offsets, total, int(u), 1)
        assert 0 <= good[1] < total and 0 < good[2] <= 16 and good[1] + good[2] <= total
        outside += bad is None or bad[1] < 0 or bad[1] >= total
    assert outside > 0


@pytest.mark.parametrize("m,off,want", [(5, 0, 5), (5, 90, 5), (20, 90, 10), (-1, 3, 0), (5, -1, 0), (5, 100, 0), (2 ** 31 - 1, 99, 1), (3, 2 ** 31 - 1, 0)])
def test_rows_are_cut_at_the_tensor(host, m, off, want):
    n = _units(host, [m], [off], 100)
    assert n == (want + 15) // 16
    if n:
        assert _unit(host, [m], [off], 100, 0) == (0, off, min(want, 16))
