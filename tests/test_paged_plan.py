"""Where the paged cache keeps positions (csrc/paged_plan.h), on the CPU: the
value slots of a block are each used once and in the order the matrix-core
lanes take them, and no position, page or length leads outside the table or
the cache."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = """
#include "paged_plan.h"
extern "C" {
int block_positions(int e) { return pkv::block_positions(e); }
int value_slot(int e, int p) { return pkv::value_slot(e, p); }
int page_of(const int32_t *row, int64_t w, int page, int64_t pages, int64_t pos) {
    return pkv::page_of(row, w, page, pages, pos); }
int64_t clamp_len(int64_t n, int64_t w, int page) { return pkv::clamp_len(n, w, page); }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SRC)
    out = d / "plan.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "llm_mojo_amd", "csrc"),
                    str(d / "plan.cpp"), "-o", str(out)], check=True)
    L = ctypes.CDLL(str(out))
    i64 = ctypes.c_int64
    L.page_of.argtypes = [ctypes.c_void_p, i64, ctypes.c_int, i64, i64]
    L.clamp_len.argtypes, L.clamp_len.restype = [i64, i64, ctypes.c_int], i64
    return L


@pytest.mark.parametrize("elem", [1, 2])
def test_value_slots(plan, elem):
    b = plan.block_positions(elem)
    nt = b // 16
    assert b * elem == 64
    slots = [plan.value_slot(elem, p) for p in range(b)]
    assert sorted(slots) == list(range(b))
    for q in range(4):  # quarter q's bytes: its positions of tile 0, 1, ..
        mine = [slots.index(s) for s in range(q * 4 * nt, (q + 1) * 4 * nt)]
        assert mine == [16 * t + 4 * q + i for t in range(nt) for i in range(4)]


def test_pages_stay_inside(plan):
    rng = np.random.default_rng(0)
    for page in (64, 192, 4096):
        for width in (1, 2, 7):
            pages = 5
            row = rng.integers(-2, pages + 2, width).astype(np.int32)
            row[0] = np.iinfo(np.int32).max if width > 2 else row[0]
            for pos in (-2 ** 31, -page, -1, 0, 1, page - 1, page, width * page - 1, width * page, 2 ** 31 - 1, 2 ** 40):
                got = plan.page_of(row.ctypes.data, width, page, pages, pos)
                if not 0 <= pos < width * page:
                    assert got == -1
                else:
                    want = row[pos // page]
                    assert got == (want if 0 <= want < pages else -1)


def test_lengths(plan):
    for n, want in ((-2 ** 31, 0), (-1, 0), (0, 0), (1, 1), (640, 640), (641, 640), (2 ** 31 - 1, 640)):
        assert plan.clamp_len(n, 10, 64) == want
