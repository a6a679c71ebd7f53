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
int value_slot(int p) { return pkv::value_slot(p); }
int page_of(const int32_t *row, int64_t w, int page, int64_t pages, int64_t pos) {
    return pkv::page_of(row, w, page, pages, pos); }
int64_t clamp_len(int64_t n, int64_t w, int page) { return pkv::clamp_len(n, w, page); }
void plan(int64_t rows, int n_head, int n_kv, int hd, int64_t *out) {  // 7 numbers
    const pkv::Plan p = pkv::plan_of(rows, n_head, n_kv);
    const pkv::Work w = pkv::work_of(p, rows, n_head, hd);
    out[0] = p.tiles; out[1] = p.columns; out[2] = pkv::slots_of(p, rows); out[3] = w.ml; out[4] = w.sums; out[5] = w.bytes;
    out[6] = p.least;
}
uint32_t per_of(uint32_t total, int columns, uint32_t least) { return pkv::per_of(total, columns, least); }
uint32_t segments_of(uint32_t blocks, uint32_t per) { return pkv::segments_of(blocks, per); }
uint32_t segment_blocks(uint32_t blocks, uint32_t segments) { return pkv::segment_blocks(blocks, segments); }
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
    L.plan.argtypes = [i64, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    u32 = ctypes.c_uint32
    L.per_of.argtypes, L.per_of.restype = [u32, ctypes.c_int, u32], u32
    L.segments_of.argtypes, L.segments_of.restype = [u32, u32], u32
    L.segment_blocks.argtypes, L.segment_blocks.restype = [u32, u32], u32
    L.clamp_len.argtypes, L.clamp_len.restype = [i64, i64, ctypes.c_int], i64
    return L


def test_value_slots(plan):
    slots = [plan.value_slot(p) for p in range(32)]
    assert sorted(slots) == list(range(32))
    for q in range(4):  # quarter q's: its positions of tile 0, then of tile 1
        assert [slots.index(s) for s in range(8 * q, 8 * q + 8)] == [16 * t + 4 * q + i for t in (0, 1) for i in range(4)]


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


def blocks(rng, rows):
    kind = rng.integers(0, 4)
    if kind == 0:
        return np.zeros(rows, np.int64)
    nb = (2.0 ** rng.uniform(0, (6, 12, 22)[kind - 1], rows)).astype(np.int64)
    nb[rng.random(rows) < 0.2] = 0
    if kind == 3:
        nb[rng.integers(0, rows)] = 2 ** 31 - 1 - nb.sum()
    return nb


def test_segments_cover_the_rows_and_fit(plan):
    """Any lengths: a row's segments cover its blocks, and the slots of all rows fit the grid and the workspace."""
    rng = np.random.default_rng(1)
    out = np.zeros(7, np.int64)
    for _ in range(1500):
        rows = int(2 ** rng.uniform(0, 10))
        n_kv = int(rng.choice([1, 2, 3, 4, 8, 12, 32, 129, 600, 2000]))
        n_head = n_kv * int(rng.choice([1, 2, 7, 8, 9, 16, 71]))
        hd = int(rng.choice([64, 128]))
        plan.plan(rows, n_head, n_kv, hd, out.ctypes.data)
        tiles, columns, slots, ml, sums, size, least = (int(x) for x in out)
        assert tiles * 8 >= n_head // n_kv > (tiles - 1) * 8
        assert columns >= 1 and (columns == 1 or n_kv * tiles * columns <= 2048) and slots == rows + columns
        assert ml >= rows * 8 and sums >= ml + slots * n_head * 8 and size == sums + slots * n_head * hd * 4
        assert ml % 256 == 0 and sums % 256 == 0
        nb = blocks(rng, rows)
        per = plan.per_of(int(nb.sum()), columns, least)
        assert per >= least >= 8 and per % 4 == 0 and per <= 2 ** 31
        used = 0
        for n in (int(x) for x in nb):
            segments = plan.segments_of(n, per)
            used += segments
            assert segments == -(-n // per)
            if n == 0:
                continue
            seg = plan.segment_blocks(n, segments)
            count = plan.segments_of(n, seg)
            assert seg % 4 == 0 and 1 <= count <= segments and (segments - 1) * seg < 2 ** 32
            assert (count - 1) * seg < n <= count * seg  # the slots from count on are empty
            assert n > least or segments == 1
        assert used <= slots
    plan.plan(1025, 12, 12, 64, out.ctypes.data)
    assert out[1] == 0 and out[2] == 0 and out[5] == out[4]
