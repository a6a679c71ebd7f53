"""The paged cache's attention at the ends of its types' ranges: scores far
from zero, whose differences float32 still holds; queries and values of very unlike sizes."""
import math

import numpy as np
import pytest

from tests.test_gpu_paged import KINDS, Case, dev, held, want

pytestmark = pytest.mark.gpu


def put(c):
    """The case's rows, changed after it was made, into its cache."""
    t = c.torch
    c.cache.store(c.layer, dev(t, c.k), dev(t, c.v), dev(t, c.seq), dev(t, c.pos), c.table)


@pytest.mark.parametrize("lens,width", [([300, 1], None), ([3000, 40, 1100], 50)])  # whole rows, and rows cut and joined
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", [10, 16, 19, 20, 30, 80, 121])
@pytest.mark.parametrize("kind", KINDS)
def test_scores_far_from_zero(gpu, kind, exponent, sign, lens, width):
    """Scores +-127 2^e + j 2^(e - 17), small j: whole units in the last place
    of float32, which the kernel forms exactly (keys and queries are whole
    numbers times powers of two, int8 scales 1).

    A weight is then off by the rounding of its exponent, at most 40 in
    magnitude where it counts: 40 2^-24 ln 2 twice (from the wave's reference,
    and that from the row's) and the constant's share of as much, below
    2^-18; the quotient has two such.  The sums' roundings are those of the
    other tests: 2^-17 + 2^-20 + (len / 16 + 64) 2^-24 of sum p |v|.
    """
    c = Case(gpu, kind, 64, 1, lens, width=width)
    c.k[:] = 0
    c.k[:, 0, 0] = sign * 127
    step = c.pos // 128 + c.rng.integers(0, 4, len(c.pos))  # larger along the row: the reference moves
    c.k[:, 0, 1] = step
    put(c)
    q = np.zeros((len(lens), 2, 64), np.float32)
    q[:, :, 0] = 2.0 ** exponent
    q[:, 0, 1], q[:, 1, 1] = 2.0 ** (exponent - 17), -(2.0 ** (exponent - 17))
    _, got = c.attend(2, scale=1.0, q=q)
    v = held(kind, c.v)[:, 0].astype(np.float64)
    for r, n in enumerate(lens):
        at = c.rows(r)
        for h, way in enumerate((1, -1)):
            s = way * step[at] * 2.0 ** (exponent - 17)
            p = np.exp(s - s.max())
            p /= p.sum()
            bar = (2.0 ** -17 + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -24) * (p @ np.abs(v[at])) + 1e-37
            assert np.all(np.abs(got[r, h] - p @ v[at]) <= bar), (r, h)


@pytest.mark.parametrize("where", ["one", "first", "last", "spread"])
@pytest.mark.parametrize("r", [20, 28, 36, 50, 80])
def test_large_values_behind_low_scores(gpu, r, where):
    """Positions whose values are 2^r times the others' and whose scores lie
    100 below them take nothing from the others, for half of the heads; for
    the other half they are all there is.  The bar is the other tests': a
    share of sum p |v|."""
    for lens, width in (([260, 40], None), ([2500, 33, 700], 50)):
        c = Case(gpu, "int8", 64, 2, lens, width=width, seed=r)
        n = np.array(lens)[c.seq]
        large = {"one": c.pos == n * 2 // 3, "first": c.pos < n // 2, "last": c.pos >= n // 2, "spread": c.pos % 5 == 1}[where]
        w = c.rng.normal(0, 1, 64).astype(np.float32)
        c.k *= np.float32(0.3)
        c.k[large] = (-800 / (w @ w)) * w
        c.v *= np.where(large, np.float32(2.0 ** (r / 2)), np.float32(2.0 ** (-r / 2)))[:, None, None]
        put(c)
        q = (c.rng.normal(0, 0.01, (len(lens), 8, 64)) + w * np.array([1, -1] * 4)[:, None]).astype(np.float32)
        _, got = c.attend(8, q=q)
        k, v = held("int8", c.k), held("int8", c.v)
        for i in range(len(lens)):
            at = c.rows(i)
            o, bar = want(q[i], k[at], v[at], 0.125, 0.0, None)
            assert np.all(np.abs(got[i] - o) <= bar), (lens, i)


def test_values_outgrown_as_scores_rise(gpu):
    """Scores that rise by 3 a block while the values' scale falls by 2^5 a
    block: the largest weight is a new position's, then an old one's."""
    for step, fall in ((3.0, 5.0), (3.0, 4.0), (6.0, 5.0), (-3.0, -5.0), (-6.0, -5.0)):
        c = Case(gpu, "int8", 64, 1, [640, 900], width=40)
        block = c.pos // 32
        c.k *= np.float32(0.05)
        c.k[:, 0, 0] = block * step
        c.v *= (2.0 ** (-fall * (block - 14))).astype(np.float32)[:, None, None]
        put(c)
        q = c.rng.normal(0, 1, (2, 3, 64)).astype(np.float32)
        q[:, :, 0] = 8
        _, got = c.attend(3, q=q)
        k, v = held("int8", c.k), held("int8", c.v)
        for i in range(2):
            at = c.rows(i)
            o, bar = want(q[i], k[at], v[at], 0.125, 0.0, None)
            assert np.all(np.abs(got[i] - o) <= bar), (step, fall, i)


@pytest.mark.parametrize("down", [16, 20, 24, 28])
@pytest.mark.parametrize("kind", KINDS)
def test_small_queries_beside_a_large_one(gpu, kind, down):
    """A head's largest query meets keys of zero: the scores come from queries
    2^-down of it, held as well as any other."""
    c = Case(gpu, kind, 64, 2, [300, 5, 64])
    c.k[:, :, 7] = 0
    put(c)
    q = c.rng.normal(0, 1.5 * 2.0 ** -down, (3, 4, 64)).astype(np.float32)
    q[:, :, 7] = 3.0
    scale = 2.0 ** down / 8
    _, got = c.attend(4, scale=scale, q=q)
    k, v = held(kind, c.k), held(kind, c.v)
    for r in range(3):
        at = c.rows(r)
        o, bar = want(q[r], k[at], v[at], scale, 0.0, None)
        assert np.all(np.abs(got[r] - o) <= bar), r


def test_large_keys_and_small_queries(gpu):
    """int8 keys near float32's end and queries as small: neither factor of a score may overflow before both are in."""
    for up, scale in ((-100, 0.125), (100, 0.125), (117, 0.125), (117, 0.1), (112, 0.003)):
        c = Case(gpu, "int8", 64, 1, [200, 33])
        c.k *= np.float32(2.0 ** up)
        put(c)
        q = (c.rng.normal(0, 1.5, (2, 4, 64)) * 2.0 ** -up).astype(np.float32)
        _, got = c.attend(4, q=q, scale=scale)
        k, v = held("int8", c.k), held("int8", c.v)
        for r in range(2):
            at = c.rows(r)
            o, bar = want(q[r], k[at], v[at], scale, 0.0, None)
            assert np.all(np.abs(got[r] - o) <= bar), (up, r)


@pytest.mark.parametrize("kind", KINDS)
def test_largest_floats(gpu, kind):
    """Finite rows up to float32's largest, by store and by a step: float16
    keeps its own largest for them, int8 their codes; infinities stay apart."""
    torch, lm, ctx = gpu
    big = [65504.0, 65519.0, 65520.0, 3e38, 3.1e38, 3.4028234663852886e38]
    x = np.ones((2 * len(big), 1, 64), np.float32)
    x[:, 0, 5] = np.array(big + [-b for b in big], np.float32)
    n = len(x)
    c = Case(gpu, kind, 64, 1, [n + 1])
    c.cache.store(0, dev(torch, x), dev(torch, x), dev(torch, np.zeros(n, np.int32)), dev(torch, np.arange(n, dtype=np.int32)),
                  c.table)
    k, v = (torch.zeros(n, 1, 64, device="cuda") for _ in range(2))
    c.cache.fetch(0, k, v, dev(torch, np.zeros(n, np.int32)), dev(torch, np.arange(n, dtype=np.int32)), c.table)
    assert np.array_equal(k.cpu().numpy(), held(kind, x)) and np.array_equal(v.cpu().numpy(), held(kind, x))
    w, _ = c.work(1, 1)
    pos, zero = (dev(torch, np.array([i], np.int32)) for i in (n, 0))
    for row in x:
        r = dev(torch, row[None])
        out = torch.zeros(1, 1, 64, device="cuda")
        c.cache.step(0, out, torch.zeros(1, 1, 64, device="cuda"), r, r, pos, c.table, w)
        c.cache.fetch(0, k[:1], v[:1], zero, pos, c.table)
        assert np.array_equal(k[:1].cpu().numpy(), held(kind, row[None])) and torch.equal(k[:1], v[:1])
        assert bool(out.isfinite().all()) or kind == "int8"  # (a sum of 13 values near float32's end)
    if kind == "f16":
        inf = torch.full((1, 1, 64), float("inf"), device="cuda")
        c.cache.store(0, inf, -inf, zero, pos, c.table)
        c.cache.fetch(0, k[:1], v[:1], zero, pos, c.table)
        assert torch.equal(k[:1], inf) and torch.equal(v[:1], -inf)


def test_old_values_beside_slowly_rising_scores(gpu):
    """One head's scores rise by an eighth from each of a wave's blocks to the
    next, the other's by more than 1, so that the reference moves each time;
    the values of the first blocks are 2^200 times the others' and stay what
    the first head's result is made of.  1025 rows, so that none is cut and a
    wave has close to two hundred blocks."""
    lens = [0] * 1025
    lens[7] = 24000
    c = Case(gpu, "int8", 64, 1, lens, page=256)
    block = (c.pos // 32).astype(np.float32)
    c.k[:] = 0
    c.k[:, 0, 0] = c.k[:, 0, 1] = block
    c.v *= np.where(block < 8, np.float32(2.0 ** 100), np.float32(2.0 ** -100))[:, None, None]
    put(c)
    q = np.zeros((1025, 2, 64), np.float32)
    q[7, 0, 0], q[7, 1, 1] = 0.03125, 0.3
    _, got = c.attend(2, scale=1.0, q=q)
    at = c.rows(7)
    o, bar = want(q[7], held("int8", c.k[at]), held("int8", c.v[at]), 1.0, 0.0, None)
    assert np.all(np.abs(got[7] - o) <= bar)
    assert not got[:7].any() and not got[8:].any()


def test_large_queries_across_large_keys(gpu):
    """Queries whose products with the keys' scales pass float32's range, and meet keys of zero: scores of 0."""
    c = Case(gpu, "int8", 64, 1, [200, 33])
    c.k *= np.float32(2.0 ** 30)
    c.k[:, :, 9] = 0
    put(c)
    q = np.zeros((2, 4, 64), np.float32)
    q[:, :, 9] = 2.0 ** 120
    q[1, 2, 8] = 2.0 ** -30  # less than what the head's largest leaves of it: no score either
    _, got = c.attend(4, q=q)
    v = held("int8", c.v)
    for r in range(2):
        at = c.rows(r)
        o, bar = want(np.zeros((4, 64), np.float32), 0 * v[at], v[at], 0.125, 0.0, None)
        assert np.all(np.abs(got[r] - o) <= bar), r
