"""The paged cache's attention at the ends of its types' ranges: scores far
from zero, whose differences float32 still holds."""
import math

import numpy as np
import pytest

from tests.test_gpu_paged import KINDS, Case, dev, held

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
