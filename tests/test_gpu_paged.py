"""The paged key / value cache and one token's attention over it (llmq_pkv_*)
against its definition in float64.

Rows: what fetch gives is compared bit by bit with the definition's rounding
(scale max|x| times the float 1 / 127, codes away from zero at ties; or
float16's).  Attention: over the fetched rows in float64.  With S the sum
of |q_d k_d| times |scale| (a bar has no sign), a score is off by at most
  d = S (2^-22 + (hd + 8) 2^-24) + 4 2^-24 |s| (+ 2^-22 cap; + 2^-23 |bias|)
(queries held to 22 bits, the products added in float32, a few roundings of
the score itself), a weight by the factor 1 + 2^-21 + d of the row's largest d,
twice (in the sums of p v and of p), and the sums by a rounding per 16
positions and 64 more: the bar is (2 d + 2^-20 + (len / 16 + 64) 2^-24) times
the sum of p |v|.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def held(kind, x):
    """Rows as the cache holds them, float32."""
    if kind == "f16":
        return np.clip(x, -65504, 65504).astype(np.float16).astype(np.float32)
    m = np.abs(x).max(-1, keepdims=True)
    s = np.where(m < np.float32(2.0 ** -120), np.float32(1), m * (np.float32(1) / np.float32(127))).astype(np.float32)
    y = x * (np.float32(1) / s)
    return (np.sign(y) * np.floor(np.abs(y) + np.float32(0.5))).astype(np.float32) * s


class Case:
    """Ragged sequences over scattered pages; every other position of the
    pages, and the spare pages, hold NaN (what an earlier user may leave)."""

    def __init__(self, gpu, kind, hd, n_kv, lens, page=64, layers=1, layer=0, seed=0, big=1.0, width=None):
        self.torch, self.lm, self.ctx = gpu
        torch = self.torch
        rng = np.random.default_rng(seed + hd + n_kv + sum(lens))
        self.rng, self.kind, self.hd, self.n_kv, self.lens, self.layer = rng, kind, hd, n_kv, list(lens), layer
        need = [-(-max(n, 1) // page) for n in lens]
        self.width = width or max(need) + 1
        n_pages = sum(need) + 2
        ids = rng.permutation(n_pages).astype(np.int32)
        self.table_np = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table_np[r, :n] = ids[at:at + n]
            at += n
        self.cache = self.lm.PagedKV(self.ctx, layers, n_pages, page, n_kv, hd, kind)
        self.table = dev(torch, self.table_np)
        # NaN everywhere first
        every = dev(torch, np.arange(n_pages, dtype=np.int32)[:, None])
        sq = np.repeat(np.arange(n_pages, dtype=np.int32), page)
        ps = np.tile(np.arange(page, dtype=np.int32), n_pages)
        nan = torch.full((len(sq), n_kv, hd), float("nan"), device="cuda")
        self.cache.store(layer, nan, nan, dev(torch, sq), dev(torch, ps), every)
        self.seq = np.concatenate([np.full(n, r, np.int32) for r, n in enumerate(lens)])
        self.pos = np.concatenate([np.arange(n, dtype=np.int32) for n in lens])
        order = rng.permutation(len(self.seq))
        self.seq, self.pos = self.seq[order], self.pos[order]
        n = len(self.seq)
        self.k = (rng.normal(0, 1, (n, n_kv, hd)) * rng.uniform(0.2, 2, (1, n_kv, hd)) * big).astype(np.float32)
        self.v = (rng.normal(0, 1, (n, n_kv, hd)) * big).astype(np.float32)
        self.cache.store(layer, dev(torch, self.k), dev(torch, self.v), dev(torch, self.seq), dev(torch, self.pos),
                         self.table)

    def rows(self, r):
        at = np.where(self.seq == r)[0]
        at = at[np.argsort(self.pos[at])]
        return at

    def work(self, rows, heads):
        # a workspace of stale NaN, with a guard behind it
        n = self.cache.work_bytes(rows, heads)
        w = self.torch.full((n + 64,), 0xFF, dtype=self.torch.uint8, device="cuda")
        return w[:n], w

    def attend(self, heads, lens=None, scale=None, cap=0.0, slopes=None, q=None):
        torch = self.torch
        n = len(self.lens)
        q = self.rng.normal(0, 1.5, (n, heads, self.hd)).astype(np.float32) if q is None else q
        out = torch.full((n, heads, self.hd), float("nan"), device="cuda")
        w, whole = self.work(n, heads)
        ln = dev(torch, np.asarray(self.lens if lens is None else lens, np.int32))
        self.cache.attend(self.layer, out, dev(torch, q), ln, self.table, w, scale=scale, cap=cap,
                          slopes=None if slopes is None else dev(torch, slopes))
        torch.cuda.synchronize()
        assert bool((whole[w.numel():] == 0xFF).all()), "wrote past its workspace"
        return q, out.cpu().numpy()


def want(q, k, v, scale, cap, slopes):
    """(out, bar) of one row in float64: q [H, hd], k and v [n, n_kv, hd]."""
    H, hd = q.shape
    n, n_kv, _ = k.shape
    if n == 0:
        return np.zeros((H, hd)), np.zeros((H, hd))
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    out, bar = np.zeros((H, hd)), np.zeros((H, hd))
    for h in range(H):
        kh, vh = k[:, h // (H // n_kv)], v[:, h // (H // n_kv)]
        s = kh @ q[h] * scale
        d = np.abs(kh) @ np.abs(q[h]) * abs(scale) * (2.0 ** -22 + (hd + 8) * 2.0 ** -24) + 2.0 ** -22 * np.abs(s)
        if cap:
            s, d = cap * np.tanh(s / cap), d + 2.0 ** -22 * cap
        if slopes is not None:
            b = float(slopes[h]) * (np.arange(n) - (n - 1))
            s, d = s + b, d + 2.0 ** -23 * np.abs(b)
        p = np.exp(s - s.max())
        live = p > 2.0 ** -40  # below, a position adds nothing that a rounding does not
        out[h] = p @ vh / p.sum()
        bar[h] = (2 * d[live].max() + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -24) * (p @ np.abs(vh) / p.sum())
    return out, bar + 1e-37


def check(c, heads, lens=None, scale=None, cap=0.0, slopes=None):
    q, got = c.attend(heads, lens, scale, cap, slopes)
    sc = 1 / math.sqrt(c.hd) if scale is None else scale
    k, v = held(c.kind, c.k), held(c.kind, c.v)
    worst = 0.0
    for r in range(len(c.lens)):
        at = c.rows(r)[:max(0, c.lens[r] if lens is None else lens[r])]
        o, bar = want(q[r], k[at], v[at], sc, cap, slopes)
        assert np.isfinite(got[r]).all(), r
        worst = max(worst, np.max(np.abs(got[r] - o) / np.maximum(bar, 1e-37)))
    assert worst <= 1.0, worst


KINDS = ["int8", "f16"]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_store_and_fetch(gpu, kind, hd):
    torch, lm, ctx = gpu
    c = Case(gpu, kind, hd, 3, [1, 64, 65, 130], page=128, layers=2, layer=1)
    ko, vo = (torch.full(c.k.shape, float("nan"), device="cuda") for _ in range(2))
    sq, ps = dev(torch, c.seq), dev(torch, c.pos)
    c.cache.fetch(1, ko, vo, sq, ps, c.table)
    assert np.array_equal(ko.cpu().numpy(), held(kind, c.k)) and np.array_equal(vo.cpu().numpy(), held(kind, c.v))
    c.cache.fetch(0, ko, vo, sq, ps, c.table)  # the other layer has nothing
    assert not ko.any() and not vo.any()
    # strided rows (views of a wider tensor), values past float16's range, rows of zeros, tiny rows
    wide = torch.zeros(len(c.seq), 9, hd, device="cuda")
    x = c.k.copy()
    x[0], x[1], x[2] = 0.0, 1e-39, 1e5
    x[3, 0, 0], x[4, 0, 1] = -7e4, 3e38
    wide[:, 3:6] = dev(torch, x)
    wide[:, 6:] = dev(torch, c.v)
    c.cache.store(1, wide[:, 3:6], wide[:, 6:], sq, ps, c.table)
    c.cache.fetch(1, ko, vo, sq, ps, c.table)
    assert np.array_equal(ko.cpu().numpy(), held(kind, x)) and np.array_equal(vo.cpu().numpy(), held(kind, c.v))


@pytest.mark.parametrize("kind", KINDS)
def test_store_runs_of_rows(gpu, kind):
    """Rows in order (as prompts come), of sequences that begin and end
    anywhere: runs from one row to several blocks, at every offset in a block,
    with padding rows and jumps between them."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(11)
    for trial in range(6):
        n_seq, width, page = 7, 5, 64
        table = rng.permutation(n_seq * width + 2)[:n_seq * width].astype(np.int32).reshape(n_seq, width)
        cache = lm.PagedKV(ctx, 1, n_seq * width + 2, page, 2, 64, kind)
        seq, pos = [], []
        for s in range(n_seq):
            at = int(rng.integers(0, 70))
            while at < width * page:
                n = int(rng.choice([1, 2, 31, 32, 33, 64, 100]))
                run = list(range(at, min(at + n, width * page)))
                seq += [s] * len(run)
                pos += run
                at = run[-1] + 1 + int(rng.choice([0, 0, 1, 40]))
                if rng.random() < 0.3:
                    pad = int(rng.integers(1, 40))
                    seq += [-1] * pad
                    pos += list(range(pad))
        seq, pos = np.array(seq, np.int32), np.array(pos, np.int32)
        k, v = (rng.normal(0, 1, (len(seq), 2, 64)).astype(np.float32) for _ in range(2))
        d = lambda a: dev(torch, a)  # noqa: E731
        cache.store(0, d(k), d(v), d(seq), d(pos), d(table))
        ko, vo = (torch.full(k.shape, float("nan"), device="cuda") for _ in range(2))
        cache.fetch(0, ko, vo, d(seq), d(pos), d(table))
        live = (seq >= 0)[:, None, None]
        assert np.array_equal(ko.cpu().numpy(), np.where(live, held(kind, k), 0))
        assert np.array_equal(vo.cpu().numpy(), np.where(live, held(kind, v), 0))
        # and one row at a time
        back = rng.permutation(len(seq))
        cache.fetch(0, ko, vo, d(seq[back]), d(pos[back]), d(table))
        assert np.array_equal(ko.cpu().numpy(), np.where(live, held(kind, k), 0)[back])


@pytest.mark.parametrize("kind", KINDS)
def test_store_leaves_out_and_overwrites_nothing_else(gpu, kind):
    """Padding rows, positions past the table, pages that are none: nothing is
    written; fetch gives zeros for them."""
    torch, lm, ctx = gpu
    c = Case(gpu, kind, 64, 2, [70, 200, 3])
    sq, ps = dev(torch, c.seq), dev(torch, c.pos)
    bad = [(-1, 0), (3, 0), (0, -1), (0, c.width * 64), (0, 64 * (c.width - 1)), (2, 64), (1, 2 ** 31 - 1),
           (-2 ** 31, 5)]
    bs, bp = (dev(torch, np.array([b[i] for b in bad], np.int32)) for i in range(2))
    one = torch.full((len(bad), 2, 64), 5.0, device="cuda")
    c.cache.store(0, one, one, bs, bp, c.table)
    c.cache.fetch(0, one, one.clone(), bs, bp, c.table)
    assert not one.any()
    table = c.table.clone()
    table[0, 0], table[1, 1], table[1, 2] = 10 ** 6, -5, c.cache.n_pages  # none of the cache's
    two = torch.full((3, 2, 64), 5.0, device="cuda")
    s3, p3 = dev(torch, np.array([0, 1, 1], np.int32)), dev(torch, np.array([3, 64, 190], np.int32))
    c.cache.store(0, two, two, s3, p3, table)
    ko, vo = (torch.full(c.k.shape, float("nan"), device="cuda") for _ in range(2))
    c.cache.fetch(0, ko, vo, sq, ps, c.table)
    assert np.array_equal(ko.cpu().numpy(), held(kind, c.k)) and np.array_equal(vo.cpu().numpy(), held(kind, c.v))


def test_nonfinite_rows(gpu):
    torch, lm, ctx = gpu
    for kind in KINDS:
        c = Case(gpu, kind, 64, 1, [8])
        x = torch.ones(3, 1, 64, device="cuda")
        x[0, 0, 5], x[1, 0, 63] = float("nan"), float("inf")
        z = torch.zeros(3, dtype=torch.int32, device="cuda")
        p = dev(torch, np.arange(3, dtype=np.int32))
        c.cache.store(0, x, x, z, p, c.table)
        k, v = torch.zeros_like(x), torch.zeros_like(x)
        c.cache.fetch(0, k, v, z, p, c.table)
        for t in (k, v):
            if kind == "int8":
                assert bool(t[:2].isnan().all())
            else:
                assert bool(t[0, 0, 5].isnan()) and bool(t[1, 0, 63].isinf()) and bool(t[0, 0, :5].eq(1).all())
            assert bool(t[2].eq(1).all())


LENS = [[1], [0, 1, 2, 15, 16, 17], [63, 64, 65, 0], [31, 32, 33, 127, 128, 129], [700, 1, 255, 257]]


@pytest.mark.parametrize("heads,n_kv", [(1, 1), (12, 12), (8, 1), (9, 1), (21, 3), (32, 4), (17, 1)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_attend(gpu, kind, hd, heads, n_kv):
    for i, lens in enumerate(LENS):
        print("attend", kind, hd, heads, n_kv, lens, flush=True)
        c = Case(gpu, kind, hd, n_kv, lens, page=(64, 128, 192)[i % 3], layers=1 + i % 2, layer=i % 2, seed=i)
        check(c, heads)


@pytest.mark.parametrize("kind", KINDS)
def test_attend_long_and_ragged(gpu, kind):
    c = Case(gpu, kind, 128, 2, [20001, 5, 0, 4096, 1023], page=256)
    check(c, 8)
    c = Case(gpu, kind, 64, 1, [70000], page=512)
    check(c, 4)


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("kind", KINDS)
def test_attend_weights_hold_22_bits(gpu, kind, n):
    """Sequences of one or two positions, 32000 weights: with so few terms a
    weight's own error shows.  A weight is held to 22 bits (2^-22 of it), its
    scale, exponential, sum and quotient round a few times: 2^-20 of sum p |v|
    in all, besides the scores' error, which one position does not have."""
    torch, lm, ctx = gpu
    rows, heads = 4000, 8
    c = Case(gpu, kind, 64, heads, [n] * rows)
    q, got = c.attend(heads)
    order = np.lexsort((c.pos, c.seq))
    k, v = (held(kind, x)[order].reshape(rows, n, heads, 64).astype(np.float64) for x in (c.k, c.v))
    s = np.einsum("rnhd,rhd->rnh", k, q.astype(np.float64)) / 8
    d = np.einsum("rnhd,rhd->rnh", np.abs(k), np.abs(q.astype(np.float64))) / 8 * (2.0 ** -22 + 72 * 2.0 ** -24)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    out = np.einsum("rnh,rnhd->rhd", p, v)
    size = np.einsum("rnh,rnhd->rhd", p, np.abs(v))
    bar = (2.0 ** -20 + (2 * d.max(1) if n > 1 else 0 * d.max(1)))[..., None] * size + 1e-37
    assert np.max(np.abs(got - out) / bar) <= 1.0


@pytest.mark.parametrize("kind", KINDS)
def test_attend_many_rows(gpu, kind):
    rng = np.random.default_rng(5)
    c = Case(gpu, kind, 64, 2, [int(x) for x in rng.integers(0, 90, 300)])
    check(c, 4)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 128, 129, 700, 1024, 1025])
@pytest.mark.parametrize("kind", KINDS)
def test_attend_rows_cut_into_segments(gpu, kind, rows):
    """Tables for more than a row that is never cut, at the edges of the rows
    that a lane and the plan hold: short rows, empty ones and a few long ones,
    whose segments are joined."""
    rng = np.random.default_rng(rows)
    for heads, n_kv in ((8, 1), (18, 2)):
        print("segments", kind, rows, heads, flush=True)
        lens = rng.integers(0, 70, rows)
        lens[rng.random(rows) < 0.1] = 0
        for n in (2500, 1057, 3001, 300)[:rows]:
            lens[rng.integers(0, rows)] = n
        c = Case(gpu, kind, 64, n_kv, [int(x) for x in lens], width=50)
        check(c, heads)
        c.cache.free()


@pytest.mark.parametrize("kind", KINDS)
def test_step_rows_cut_into_segments(gpu, kind):
    """Steps whose new token is in a segment's first, last and only block, and attend after them."""
    torch, lm, ctx = gpu
    lens = [2048, 2047, 1, 33, 511, 512, 513, 1024, 0, 1999]
    c = Case(gpu, kind, 128, 2, [n + 1 for n in lens], width=40)
    n, heads = len(lens), 18
    x = dev(torch, c.rng.normal(0, 1, (n, heads + 4, 128)).astype(np.float32))
    pos = dev(torch, np.array(lens, np.int32))
    out, again = (torch.full((n, heads, 128), float("nan"), device="cuda") for _ in range(2))
    w, _ = c.work(n, heads)
    c.cache.step(0, out, x[:, :heads], x[:, heads:heads + 2], x[:, heads + 2:], pos, c.table, w)
    c.cache.attend(0, again, x[:, :heads], pos + 1, c.table, w)
    for r, p in enumerate(lens):
        at = [torch.full((p + 1,), r, dtype=torch.int32, device="cuda"),
              torch.arange(p + 1, dtype=torch.int32, device="cuda")]
        k, v = (torch.empty(p + 1, 2, 128, device="cuda") for _ in range(2))
        c.cache.fetch(0, k, v, *at, c.table)
        k, v = k.cpu().numpy(), v.cpu().numpy()
        assert np.array_equal(k[p], held(kind, x[r, heads:heads + 2].cpu().numpy()))
        o, bar = want(x[r, :heads].cpu().numpy(), k, v, 1 / math.sqrt(128), 0.0, None)
        for y in (out, again):
            assert np.all(np.abs(y[r].cpu().numpy() - o) <= bar), r


@pytest.mark.parametrize("cap,bias,scale", [(30.0, False, None), (0.0, True, None), (5.0, True, 0.3), (0.0, False, 1e-9),
                                            (0.0, False, -0.125), (0.0, False, 3.0)])
@pytest.mark.parametrize("kind", KINDS)
def test_attend_cap_bias_scale(gpu, kind, cap, bias, scale):
    c = Case(gpu, kind, 64, 3, [300, 1, 64, 129], page=64)
    slopes = (2.0 ** (-8.0 * np.arange(1, 7) / 6)).astype(np.float32) if bias else None
    check(c, 6, scale=scale, cap=cap, slopes=slopes)


@pytest.mark.parametrize("big", [1e-6, 1e4])
@pytest.mark.parametrize("kind", KINDS)
def test_attend_sizes_of_values(gpu, kind, big):
    """Keys and values far from 1 (float16's subnormals and its range's end)."""
    c = Case(gpu, kind, 64, 2, [200, 70], big=big)
    check(c, 4, scale=0.125 / big)


def test_attend_uneven_value_scales(gpu):
    """Value rows 2^-60 to 2^60 apart in one sequence: the int8 scales span it."""
    torch, lm, ctx = gpu
    c = Case(gpu, "int8", 64, 1, [260])
    at = c.rows(0)
    c.v[at] *= (2.0 ** np.linspace(-60, 60, 260)).astype(np.float32)[:, None, None]
    c.cache.store(0, dev(torch, c.k), dev(torch, c.v), dev(torch, c.seq), dev(torch, c.pos), c.table)
    check(c, 2)
    c.v[at] = c.v[at][::-1]
    c.cache.store(0, dev(torch, c.k), dev(torch, c.v), dev(torch, c.seq), dev(torch, c.pos), c.table)
    check(c, 2)


def test_attend_zero_rows_among_small(gpu):
    """Rows of zeros, whose int8 scale says nothing, beside values near 2^-60."""
    torch, lm, ctx = gpu
    c = Case(gpu, "int8", 64, 1, [100])
    at = c.rows(0)
    c.v[at] *= np.float32(2.0 ** -60)
    c.v[at[::3]] = 0
    c.k[at[1::3]] = 0
    c.cache.store(0, dev(torch, c.k), dev(torch, c.v), dev(torch, c.seq), dev(torch, c.pos), c.table)
    check(c, 2)


@pytest.mark.parametrize("kind", KINDS)
def test_attend_lengths_past_the_table_and_bad_pages(gpu, kind):
    torch, lm, ctx = gpu
    c = Case(gpu, kind, 64, 2, [128, 200, 64], width=4)
    q, got = c.attend(4, lens=[-7, 200, 64])
    assert not got[0].any()
    # row 1's second page is none of the cache's: its positions are left out
    for bad in (-1, c.cache.n_pages, 2 ** 31 - 1):
        table = c.table.clone()
        table[1, 1] = bad
        keep = c.table
        c.table = table
        q, got = c.attend(4)
        c.table = keep
        k, v = held(kind, c.k), held(kind, c.v)
        at = np.concatenate([c.rows(1)[:64], c.rows(1)[128:]])
        o, bar = want(q[1], k[at], v[at], 0.125, 0.0, None)
        assert np.all(np.abs(got[1] - o) <= bar)
    table = torch.full_like(c.table, -1)
    c.table = table
    q, got = c.attend(4)
    assert not got.any()
    # a length past the table's row ends with it
    c = Case(gpu, kind, 64, 2, [128, 64], width=2)
    q, got = c.attend(4, lens=[2 ** 31 - 1, 64])
    k, v = held(kind, c.k), held(kind, c.v)
    o, bar = want(q[0], k[c.rows(0)], v[c.rows(0)], 0.125, 0.0, None)
    assert np.all(np.abs(got[0] - o) <= bar)


@pytest.mark.parametrize("kind", KINDS)
def test_attend_nan_and_inf(gpu, kind):
    """A NaN or infinite query or key gives NaN to its own rows and heads only."""
    torch, lm, ctx = gpu
    c = Case(gpu, kind, 64, 2, [70, 70, 70])
    q = c.rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    q[0, 1, 3], q[2, 2, 60] = np.nan, np.inf
    clean = np.nan_to_num(q, nan=0.0, posinf=0.0)
    _, base = c.attend(4, q=clean)
    _, got = c.attend(4, q=q)
    hit = np.zeros((3, 4), bool)
    hit[0, 1] = hit[2, 2] = True
    assert np.isnan(got[hit]).all()
    assert np.array_equal(got[~hit], base[~hit])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,heads,n_kv", [(64, 12, 12), (64, 8, 1), (128, 32, 8), (128, 18, 1)])
def test_step(gpu, kind, hd, heads, n_kv):
    """A step is store then attend; rows without a token give zeros and store nothing."""
    torch, lm, ctx = gpu
    lens = [1, 0, 64, 65, 500, 128]
    c = Case(gpu, kind, hd, n_kv, lens, page=64)
    n = len(lens)
    qkv = c.rng.normal(0, 1, (n, heads + 2 * n_kv, hd)).astype(np.float32)
    x = dev(torch, qkv)
    pos = dev(torch, np.array(lens, np.int32) - 1)
    seq = dev(torch, np.arange(n, dtype=np.int32))
    w, _ = c.work(n, heads)
    out = torch.full((n, heads, hd), float("nan"), device="cuda")
    c.cache.step(0, out, x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:], pos, c.table, w)
    ko, vo = (torch.zeros(n, n_kv, hd, device="cuda") for _ in range(2))
    c.cache.fetch(0, ko, vo, seq, pos, c.table)
    live = np.array(lens) > 0
    assert np.array_equal(ko.cpu().numpy()[live], held(kind, qkv[:, heads:heads + n_kv])[live])
    assert np.array_equal(vo.cpu().numpy()[live], held(kind, qkv[:, heads + n_kv:])[live])
    got = out.cpu().numpy()
    for r in range(n):
        at = c.rows(r)
        if lens[r]:
            c.k[at[-1]], c.v[at[-1]] = qkv[r, heads:heads + n_kv], qkv[r, heads + n_kv:]
        o, bar = want(qkv[r, :heads], held(kind, c.k[at]), held(kind, c.v[at]), 1 / math.sqrt(hd), 0.0, None)
        assert np.all(np.abs(got[r] - o) <= bar), r
    # everything else in the cache is as it was
    ka, va = (torch.zeros(c.k.shape, device="cuda") for _ in range(2))
    c.cache.fetch(0, ka, va, dev(torch, c.seq), dev(torch, c.pos), c.table)
    assert np.array_equal(ka.cpu().numpy(), held(kind, c.k)) and np.array_equal(va.cpu().numpy(), held(kind, c.v))
    again = torch.zeros_like(out)
    c.cache.attend(0, again, x[:, :heads].contiguous(), dev(torch, np.array(lens, np.int32)), c.table, w)
    assert torch.equal(again, out)


def test_results_do_not_depend_on_neighbours_or_repeats(gpu):
    """Twice the same bits."""
    torch, lm, ctx = gpu
    c = Case(gpu, "int8", 128, 2, [3000, 10, 777])
    q, a = c.attend(8)
    _, b = c.attend(8, q=q)
    assert np.array_equal(a, b)


def test_cache_past_32_bits(gpu):
    """Offsets past 2^32 bytes: the last layer's last pages."""
    torch, lm, ctx = gpu
    cache = lm.PagedKV(ctx, 3, 700, 4096, 4, 128, "int8")  # 1.47e9 codes a layer
    assert cache.nbytes() > 2 * 2 ** 32
    table = torch.tensor([[699, 698]], dtype=torch.int32, device="cuda")
    n = 4096 + 77
    rng = np.random.default_rng(1)
    k, v = (rng.normal(0, 1, (n, 4, 128)).astype(np.float32) for _ in range(2))
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    cache.store(2, dev(torch, k), dev(torch, v), seq, pos, table)
    q = rng.normal(0, 1, (1, 8, 128)).astype(np.float32)
    out = torch.zeros(1, 8, 128, device="cuda")
    w = torch.empty(cache.work_bytes(1, 8), dtype=torch.uint8, device="cuda")
    cache.attend(2, out, dev(torch, q), dev(torch, np.array([n], np.int32)), table, w)
    o, bar = want(q[0], held("int8", k), held("int8", v), 1 / math.sqrt(128), 0.0, None)
    assert np.all(np.abs(out.cpu().numpy()[0] - o) <= bar)
    cache.free()


@pytest.mark.parametrize("kind", KINDS)
def test_step_in_a_graph(gpu, kind):
    """A captured step follows the positions and tables in device memory: ten
    replays, with eager work between, equal eager steps on another cache."""
    torch, lm, ctx = gpu
    lens = [60, 5, 1]
    a, b = (Case(gpu, kind, 64, 2, lens, width=3, seed=9) for _ in range(2))
    n, heads = 3, 8
    x = torch.zeros(n, heads + 4, 64, device="cuda")
    pos = dev(torch, np.array(lens, np.int32))
    table = a.table.clone()
    table[0, 1] = table[0, 0].item() + 0  # the first row's second page: set below
    spare = [p for p in range(a.cache.n_pages) if p not in set(a.table_np.ravel().tolist())]
    table[0, 1] = spare[0]
    tb = b.table.clone()
    spare_b = [p for p in range(b.cache.n_pages) if p not in set(b.table_np.ravel().tolist())]
    tb[0, 1] = spare_b[0]
    w, _ = a.work(n, heads)
    out = torch.zeros(n, heads, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin()
            a.cache.step(0, out, x[:, :heads], x[:, heads:heads + 2], x[:, heads + 2:], pos, table, w, cap=20.0)
            pos.add_(1)
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    pb = dev(torch, np.array(lens, np.int32))
    wb, _ = b.work(n, heads)
    ob = torch.zeros_like(out)
    for i in range(10):
        x.copy_(dev(torch, a.rng.normal(0, 1, tuple(x.shape)).astype(np.float32)))
        graph.replay()
        b.cache.step(0, ob, x[:, :heads], x[:, heads:heads + 2], x[:, heads + 2:], pb, tb, wb, cap=20.0)
        pb.add_(1)
        torch.cuda.synchronize()
        assert torch.equal(out, ob), i


@pytest.mark.parametrize("kind", KINDS)
def test_store_and_fetch_in_a_graph(gpu, kind):
    """A captured store and fetch take the rows, positions and tables that are there at each replay."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(4)
    c = lm.PagedKV(ctx, 1, 12, 64, 2, 64, kind)
    T = 70
    k, v, ko, vo = (torch.zeros(T, 2, 64, device="cuda") for _ in range(4))
    seq, pos = (torch.zeros(T, dtype=torch.int32, device="cuda") for _ in range(2))
    table = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin()
            c.store(0, k, v, seq, pos, table)
            c.fetch(0, ko, vo, seq, pos, table)
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in range(5):
        table.copy_(dev(torch, rng.permutation(12).reshape(3, 4).astype(np.int32)))
        s, first = rng.integers(0, 3), rng.integers(0, 180)
        seq.fill_(int(s))
        pos.copy_(torch.arange(T, dtype=torch.int32) + int(first))
        x, y = (rng.normal(0, 1, (T, 2, 64)).astype(np.float32) for _ in range(2))
        k.copy_(dev(torch, x))
        v.copy_(dev(torch, y))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(ko.cpu().numpy(), held(kind, x)) and np.array_equal(vo.cpu().numpy(), held(kind, y)), i


def test_streams(gpu):
    """Two caches on two streams, and a context moved between them."""
    torch, lm, ctx = gpu
    c = Case(gpu, "int8", 64, 2, [900, 3])
    q, base = c.attend(8)
    torch.cuda.synchronize()
    outs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        try:
            with torch.cuda.stream(s):
                ctx.set_stream(s)
                outs.append(c.attend(8, q=q)[1])
        finally:
            ctx.set_stream(torch.cuda.current_stream())
    assert all(np.array_equal(o, base) for o in outs)


def test_cache_outlives_its_context(gpu):
    torch, lm, ctx = gpu
    other = lm.Context(0)
    c = lm.PagedKV(other, 1, 4, 64, 2, 64)
    other.close()
    assert c.nbytes() == 2 * 4 * 2 * 64 * (64 + 4)
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    i = z(1, dtype=torch.int32)
    with pytest.raises(lm.LlmqError):  # no context, no call
        c.store(0, z(1, 2, 64), z(1, 2, 64), i, i, i[None])
    c.ctx = ctx
    c.store(0, z(1, 2, 64) + 3, z(1, 2, 64), i, i, i[None])
    k, v = z(1, 2, 64), z(1, 2, 64)
    c.fetch(0, k, v, i, i, i[None])
    assert np.allclose(k.cpu().numpy(), 3)
    c.free()
    with pytest.raises(lm.LlmqError):
        c.fetch(0, k, v, i, i, i[None])
    c.free()


def test_refusals(gpu):
    torch, lm, ctx = gpu
    for args in ((0, 4, 64, 2, 64), (1, 0, 64, 2, 64), (1, 4, 32, 2, 64), (1, 4, 96, 2, 64), (1, 4, 8192, 2, 64),
                 (1, 4, 64, 0, 64), (1, 4, 64, 2, 80)):
        with pytest.raises(lm.LlmqError):
            lm.PagedKV(ctx, *args)
    with pytest.raises(ValueError):
        lm.PagedKV(ctx, 1, 4, 64, 2, 64, "int4")
    c = lm.PagedKV(ctx, 1, 4, 64, 2, 64)
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    i32 = dict(dtype=torch.int32)
    table, ln, w = z(3, 2, **i32), z(3, **i32), z(c.work_bytes(3, 4), dtype=torch.uint8)
    q, out = z(3, 4, 64), z(3, 4, 64)
    c.attend(0, out, q, ln, table, w)
    bad = [
        lambda: c.attend(1, out, q, ln, table, w),
        lambda: c.attend(0, out, z(3, 5, 64), ln, table, w),
        lambda: c.attend(0, z(3, 3, 64), z(3, 3, 64), ln, table, w),
        lambda: c.attend(0, out, q.half(), ln, table, w),
        lambda: c.attend(0, out, z(3, 64, 4).transpose(1, 2), ln, table, w),
        lambda: c.attend(0, out, q, ln.long(), table, w),
        lambda: c.attend(0, out, q, ln[:2], table, w),
        lambda: c.attend(0, out, q, ln, table[:2], w),
        lambda: c.attend(0, out, q, ln, table, w[:-1]),
        lambda: c.attend(0, out, q, ln, table, w, cap=-1.0),
        lambda: c.attend(0, out, q, ln, table, w, cap=float("nan")),
        lambda: c.attend(0, out, q, ln, table, w, cap=1e-40),
        lambda: c.attend(0, out, q, ln, table, w, scale=float("nan")),
        lambda: c.attend(0, out, q, ln, table, w, slopes=z(3)),
        lambda: c.attend(0, out, q.cpu(), ln, table, w),
        lambda: c.store(0, z(2, 2, 64), z(3, 2, 64), ln[:2], ln[:2], table),
        lambda: c.store(0, z(2, 3, 64), z(2, 3, 64), ln[:2], ln[:2], table),
        lambda: c.store(-1, z(2, 2, 64), z(2, 2, 64), ln[:2], ln[:2], table),
        lambda: c.step(0, out, q, z(3, 2, 64), z(3, 2, 64), ln, table, w),  # strides differ
        lambda: c.step(0, out, q, z(3, 2, 32), z(3, 2, 32), ln, table, w),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, lm.LlmqError)):
            f()
            print("not refused:", i)
    # nothing to do is no error
    e = z(0, **i32)
    c.store(0, z(0, 2, 64), z(0, 2, 64), e, e, table)
    c.attend(0, z(0, 4, 64), z(0, 4, 64), e, z(0, 2, **i32), w)
    torch.cuda.synchronize()
