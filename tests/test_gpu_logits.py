"""Rules on logits and the greedy pick (llmq_adjust_logits).

The definition is a fixed order of float32 operations on each logit, so the
outputs are compared bit by bit with NumPy's (each operation rounded once,
the biases of a token added in the list's order), and the picks with the
first largest value.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F = np.float32


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def want(x, hist=None, hoff=None, rep=None, pres=None, freq=None, bias=None, mask=None):
    out = x.copy()
    rows, V = x.shape
    with np.errstate(all="ignore"):
        for r in range(rows):
            l = out[r]
            if hist is not None:
                ids = hist[hoff[r]:hoff[r + 1]]
                ids = ids[(ids >= 0) & (ids < V)]
                c = np.bincount(ids, minlength=V)
                at = c > 0
                y = l[at]
                if rep is not None:
                    y = np.where(y > 0, y / rep[r], y * rep[r]).astype(F)
                f, p = (F(0) if a is None else a[r] for a in (freq, pres))
                l[at] = y - (f * c[at].astype(F) + p)
            if bias is not None:
                ids, val, off = bias
                add = np.zeros(V, F)
                for i, b in zip(ids[off[r]:off[r + 1]], val[off[r]:off[r + 1]]):
                    if 0 <= i < V:
                        add[i] = add[i] + b
                l[:] = l + add
            if mask is not None:
                bits = (mask[r].view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1
                l[bits.reshape(-1)[:V] == 0] = -np.inf
    pick = np.full(rows, -1, np.int64)
    for r in range(rows):
        y = np.where(np.isnan(out[r]), F(-np.inf), out[r])
        if y.max() > -np.inf:
            pick[r] = np.argmax(y)
    return out, pick


def ragged(rng, rows, most, V, lo=0):
    n = rng.integers(0, most + 1, rows)
    n[rng.integers(0, rows)] = most
    off = np.concatenate([[0], np.cumsum(n)]).astype(np.int64)
    return rng.integers(lo, V, off[-1]).astype(np.int32), off


def run(gpu, x, pad=0, inplace=False, hist=None, hoff=None, rep=None, pres=None, freq=None, bias=None, mask=None,
        pick=True):
    torch, lm, ctx = gpu
    rows, V = x.shape
    buf = torch.full((rows, V + pad), 7.0, device="cuda")
    buf[:, :V] = dev(torch, x)
    src = buf[:, :V]
    dst = src if inplace else torch.full((rows, V + pad), 7.0, device="cuda")[:, :V]
    d = lambda a: None if a is None else dev(torch, a)  # noqa: E731
    pk = torch.full((rows,), -5, dtype=torch.int64, device="cuda") if pick else None
    n = lm.logits_work_bytes(rows, V)
    work = torch.full((n + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    lm.adjust_logits(ctx, dst, src, history=None if hist is None else (d(hist), d(hoff)), repetition=d(rep),
                     presence=d(pres), frequency=d(freq), bias=None if bias is None else tuple(d(b) for b in bias),
                     mask=d(mask), pick=pk, work=work[:n])
    torch.cuda.synchronize()
    assert bool((work[n:] == 0xFF).all())
    if pad:
        assert bool((dst._base[:, V:] == 7.0).all()), "wrote past a row"
    return dst.cpu().numpy(), pk.cpu().numpy() if pick else None


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32)) or (
        np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)]))


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("V", [1, 31, 32, 33, 4095, 4096, 4097, 32000, 50257])
def test_all_rules(gpu, rows, V):
    rng = np.random.default_rng(rows * 1000 + V)
    print("rules", rows, V, flush=True)
    x = rng.normal(0, 4, (rows, V)).astype(F)
    hist, hoff = ragged(rng, rows, 700, V)
    hist[::7] = hist[0] if len(hist) else 0  # one token many times
    rep, pres, freq = (rng.uniform(a, b, rows).astype(F) for a, b in ((0.8, 1.5), (-0.5, 0.5), (-0.2, 0.4)))
    ids, off = ragged(rng, rows, 50, V)
    ids[1::3] = ids[::3][:len(ids[1::3])]  # tokens twice
    bias = (ids, rng.normal(0, 3, len(ids)).astype(F), off)
    mask = rng.integers(-2 ** 31, 2 ** 31, (rows, -(-V // 32) + 2)).astype(np.int32)
    kw = dict(hist=hist, hoff=hoff, rep=rep, pres=pres, freq=freq, bias=bias, mask=mask)
    o, p = want(x, **kw)
    got, pick = run(gpu, x, pad=3, **kw)
    assert same(got, o) and np.array_equal(pick, p)
    got, pick = run(gpu, x, pad=1, inplace=True, **kw)
    assert same(got, o) and np.array_equal(pick, p)


@pytest.mark.parametrize("part", ["none", "rep", "pres", "freq", "bias", "mask", "hist", "nopick"])
def test_each_rule_alone(gpu, part):
    rng = np.random.default_rng(3)
    rows, V = 5, 9001
    x = rng.normal(0, 2, (rows, V)).astype(F)
    hist, hoff = ragged(rng, rows, 3000, 500)
    kw = {}
    if part in ("rep", "pres", "freq", "hist"):
        kw = dict(hist=hist, hoff=hoff)
        if part != "hist":
            kw[part] = rng.uniform(0.5, 2, rows).astype(F)
    if part == "bias":
        ids, off = ragged(rng, rows, 400, V)
        kw = dict(bias=(ids, rng.normal(0, 1, len(ids)).astype(F), off))
    if part == "mask":
        kw = dict(mask=rng.integers(-2 ** 31, 2 ** 31, (rows, 282)).astype(np.int32))
    o, p = want(x, **kw)
    got, pick = run(gpu, x, pick=part != "nopick", **kw)
    assert same(got, o)
    if part != "nopick":
        assert np.array_equal(pick, p)


def test_edges(gpu):
    """Rows with nothing left, NaN, infinities, ties, ids that are none."""
    rng = np.random.default_rng(4)
    V = 5000
    x = rng.normal(0, 1, (9, V)).astype(F)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 100], x[2, 4999] = np.nan, np.inf
    x[3] = 1.5  # all equal: the first
    x[4, 77] = x[4, 4500] = 50.0
    x[5, 0] = np.finfo(F).max
    x[6] = np.finfo(F).min
    mask = np.full((9, 157), -1, np.int32)
    mask[7] = 0  # a grammar that allows nothing
    mask[8] = 0
    mask[8, 150] = 1 << 7  # one token
    mask[2, 4999 // 32] &= ~(1 << (4999 % 32))  # an infinity that is masked
    x[8, 150 * 32 + 7] = -1e30
    o, p = want(x, mask=mask)
    got, pick = run(gpu, x, mask=mask)
    assert same(got, o) and np.array_equal(pick, p)
    assert list(pick[[0, 1, 3, 4, 7, 8]]) == [-1, -1, 0, 77, -1, 4807]
    hist = np.array([-1, V, 2 ** 31 - 1, -2 ** 31, 3, 3, 4999], np.int32)
    hoff = np.array([0, 7, 7, 7, 7, 7, 7, 7, 7, 7], np.int64)
    bias = (np.array([-1, 5, V, 2 ** 31 - 1], np.int32), np.ones(4, F), np.array([0, 4] + [4] * 8, np.int64))
    one = np.full(9, 1.25, F)
    kw = dict(hist=hist, hoff=hoff, rep=one, pres=one, freq=one, bias=bias)
    o, p = want(x, **kw)
    got, pick = run(gpu, x, **kw)
    assert same(got, o) and np.array_equal(pick, p)


def test_offsets_outside_the_lists(gpu):
    """Offsets that lead outside their list are taken to its ends."""
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (3, 600)).astype(F)
    hist = rng.integers(0, 600, 40).astype(np.int32)
    ids, val = rng.integers(0, 600, 10).astype(np.int32), rng.normal(0, 1, 10).astype(F)
    one = np.full(3, 1.5, F)
    bad = dict(hoff=np.array([-2 ** 40, 20, 2 ** 50, 7], np.int64))
    good = np.array([0, 20, 40, 40], np.int64)
    got, _ = run(gpu, x, hist=hist, rep=one, bias=(ids, val, np.array([-9, 4, 10 ** 12, 3], np.int64)), **bad)
    o, _ = want(x, hist=hist, hoff=good, rep=one, bias=(ids, val, np.array([0, 4, 10, 10], np.int64)))
    assert same(got, o)


@pytest.mark.parametrize("lo", [2 ** 63 - 1, 2 ** 63 - 300, 41])
def test_offsets_at_the_type_s_end(gpu, lo):
    """A row that begins past its list, also where its next entries' positions would wrap, is empty."""
    rng = np.random.default_rng(11)
    x = rng.normal(0, 1, (2, 600)).astype(F)
    hist = rng.integers(0, 600, 40).astype(np.int32)
    one = np.full(2, 1.5, F)
    got, _ = run(gpu, x, hist=hist, rep=one, hoff=np.array([0, lo, 2 ** 63 - 1], np.int64),
                 bias=(hist[:10], x[0, :10], np.array([0, lo, 2 ** 63 - 1], np.int64)))
    o, _ = want(x, hist=hist, rep=one, hoff=np.array([0, 40, 40], np.int64),
                bias=(hist[:10], x[0, :10], np.array([0, 10, 10], np.int64)))
    assert same(got, o)


def test_empty_lists(gpu):
    torch, lm, ctx = gpu
    x = np.random.default_rng(6).normal(0, 1, (2, 100)).astype(F)
    z = np.zeros(0, np.int32)
    off = np.zeros(3, np.int64)
    got, pick = run(gpu, x, hist=z, hoff=off, rep=np.full(2, 2, F), bias=(z, np.zeros(0, F), off))
    assert same(got, x) and np.array_equal(pick, x.argmax(1))
    e = torch.zeros(0, 100, device="cuda")
    lm.adjust_logits(ctx, e, e.clone())


def test_long_history_and_bias_list(gpu):
    rng = np.random.default_rng(7)
    V = 128256
    x = rng.normal(0, 1, (2, V)).astype(F)
    hist = np.concatenate([np.full(100000, V - 1, np.int32), rng.integers(0, V, 31000).astype(np.int32)])
    hoff = np.array([0, 110000, 131000], np.int64)
    ids = rng.integers(0, 40, 3000).astype(np.int32)  # tokens 75 times each
    bias = (ids, rng.normal(0, 1, 3000).astype(F), np.array([0, 2900, 3000], np.int64))
    kw = dict(hist=hist, hoff=hoff, rep=np.full(2, 1.3, F), freq=np.full(2, 0.01, F), bias=bias)
    o, p = want(x, **kw)
    got, pick = run(gpu, x, **kw)
    assert same(got, o) and np.array_equal(pick, p)


def test_in_a_graph(gpu):
    torch, lm, ctx = gpu
    rng = np.random.default_rng(8)
    rows, V = 4, 32000
    x = torch.zeros(rows, V, device="cuda")
    hist, hoff = ragged(rng, rows, 300, V)
    h = (dev(torch, hist), dev(torch, hoff))
    rep = torch.full((rows,), 1.2, device="cuda")
    out, pick = torch.zeros_like(x), torch.zeros(rows, dtype=torch.int64, device="cuda")
    work = torch.empty(lm.logits_work_bytes(rows, V), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin()
            lm.adjust_logits(ctx, out, x, history=h, repetition=rep, pick=pick, work=work)
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in range(6):
        a = rng.normal(0, 3, (rows, V)).astype(F)
        x.copy_(dev(torch, a))
        hist = rng.integers(0, V, len(hist)).astype(np.int32)
        h[0].copy_(dev(torch, hist))
        graph.replay()
        torch.cuda.synchronize()
        o, p = want(a, hist=hist, hoff=hoff, rep=np.full(rows, 1.2, F))
        assert same(out.cpu().numpy(), o) and np.array_equal(pick.cpu().numpy(), p), i


def test_refusals(gpu):
    torch, lm, ctx = gpu
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    x, i32, i64 = z(3, 100), dict(dtype=torch.int32), dict(dtype=torch.int64)
    w = z(lm.logits_work_bytes(3, 100), dtype=torch.uint8)
    h = (z(4, **i32), z(4, **i64))
    bad = [
        lambda: lm.adjust_logits(ctx, z(3, 99), x),
        lambda: lm.adjust_logits(ctx, z(3, 100).half(), x),
        lambda: lm.adjust_logits(ctx, z(100, 3).t(), x),
        lambda: lm.adjust_logits(ctx, x, x, history=(h[0].long(), h[1])),
        lambda: lm.adjust_logits(ctx, x, x, history=(h[0], h[1][:3])),
        lambda: lm.adjust_logits(ctx, x, x, history=h, repetition=z(2)),
        lambda: lm.adjust_logits(ctx, x, x, bias=(h[0], z(3), h[1])),
        lambda: lm.adjust_logits(ctx, x, x, mask=z(3, 3, **i32)),
        lambda: lm.adjust_logits(ctx, x, x, mask=z(2, 4, **i32)),
        lambda: lm.adjust_logits(ctx, x, x, pick=z(3, **i64)),
        lambda: lm.adjust_logits(ctx, x, x, pick=z(3, **i64), work=w[:-1]),
        lambda: lm.adjust_logits(ctx, x, x, pick=z(3, **i32), work=w),
        lambda: lm.adjust_logits(ctx, x.cpu(), x),
    ]
    for f in bad:
        with pytest.raises((ValueError, lm.LlmqError)):
            f()
    lm.adjust_logits(ctx, x, x, history=h, repetition=z(3) + 1, mask=z(3, 4, **i32), pick=z(3, **i64), work=w)
    torch.cuda.synchronize()
