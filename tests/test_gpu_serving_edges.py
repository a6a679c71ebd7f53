"""The serving operators where one form of a kernel ends and the next begins,
on several streams at once, and beside other rows: the paged attention with
more rows than are cut, two caches of two contexts at work together, and one
token's microscaled product at the longest row that its own kernel takes."""

import numpy as np
import pytest

from tests.test_gpu_mx4 import bar as bar_mx4
from tests.test_gpu_mx4 import inputs, quant, values
from tests.test_gpu_paged import KINDS, Case, dev, held, want

pytestmark = pytest.mark.gpu

F = np.float32


@pytest.mark.parametrize("rows", [1024, 1025])
@pytest.mark.parametrize("kind", KINDS)
def test_step_of_many_rows(gpu, kind, rows):
    """The most rows whose lengths a step looks through to cut them, and one more, which are taken whole."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, 60, rows)
    lens[rng.random(rows) < 0.1] = 0
    lens[[3, rows // 2, rows - 1]] = 1500, 2999, 700
    c = Case(gpu, kind, 64, 1, [int(n) for n in lens], width=50)
    heads = 9
    x = rng.normal(0, 1, (rows, heads + 2, 64)).astype(F)
    d = dev(torch, x)
    out = torch.full((rows, heads, 64), float("nan"), device="cuda")
    w, whole = c.work(rows, heads)
    c.cache.step(0, out, d[:, :heads], d[:, heads:heads + 1], d[:, heads + 1:], dev(torch, (lens - 1).astype(np.int32)),
                 c.table, w)
    torch.cuda.synchronize()
    assert bool((whole[w.numel():] == 0xFF).all())
    got = out.cpu().numpy()
    for r in range(rows):
        at = c.rows(r)
        if lens[r]:
            c.k[at[-1]], c.v[at[-1]] = x[r, heads:heads + 1], x[r, heads + 1:]
        o, bar = want(x[r, :heads], held(kind, c.k[at]), held(kind, c.v[at]), 0.125, 0.0, None)
        assert np.all(np.abs(got[r] - o) <= bar), r
    ko, vo = (torch.zeros(c.k.shape, device="cuda") for _ in range(2))
    c.cache.fetch(0, ko, vo, dev(torch, c.seq), dev(torch, c.pos), c.table)
    assert np.array_equal(ko.cpu().numpy(), held(kind, c.k)) and np.array_equal(vo.cpu().numpy(), held(kind, c.v))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width", [None, 50])  # rows whole, and cut and joined
def test_other_rows_do_not_change_a_row(gpu, kind, width):
    """Other queries, keys and values in the other rows, of the same lengths: the same bits."""
    torch, lm, ctx = gpu
    lens = [333, 900, 17, 64] if width is None else [2500, 900, 17, 3100]
    c = Case(gpu, kind, 128, 2, lens, width=width)
    q, a = c.attend(12)
    other = (c.seq != 1) & (c.seq != 2)
    c.k[other] = c.rng.normal(0, 3, c.k[other].shape)
    c.v[other] = c.rng.normal(0, 90, c.v[other].shape)
    c.cache.store(0, dev(torch, c.k), dev(torch, c.v), dev(torch, c.seq), dev(torch, c.pos), c.table)
    p = q.copy()
    p[[0, 3]] = c.rng.normal(0, 2, p[[0, 3]].shape)
    _, b = c.attend(12, q=p)
    assert np.array_equal(a[[1, 2]], b[[1, 2]]) and not np.array_equal(a[[0, 3]], b[[0, 3]])


@pytest.mark.parametrize("kind", KINDS)
def test_two_caches_at_once(gpu, kind):
    """Two contexts, each with its cache, stream and workspace: their stores, steps and attends are all enqueued
    before anything is waited for, and equal the same calls one after another."""
    torch, lm, _ = gpu
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [lm.Context(0, s) for s in streams]
    lens, heads, n_kv = [4000, 70, 1999], 16, 2
    cases, xs, ws, poss, outs = [], [], [], [], []
    for i, (s, ctx) in enumerate(zip(streams, ctxs)):
        with torch.cuda.stream(s):
            c = Case((torch, lm, ctx), kind, 128, n_kv, [n + 8 for n in lens], width=40, page=128, seed=i)
            cases.append(c)
            xs.append([dev(torch, c.rng.normal(0, 1, (3, heads + 2 * n_kv, 128)).astype(F)) for _ in range(8)])
            ws.append(c.work(3, heads)[0])
            poss.append([dev(torch, np.array(lens, np.int32) + t) for t in range(8)])
            outs.append([[torch.zeros(3, heads, 128, device="cuda") for _ in range(8)] for _ in range(2)])
    torch.cuda.synchronize()

    def step(i, t, way):
        x, c = xs[i][t], cases[i]
        c.cache.step(0, outs[i][way][t], x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:], poss[i][t], c.table,
                     ws[i])

    for t in range(8):
        for i in range(2):
            step(i, t, 0)
    torch.cuda.synchronize()
    for i in range(2):
        for t in range(8):
            step(i, t, 1)
            torch.cuda.synchronize()
    for i in range(2):
        for t in range(8):
            assert torch.equal(outs[i][0][t], outs[i][1][t]), (i, t)
        assert not torch.equal(outs[0][0][0], outs[1][0][0])
    for c in cases:
        c.cache.free()
    for ctx in ctxs:
        ctx.close()


@pytest.mark.parametrize("k", [122880, 122912])
def test_one_token_of_the_longest_rows(gpu, k):
    """One token of 122880 inputs is quantized in the product's own kernel, of
    more by way of a record: the same bits as mx4_quantize and mx4_linear."""
    torch, lm, ctx = gpu
    n = 40
    x, w = inputs(np.random.default_rng(k), 1, k, n)
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    xd = dev(torch, x)
    outs = [torch.full((2, n), 7.0, device="cuda") for _ in range(3)]
    lm.linear(ctx, outs[0][:1], xd, m)
    assert lm.lib().llmq_linear_noalloc(ctx.h, outs[1].data_ptr(), xd.data_ptr(), m.h, None, 1, k, n, 0) == 0
    codes = torch.zeros(1, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(1, k // 32, dtype=torch.uint8, device="cuda")
    lm.mx4_quantize(ctx, xd, codes, scales)
    lm.mx4_linear(ctx, outs[2][:1], codes, scales, m)
    torch.cuda.synchronize()
    assert all(bool((o[1] == 7.0).all()) for o in outs)
    xv, wv = values(*quant(x)), values(*quant(w))
    assert np.all(np.abs(outs[0][:1].cpu().numpy() - xv @ wv.T) <= bar_mx4(xv, wv))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    # under capture the first needs no workspace, the second is refused
    graph, out = torch.cuda.CUDAGraph(), torch.zeros(1, n, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin()
            if k == 122880:
                lm.linear(ctx, out, xd, m)
            else:
                with pytest.raises(lm.LlmqError, match="mx4_linear"):
                    lm.linear(ctx, out, xd, m)
                lm.mx4_linear(ctx, out, codes, scales, m)
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], outs[0][0])
