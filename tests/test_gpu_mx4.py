"""Microscaled 4-bit floating point: quantizing is compared bit by bit with
its definition in NumPy, the products with float64 over the values the codes
stand for.

The bar of a product: two codes' product times two powers of two is exact, so
an output's error is that of adding K terms in float32: at most K / 128 + 32
roundings on any path (a step of the instruction adds 128 products into 4
partial sums and the accumulator), each within 2^-23 (the instruction may
truncate) of the sum of the absolute products; bias, GELU and residual as the
epilogue rounds them, 8 2^-24 of their sizes.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F = np.float32
VAL = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
VALS = np.concatenate([VAL, -VAL])


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def quant(x):
    """(codes [T, K / 2], scales [T, K / 32]) by the definition, in float64."""
    T, K = x.shape
    b = x.reshape(T, K // 32, 32).astype(np.float64)
    bad = ~np.isfinite(b).all(-1)
    with np.errstate(all="ignore"):
        m = np.where(np.isfinite(b), np.abs(b), 0).max(-1)
        e = np.where(m > 0, np.frexp(m)[1] - 1 - 2 + 127, 0)
    e = np.maximum(e, 0)
    y = np.abs(np.where(np.isfinite(b), b, 0)) / 2.0 ** (e[..., None] - 127.0)
    near = np.abs(y[..., None] - VAL)
    best = near.min(-1, keepdims=True)
    tied = near == best
    even = tied & (np.arange(8) % 2 == 0)
    c = np.where(even.any(-1), even.argmax(-1), tied.argmax(-1))
    c = c + 8 * np.signbit(b)
    c[bad] = 0
    e[bad] = 255
    c = c.reshape(T, K).astype(np.uint8)
    return c[:, ::2] | c[:, 1::2] << 4, e.astype(np.uint8)


def values(codes, scales):
    """float64 values of packed rows."""
    T, half = codes.shape
    c = np.stack([codes & 15, codes >> 4], -1).reshape(T, half // 16, 32)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (VALS[c] * s[..., None]).reshape(T, 2 * half)


def edges():
    """Rows of blocks whose values are ties, the grid, near-ties, at many sizes."""
    g = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], F)
    up, down = np.nextafter(g, F(9)), np.nextafter(g, F(-9))
    rows = []
    for top in (4.0, 5.0, 6.0, 7.0, 7.9999995):
        for a in (g, up, down):
            blk = np.concatenate([a, -a]).astype(F)
            blk = np.clip(blk, -F(top), F(top))
            blk[0] = top
            for e in (-126, -125, -100, -3, 0, 1, 60, 124):
                with np.errstate(all="ignore"):
                    rows.append((blk.astype(np.float64) * 2.0 ** e).astype(F))
    return np.stack(rows)


def test_quantize_edges(gpu):
    torch, lm, ctx = gpu
    x = edges()
    tiny = np.float64(2.0) ** -149 * np.arange(32).reshape(1, 32)
    x = np.concatenate([x, np.zeros((1, 32), F), -np.zeros((1, 32), F), tiny.astype(F),
                        (tiny * 2.0 ** 20).astype(F), np.full((1, 32), 3.4e38, F), np.full((1, 32), -1e-38, F)])
    x = np.concatenate([x, x[:4], x[:4]])
    x[-1, 3], x[-2, 31], x[-3, 0], x[-4, 7] = np.nan, np.inf, -np.inf, np.nan
    codes = torch.zeros(len(x), 16, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(len(x), 1, dtype=torch.uint8, device="cuda")
    lm.mx4_quantize(ctx, dev(torch, x), codes, scales)
    c, s = quant(x)
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), c)
    out = torch.zeros(len(x), 32, device="cuda")
    lm.mx4_dequantize(ctx, codes, scales, out)
    v = values(c, s).astype(F)
    got = out.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(v)) and np.array_equal(got[~np.isnan(v)], v[~np.isnan(v)])


@pytest.mark.parametrize("T,K", [(1, 32), (1, 11008), (3, 96), (16, 2048), (37, 160), (257, 1056), (1000, 64),
                                 (5, 32768)])
def test_quantize_shapes(gpu, T, K):
    torch, lm, ctx = gpu
    rng = np.random.default_rng(T + K)
    x = (rng.normal(0, 1, (T, K)) * 2.0 ** rng.integers(-20, 20, (T, 1))).astype(F)
    wide = torch.full((T, K + 7), float("nan"), device="cuda")  # rows 4-byte aligned only
    wide[:, 3:K + 3] = dev(torch, x)
    codes = torch.zeros(T, K // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(T, K // 32, dtype=torch.uint8, device="cuda")
    for src in (dev(torch, x), wide[:, 3:K + 3]):
        codes.fill_(0xAA)
        scales.fill_(0xAA)
        lm.mx4_quantize(ctx, src, codes, scales)
        c, s = quant(x)
        assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)
    out = torch.full((T, K + 5), 7.0, device="cuda")
    lm.mx4_dequantize(ctx, codes, scales, out[:, 1:K + 1])
    assert np.array_equal(out[:, 1:K + 1].cpu().numpy(), values(c, s).astype(F))
    assert bool((out[:, 0] == 7).all()) and bool((out[:, K + 1:] == 7).all())


def test_dequantize_every_code_and_scale(gpu):
    torch, lm, ctx = gpu
    codes = np.tile((np.arange(16) * 17 % 256).astype(np.uint8), (256, 1))
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    out = torch.zeros(256, 32, device="cuda")
    lm.mx4_dequantize(ctx, dev(torch, codes), dev(torch, scales), out)
    with np.errstate(all="ignore"):
        v = values(codes, scales).astype(F)
    got = out.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(v)) and np.array_equal(got[~np.isnan(v)], v[~np.isnan(v)])


@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (17, 160), (300, 544), (70, 2048)])
def test_matrix(gpu, n, k):
    torch, lm, ctx = gpu
    rng = np.random.default_rng(n + k)
    w = rng.normal(0, 0.05, (n, k)).astype(F)
    w[0, :32] = 0
    c, s = quant(w)
    mats = [lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False),
            lm.HipMX4Matrix.from_f32(ctx, np.ascontiguousarray(w.T), reduce_rows=True),
            lm.HipMX4Matrix.from_f32(ctx, dev(torch, w), reduce_rows=False),
            lm.HipMX4Matrix.from_f32(ctx, dev(torch, w.T), reduce_rows=True),
            lm.HipMX4Matrix.restore(ctx, c, s)]
    for m in mats:
        gc, gs = m.export()
        assert (m.rows, m.cols, m.nbytes(), m.group_size(), m.has_i16()) == (n, k, n * k // 2 + n * k // 32, 32, False)
        assert np.array_equal(gc, c) and np.array_equal(gs, s)
        for r in {0, n // 2, n - 1}:
            assert np.array_equal(m.dequant_row(r), values(c, s)[r].astype(F))
        m.free()


def bar(x, w, bias=None):
    size = np.abs(x) @ np.abs(w).T
    return (x.shape[1] / 128 + 32) * 2.0 ** -23 * size + 8 * 2.0 ** -24 * (0 if bias is None else np.abs(bias))


def inputs(rng, T, k, n):
    x = rng.normal(0, 1, (T, k)).astype(F)
    x[:, rng.integers(0, k)] *= 30
    w = rng.normal(0, 0.05, (n, k)).astype(F)
    return x, w


TS = [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 64, 65, 100, 128, 129, 257]


@pytest.mark.parametrize("n,k", [(1, 32), (15, 64), (16, 96), (17, 128), (70, 160), (64, 256), (300, 480), (129, 512),
                                 (1000, 544), (256, 1024), (200, 2080), (48, 11008), (513, 4096)])
def test_linear(gpu, n, k):
    """Every number of tokens at the edges of the tiles, through linear,
    linear_noalloc and mx4_linear (which agree bit for bit)."""
    torch, lm, ctx = gpu
    for T in TS:
        print("mx4 linear", T, k, n, flush=True)
        rng = np.random.default_rng(T + n + k)
        x, w = inputs(rng, T, k, n)
        m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
        xv, wv = values(*quant(x)), values(*quant(w))
        xd = dev(torch, x)
        outs = [torch.full((T + 1, n), 7.0, device="cuda") for _ in range(3)]
        lm.linear(ctx, outs[0][:T], xd, m)
        assert lm.lib().llmq_linear_noalloc(ctx.h, outs[1].data_ptr(), xd.data_ptr(), m.h, None, T, k, n, 0) == 0
        codes = torch.zeros(T, k // 2, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(T, k // 32, dtype=torch.uint8, device="cuda")
        lm.mx4_quantize(ctx, xd, codes, scales)
        lm.mx4_linear(ctx, outs[2][:T], codes, scales, m)
        torch.cuda.synchronize()
        for o in outs:
            assert bool((o[T] == 7.0).all()), "wrote past the last token"
        got = outs[0][:T].cpu().numpy()
        assert np.all(np.abs(got - xv @ wv.T) <= bar(xv, wv))
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        m.free()


@pytest.mark.parametrize("T,k,n", [(33, 512, 21000), (65, 2080, 11008), (300, 160, 4113), (321, 32, 4200),
                                   (1000, 544, 1300), (4001, 1056, 350), (2048, 160, 2816), (1537, 672, 3001),
                                   (1600, 1024, 2820)])
def test_linear_many_workgroups(gpu, T, k, n):
    """Sizes that the large tiles take (of 64 and of 96 tokens), odd ones
    among them, with each epilogue, through linear, linear_noalloc and
    mx4_linear; a NaN token and a NaN output row stay by themselves."""
    torch, lm, ctx = gpu
    print("mx4 many", T, k, n, flush=True)
    rng = np.random.default_rng(T + k + n)
    x, w = inputs(rng, T, k, n)
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    xv, wv = values(*quant(x)), values(*quant(w))
    xd = dev(torch, x)
    size = bar(xv, wv)
    y = xv @ wv.T
    outs = [torch.full((T + 1, n), 7.0, device="cuda") for _ in range(3)]
    lm.linear(ctx, outs[0][:T], xd, m)
    assert lm.lib().llmq_linear_noalloc(ctx.h, outs[1].data_ptr(), xd.data_ptr(), m.h, None, T, k, n, 0) == 0
    codes = torch.zeros(T, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(T, k // 32, dtype=torch.uint8, device="cuda")
    lm.mx4_quantize(ctx, xd, codes, scales)
    lm.mx4_linear(ctx, outs[2][:T], codes, scales, m)
    for o in outs:
        assert bool((o[T] == 7.0).all()), "wrote past the last token"
        assert np.all(np.abs(o[:T].cpu().numpy() - y) <= size)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    b, r = rng.normal(0, 1, n).astype(F), rng.normal(0, 1, (T, n)).astype(F)
    out = torch.zeros(T, n, device="cuda")
    lm.linear(ctx, out, xd, m, dev(torch, b))
    assert np.all(np.abs(out.cpu().numpy() - (y + b)) <= size + 8 * 2.0 ** -24 * np.abs(b) + 2.0 ** -24 * np.abs(y + b))
    out = dev(torch, r)
    lm.linear(ctx, out, xd, m, resid=True)
    assert np.all(np.abs(out.cpu().numpy() - (y + r)) <= size + 2.0 ** -23 * (np.abs(y) + np.abs(r)))
    x[T - 2, 3], w[n - 1, 5] = np.nan, np.inf
    m2 = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    lm.linear(ctx, out, dev(torch, x), m2)
    bad = np.zeros((T, n), bool)
    bad[T - 2], bad[:, n - 1] = True, True
    got = out.cpu().numpy()
    assert np.array_equal(np.isnan(got), bad)
    assert np.array_equal(got[~bad], outs[0][:T].cpu().numpy()[~bad])
    m.free()
    m2.free()


@pytest.mark.parametrize("T", [1, 3, 16, 40, 150, 300])
@pytest.mark.parametrize("flags", ["bias", "gelu", "resid", "bias gelu", "bias resid", "bias gelu resid"])
def test_epilogues(gpu, T, flags):
    torch, lm, ctx = gpu
    rng = np.random.default_rng(T)
    k, n = 352, 203
    x, w = inputs(rng, T, k, n)
    b = rng.normal(0, 1, n).astype(F) if "bias" in flags else None
    r = rng.normal(0, 1, (T, n)).astype(F)
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    xv, wv = values(*quant(x)), values(*quant(w))
    out = dev(torch, r)
    lm.linear(ctx, out, dev(torch, x), m, None if b is None else dev(torch, b), resid="resid" in flags,
              gelu="gelu" in flags)
    y = xv @ wv.T
    d = bar(xv, wv, b)
    if b is not None:
        y = y + b
    if "gelu" in flags:  # its slope stays below 1.13
        y, d = 0.5 * y * (1 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3))), 1.13 * d + 2.0 ** -20 * np.abs(y)
    if "resid" in flags:
        y, d = y + r, d + 2.0 ** -23 * (np.abs(y) + np.abs(r))
    assert np.all(np.abs(out.cpu().numpy() - y) <= d)


@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_head_and_scales_far_apart(gpu, T):
    """llmq_head; weights and activations from 2^-60 to 2^60 in one product,
    rows of zeros."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(T)
    k, n = 512, 321
    x, w = inputs(rng, T, k, n)
    w[7] = 0
    x[0] = 0
    x *= 2.0 ** rng.integers(-60, 60, (T, k // 32)).repeat(32, 1).astype(F)
    w *= 2.0 ** rng.integers(-60, 60, (n, k // 32)).repeat(32, 1).astype(F)
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    xv, wv = values(*quant(x)), values(*quant(w))
    out = torch.full((T, n), float("nan"), device="cuda")
    lm.head(ctx, out, dev(torch, x), m)
    assert np.all(np.abs(out.cpu().numpy() - xv @ wv.T) <= bar(xv, wv))


@pytest.mark.parametrize("T", [1, 6, 40, 200])
def test_nan_stays_in_its_row(gpu, T):
    torch, lm, ctx = gpu
    rng = np.random.default_rng(T)
    k, n = 288, 70
    x, w = inputs(rng, T, k, n)
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    base = torch.zeros(T, n, device="cuda")
    lm.linear(ctx, base, dev(torch, x), m)
    hit = sorted({T // 2, T - 1})
    y = x.copy()
    y[hit, 287], w[[3, 69], 40] = np.nan, np.inf
    m2 = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    for mm, rows in ((m, []), (m2, [3, 69])):
        out = torch.zeros(T, n, device="cuda")
        lm.linear(ctx, out, dev(torch, y), mm)
        bad = np.zeros((T, n), bool)
        bad[hit] = True
        bad[:, rows] = True
        got = out.cpu().numpy()
        assert np.array_equal(np.isnan(got), bad)
        assert np.array_equal(got[~bad], base.cpu().numpy()[~bad])


def test_results_do_not_depend_on_neighbours(gpu):
    """A token's outputs are the same bits whatever other tokens a call of the
    same number of tokens holds."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(1)
    for T in (1, 7, 48, 300):
        x, w = inputs(rng, T, 1024, 256)
        m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
        a, b = torch.zeros(T, 256, device="cuda"), torch.zeros(T, 256, device="cuda")
        lm.linear(ctx, a, dev(torch, x), m)
        y = x.copy()
        y[:T - 1] = rng.normal(0, 100, (T - 1, 1024))
        lm.linear(ctx, b, dev(torch, y), m)
        assert torch.equal(a[T - 1], b[T - 1])


def test_in_a_graph(gpu):
    """quantize and mx4_linear into the caller's memory are captured; linear
    of several tokens, whose workspace is the context's, is refused there."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(2)
    T, k, n = 33, 1024, 512
    x, w = inputs(rng, T, k, n)
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    xd, out, one = torch.zeros(T, k, device="cuda"), torch.zeros(T, n, device="cuda"), torch.zeros(1, n, device="cuda")
    codes = torch.zeros(T, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(T, k // 32, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin()
            lm.mx4_quantize(ctx, xd, codes, scales)
            lm.mx4_linear(ctx, out, codes, scales, m)
            lm.mx4_linear(ctx, one, codes[:1], scales[:1], m)
            with pytest.raises(lm.LlmqError, match="mx4_linear"):
                lm.linear(ctx, out, xd, m)
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    want = torch.zeros(T, n, device="cuda")
    want1 = torch.zeros(1, n, device="cuda")
    for i in range(5):
        xd.copy_(dev(torch, rng.normal(0, 1, (T, k)).astype(F)))
        graph.replay()
        lm.linear(ctx, want, xd, m)
        lm.linear(ctx, want1, xd[:1], m)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(one, want1), i


def test_refusals(gpu):
    torch, lm, ctx = gpu
    from llm_mojo_amd._lib import check

    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    u8 = dict(dtype=torch.uint8)
    m = lm.HipMX4Matrix.from_f32(ctx, z(16, 64), reduce_rows=False)
    q = lm.HipQuantMatrix.from_f32(ctx, np.zeros((64, 16), F), 8, 0)
    L = lm.lib()
    bad = [
        lambda: lm.HipMX4Matrix.from_f32(ctx, z(16, 40), reduce_rows=False),
        lambda: lm.HipMX4Matrix.from_f32(ctx, z(16, 0), reduce_rows=False),
        lambda: lm.HipMX4Matrix.from_f32(ctx, np.zeros((16, 48), F), reduce_rows=False),
        lambda: lm.HipMX4Matrix.from_f32(ctx, z(16, 64).half(), reduce_rows=False),
        lambda: lm.HipMX4Matrix.restore(ctx, np.zeros((16, 24), np.uint8), np.zeros((16, 1), np.uint8)),
        lambda: lm.HipMX4Matrix.restore(ctx, np.zeros((16, 32), np.uint8), np.zeros((16, 1), np.uint8)),
        lambda: lm.mx4_quantize(ctx, z(2, 64), z(2, 32, **u8), z(2, 1, **u8)),
        lambda: lm.mx4_quantize(ctx, z(2, 48), z(2, 24, **u8), z(2, 1, **u8)),
        lambda: lm.mx4_quantize(ctx, z(64, 2).t(), z(2, 32, **u8), z(2, 2, **u8)),
        lambda: lm.mx4_linear(ctx, z(2, 16), z(2, 48, **u8), z(2, 3, **u8), m),
        lambda: lm.mx4_linear(ctx, z(2, 15), z(2, 32, **u8), z(2, 2, **u8), m),
        lambda: lm.mx4_linear(ctx, z(2, 16), z(2, 32, **u8), z(2, 2, **u8), q),
        lambda: lm.linear(ctx, z(2, 16), z(2, 32), m),
        lambda: lm.linear(ctx, z(2, 16), z(2, 64), m, ln=(z(64), z(64))),
        lambda: m.dequant_row(16),
        lambda: m.dequant_row(-1),
        lambda: check(L.llmq_mat_export(ctx.h, m.h, None, None, None)),
        lambda: check(L.llmq_mat_export_mx4(ctx.h, q.h, None, None)),
        lambda: lm.linear_act(ctx, z(1, 16), z(lm.act_bytes(64), **u8), m),
        lambda: lm.HipQuantMatrix.dot_row_i16(m, 0, z(64, dtype=torch.int16), z(1)),
        lambda: lm.debug_chunk_sums(ctx, z(1, 64), m, z(1, 16), z(16, 2, dtype=torch.int32), z(64, dtype=torch.int16),
                                    z(1)),
    ]
    keep = []
    for i, f in enumerate(bad):
        print("refusal", i, flush=True)
        with pytest.raises((ValueError, lm.LlmqError)) as e:
            keep.append(f())
        assert "HIP" not in str(e.value)
    # flags and pointers that are none, at the C entry
    x, o = z(2, 64), z(2, 16)
    for rc in (L.llmq_linear(ctx.h, o.data_ptr(), x.data_ptr(), m.h, None, 2, 64, 16, lm.LLMQ_BIAS),
               L.llmq_linear(ctx.h, o.data_ptr(), x.data_ptr(), m.h, None, 2, 64, 16, 8),
               L.llmq_linear(ctx.h, o.data_ptr(), None, m.h, None, 2, 64, 16, 0),
               L.llmq_linear(ctx.h, None, x.data_ptr(), m.h, None, 2, 64, 16, 0),
               L.llmq_linear(ctx.h, o.data_ptr(), x.data_ptr(), m.h, None, -1, 64, 16, 0),
               L.llmq_linear_noalloc(ctx.h, o.data_ptr(), x.data_ptr(), m.h, None, 1 << 20, 64, 16, 0),
               L.llmq_mx4_quantize(ctx.h, x.data_ptr(), 63, 2, 64, o.data_ptr(), o.data_ptr()),
               L.llmq_mx4_linear(ctx.h, o.data_ptr(), x.data_ptr() + 4, x.data_ptr(), m.h, None, 1, 64, 16, 0)):
        assert rc == -1
    lm.linear(ctx, z(0, 16), z(0, 64), m)  # nothing to do is no error
    lm.mx4_quantize(ctx, z(0, 64), z(0, 32, **u8), z(0, 2, **u8))
    lm.mx4_linear(ctx, z(0, 16), z(0, 32, **u8), z(0, 2, **u8), m)
    torch.cuda.synchronize()
