"""Microscaled matrices beside contexts that end before them, are another GPU's, or are
made while a stream is being captured."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F = np.float32


def product(gpu, ctx, w, x):
    torch, lm, _ = gpu
    out = torch.full((x.shape[0], w.rows), float("nan"), device="cuda")
    lm.linear(ctx, out, x, w)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def test_matrix_outlives_its_context(gpu):
    """Used through another context, and freed, after its own has gone; quantized integer matrices too."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(0)
    w = rng.normal(0, 1, (48, 256)).astype(F)
    x = torch.from_numpy(rng.normal(0, 1, (3, 256)).astype(F)).cuda()
    makers = [lambda c: lm.HipMX4Matrix.from_f32(c, w, reduce_rows=False),
              lambda c: lm.HipMX4Matrix.from_f32(c, torch.from_numpy(w).cuda(), reduce_rows=False),
              lambda c: lm.HipMX4Matrix.restore(c, *lm.HipMX4Matrix.from_f32(c, w, reduce_rows=False).export()),
              lambda c: lm.HipQuantMatrix.from_f32(c, w, 4, 32, False, True, reduce_rows=False)]
    for make in makers:
        kept = make(ctx)
        want = product(gpu, ctx, kept, x)
        other = lm.Context(0)
        m = make(other)
        other.sync()
        other.close()
        assert np.array_equal(product(gpu, ctx, m, x), want)
        m.free()
        m.free()
        assert np.array_equal(product(gpu, ctx, kept, x), want)
        kept.free()


def test_matrix_of_another_gpu(gpu):
    """Every call with a context of another GPU than the matrix's is refused.
    (The context is memory that says GPU 1 and nothing else: a refused call looks no further.)"""
    torch, lm, ctx = gpu
    L = lm.lib()
    m = lm.HipMX4Matrix.from_f32(ctx, np.ones((16, 64), F), reduce_rows=False)
    far = ctypes.create_string_buffer(1 << 16)
    ctypes.c_int.from_buffer(far).value = 1
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    x, out, codes, scales = z(2, 64), z(2, 16), z(2, 32, dtype=torch.uint8), z(2, 2, dtype=torch.uint8)
    row, c, s = np.zeros(64, F), np.zeros((16, 32), np.uint8), np.zeros((16, 2), np.uint8)
    for T in (1, 2):
        assert L.llmq_linear(far, out.data_ptr(), x.data_ptr(), m.h, None, T, 64, 16, 0) == -1
        assert b"device" in L.llmq_last_error()
        assert L.llmq_head(far, out.data_ptr(), x.data_ptr(), m.h, T, 16, 64) == -1
        assert L.llmq_mx4_linear(far, out.data_ptr(), codes.data_ptr(), scales.data_ptr(), m.h, None, T, 64, 16, 0) == -1
        assert b"device" in L.llmq_last_error()
    assert L.llmq_mat_dequant_row(far, m.h, 0, row.ctypes.data) == -1 and b"device" in L.llmq_last_error()
    assert L.llmq_mat_export_mx4(far, m.h, c.ctypes.data, s.ctypes.data) == -1 and b"device" in L.llmq_last_error()
    assert np.array_equal(m.dequant_row(0), np.ones(64, F))


def test_matrices_are_not_made_under_capture(gpu):
    """A matrix is made, and copied to the host, outside of graphs only: the
    calls are refused before they touch the capture, which goes on."""
    torch, lm, ctx = gpu
    rng = np.random.default_rng(1)
    w = rng.normal(0, 1, (16, 64)).astype(F)
    wd = torch.from_numpy(w).cuda()
    m = lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False)
    codes, scales = m.export()
    x, out, want = torch.zeros(1, 64, device="cuda"), torch.zeros(1, 16, device="cuda"), torch.zeros(1, 16, device="cuda")
    calls = [lambda: lm.HipMX4Matrix.from_f32(ctx, w, reduce_rows=False),
             lambda: lm.HipMX4Matrix.from_f32(ctx, wd, reduce_rows=False),
             lambda: lm.HipMX4Matrix.restore(ctx, codes, scales), m.export, lambda: m.dequant_row(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            ctx.set_stream(side)
            graph.capture_begin(capture_error_mode="relaxed")
            for f in calls:
                with pytest.raises(lm.LlmqError, match="capture"):
                    f()
            lm.linear(ctx, out, x, m)
            graph.capture_end()
    finally:
        ctx.set_stream(torch.cuda.current_stream())
    for i in range(3):
        x.copy_(torch.from_numpy(rng.normal(0, 1, (1, 64)).astype(F)))
        graph.replay()
        lm.linear(ctx, want, x, m)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
