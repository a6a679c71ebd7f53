"""Microscaled matrices beside contexts that end before them, or are another GPU's."""
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
