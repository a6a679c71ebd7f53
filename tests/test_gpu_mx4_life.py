"""Microscaled matrices beside contexts that end before them."""
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
