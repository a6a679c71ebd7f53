"""Refusals of the paged cache, the microscaled products and the logits'
rules, on the CPU: the C entries' argument checks come before anything of the
GPU (their context is memory of zeros here), and the wrappers' checks of types,
shapes and strides are those of tensors on any device."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
import llm_mojo_amd as lm  # noqa: E402
from llm_mojo_amd import serving  # noqa: E402
from llm_mojo_amd._lib import LogitRules  # noqa: E402

EINVAL = -1


@pytest.fixture(scope="module")
def L():
    return lm.lib()


@pytest.fixture(scope="module")
def ctx():
    """A context that no refused call looks into."""
    return ctypes.create_string_buffer(1 << 16)


def refused(L, rc):
    assert rc == EINVAL
    assert b"HIP" not in L.llmq_last_error()


def test_cache_creation(L, ctx):
    h = ctypes.c_void_p()
    for args in ((2, 1, 4, 64, 2, 64), (0, 0, 4, 64, 2, 64), (0, 1, 0, 64, 2, 64), (0, 1, 1 << 31, 64, 2, 64),
                 (0, 1, 4, 32, 2, 64), (0, 1, 4, 8192, 2, 64), (0, 1, 4, 80, 2, 64), (0, 1, 4, 0, 2, 64),
                 (0, 1, 4, -64, 2, 64), (0, 1, 4, 64, 0, 64), (0, 1, 4, 64, 65536, 64),
                 (0, 1 << 30, 1 << 30, 4096, 65535, 128)):
        assert L.llmq_pkv_create(ctx, *args, ctypes.byref(h)) < 0 and not h.value, args
    assert L.llmq_pkv_create(ctx, 0, 1, 4, 64, 2, 96, ctypes.byref(h)) < 0
    refused(L, L.llmq_pkv_create(None, 0, 1, 4, 64, 2, 64, ctypes.byref(h)))
    refused(L, L.llmq_pkv_create(ctx, 0, 1, 4, 64, 2, 64, None))


def test_no_cache(L, ctx):
    assert L.llmq_pkv_free(None) == 0 and L.llmq_pkv_nbytes(None) == 0
    assert L.llmq_pkv_work_bytes(None, 1, 1) == -1
    p = ctypes.addressof(ctx)
    for f in (L.llmq_pkv_store, L.llmq_pkv_fetch):
        refused(L, f(ctx, None, 0, p, p, 128, 1, p, p, p, 1, 1))
    refused(L, L.llmq_pkv_attend(ctx, None, 0, p, 128, p, 128, 1, 2, p, p, 1, 1.0, 0.0, None, p, 1 << 16))
    refused(L, L.llmq_pkv_step(ctx, None, 0, p, 128, p, p, p, 128, 1, 2, p, p, 1, 1.0, 0.0, None, p, 1 << 16))
    refused(L, L.llmq_pkv_step(ctx, None, 0, p, 128, p, None, p, 128, 1, 2, p, p, 1, 1.0, 0.0, None, p, 1 << 16))


def test_microscaled(L, ctx):
    p = ctypes.addressof(ctx)
    p += -p % 16
    h = ctypes.c_void_p()
    for rows, cols in ((0, 32), (4, 0), (4, 48), (-1, 32), (1 << 31, 32), (1, 1 << 25)):
        refused(L, L.llmq_mat_from_f32_mx4(ctx, p, rows, cols, 0, ctypes.byref(h)))
        refused(L, L.llmq_mat_from_f32_mx4_device(ctx, p, rows, cols, 0, ctypes.byref(h)))
        refused(L, L.llmq_mat_from_f32_mx4(ctx, p, cols, rows, 1, ctypes.byref(h)))
        refused(L, L.llmq_mat_restore_mx4(ctx, rows, cols, p, p, ctypes.byref(h)))
    refused(L, L.llmq_mat_restore_mx4(ctx, 4, 32, None, p, ctypes.byref(h)))
    refused(L, L.llmq_mat_export_mx4(ctx, None, p, p))
    for call in (lambda ld, T, K, c, s: L.llmq_mx4_quantize(ctx, p, ld, T, K, c, s),
                 lambda ld, T, K, c, s: L.llmq_mx4_dequantize(ctx, c, s, T, K, p, ld)):
        for args in ((31, 1, 32, p, p), (48, 1, 48, p, p), (32, -1, 32, p, p), (32, 1, 0, p, p), (32, 1, 32, p + 4, p),
                     (32, 1, 32, None, p), (32, 1, 32, p, None), (1 << 25, 1, 1 << 25, p, p)):
            refused(L, call(*args))
    refused(L, L.llmq_mx4_linear(ctx, p, p, p, None, None, 1, 32, 16, 0))


def test_logits(L, ctx):
    p = ctypes.addressof(ctx)
    p += -p % 16
    for rows, V in ((-1, 10), (65536, 10), (1, 0), (1, 1 << 30)):
        assert L.llmq_adjust_logits_work_bytes(rows, V) == -1
        refused(L, L.llmq_adjust_logits(ctx, p, V, p, V, rows, V, None, None, None, 0))
    call = lambda out=p, ldo=100, x=p, ldl=100, rows=1, rules=None, pick=None, work=p, nw=1 << 15: (  # noqa: E731
        L.llmq_adjust_logits(ctx, out, ldo, x, ldl, rows, 100, None if rules is None else ctypes.byref(rules), pick,
                             work, nw))
    for kw in (dict(out=None), dict(x=None), dict(ldo=99), dict(ldl=99), dict(pick=p, work=None), dict(pick=p, nw=8),
               dict(pick=p, work=p + 4), dict(rules=LogitRules(history_len=-1)), dict(rules=LogitRules(bias_len=-1)),
               dict(rules=LogitRules(history_len=1, history=p)), dict(rules=LogitRules(bias_len=1, bias_ids=p, bias=p)),
               dict(rules=LogitRules(mask=p, mask_ld=3))):
        refused(L, call(**kw))


class Nowhere:
    """A context whose device is that of CPU tensors, so that the wrappers' other checks are reached."""

    h, device = None, -1


def paged():
    serving._torch()
    kv = lm.PagedKV.__new__(lm.PagedKV)
    kv.ctx, kv.h, kv._dev, kv._scale = Nowhere, None, -1, 0.125
    kv.n_layer, kv.n_pages, kv.page, kv.n_kv, kv.head_dim = 1, 4, 64, 2, 64
    return kv


def test_wrapper_of_the_cache():
    c = paged()
    z, i32 = torch.zeros, dict(dtype=torch.int32)
    table, ln, w, q, out = z(3, 2, **i32), z(3, **i32), z(64, dtype=torch.uint8), z(3, 4, 64), z(3, 4, 64)
    k = z(3, 2, 64)
    bad = [
        lambda: c.attend(0, z(2, 4, 64), q, ln, table, w),
        lambda: c.attend(0, out, q.half(), ln, table, w),
        lambda: c.attend(0, out, z(3, 64, 4).transpose(1, 2), ln, table, w),
        lambda: c.attend(0, out, q, ln.long(), table, w),
        lambda: c.attend(0, out, q, ln[:2], table, w),
        lambda: c.attend(0, out, q, z(6, **i32)[::2], table, w),
        lambda: c.attend(0, out, q, ln, table[:2], w),
        lambda: c.attend(0, out, q, ln, z(2, 3, **i32).t(), w),
        lambda: c.attend(0, out, q, ln, table, z(128, dtype=torch.uint8)[::2]),
        lambda: c.attend(0, out, q, ln, table, w, slopes=z(3)),
        lambda: c.store(0, z(2, 2, 64), k, ln[:2], ln[:2], table),
        lambda: c.store(0, z(2, 3, 64), z(2, 3, 64), ln[:2], ln[:2], table),
        lambda: c.store(0, k, z(3, 4, 64)[:, :2], ln, ln, table),
        lambda: c.step(0, out, q, k, k, ln, table, w),
        lambda: c.step(0, out, q, z(3, 2, 32), z(3, 2, 32), ln, table, w),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    c._dev = 0  # a GPU's cache takes no tensors of the CPU
    for f in (lambda: c.attend(0, out, q, ln, table, w), lambda: c.store(0, k, k, ln, ln, table),
              lambda: c.fetch(0, k, k, ln, ln, table)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ValueError):
        lm.PagedKV(Nowhere, 1, 4, 64, 2, 64, "int4")


def test_wrapper_of_the_logits():
    z, i32, i64 = torch.zeros, dict(dtype=torch.int32), dict(dtype=torch.int64)
    x, h, w = z(3, 100), (z(4, **i32), z(4, **i64)), z(4096, dtype=torch.uint8)
    ctx = Nowhere
    bad = [
        dict(out=z(3, 99)), dict(out=z(3, 100).half()), dict(out=z(100, 3).t()), dict(history=(h[0].long(), h[1])),
        dict(history=(h[0], h[1][:3])), dict(history=h, repetition=z(2)), dict(bias=(h[0], z(3), h[1])),
        dict(mask=z(3, 3, **i32)), dict(mask=z(2, 4, **i32)), dict(pick=z(3, **i64)),
        dict(pick=z(3, **i32), work=w), dict(pick=z(3, **i64), work=w[::2]),
    ]
    for kw in bad:
        with pytest.raises(ValueError):
            lm.adjust_logits(ctx, kw.pop("out", x), x, **kw)

    class Gpu:
        h, device = None, 0

    with pytest.raises(ValueError):
        lm.adjust_logits(Gpu, x, x)


def test_wrappers_of_the_products():
    z, u8 = torch.zeros, dict(dtype=torch.uint8)

    class W:
        h, rows, cols = None, 16, 64

    ok = (z(2, 32, **u8), z(2, 2, **u8))
    bad = [
        lambda: lm.mx4_quantize(Nowhere, z(2, 64), z(2, 32, **u8), z(2, 1, **u8)),
        lambda: lm.mx4_quantize(Nowhere, z(64, 2).t(), *ok),
        lambda: lm.mx4_quantize(Nowhere, z(2, 64).half(), *ok),
        lambda: lm.mx4_dequantize(Nowhere, ok[0].int(), ok[1], z(2, 64)),
        lambda: lm.mx4_linear(Nowhere, z(2, 16), z(2, 48, **u8), z(2, 3, **u8), W),
        lambda: lm.mx4_linear(Nowhere, z(2, 15), *ok, W),
        lambda: lm.mx4_linear(Nowhere, z(16, 2).t(), *ok, W),
        lambda: lm.mx4_linear(Nowhere, z(2, 16), *ok, W, bias=z(15)),
        lambda: lm.mx4_linear(Nowhere, z(2, 16), *ok, W, bias=z(16).half()),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
