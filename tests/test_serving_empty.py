"""Calls of no rows: tensors without elements may have any strides (numpy's
have zeros), which the wrappers of the serving operators must not refuse.  On
the CPU: the calls get past the wrappers and are refused by the library, for
their missing context."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import llm_mojo_amd as lm  # noqa: E402
from llm_mojo_amd import serving  # noqa: E402
from tests.test_serving_refusals import Nowhere, paged  # noqa: E402


def none(*shape, dtype=np.float32):
    t = torch.from_numpy(np.zeros(shape, dtype))
    assert t.numel() == 0 and t.stride(-1) != 1  # as numpy gives them
    return t


def test_no_rows():
    serving._torch()
    c = paged()
    i, table, w = torch.zeros(0, dtype=torch.int32), torch.zeros(0, 2, dtype=torch.int32), torch.zeros(64, dtype=torch.uint8)
    k, q = none(0, 2, 64), none(0, 4, 64)
    calls = [
        lambda: c.store(0, k, k, i, i, table),
        lambda: c.fetch(0, none(0, 128), none(0, 128), i, i, table),
        lambda: c.attend(0, none(0, 256), q, i, table, w),
        lambda: c.step(0, q, q, k, k, i, table, w),
        lambda: lm.adjust_logits(Nowhere, none(0, 100), none(0, 100), mask=none(0, 4, dtype=np.int32)),
        lambda: lm.mx4_quantize(Nowhere, none(0, 64), none(0, 32, dtype=np.uint8), none(0, 2, dtype=np.uint8)),
    ]
    for f in calls:
        with pytest.raises(lm.LlmqError, match="null argument"):
            f()
    # their shapes still count
    for f in (lambda: c.store(0, none(0, 2, 32), none(0, 2, 32), i, i, table),
              lambda: c.store(0, none(0, 64), none(0, 64), i, i, table),
              lambda: lm.adjust_logits(Nowhere, none(0, 99), none(0, 100))):
        with pytest.raises(ValueError):
            f()
