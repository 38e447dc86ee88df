"""Norms between blocks: calls without rows or columns, whose tensors are nobody's afterwards."""
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 100), (3, 0), (0, 0), (0, 70000)])
def test_empty_calls_keep_nothing(cuda, shape):
    import gc
    import weakref

    import torch
    x, out, h = (torch.zeros(shape, device="cuda") for _ in range(3))
    before = sys.getrefcount(out), sys.getrefcount(h)
    for _ in range(10):
        y, z = cuda.block_norm(x, out=out, h_out=h)
        assert y is out and z is h
    del y, z
    assert (sys.getrefcount(out), sys.getrefcount(h)) == before
    y, z = cuda.block_norm(x, dtype=torch.float16)
    assert y.shape == z.shape == shape and y.dtype == torch.float16
    gone = weakref.ref(y), weakref.ref(z)
    assert sys.getrefcount(y) == sys.getrefcount(out)
    del y, z
    gc.collect()
    assert gone[0]() is None and gone[1]() is None
