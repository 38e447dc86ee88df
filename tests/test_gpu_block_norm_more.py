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


@pytest.mark.parametrize("n", [2044, 2048, 2560, 2564, 3000])
@pytest.mark.parametrize("rows", [600, 1100])
def test_many_rows_either_side_of_a_width(cuda, n, rows):
    """Widths about those from which a thread has two groups of values, and from which blocks stay, as in test_gpu_block_norm.py."""
    from test_gpu_block_norm import test_many_rows
    test_many_rows(cuda, n, rows)
