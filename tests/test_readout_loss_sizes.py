"""Workspace sizes of the read-out's cross-entropy at the ends of its range (no GPU)."""
import pytest

from gncde import _lib

LIB = _lib.load()
P = 0x10000  # an aligned address that is never read


@pytest.mark.parametrize("dtype", [_lib.DTYPE_FP32, _lib.DTYPE_BF16])
@pytest.mark.parametrize("hidden,classes", [(16, 30), (64, 300), (64, 5000), (72, 513), (256, 1000), (4096, 1000),
                                            (333, 50021), (4096, 131072), (1, 1 << 26), (1 << 16, 1)])
def test_no_rows(hidden, classes, dtype):
    """An empty batch has a workspace for the loss and for the gradient, and its gradient without outputs is nothing."""
    for grad in (0, 1):
        n = LIB.gncde_linear_cross_entropy_workspace_bytes(0, hidden, classes, dtype, grad)
        assert 0 < n <= LIB.gncde_linear_cross_entropy_workspace_bytes(1, hidden, classes, dtype, grad)
    assert LIB.gncde_linear_cross_entropy(0, hidden, classes, dtype, None, P, None, _lib.TARGET_INDEX64, None, None, None,
                                          None, None, 0, None) == 0


@pytest.mark.parametrize("dtype", [_lib.DTYPE_FP32, _lib.DTYPE_BF16])
def test_every_accepted_size_has_a_workspace(dtype):
    """Rows, hidden and classes at and around the limits: a size or 0, never an end of the process."""
    f = LIB.gncde_linear_cross_entropy_workspace_bytes
    for rows in (0, 1, 2, 16, 17, 31, 64, 255, 4097, 1 << 21, (1 << 21) + 1):
        for hidden in (1, 2, 7, 63, 64, 129, 4096, 1 << 16):
            for classes in (1, 2, 3, 255, 513, 4097, 1 << 17, 1 << 26):
                for grad in (0, 1):
                    ok = rows <= 1 << 21 and rows * hidden <= 1 << 35 and classes * hidden <= 1 << 35
                    assert (f(rows, hidden, classes, dtype, grad) > 0) == ok, (rows, hidden, classes, grad)
