"""Which weight gradients are split over blocks, seen from the workspace that their sums need (host-only handle)."""
import ctypes

import pytest

FLOAT, HALF, ARRAY = 2, 1, 4


@pytest.fixture(scope="module")
def handle(ops):
    h = ops.Handle(0)
    yield h
    h.destroy()


def partial_tiles(ops, handle, dtype, rows, groups, ci, co):
    d = [ops.TensorDesc(ARRAY, dtype, dims) for dims in ((rows, ci), (rows, co), (groups, ci, co))]
    size = ctypes.c_size_t(0)
    assert ops.lib().mluOpGetGroupedMatMulBackwardWeightWorkspaceSize(handle.ptr, *d, ctypes.byref(size)) == 0
    return size.value // (4 * ci * co)


@pytest.mark.parametrize("rows", [4000, 8192, 8193])
@pytest.mark.parametrize("groups", [4, 13, 32])
def test_float_gradients_of_few_rows_are_split(ops, handle, rows, groups):
    """All rows may lie in one group, whose products one block would walk alone."""
    assert partial_tiles(ops, handle, FLOAT, rows, groups, 64, 64) >= rows // 512
