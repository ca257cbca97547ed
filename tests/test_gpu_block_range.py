"""kd_block_rows and its backward over more rows than a launch of a workgroup for each can have, which one kernel takes in turns."""
import ctypes

import numpy as np
import pytest

import block
import kd
from test_gpu_block import R, check_block, random_case

pytestmark = pytest.mark.gpu


def test_more_short_rows_than_workgroups(kdb):
    rng = np.random.default_rng(1)
    check_block(kdb, random_case(rng, 2 ** 25 + 3, 2, np.float32, None, R, 1, 1.0), forward_only=True)


@pytest.mark.parametrize("shape", [(2 ** 23 + 3, 520), (2 ** 21 + 3, 2052)], ids=lambda s: "x".join(map(str, s)))
def test_more_rows_than_workgroups_in_place(kdb, shape):
    """Two rows at each end and about the border, of 2^32 elements and more: a scaled sum with dropout, h in the place of x."""
    rows, cols = shape
    rng = np.random.default_rng(cols)
    x = kdb.empty(shape, np.float32)
    some = [0, 1, rows - 5, rows - 4, rows - 2, rows - 1]
    values = rng.normal(size=(6, cols)).astype(np.float32)
    copy(kdb, x, some, values)
    b = kd.Block(x.ptr, None, None, rows, cols, 0, 1.0, 0.75, 0.5, kd.Norm(), kd.Norm(), kd.Counter(9, 8, 7, 6, None))
    kdb.call("block_rows", kd.F32, x.ptr, None, None, b)
    want = np.stack([np.where(block.kept(1, cols, 0.5, seed=9, stream=8, step=7, row=6 + r)[0], np.float32(1.5) * v, 0) for r, v in zip(some, values)])
    np.testing.assert_array_equal(copy(kdb, x, some), want.astype(np.float32))


def test_gradients_of_more_rows_than_workgroups(kdb):
    """2^21 rows of more than 4096, whose gradient is another dropout with the same mask, in place."""
    rows, cols = 2 ** 21 + 3, 4100
    rng = np.random.default_rng(2)
    grad = kdb.empty((rows, cols), np.float32)
    some = [0, 1, 2 ** 21 - 1, 2 ** 21, rows - 1]
    values = rng.normal(size=(5, cols)).astype(np.float32)
    copy(kdb, grad, some, values)
    b = kd.Block(None, None, None, rows, cols, 0, 1.0, 0.75, 0.5, kd.Norm(), kd.Norm(), kd.Counter(9, 8, 7, 6, None))
    stats = kdb.to_device(np.tile([0.0, 1.0, 0.0, 1.0], (rows, 1)))
    kdb.call("block_rows_backward", kd.F32, kd.BlockGrads(x=grad.ptr), b, None, stats.ptr, grad.ptr, None, None, 0)
    want = np.stack([np.where(block.kept(1, cols, 0.5, seed=9, stream=8, step=7, row=6 + r)[0], np.float32(1.5) * v, 0) for r, v in zip(some, values)])
    np.testing.assert_array_equal(copy(kdb, grad, some), want.astype(np.float32))


def copy(kdb, on, rows, values=None):
    """Some rows of a large array, to the device or back."""
    out = np.empty((len(rows), on.shape[1]), np.float32) if values is None else values
    for r, row in zip(rows, out):
        at = ctypes.c_void_p(on.ptr + r * row.nbytes)
        here = row.ctypes.data_as(ctypes.c_void_p)
        if values is None:
            kdb.check(kdb.lib.kd_copy_d2h(here, at, row.nbytes), "kd_copy_d2h")
        else:
            kdb.check(kdb.lib.kd_copy_h2d(at, here, row.nbytes), "kd_copy_h2d")
    return out
