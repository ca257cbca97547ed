"""The backend's shared workspace after its last user's stream is gone: a stream is created, a call that splits its work over
the workspace runs on it, the stream is destroyed, and calls on the null stream and on new streams go on.
"""
import ctypes

import numpy as np
import pytest

import kd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", ["reduce", "reduce_noalloc"])  # the growable workspace, the static scratch
@pytest.mark.parametrize("rounds", [1, 6])
def test_the_workspace_outlives_its_last_stream(kdb, rounds, entry):
    lib = kdb.lib
    rng = np.random.default_rng(rounds)
    x = rng.integers(-1000, 1000, (3, 200000)).astype(np.int64)
    dx, out = kdb.to_device(x), kdb.empty((3,), np.int64)

    def total():
        kdb.call(entry, kd.REDUCE_SUM, kd.I64, kd.I64, out.ptr, dx.ptr, x.shape[1], 3)  # few long rows: in split sums
        return out.numpy()

    want = x.sum(1)
    np.testing.assert_array_equal(total(), want)
    before = ctypes.c_void_p(lib.kd_get_stream())
    for _ in range(rounds):
        stream = ctypes.c_void_p()
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        try:
            lib.kd_set_stream(stream)
            np.testing.assert_array_equal(total(), want)
        finally:
            lib.kd_set_stream(before)
            assert lib.hipStreamDestroy(stream) == 0
        held = [kdb.empty((1 << 16,), np.float32) for _ in range(8)]  # host and device memory taken up meanwhile
        np.testing.assert_array_equal(total(), want)
        del held
