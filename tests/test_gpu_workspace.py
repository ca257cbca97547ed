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


@pytest.mark.parametrize("entry", ["reduce", "reduce_noalloc"])
def test_a_stream_that_goes_with_work_in_flight(kdb, entry):
    """Streams that are destroyed behind calls of theirs that still run, each followed by a new one, which may have the same
    address: every call's sums are its own."""
    lib = kdb.lib
    rng = np.random.default_rng(7)
    long, short = (rng.integers(-1000, 1000, (3, n)).astype(np.int64) for n in (4000000, 60000))
    dl, ds = kdb.to_device(long), kdb.to_device(short)
    want = long.sum(1), short.sum(1)
    before = ctypes.c_void_p(lib.kd_get_stream())
    outs = [kdb.to_device(np.full(3, -777, np.int64)) for _ in range(40)]
    kdb.synchronize()
    for i in range(0, 40, 5):
        stream = ctypes.c_void_p()
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        try:
            lib.kd_set_stream(stream)
            for j in range(i, i + 5):  # the short one first: it is what follows the other stream's long ones
                data, n = (dl, 4000000) if j > i else (ds, 60000)
                kdb.call(entry, kd.REDUCE_SUM, kd.I64, kd.I64, outs[j].ptr, data.ptr, n, 3)
        finally:
            lib.kd_set_stream(before)
            assert lib.hipStreamDestroy(stream) == 0
    assert lib.hipDeviceSynchronize() == 0
    for j, out in enumerate(outs):
        np.testing.assert_array_equal(out.numpy(), want[0 if j % 5 else 1], err_msg=f"call {j}")


@pytest.mark.parametrize("entry", ["reduce", "reduce_noalloc"])
def test_a_captured_call_after_another_streams(kdb, entry):
    """A call on one stream, then the same captured on a second: replays with eager calls between give the eager sums."""
    lib = kdb.lib
    rng = np.random.default_rng(9)
    x = rng.integers(-1000, 1000, (3, 200000)).astype(np.int64)
    dx, out, captured = kdb.to_device(x), kdb.empty((3,), np.int64), kdb.empty((3,), np.int64)

    def call(to):
        kdb.call(entry, kd.REDUCE_SUM, kd.I64, kd.I64, to.ptr, dx.ptr, x.shape[1], 3)

    before = ctypes.c_void_p(lib.kd_get_stream())
    first, second = ctypes.c_void_p(), ctypes.c_void_p()
    for stream in (first, second):
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    try:
        lib.kd_set_stream(first)
        call(out)
        lib.kd_set_stream(second)
        assert lib.hipStreamBeginCapture(second, 1) == 0  # thread-local
        call(captured)
        assert lib.hipStreamEndCapture(second, ctypes.byref(graph)) == 0
        assert lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
        for stream in (second, first, second):
            x = rng.integers(-1000, 1000, x.shape).astype(np.int64)
            dx.upload(x)
            lib.kd_set_stream(stream)
            call(out)
            assert lib.hipStreamSynchronize(stream) == 0
            assert lib.hipGraphLaunch(run, second) == 0
            assert lib.hipStreamSynchronize(second) == 0
            np.testing.assert_array_equal(out.numpy(), x.sum(1))
            np.testing.assert_array_equal(captured.numpy(), x.sum(1))
    finally:
        lib.kd_set_stream(before)
        if run:
            lib.hipGraphExecDestroy(run)
        if graph:
            lib.hipGraphDestroy(graph)
        for stream in (first, second):
            lib.hipStreamDestroy(stream)
