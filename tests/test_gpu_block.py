"""kd_counter_dropout and kd_block_rows / kd_block_rows_backward against their definitions in 64 bits (tests/block.py)."""
import ctypes

import numpy as np
import pytest

import block
import kd

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]
IDS = ["f32", "f64"]
SHAPES = [(1, 1), (1, 2), (3, 5), (7, 63), (5, 64), (4, 255), (9, 256), (33, 257), (2, 512), (6, 768), (2, 1000), (3, 1024),
          (5, 1537), (2, 2048), (3, 2051), (2, 4096), (2, 4099), (40, 4096), (3, 8192), (2, 8195), (2, 12288), (1, 16384), (2, 16387),
          (1, 33001), (700, 96), (300, 1)]


def counter_of(seed=0, stream=0, step=0, row=0, more=None):
    return kd.Counter(seed, stream, step, row, more.ptr if more is not None else None)


def place(kdb, array, shift=0):
    """The array on the device, `shift` elements behind a 16-byte boundary; (pointer, owner)."""
    raw = np.zeros(array.size + shift, array.dtype)
    raw[shift:] = array.ravel()
    on = kdb.to_device(raw)
    return on.ptr + shift * array.itemsize, on


class Out:
    """An output with a border of its own on either side, which stays as it was."""

    def __init__(self, kdb, shape, dtype, shift=0):
        self.shape, self.count, self.shift = shape, int(np.prod(shape)), 64 + shift
        self.on = kdb.to_device(np.full(self.count + 128 + shift, 777, dtype))
        self.ptr = self.on.ptr + self.shift * self.on.dtype.itemsize

    def numpy(self):
        raw = self.on.numpy()
        assert (raw[:self.shift] == 777).all() and (raw[self.shift + self.count:] == 777).all()
        return raw[self.shift:self.shift + self.count].reshape(self.shape)


# ---- dropout --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES + [(1, 4096 * 1024 + 3), (70001, 3)], ids=lambda s: "x".join(map(str, s)))
def test_dropout_is_its_definition(kdb, shape, dtype):
    rng = np.random.default_rng(shape[0] * 7 + shape[1])
    x = rng.normal(size=shape).astype(dtype)
    for keep, shift in ((0.9, 0), (0.25, 1), (1.0, 2)):
        counter = dict(seed=0x123456789abcdef0 + shape[1], stream=3, step=2 ** 32 - 2, row=17)
        more = kdb.to_device(np.array([5], np.int64))  # the step passes 2^32
        out = Out(kdb, shape, dtype, shift)
        ptr, on = place(kdb, x, shift)
        kdb.call("counter_dropout", kd.DTYPE_OF[x.dtype], out.ptr, ptr, *shape, keep, counter_of(**counter, more=more))
        want = np.where(block.kept(*shape, keep, **counter, more=5), x * dtype(1 / keep), dtype(0))
        np.testing.assert_array_equal(out.numpy(), want)


def test_dropout_in_place_in_parts_and_of_what_is_not_finite(kdb):
    rng = np.random.default_rng(1)
    x = rng.normal(size=(40, 37)).astype(np.float32)
    x[rng.random(x.shape) < 0.3] = np.nan
    x[rng.random(x.shape) < 0.3] = np.inf
    mask = block.kept(40, 37, 0.5, seed=9, row=100)
    want = np.where(mask, x * np.float32(2), 0)
    whole = kdb.to_device(x)
    kdb.call("counter_dropout", kd.F32, whole.ptr, whole.ptr, 40, 37, 0.5, counter_of(9, row=100))
    np.testing.assert_array_equal(whole.numpy(), want)
    parts = kdb.to_device(x)
    for first, rows in ((30, 10), (0, 13), (13, 17)):
        at = parts.ptr + first * 37 * 4
        kdb.call("counter_dropout", kd.F32, at, at, rows, 37, 0.5, counter_of(9, row=100 + first))
    np.testing.assert_array_equal(parts.numpy(), want)


def test_dropout_at_the_ends_of_the_counter(kdb):
    """The last rows that have a mask, the least keep, and a step and stream of 2^32 - 1."""
    x = np.ones((3, 4001), np.float64)
    for keep in (2.0 ** -32, 1 - 2.0 ** -32, 0.5):
        counter = dict(seed=2 ** 64 - 1, stream=2 ** 32 - 1, step=2 ** 32 - 1, row=2 ** 32 - 3)
        out = kdb.empty(x.shape, np.float64)
        kdb.call("counter_dropout", kd.F64, out.ptr, kdb.to_device(x).ptr, 3, 4001, keep, counter_of(**counter))
        np.testing.assert_array_equal(out.numpy() != 0, block.kept(3, 4001, keep, **counter))


# ---- the end of a block ---------------------------------------------------------------------------


class Run:
    """A case's operands on the device, and its calls."""

    def __init__(self, kdb, case, shift=0, device_step=None):
        self.kdb, self.case, self.dtype = kdb, case, case.x.dtype
        self.own = []

        def on(array):
            if array is None:
                return None
            ptr, owner = place(kdb, array, shift)
            self.own.append(owner)
            return ptr

        norms = [kd.Norm(on(n["weight"]), on(n["bias"]), n["eps"], n["kind"]) if n else kd.Norm() for n in (case.after, case.before)]
        counter = {k: v for k, v in case.counter.items() if k != "more"}
        gate = case.gate
        self.x, self.residual = on(case.x), on(case.residual)
        self.block = kd.Block(self.x, self.residual, on(gate), case.rows, case.cols,
                              0 if gate is None else 1 if gate.ndim == 1 else case.rows, case.residual_scale, case.block_scale,
                              case.keep, *norms, counter_of(**counter, more=device_step))
        shape = (case.rows, case.cols)
        self.h, self.y = Out(kdb, shape, self.dtype, shift), Out(kdb, shape, self.dtype, shift)
        self.stats = Out(kdb, (case.rows, 4), np.float64)

    def forward(self):
        self.kdb.call("block_rows", kd.DTYPE_OF[self.dtype], self.h.ptr, self.y.ptr if self.case.before else None,
                      self.stats.ptr, self.block)
        return self.h.numpy(), self.y.numpy() if self.case.before else None

    def room(self):
        n = ctypes.c_int64()
        self.kdb.call("block_rows_workspace", ctypes.byref(n), kd.DTYPE_OF[self.dtype], self.case.rows, self.case.cols)
        return self.kdb.to_device(np.full(max(n.value, 16), 0xff, np.uint8)), n.value

    def wanted(self):
        case, row = self.case, (self.case.cols,)
        shapes = {"x": case.x.shape, "residual": case.x.shape}
        if case.gate is not None:
            shapes["gate"] = case.gate.shape
        for name, norm in (("after", case.after), ("before", case.before)):
            if norm is not None:
                shapes.update({name + "_weight": row, name + "_bias": row})
        return shapes

    def backward(self, grad_h, grad_y, names=None, shift=0):
        outs = {n: Out(self.kdb, s, self.dtype, shift) for n, s in self.wanted().items() if names is None or n in names}
        grads = kd.BlockGrads(*(outs[n].ptr if n in outs else None for n, _ in kd.BlockGrads._fields_))
        given = [place(self.kdb, g, shift) if g is not None else (None, None) for g in (grad_h, grad_y)]
        room, size = self.room()
        self.kdb.call("block_rows_backward", kd.DTYPE_OF[self.dtype], grads, self.block, self.h.ptr, self.stats.ptr, given[0][0],
                      given[1][0], room.ptr, size)
        return {n: o.numpy() for n, o in outs.items()}


def noise(case):
    """What a row's 64-bit arithmetic may be off by, in units of its terms' size: a norm's mean square is a sum of n terms of
    three roundings each, whose distance from the pivot costs a factor n more at the worst."""
    return (32 + 8 * case.cols) * 2.0 ** -53


def check(got, want, size, eps, parts=0.0, what=""):
    """Half a step of the result and the terms' roundings; `parts`: those of sums in the element type, per term."""
    bound = eps / 2 * np.abs(want) * (1 + 2 ** -20) + parts * size + np.finfo(got.dtype).tiny
    off = np.abs(got - want)
    assert got.shape == want.shape and (off <= bound).all(), (what, np.nanmax(off / bound), np.isnan(got).sum())


def check_block(kdb, case, grad_h=None, grad_y=None, shift=0, forward_only=False):
    """The rows' own arithmetic is 64 bits; the sums over rows have up to 32 roundings of the element type a term in a
    part, and f64's behind that."""
    eps, run, low = np.finfo(case.x.dtype).eps, Run(kdb, case, shift), noise(case)
    h, y = run.forward()
    want, size = case.sum()
    check(h, want, size, eps, low, "h")
    if case.before:
        check(y, *case.next(h), eps, low, "y")
    for at, norm, v in ((0, case.after, case.x), (2, case.before, h)):
        mean, rate = block.norm_stats(v.astype(np.float64), norm)
        stats = run.stats.numpy()
        np.testing.assert_allclose(stats[:, at], mean, rtol=0, atol=low * (1 + np.abs(v).max()))
        np.testing.assert_allclose(stats[:, at + 1], rate, rtol=max(low, 1e-12))
    if forward_only:
        return run
    got = run.backward(grad_h, grad_y, shift=shift)
    for name, (want, size) in case.backward(h, grad_h, grad_y).items():
        if name in got:
            summed = want.ndim == 1
            check(got[name], want, size, eps, 4 * low + (34 * eps / 2 if summed else 0), name)
    return run


def norm(rng, kind, cols, dtype, weight=True, bias=True, eps=1e-5):
    return kind and dict(kind=kind, eps=eps, weight=(1 + 0.3 * rng.normal(size=cols)).astype(dtype) if weight else None,
                         bias=(0.5 * rng.normal(size=cols)).astype(dtype) if bias else None)


def random_case(rng, rows, cols, dtype, after, before, gate, keep, residual=True, **more):
    def normal(*shape):
        return rng.normal(size=shape).astype(dtype)

    return block.Case(normal(rows, cols) * dtype(3) + dtype(0.5), normal(rows, cols) if residual else None,
                      [None, normal(cols), normal(rows, cols)][gate], norm(rng, after, cols, dtype), norm(rng, before, cols, dtype),
                      0.7, -1.25, keep, seed=rows * 1000 + cols, stream=1, step=2, row=3, **more)


L, R = kd.NORM_LAYER, kd.NORM_RMS
KINDS = [(None, L, 0, 1.0), (None, L, 0, 0.9), (R, R, 1, 0.8), (L, R, 2, 0.6), (R, None, 1, 0.5), (L, L, 1, 1.0), (None, None, 2, 0.5),
         (L, None, 0, 1.0), (None, R, 1, 1.0)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_a_block_is_its_definition(kdb, shape, dtype):
    rng = np.random.default_rng(shape[0] + 3 * shape[1])
    kinds = KINDS if shape[0] * shape[1] < 5000 else [KINDS[i] for i in rng.permutation(len(KINDS))[:3]]
    for i, (after, before, gate, keep) in enumerate(kinds):
        case = random_case(rng, *shape, dtype, after, before, gate, keep, residual=i % 4 != 3)
        grad_h, grad_y = (rng.normal(size=shape).astype(dtype) for _ in range(2))
        check_block(kdb, case, grad_h if i % 5 != 4 else None, grad_y if before and i % 6 != 5 else None, shift=i % 4)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 96), (4096, 64), (5000, 250), (1100, 768), (2500, 1030), (600, 4100), (257, 9000), (300, 4096),
                                   (9000, 30)], ids=lambda s: "x".join(map(str, s)))
def test_sums_over_many_rows(kdb, shape, dtype):
    """Parts of the rows, of each plan; a pass with one exchange a row (a norm on one side) as well as two."""
    rng = np.random.default_rng(shape[0])
    for after, before, gate, keep in ((R, L, 1, 0.9), (L, R, 2, 1.0), (None, L, 0, 0.9), (R, None, 0, 1.0)):
        case = random_case(rng, *shape, dtype, after, before, gate, keep)
        grad_h, grad_y = (rng.normal(size=shape).astype(dtype) for _ in range(2))
        check_block(kdb, case, grad_h, grad_y if before else None)


@pytest.mark.parametrize("shape", [(2100, 4096), (4200, 1102), (10300, 520)], ids=lambda s: "x".join(map(str, s)))
def test_rows_one_after_another(kdb, shape):
    """As many rows as make the forward kernel hold the weights, with one exchange a row and with two, whole quads and others."""
    rng = np.random.default_rng(shape[0])
    for after, before, gate, keep in ((L, L, 1, 1.0), (L, None, 1, 1.0), (R, R, 1, 0.5)):
        check_block(kdb, random_case(rng, *shape, np.float32, after, before, gate, keep), forward_only=True)


@pytest.mark.parametrize("shape", [(5, 96), (5, 768), (5, 4096), (3, 40000)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_far_from_zero_constant_rows_and_outliers(kdb, shape, dtype):
    """A mean of 1e4 deviations, rows of one value (their norm is the bias), a first value of 1e6 deviations, eps of 0 beside a
    large one."""
    rng = np.random.default_rng(4)
    for kind in (L, R):
        case = random_case(rng, *shape, dtype, kind, kind, 0, 1.0)
        case.x[0] += dtype(3e4)
        case.x[1], case.residual[1] = dtype(12345.678), dtype(-3.25)
        case.x[2, 0] = dtype(1e6)
        case.x[3:] *= dtype(1e-3)
        case.after["eps"], case.before["eps"] = 1e-12, 100.0
        if kind == L:
            run = Run(kdb, case)
            h, _ = run.forward()
            bias = case.after["bias"].astype(np.float64)
            # each product is off by half a step of itself, however near to 0 their sum is, and the sum by half a step of itself
            want, terms = -1.25 * bias + 0.7 * -3.25, np.abs(1.25 * bias) + 0.7 * 3.25
            assert (np.abs(h[1] - want) <= np.finfo(dtype).eps / 2 * np.abs(want) + 2.0 ** -52 * terms).all()
        check_block(kdb, case, *(rng.normal(size=shape).astype(dtype) for _ in range(2)))


def test_what_is_not_finite_stays_in_its_row(kdb):
    """A NaN or infinity spoils its own row and the sums over rows, nothing else; where dropout takes it out, without a norm
    ahead of it, it spoils nothing."""
    rng = np.random.default_rng(5)
    case = random_case(rng, 6, 300, np.float32, None, R, 0, 0.5)
    out = ~block.kept(6, 300, 0.5, **case.counter)
    case.x[1][out[1]] = np.nan
    case.x[2][out[2]] = np.inf
    run = check_block(kdb, case, *(rng.normal(size=(6, 300)).astype(np.float32) for _ in range(2)))
    case.x[3, np.flatnonzero(~out[3])[0]] = np.nan
    run = Run(kdb, case)
    h, y = run.forward()
    assert np.isnan(y[3]).all() and np.isfinite(np.delete(y, 3, 0)).all() and np.isfinite(np.delete(h, 3, 0)).all()
    grads = run.backward(*(rng.normal(size=(6, 300)).astype(np.float32) for _ in range(2)))
    assert np.isfinite(np.delete(grads["x"], 3, 0)).all() and np.isnan(grads["residual"][3]).all()


@pytest.mark.parametrize("cols", [90, 1100, 6000, 9001, 20003])
def test_dropped_places_of_an_infinite_gate_have_no_gradient(kdb, cols):
    rng = np.random.default_rng(cols)
    case = random_case(rng, 3, cols, np.float64, R, None, 2, 0.5)
    out = ~block.kept(3, cols, 0.5, **case.counter)
    grad = rng.normal(size=(3, cols))
    want = case.backward(case.sum()[0], grad, None)
    case.gate[out] = np.inf
    run = Run(kdb, case)
    run.forward()
    got = run.backward(grad, None)
    for name in ("x", "gate", "after_weight", "after_bias"):
        check(got[name], *want[name], 2.0 ** -52, 4 * noise(case) + 2.0 ** -48, name)


def test_millions_of_short_rows(kdb):
    """More rows than a launch has workgroups of 1024 threads."""
    rng = np.random.default_rng(11)
    rows, cols = (1 << 22) + 3, 5
    case = random_case(rng, rows, cols, np.float32, None, R, 0, 1.0)
    grad = rng.normal(size=(rows, cols)).astype(np.float32)
    check_block(kdb, case, grad, grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(4, 100), (3, 4096), (2, 40001)], ids=lambda s: "x".join(map(str, s)))
def test_in_place(kdb, shape, dtype):
    """h over x or the residual, y over the other; the gradients over those that they are made from, or over x."""
    rng = np.random.default_rng(6)
    case = random_case(rng, *shape, dtype, L, R, 2, 0.7)
    grad_h, grad_y = (rng.normal(size=shape).astype(dtype) for _ in range(2))
    plain = Run(kdb, case)
    h, y = plain.forward()
    grads = plain.backward(grad_h, grad_y)
    for swap in (False, True):
        run = Run(kdb, case)
        places = [run.x, run.residual]
        at_h, at_y = places[::-1] if swap else places
        kdb.call("block_rows", kd.DTYPE_OF[h.dtype], at_h, at_y, run.stats.ptr, run.block)
        held = {o.ptr: o.numpy().reshape(shape) for o in run.own if o.nbytes == h.nbytes}
        np.testing.assert_array_equal(held[at_h], h)
        np.testing.assert_array_equal(held[at_y], y)
        np.testing.assert_array_equal(run.stats.numpy(), plain.stats.numpy())
        for over in ("gradients", "x"):
            run = Run(kdb, case)
            run.forward()
            dh, dy = kdb.to_device(grad_h), kdb.to_device(grad_y)
            at = dict(zip(("residual", "x"), (dy.ptr, dh.ptr) if swap else (dh.ptr, dy.ptr)))
            if over == "x":
                at["x"] = run.x
            outs = {n: Out(kdb, s, dtype) for n, s in run.wanted().items() if n not in at}
            at.update({n: o.ptr for n, o in outs.items()})
            room, size = run.room()
            kdb.call("block_rows_backward", kd.DTYPE_OF[h.dtype], kd.BlockGrads(*(at.get(n) for n, _ in kd.BlockGrads._fields_)),
                     run.block, run.h.ptr, run.stats.ptr, dh.ptr, dy.ptr, room.ptr, size)
            held = {o.ptr: o for o in (dh, dy, *run.own)}
            for name, want in grads.items():
                got = outs[name].numpy() if name in outs else held[at[name]].numpy().reshape(shape)
                np.testing.assert_array_equal(got, want, err_msg=name)


def test_a_part_of_the_outputs(kdb):
    """Outputs that are left out change no bit of the others; without summed gradients no workspace is needed."""
    rng = np.random.default_rng(7)
    for cols in (200, 5000, 20000):
        case = random_case(rng, 9, cols, np.float32, R, L, 1, 0.9)
        grad_h, grad_y = (rng.normal(size=(9, cols)).astype(np.float32) for _ in range(2))
        run = Run(kdb, case)
        h, y = run.forward()
        grads = run.backward(grad_h, grad_y)
        for name in grads:
            np.testing.assert_array_equal(run.backward(grad_h, grad_y, [name])[name], grads[name], err_msg=name)
        for keep_h, keep_y in ((True, False), (False, True)):
            again = Run(kdb, case)
            kdb.call("block_rows", kd.F32, again.h.ptr if keep_h else None, again.y.ptr if keep_y else None, None, again.block)
            if keep_h:
                np.testing.assert_array_equal(again.h.numpy(), h)
            if keep_y:
                np.testing.assert_array_equal(again.y.numpy(), y)
        again = Run(kdb, case)
        kdb.call("block_rows", kd.F32, None, None, again.stats.ptr, again.block)
        np.testing.assert_array_equal(again.stats.numpy(), run.stats.numpy())
        out, dh, dy = Out(kdb, (9, cols), np.float32), kdb.to_device(grad_h), kdb.to_device(grad_y)
        kdb.call("block_rows_backward", kd.F32, kd.BlockGrads(x=out.ptr), run.block, run.h.ptr, run.stats.ptr, dh.ptr, dy.ptr, None, 0)
        np.testing.assert_array_equal(out.numpy(), grads["x"])


def test_no_rows(kdb):
    """Sums over no rows are 0; nothing else is written."""
    row = np.ones(300, np.float32)
    case = block.Case(np.zeros((0, 300), np.float32), None, row, *(dict(kind=L, eps=0.1, weight=row, bias=row) for _ in range(2)), keep=0.5)
    run = Run(kdb, case)
    run.forward()
    got = run.backward(np.zeros((0, 300), np.float32), None)
    assert all((got[n] == 0).all() for n in ("gate", "after_weight", "after_bias", "before_weight", "before_bias"))


def test_offsets_past_32_bits(kdb):
    """The last rows of 2^32 + elements, f32, forward and backward, against the same rows alone."""
    rng = np.random.default_rng(8)
    cols = 8200
    rows = 2 ** 32 // cols + 5
    case = random_case(rng, 4, cols, np.float32, R, L, 1, 0.9)
    near = Run(kdb, case)
    h, y = near.forward()
    grad = rng.normal(size=(4, cols)).astype(np.float32)
    grads = near.backward(grad, None, ["x", "residual"])
    far = [kdb.empty((rows, cols), np.float32) for _ in range(3)]
    first = (rows - 4) * cols * 4

    def put(at, array):
        kdb.check(kdb.lib.kd_copy_h2d(ctypes.c_void_p(at), array.ctypes.data_as(ctypes.c_void_p), array.nbytes), "kd_copy_h2d")

    def last(on):
        out = np.empty((4, cols), np.float32)
        kdb.check(kdb.lib.kd_copy_d2h(out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(on.ptr + first), out.nbytes), "kd_copy_d2h")
        return out

    put(far[0].ptr + first, case.x)
    put(far[1].ptr + first, case.residual)
    b = kd.Block.from_buffer_copy(near.block)
    b.x, b.residual, b.rows = far[0].ptr, far[1].ptr, rows
    b.counter.row -= rows - 4
    b.counter.row += 2 ** 31
    b2 = kd.Block.from_buffer_copy(near.block)
    b2.counter.row += 2 ** 31
    kdb.call("block_rows", kd.F32, near.h.ptr, near.y.ptr, near.stats.ptr, b2)
    h, y = near.h.numpy(), near.y.numpy()
    near.block = b2
    grads = near.backward(grad, None, ["x", "residual"])
    stats = kdb.empty((rows, 4), np.float64)
    kdb.call("block_rows", kd.F32, far[2].ptr, far[1].ptr, stats.ptr, b)
    np.testing.assert_array_equal(last(far[2]), h)
    np.testing.assert_array_equal(last(far[1]), y)
    put(far[1].ptr + first, grad)
    kdb.call("block_rows_backward", kd.F32, kd.BlockGrads(x=far[2].ptr, residual=far[1].ptr), b, far[2].ptr, stats.ptr, far[1].ptr, None, None, 0)
    np.testing.assert_array_equal(last(far[1]), grads["residual"])
    np.testing.assert_array_equal(last(far[2]), grads["x"])


@pytest.mark.parametrize("cols", [4065, 4068, 4069, 4072])
def test_sums_that_fill_the_local_memory(kdb, cols):
    """Five f64 sums of rows that just fit a workgroup's local memory, and of rows that just do not."""
    rng = np.random.default_rng(cols)
    case = random_case(rng, 300, cols, np.float64, L, R, 1, 0.9)
    check_block(kdb, case, *(rng.normal(size=(300, cols)) for _ in range(2)))


@pytest.mark.parametrize("shape", [(8193, 4096), (8705, 1100), (33000, 520), (140001, 31), (4100, 5120), (900, 16001)],
                         ids=lambda s: "x".join(map(str, s)))
def test_sums_of_more_rows_than_one_round(kdb, shape):
    """Parts of the rows in two rounds and more; segments that are not as many as the rows' parts; gradients past the caches."""
    rng = np.random.default_rng(shape[0])
    case = random_case(rng, *shape, np.float32, R, L, 1, 0.9)
    check_block(kdb, case, *(rng.normal(size=shape).astype(np.float32) for _ in range(2)))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [769, 1001, 1281, 1285, 1793, 2305, 2561, 4097, 5121, 6145, 7169, 8193, 12289, 16384, 640, 1280, 2560, 5120, 12292])
def test_teams_of_any_number_of_waves(kdb, cols, dtype):
    """Rows that need one wave more, and whole quads; many rows and few, which divide otherwise."""
    rng = np.random.default_rng(cols)
    for rows, (after, before, gate, keep) in ((3, (L, R, 1, 0.9)), (300, (R, L, 1, 0.8)), (290, (None, L, 0, 0.7))):
        case = random_case(rng, rows, cols, dtype, after, before, gate, keep)
        check_block(kdb, case, *(rng.normal(size=(rows, cols)).astype(dtype) for _ in range(2)))


@pytest.mark.parametrize("shape", [(12400, 640), (16400, 1281), (8300, 1797), (8200, 2304), (4100, 2572)], ids=lambda s: "x".join(map(str, s)))
def test_rows_one_after_another_in_teams_of_any_number_of_waves(kdb, shape):
    rng = np.random.default_rng(shape[1])
    for after, before, gate in ((L, L, 1), (R, R, 1), (L, R, 2)):
        check_block(kdb, random_case(rng, *shape, np.float32, after, before, gate, 0.9), forward_only=True)
