"""Operands of the losses that stand elsewhere than a test's usually do: in each other's place, behind an odd element, in logits that
pass the caches or 32 bits of offsets. A row's bits depend on none of that."""
import ctypes

import numpy as np
import pytest

import answers
import kd
from test_gpu_answers import grad_tolerance, logits_of, policy_of, run_policy, same
from test_gpu_answers_precision import by_shares

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]
IDS = ["f32", "f64"]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(70, 96), (301, 700), (33, 3000), (5, 20000), (20001, 50)], ids=lambda s: "x".join(map(str, s)))
def test_numbers_of_rows_in_each_others_place(kdb, shape, dtype):
    """Losses over advantages or weights, log-probabilities over the old or the reference's, f64 slopes over log-probabilities."""
    rng = np.random.default_rng(sum(shape))
    rows, cols = shape
    z, targets = logits_of(rng, rows, cols, dtype)
    lp = answers.token_logps(z, targets, 1.0)
    old, reference = policy_of(rng, lp, targets, cols, 0.2, 0.3)
    advantages, weights = rng.normal(size=(2, rows)).astype(dtype)
    for grad in (True, False):
        want = run_policy(kdb, z, targets, old, reference, advantages, weights, 1.0, 0.2, 0.3, 0.1, grad=grad)
        for to_losses, to_logps in (("a", "old"), ("w", "reference")):
            on = {n: kdb.to_device(v) for n, v in dict(z=z, t=targets, old=old, reference=reference, a=advantages, w=weights).items()}
            out = kdb.empty(z.shape, z.dtype)
            policy = kd.Policy(on["old"].ptr, on["reference"].ptr, on["a"].ptr, 1.0, 0.2, 0.3, 0.1)
            kdb.call("policy_rows", kd.DTYPE_OF[z.dtype], on[to_losses].ptr, on[to_logps].ptr, out.ptr if grad else None, on["z"].ptr, on["t"].ptr,
                     policy, on["w"].ptr, rows, cols)
            np.testing.assert_array_equal(on[to_losses].numpy(), want[0])
            np.testing.assert_array_equal(on[to_logps].numpy(), want[1])
            if grad:
                np.testing.assert_array_equal(out.numpy(), want[2])
    if dtype is np.float64:
        starts = np.array([0, rows // 3, rows // 2, rows // 2, rows - 1], np.int64)
        two = [kdb.to_device(v) for v in (lp, reference, targets, starts, np.ones(2))]
        losses, slopes = kdb.empty((2,), dtype), kdb.empty((rows,), dtype)
        rest = [a.ptr for a in two] + [2, rows, cols, 0.1, 0.1]
        kdb.call("preference_pairs", kd.F64, losses.ptr, None, slopes.ptr, *rest)
        want = losses.numpy(), slopes.numpy()
        for place in (1, 0):
            again = kdb.to_device((lp, reference)[place])
            rest[place] = again.ptr
            kdb.call("preference_pairs", kd.F64, losses.ptr, None, again.ptr, *rest)
            rest[place] = two[place].ptr
            np.testing.assert_array_equal(losses.numpy(), want[0])
            np.testing.assert_array_equal(again.numpy(), want[1])


class Operands:
    """Numbers a row on the device, for calls on any part of the rows."""

    def __init__(self, kdb, dtype, rows, cols, targets, rng):
        self.kdb, self.dtype, self.rows, self.cols, self.targets = kdb, np.dtype(dtype), rows, cols, targets
        lp = -12 * rng.random(rows)
        self.old, self.reference = lp, lp + 0.5 * rng.normal(size=rows)
        self.advantages, self.weights = rng.normal(size=(2, rows)).astype(dtype)
        self.t, self.o, self.r, self.a, self.w = (kdb.to_device(v) for v in (targets, self.old, self.reference, self.advantages, self.weights))
        self.lp, self.losses, self.stats = kdb.empty((rows,), np.float64), kdb.empty((rows,), dtype), kdb.empty((rows, 2), dtype)

    def policy(self, grad, logits, first=0, rows=None):
        rows, size = self.rows if rows is None else rows, self.dtype.itemsize
        policy = kd.Policy(self.o.ptr + 8 * first, self.r.ptr + 8 * first, self.a.ptr + size * first, 0.9, 0.2, 0.3, 0.1)
        at = first * self.cols * size
        self.kdb.call("policy_rows", kd.DTYPE_OF[self.dtype], self.losses.ptr + size * first, self.lp.ptr + 8 * first,
                      grad + at if grad else None, logits + at, self.t.ptr + 8 * first, policy, self.w.ptr + size * first, rows, self.cols)

    def token(self, logits, first=0, rows=None):
        rows, size = self.rows if rows is None else rows, self.dtype.itemsize
        self.kdb.call("token_logps", kd.DTYPE_OF[self.dtype], self.lp.ptr + 8 * first, self.stats.ptr + 2 * size * first,
                      logits + first * self.cols * size, self.t.ptr + 8 * first, rows, self.cols, 0.9)

    def token_grad(self, out, logits, first=0, rows=None):
        rows, size = self.rows if rows is None else rows, self.dtype.itemsize
        at = first * self.cols * size
        self.kdb.call("token_logps_grad", kd.DTYPE_OF[self.dtype], out + at, logits + at, self.stats.ptr + 2 * size * first,
                      self.t.ptr + 8 * first, self.w.ptr + size * first, rows, self.cols, 0.9)

    def numbers(self):
        return self.lp.numpy(), self.losses.numpy()

    def check(self, z, rows, lp, losses=None, grad=None, by_policy=True):
        """Some rows' results against the definitions; z and grad are those rows'."""
        rows = np.asarray(rows)
        targets, weights = self.targets[rows], self.weights[rows]
        want = answers.token_logps(z, targets, 0.9)
        off, below = by_shares(z, 0.9)
        there = answers.counted(targets, self.cols)
        own = below[np.arange(len(rows)), np.where(there, targets, 0)]
        off = (off + 3 * 2.0 ** -53 * own) * there
        same(lp, want, off)
        slopes = weights.astype(np.float64)
        moved = 0
        if by_policy:
            loss, slope = answers.policy(want, targets, self.cols, self.old[rows], self.reference[rows], self.advantages[rows], 0.2, 0.3, 0.1)
            with np.errstate(over="ignore"):
                size = np.exp(want - self.old[rows]) * np.abs(self.advantages[rows]) + 0.1 * (1 + np.exp(self.reference[rows] - want))
            moved = (2 * off + 2.0 ** -48) * size * there  # the terms' derivatives, by the log-probability's error
            # a ratio at a clip's border may stand on either side of it
            clear = ~there | (np.abs(want - self.old[rows] - np.log(0.8)) > 1e-6) & (np.abs(want - self.old[rows] - np.log(1.3)) > 1e-6)
            assert clear.mean() > 0.9
            same(losses[clear], loss[clear], (moved + np.finfo(z.dtype).eps / 2 * np.abs(loss) + np.finfo(z.dtype).tiny)[clear])
            slopes = slope * slopes
            moved = moved * np.abs(weights)
            z, targets, slopes, moved, grad = z[clear], targets[clear], slopes[clear], moved[clear], grad[clear] if grad is not None else None
        if grad is not None:
            one = answers.token_logps_grad(z, targets, np.where(answers.counted(targets, self.cols), 1.0, 0.0), 0.9)
            same(grad, answers.token_logps_grad(z, targets, slopes, 0.9),
                 grad_tolerance(z, targets, slopes, 0.9) + np.abs(one) * np.broadcast_to(moved, targets.shape)[:, None])


def split(rows, cols, dtype, most):
    """Parts of the rows of at most `most` bytes of logits."""
    step = max(1, most // (cols * np.dtype(dtype).itemsize))
    return [(first, min(step, rows - first)) for first in range(0, rows, step)]


def all_calls(operands, logits, out, parts):
    """Every call's outputs, by parts of the rows; those of long rows without a gradient whole, since their workgroups, and with
    them the order of the sums, go by the number of rows."""
    got = []
    whole = [(0, operands.rows)] if operands.cols * operands.dtype.itemsize > 1024 * 16 else parts
    for grad in (True, False):
        for part in parts if grad else whole:
            operands.policy(out.ptr if grad else None, logits.ptr, *part)
        got += [*operands.numbers(), out.numpy() if grad else None]
    for part in whole:
        operands.token(logits.ptr, *part)
    for part in parts:
        operands.token_grad(out.ptr, logits.ptr, *part)
    return got + [operands.lp.numpy(), operands.stats.numpy(), out.numpy()]


def check_parts(kdb, dtype, rows, cols, parts, seed):
    """A call on all rows has the bits of calls on parts of them, and the definitions' values in a few."""
    rng = np.random.default_rng(seed)
    base, _ = logits_of(rng, min(rows, 61), cols, dtype)
    z = base[np.arange(rows) % len(base)]
    targets = rng.integers(0, cols, rows)
    targets[rng.random(rows) < 0.25] = rng.choice([-1, cols, 2 ** 40])
    targets[-1] = cols - 1
    operands = Operands(kdb, dtype, rows, cols, targets, rng)
    logits, out = kdb.to_device(z), kdb.empty((rows, cols), dtype)
    whole = all_calls(operands, logits, out, [(0, rows)])
    for got, want in zip(all_calls(operands, logits, out, parts), whole):
        if got is not None:
            np.testing.assert_array_equal(got, want)
    some = np.unique(np.concatenate((np.arange(min(rows, 9)), rng.integers(0, rows, 20), np.arange(max(rows - 9, 0), rows))))
    lp, losses, grad, lp_alone, losses_alone, _, lp_token, _, grad_token = whole
    operands.check(z[some], some, lp[some], losses[some], grad[some])
    operands.check(z[some], some, lp_alone[some], losses_alone[some])
    operands.check(z[some], some, lp_token[some], grad=grad_token[some], by_policy=False)


@pytest.mark.parametrize("cols", [1, 3, 96, 128, 250, 300, 500, 512])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_that_share_a_wave(kdb, dtype, cols):
    """Many short rows go four to a wave; the last wave has one, two or three, and rows without a target stand among all."""
    for rows in (16384, 16389, 20002, 17003):
        check_parts(kdb, dtype, rows, cols, [(0, 9000), (9000, rows - 9000)], rows + cols)


@pytest.mark.parametrize("shape", [(700, 50257), (1750, 50257), (900, 20001), (12000, 3000), (28500, 3000), (36000, 1000), (85000, 1000), (70000, 500),
                                   (170000, 500), (260, 151001)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_logits_past_the_caches(kdb, dtype, shape):
    """More than 96, 128 and 320 MiB, where loads, stores or both go past the caches, against parts that do not."""
    rows, cols = shape
    rows = rows if dtype is np.float32 else rows // 2 + 1
    check_parts(kdb, dtype, rows, cols, split(rows, cols, dtype, 60 << 20), cols)


@pytest.mark.parametrize("shape", [(2 ** 32 // 50257 + 5, 50257), (2 ** 32 // 3001 + 5, 3001), (2 ** 22 - 4, 1024)], ids=lambda s: "x".join(map(str, s)))
def test_offsets_past_32_bits(kdb, shape):
    """2^32 elements and as many rows as a call takes, in place: the first rows, the ones about the border and the last ones."""
    rows, cols = shape
    rng = np.random.default_rng(cols)
    border = min(2 ** 32 // cols, rows - 4)
    some = np.unique(np.r_[0:3, 2 ** 31 // cols - 1:2 ** 31 // cols + 2, border - 2:border + 2, rows - 3:rows])
    targets = np.full(rows, -1)
    targets[some] = rng.integers(0, cols, len(some))
    targets[some[4]] = -1
    operands = Operands(kdb, np.float32, rows, cols, targets, rng)
    z, _ = logits_of(rng, len(some), cols, np.float32)
    logits = kdb.empty(shape, np.float32)

    def put():
        for r, row in zip(some, z):
            kdb.check(kdb.lib.kd_copy_h2d(ctypes.c_void_p(logits.ptr + int(r) * cols * 4), row.ctypes.data_as(ctypes.c_void_p), row.nbytes), "kd_copy_h2d")

    def back(r):
        out = np.empty(cols, np.float32)
        kdb.check(kdb.lib.kd_copy_d2h(out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(logits.ptr + int(r) * cols * 4), out.nbytes), "kd_copy_d2h")
        return out

    put()
    operands.policy(None, logits.ptr)
    lp, losses = operands.numbers()
    operands.check(z, some, lp[some], losses[some])
    operands.policy(logits.ptr, logits.ptr)
    lp, losses = operands.numbers()
    operands.check(z, some, lp[some], losses[some], np.stack([back(r) for r in some]))
    put()
    operands.token(logits.ptr)
    operands.token_grad(logits.ptr, logits.ptr)
    operands.check(z, some, operands.lp.numpy()[some], grad=np.stack([back(r) for r in some]), by_policy=False)
    others = np.setdiff1d(np.arange(rows), some)
    assert (operands.lp.numpy()[others] == 0).all() and (operands.stats.numpy()[others] == [0, 1]).all()
    for r in (some[2] + 1, border + 2 if border + 2 < rows - 3 else border - 3, rows - 4):
        assert r in some or (back(r) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(70, 96), (16390, 31), (7, 1000), (3, 8200), (2, 50257), (2, 151001)], ids=lambda s: "x".join(map(str, s)))
def test_operands_behind_an_odd_element(kdb, shape, dtype):
    """Every operand one or three elements behind where a memory block begins."""
    rows, cols = shape
    rng = np.random.default_rng(cols)
    z, targets = logits_of(rng, rows, cols, dtype)
    operands = Operands(kdb, dtype, rows, cols, targets, rng)
    out = kdb.empty(shape, dtype)
    want = all_calls(operands, kdb.to_device(z), out, [(0, rows)])

    class Behind:
        def __init__(self, array, by):
            flat = np.concatenate((np.full(by, 7, array.dtype), array.ravel(), np.full(3, 7, array.dtype)))
            self.on, self.by, self.shape = kdb.to_device(flat), by, array.shape
            self.ptr = self.on.ptr + by * array.itemsize

        def numpy(self):
            flat = self.on.numpy()
            assert (flat[:self.by] == 7).all() and (flat[-3:] == 7).all()
            return flat[self.by:-3].reshape(self.shape)

    for by in (1, 3):
        for name in ("t", "o", "r", "a", "w", "lp", "losses", "stats"):
            setattr(operands, name, Behind(getattr(operands, name).numpy(), by))
        got = all_calls(operands, Behind(z, by), Behind(np.zeros(shape, dtype), 4 - by), [(0, rows)])
        for g, w in zip(got, want):
            if g is not None:
                np.testing.assert_array_equal(g, w)
