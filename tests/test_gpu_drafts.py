"""kd_verify_drafts and kd_distill_rows / kd_distill_grad against their definitions in 64 bits (tests/drafts.py), the
gradient against differences of the loss as well."""
import numpy as np
import pytest

import drafts as definition
import kd

pytestmark = pytest.mark.gpu

NUMPY = {kd.F32: np.float32, kd.F64: np.float64}


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def run_verify(kdb, target, draft, drafted, counts, uniforms):
    sequences, drafts = drafted.shape
    on = [kdb.to_device(a) if a is not None else None for a in (target, draft, drafted, counts, uniforms)]
    tokens, accepted = (kdb.to_device(np.full(s, -777, np.int64)) for s in ((sequences, drafts + 1), (sequences,)))
    ptr = [a.ptr if a is not None else None for a in on]
    kdb.call("verify_drafts", kd.DTYPE_OF[target.dtype], tokens.ptr, accepted.ptr, *ptr, sequences, drafts, target.shape[2])
    return tokens.numpy(), accepted.numpy()


def probabilities(rng, sequences, drafts, vocab, dtype, near=0.5):
    logits = 2 * rng.normal(size=(sequences, drafts + 1, vocab))
    target = softmax(logits).astype(dtype)
    draft = softmax(logits[:, :drafts] + near * rng.normal(size=(sequences, drafts, vocab))).astype(dtype)
    drafted = np.empty((sequences, drafts), np.int64)
    for s in range(sequences):
        for i in range(drafts):
            drafted[s, i] = min(np.searchsorted(np.cumsum(draft[s, i], dtype=np.float64), rng.random()), vocab - 1)
    counts = rng.integers(0, drafts + 1, sequences)
    counts[::2] = drafts
    return target, draft, drafted, counts.astype(np.int64), rng.random((sequences, drafts + 1))


@pytest.mark.parametrize("dtype", [kd.F32, kd.F64], ids=["f32", "f64"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 2), (3, 0, 17), (5, 4, 63), (9, 3, 64), (4, 7, 1025), (2, 70, 300),
                                   (3, 5, 50257), (40, 2, 4099), (1, 1, 100003), (20, 2, 16400), (16, 1, 16384), (5, 2, 40000), (33, 1, 40001)], ids=lambda s: "x".join(map(str, s)))
def test_verification_is_its_definition(kdb, shape, dtype):
    rng = np.random.default_rng(sum(shape))
    given = probabilities(rng, *shape, NUMPY[dtype], near=0.5 if shape[1] < 70 else 0.05)
    for certain in (False, True):
        target, draft, drafted, counts, uniforms = given
        draft = None if certain else draft
        want = definition.verify(target, draft, drafted, counts, uniforms)
        got = run_verify(kdb, target, draft, drafted, counts, uniforms)
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_array_equal(got[0], want[0])


@pytest.mark.parametrize("vocab", [5000, 40009])
@pytest.mark.parametrize("dtype", [kd.F32, kd.F64], ids=["f32", "f64"])
def test_verification_at_the_borders(kdb, dtype, vocab):
    """Draws of 0 and just below 1, weights at the ends alone, a draft equal to its target, tokens out of range, counts out
    of range, rows that hold nothing to draw from, NaN and infinity."""
    rng = np.random.default_rng(1)
    T = NUMPY[dtype]
    target, draft, drafted, counts, uniforms = probabilities(rng, 14, 3, vocab, T)
    counts[:] = 3
    counts[0], counts[1] = -5, 99
    uniforms[2, 3], uniforms[3, 3] = 0, np.nextafter(1, 0)
    drafted[4, 0], drafted[5, 1] = -1, vocab
    draft[6] = target[6, :3]
    uniforms[7, 0], draft[7, 0, drafted[7, 0]] = 0, 0.5  # a draw of 0 takes any token that the target may give
    target[8, 0] = 0
    target[9, 0, 17] = np.nan
    target[10, 0, 4] = np.inf
    draft[11, 0, 5] = np.nan
    uniforms[8:12, 0] = 0.999999
    for s in range(8, 12):
        drafted[s, 0], target[s, 0, 900] = 900, 0
    target[12, 0], draft[12, 0], drafted[12, 0], uniforms[12, 0] = 0, 0, 3, 0.5
    target[12, 0, vocab - 1], draft[12, 0, 3] = 1, 1
    target[13, 0], target[13, 0, 0], draft[13, 0], draft[13, 0, 3], drafted[13, 0] = 0, 1, 0, 1, 3
    for q in (draft, None):
        want = definition.verify(target, q, drafted, counts, uniforms)
        got = run_verify(kdb, target, q, drafted, counts, uniforms)
        np.testing.assert_array_equal(got[1], want[1])
        np.testing.assert_array_equal(got[0], want[0])
    assert got[0][8, 0] == -1 and got[0][9, 0] == -1 and got[0][10, 0] == -1


def test_the_kept_tokens_follow_the_target(kdb):
    """Whatever the draft proposes, the first token of a sequence is distributed as the target: 40000 sequences over five
    tokens, each count within 6 of its own deviations."""
    rng = np.random.default_rng(2)
    n = 40000
    p, q = np.array([0.1, 0.4, 0.05, 0.25, 0.2]), np.array([0.3, 0.1, 0.3, 0.1, 0.2])
    target, draft = np.broadcast_to(p, (n, 2, 5)).copy(), np.broadcast_to(q, (n, 1, 5)).copy()
    drafted = rng.choice(5, (n, 1), p=q)
    tokens, accepted = run_verify(kdb, target, draft, drafted, np.ones(n, np.int64), rng.random((n, 2)))
    counts = np.bincount(tokens[:, 0], minlength=5)
    assert (np.abs(counts - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all()
    assert abs(accepted.mean() - np.minimum(p, q).sum()) < 6 * 0.5 / np.sqrt(n)


# ---- distillation ---------------------------------------------------------------------------------


def run_distill(kdb, logits, indices, teacher, weights, temperature, in_place=False):
    rows, cols = logits.shape
    dtype, kept = kd.DTYPE_OF[logits.dtype], indices.shape[1]
    z, i, t, w = (kdb.to_device(a) for a in (logits, indices, teacher, weights))
    losses, stats = kdb.empty((rows,), logits.dtype), kdb.empty((rows, 2), logits.dtype)
    out = z if in_place else kdb.empty(logits.shape, logits.dtype)
    kdb.call("distill_rows", dtype, losses.ptr, stats.ptr, z.ptr, i.ptr, t.ptr, rows, cols, kept, temperature)
    kdb.call("distill_grad", dtype, out.ptr, z.ptr, stats.ptr, i.ptr, t.ptr, w.ptr, rows, cols, kept, temperature)
    return losses.numpy(), stats.numpy(), out.numpy()


def check_distill(kdb, logits, indices, teacher, weights, temperature, **how):
    """losses: terms of size up to (spread of z and t) / T of f64 logarithms, but the sum of exponentials has an f32
    exponential's 2 steps and the rounded argument's half step times its size, at most X = max|z - max| / T over the
    entries whose exponential is not 0 (exp(-800) is 0 in f64 too, whatever the argument's rounding): T^2 (X + 4) eps, and
    the result's own rounding. The gradient: each of sigma and pi to (X + 8) eps of itself, the
    difference and products 3 eps more."""
    eps = np.finfo(logits.dtype).eps
    want, grad = definition.distill(logits, indices, teacher, temperature)
    losses, stats, got = run_distill(kdb, logits, indices, teacher, weights, temperature, **how)
    z = logits.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        below = (z.max(1, keepdims=True) - z) / temperature
    spread = np.where(below < 800, below, 0).max(1)
    tolerance = temperature ** 2 * (spread + 4) * eps + eps * np.abs(want)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(losses[~finite], want[~finite])
    off = np.abs(losses[finite] - want[finite]) / tolerance[finite]
    assert (off <= 1).all(), off
    w = weights.astype(np.float64)[:, None]
    hit = np.zeros(z.shape)
    for r in range(len(z)):
        there = (indices[r] >= 0) & (indices[r] < z.shape[1])
        hit[r, indices[r, there]] = 1
    with np.errstate(invalid="ignore", divide="ignore"):
        x = (z - z.max(1, keepdims=True)) / temperature
        sigma = np.exp(x) / np.exp(x).sum(1, keepdims=True)
    bound = (spread[:, None] + 11) * eps * np.abs(w) * temperature * (sigma + hit) + np.finfo(logits.dtype).tiny
    assert (np.abs(got - w * grad) <= bound).all(), np.nanmax(np.abs(got - w * grad) / bound)
    return losses, stats, got


@pytest.mark.parametrize("dtype", [kd.F32, kd.F64], ids=["f32", "f64"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2, 2), (70, 96, 8), (5, 63, 63), (4, 64, 1), (7, 1023, 40), (3, 1024, 1024),
                                   (2, 1025, 1000), (6, 5001, 64), (3, 50257, 64), (300, 40, 3), (1, 100001, 17)],
                         ids=lambda s: "x".join(map(str, s)))
def test_distillation_is_its_definition(kdb, shape, dtype):
    rows, cols, kept = shape
    rng = np.random.default_rng(rows + cols)
    logits = (2 * rng.normal(size=(rows, cols))).astype(NUMPY[dtype])
    indices = np.argsort(-(logits + rng.normal(size=logits.shape)), 1)[:, :kept].astype(np.int64)
    teacher = (np.take_along_axis(logits, indices, 1) + rng.normal(size=indices.shape)).astype(NUMPY[dtype])
    weights = rng.normal(size=rows).astype(NUMPY[dtype])
    for temperature in (1.0, 2.5):
        first = check_distill(kdb, logits, indices, teacher, weights, temperature)
        again = run_distill(kdb, logits, indices, teacher, weights, temperature, in_place=True)
        for a, b in zip(first, again):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("rows", [700, 1700])
def test_distillation_of_more_than_the_caches(kdb, rows):
    """Logits of 107 and 259 MiB, whose loads and stores go past the caches: every row as in a call of 82 MB."""
    rng = np.random.default_rng(rows)
    base = rng.normal(size=(512, 40001)).astype(np.float32)
    indices = rng.integers(0, 40001, (512, 9))
    teacher = rng.normal(size=(512, 9)).astype(np.float32)
    weights = rng.normal(size=512).astype(np.float32)
    few = check_distill(kdb, base, indices, teacher, weights, 1.5)
    which = rng.integers(0, 512, rows)
    many = run_distill(kdb, base[which], indices[which], teacher[which], weights[which], 1.5, in_place=rows == 700)
    for a, b in zip(few, many):
        np.testing.assert_array_equal(a[which], b)


@pytest.mark.parametrize("rows,dtype", [(1700, np.float32), (900, np.float64)])
def test_large_distillation_in_place(kdb, rows, dtype):
    """Gradients stored past the caches over the logits that they come from, f32 and f64: every row as in a call of 512,
    which sums a row by as many threads."""
    rng = np.random.default_rng(rows)
    base = rng.normal(size=(512, 40001)).astype(dtype)
    indices = rng.integers(0, 40001, (512, 9))
    teacher, weights = rng.normal(size=(512, 9)).astype(dtype), rng.normal(size=512).astype(dtype)
    few = run_distill(kdb, base, indices, teacher, weights, 1.5)
    # As check_distill, but log sigma is of size X + log(cols), which is not below X by far here, and the definition in f64 rounds
    # as often as f64 losses do: twice T^2 (X + log(cols) + 4) eps + eps |loss|, and twice (X + log(cols) + 11) eps of sigma and pi.
    eps, z = np.finfo(dtype).eps, base.astype(np.float64)
    want, grad = definition.distill(base, indices, teacher, 1.5)
    size = (z.max(1) - z.min(1)) / 1.5 + np.log(40001)
    assert (np.abs(few[0] - want) <= 2 * eps * (1.5 ** 2 * (size + 4) + np.abs(want))).all()
    hit = np.zeros(z.shape)
    np.put_along_axis(hit, indices, 1, 1)  # the shares of a row add up to 1
    bound = 2 * eps * (size + 11)[:, None] * np.abs(weights.astype(np.float64))[:, None] * 1.5 * (softmax(z / 1.5) + hit)
    assert (np.abs(few[2] - weights.astype(np.float64)[:, None] * grad) <= bound + np.finfo(dtype).tiny).all()
    which = rng.integers(0, 512, rows)
    many = run_distill(kdb, base[which], indices[which], teacher[which], weights[which], 1.5, in_place=True)
    for a, b in zip(few, many):
        np.testing.assert_array_equal(a[which], b)


@pytest.mark.parametrize("dtype", [kd.F32, kd.F64], ids=["f32", "f64"])
@pytest.mark.parametrize("cols", [50, 3000])
def test_distillation_of_odd_rows(kdb, cols, dtype):
    """The same index twice, entries of no column, rows without entries, teacher logits of -inf, student logits of -inf and
    of the type's lowest value, in and outside the kept entries, large offsets."""
    rng = np.random.default_rng(cols)
    rows, kept, T = 9, 12, NUMPY[dtype]
    logits = rng.normal(size=(rows, cols)).astype(T)
    indices = np.stack([rng.permutation(cols)[:kept] for _ in range(rows)]).astype(np.int64)
    teacher = rng.normal(size=(rows, kept)).astype(T)
    indices[0, 1:6] = indices[0, 0]
    indices[1, ::2] = [-1, cols, 1 << 40, -(1 << 40), -7, cols + 1]
    indices[2] = -1
    teacher[3], teacher[4, 1:] = -np.inf, -np.inf
    logits[5, indices[5, 0]] = -np.inf                # a kept entry that the student excludes: the loss is infinite
    free = [c for c in range(cols) if c not in indices[6]]
    logits[6, free[:20]], logits[6, free[20]] = -np.inf, np.finfo(T).min
    logits[7] += 3e4
    teacher[7] -= 3e4
    teacher[8, 3:] = np.finfo(T).min
    weights = rng.normal(size=rows).astype(T)
    losses, stats, grad = check_distill(kdb, logits, indices, teacher, weights, 1.5)
    assert losses[2] == 0 and losses[3] == 0 and np.isposinf(losses[5])
    assert (grad[2] == 0).all() and (grad[3] == 0).all() and np.isfinite(grad).all()


@pytest.mark.parametrize("cols", [33, 2000])
def test_a_nan_stays_in_its_row(kdb, cols):
    rng = np.random.default_rng(5)
    logits = rng.normal(size=(4, cols)).astype(np.float32)
    indices = np.stack([rng.permutation(cols)[:5] for _ in range(4)]).astype(np.int64)
    teacher = rng.normal(size=(4, 5)).astype(np.float32)
    logits[1, 7], teacher[2, 3] = np.nan, np.nan
    losses, stats, grad = run_distill(kdb, logits, indices, teacher, np.ones(4, np.float32), 1.0)
    np.testing.assert_array_equal(np.isnan(losses), [False, True, True, False])
    assert np.isnan(grad[1]).all() and np.isnan(grad[2, indices[2]]).all()
    assert np.isfinite(grad[0]).all() and np.isfinite(grad[3]).all()


def test_the_gradient_against_differences(kdb):
    rng = np.random.default_rng(6)
    rows, cols, kept, h = 3, 20, 5, 1e-5
    logits = rng.normal(size=(rows, cols))
    indices = np.stack([rng.permutation(cols)[:kept] for _ in range(rows)]).astype(np.int64)
    teacher, weights = rng.normal(size=(rows, kept)), rng.normal(size=rows)
    grad = run_distill(kdb, logits, indices, teacher, weights, 1.7)[2]
    differences = np.empty_like(grad)
    for c in range(cols):
        d = np.zeros(cols)
        d[c] = h
        up, down = (run_distill(kdb, logits + x, indices, teacher, weights, 1.7)[0] for x in (d, -d))
        differences[:, c] = weights * (up - down) / (2 * h)
    # the differences' own error: h^2 / 6 of a third derivative below 2, and rounding of losses below 20 over h
    assert np.abs(grad - differences).max() <= np.abs(weights).max() * (h * h + 20 * 2.0 ** -52 / h * 8)
