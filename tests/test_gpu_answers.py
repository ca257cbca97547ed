"""kd_token_logps, kd_token_logps_grad, kd_preference_pairs and kd_policy_rows against their definitions in 64 bits
(tests/answers.py)."""
import numpy as np
import pytest

import answers
import kd

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]
IDS = ["f32", "f64"]
SHAPES = [(1, 1), (3, 2), (5, 63), (70, 96), (4, 64), (9, 256), (6, 257), (7, 1000), (3, 1024), (2, 1025), (5, 4099), (3, 8200),
          (2, 16385), (3, 32771), (4, 50257), (2, 65537), (1, 100003), (1, 151000), (600, 40), (300, 3001)]


def logits_of(rng, rows, cols, dtype):
    z = 2 * rng.normal(size=(rows, cols))
    targets = rng.integers(0, cols, rows)
    z[np.arange(rows), targets] += 4
    targets[rng.random(rows) < 0.25] = rng.choice([-1, cols, -100, 2 ** 40])
    if rows > 2:
        targets[0] = cols - 1
    return z.astype(dtype), targets.astype(np.int64)


def spread(z, temperature):
    """max|z - max| / T over the entries whose exponential counts."""
    z = z.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        below = (z.max(1, keepdims=True) - z) / temperature
    return np.where(below < 800, below, 0).max(1)


def logp_tolerance(z, temperature):
    """An exponential's own two steps, its argument's half step of the difference and one more of its product (X each, X the
    spread), the maxima that parts are moved by (another X + 2), in units of the sum; f64's logarithm and differences."""
    eps = np.finfo(z.dtype).eps
    x = spread(z, temperature)
    return (2 * x + 6) * eps + 8 * 2.0 ** -53 * (1 + x)


def grad_tolerance(z, targets, slopes, temperature):
    """The softmax to the exponential's and the sum's tolerance, the products and the difference three steps."""
    eps = np.finfo(z.dtype).eps
    soft = np.exp(answers.shares(z, temperature))
    there = answers.counted(targets, z.shape[1])
    soft[np.flatnonzero(there), targets[there]] += 1
    x = spread(z, temperature)[:, None]
    with np.errstate(invalid="ignore"):
        return (4 * x + 14) * eps * np.abs(slopes)[:, None] / temperature * soft + np.finfo(z.dtype).tiny


def same(got, want, tolerance):
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    off = np.abs(got[finite] - want[finite])
    bound = np.broadcast_to(tolerance, want.shape)[finite]
    assert (off <= bound).all(), (off / bound).max()


def token_logps(kdb, z, targets, temperature):
    rows, cols = z.shape
    logps, stats = kdb.empty((rows,), np.float64), kdb.empty((rows, 2), z.dtype)
    dz, dt = kdb.to_device(z), kdb.to_device(targets)
    kdb.call("token_logps", kd.DTYPE_OF[z.dtype], logps.ptr, stats.ptr, dz.ptr, dt.ptr, rows, cols, temperature)
    return logps, stats, dz, dt


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_log_probabilities_and_their_gradient(kdb, shape, dtype):
    rng = np.random.default_rng(sum(shape))
    for temperature, in_place in ((1.0, False), (0.37, True)):
        z, targets = logits_of(rng, *shape, dtype)
        slopes = rng.normal(size=shape[0]).astype(dtype)
        logps, stats, dz, dt = token_logps(kdb, z, targets, temperature)
        there = answers.counted(targets, shape[1])
        same(logps.numpy(), answers.token_logps(z, targets, temperature), logp_tolerance(z, temperature) * there)
        assert (stats.numpy()[~there] == [0, 1]).all()
        np.testing.assert_array_equal(stats.numpy()[there, 0], z.max(1)[there])
        out = dz if in_place else kdb.empty(shape, dtype)
        ds = kdb.to_device(slopes)
        kdb.call("token_logps_grad", kd.DTYPE_OF[z.dtype], out.ptr, dz.ptr, stats.ptr, dt.ptr, ds.ptr, *shape, temperature)
        same(out.numpy(), answers.token_logps_grad(z, targets, slopes, temperature), grad_tolerance(z, targets, slopes, temperature))


def policy_of(rng, lp, targets, cols, low, high):
    """Old log-probabilities whose ratios stand on both sides of the borders, but not at them, where rounding decides."""
    moved = 0.4 * rng.normal(size=len(lp))
    for border in (np.log1p(-low), np.log1p(high)):
        moved[np.abs(moved - border) < 1e-2] += 0.05
    return np.where(np.isfinite(lp), lp, 0) - moved, np.where(np.isfinite(lp), lp, 0) + 0.5 * rng.normal(size=len(lp))


def run_policy(kdb, z, targets, old, reference, advantages, weights, temperature, low, high, kl, grad=True, in_place=False):
    rows, cols = z.shape
    on = {n: kdb.to_device(a) if a is not None else None for n, a in dict(z=z, t=targets, old=old, ref=reference, a=advantages, w=weights).items()}
    ptr = {n: a.ptr if a is not None else None for n, a in on.items()}
    losses, logps = kdb.empty((rows,), z.dtype), kdb.empty((rows,), np.float64)
    out = on["z"] if in_place else kdb.empty(z.shape, z.dtype) if grad else None
    policy = kd.Policy(ptr["old"], ptr["ref"], ptr["a"], temperature, low, high, kl)
    kdb.call("policy_rows", kd.DTYPE_OF[z.dtype], losses.ptr, logps.ptr, out.ptr if out else None, ptr["z"], ptr["t"], policy,
             ptr["w"] if grad else None, rows, cols)
    return losses.numpy(), logps.numpy(), out.numpy() if out else None


def check_policy(kdb, z, targets, old, reference, advantages, weights, temperature, low, high, kl, **how):
    losses, logps, grad = run_policy(kdb, z, targets, old, reference, advantages, weights, temperature, low, high, kl, **how)
    eps = np.finfo(z.dtype).eps
    lp = answers.token_logps(z, targets, temperature)
    there = answers.counted(targets, z.shape[1])
    off = logp_tolerance(z, temperature)
    same(logps, lp, off * there)
    want, slopes = answers.policy(lp, targets, z.shape[1], old, reference, advantages, low, high, kl)
    # the terms' derivatives with respect to lp, by its tolerance
    with np.errstate(over="ignore", invalid="ignore"):
        ratio = np.exp(lp - old) * np.abs(advantages) if old is not None else np.abs(advantages)
        away = kl * np.exp(reference - lp) if reference is not None and kl else 0
        moved = np.where(there, 2 * off * (ratio + away + kl) + 2.0 ** -48 * (ratio + away + kl), 0)
    same(losses, want, moved + eps / 2 * np.abs(want) + np.finfo(z.dtype).tiny)
    if grad is not None:
        slopes = slopes * weights.astype(np.float64)
        grown = np.zeros(z.shape)
        soft = np.exp(answers.shares(z, temperature))
        soft[np.flatnonzero(there), targets[there]] += 1
        grown[there] = (moved * np.abs(weights.astype(np.float64)))[there, None] * soft[there] / temperature
        same(grad, answers.token_logps_grad(z, targets, slopes, temperature), grad_tolerance(z, targets, slopes, temperature) + grown)
    return losses, logps, grad


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_the_policy_loss_and_its_gradient(kdb, shape, dtype):
    rng = np.random.default_rng(2 * sum(shape))
    for temperature, given, kl, in_place in ((1.0, True, 0.1, False), (0.6, False, 0.1, True), (1.3, True, 0.0, False)):
        z, targets = logits_of(rng, *shape, dtype)
        lp = answers.token_logps(z, targets, temperature)
        old, reference = policy_of(rng, lp, targets, shape[1], 0.2, 0.3)
        advantages, weights = rng.normal(size=(2, shape[0])).astype(dtype)
        advantages[::7] = 0
        for how in (dict(in_place=in_place), dict(grad=False)):
            check_policy(kdb, z, targets, old if given else None, reference if kl else None, advantages, weights, temperature,
                         0.2, 0.3, kl, **how)


@pytest.mark.parametrize("cols", [40, 700, 3000, 50257, 120001])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_masked_logits_and_rows_without_a_distribution(kdb, dtype, cols):
    """Logits of -inf and of the type's lowest value, a target among them, rows of nothing else, infinities and NaN; rows
    without a target hold anything and give 0; far offsets cost nothing."""
    rng = np.random.default_rng(cols)
    z, targets = logits_of(rng, 12, cols, dtype)
    targets[:] = rng.integers(0, cols // 2, 12)
    z[0, cols // 2:] = -np.inf
    z[1, cols // 2:] = np.finfo(dtype).min
    z[2] = -np.inf
    z[3] = np.finfo(dtype).min
    z[4, targets[4]] = -np.inf
    z[5, 3] = np.nan
    z[6, 3] = np.inf
    z[7], targets[7] = np.nan, -1
    z[8], targets[8] = -np.inf, cols
    z[9] += dtype(1e5)
    z[10, 1:] = -np.inf
    targets[10] = 0
    slopes = rng.normal(size=12).astype(dtype)
    slopes[11] = 0
    z[11, 5] = np.nan
    logps, stats, dz, dt = token_logps(kdb, z, targets, 1.0)
    want = answers.token_logps(z, targets, 1.0)
    same(logps.numpy(), want, np.nan_to_num(logp_tolerance(z, 1.0)))
    assert logps.numpy()[10] == 0 and want[4] == -np.inf
    out, ds = kdb.empty(z.shape, dtype), kdb.to_device(slopes)
    kdb.call("token_logps_grad", kd.DTYPE_OF[z.dtype], out.ptr, dz.ptr, stats.ptr, dt.ptr, ds.ptr, *z.shape, 1.0)
    good = [0, 1, 3, 4, 7, 8, 9, 10, 11]
    grad = answers.token_logps_grad(z, targets, slopes, 1.0)
    same(out.numpy()[good], grad[good], np.nan_to_num(grad_tolerance(z, targets, slopes, 1.0))[good])
    assert all(np.isnan(out.numpy()[r]).any() for r in (2, 5, 6))
    advantages, weights = np.ones(12, dtype), np.ones(12, dtype)
    advantages[11] = 0  # neither term nor derivative, whatever the row holds
    losses, lp, grad = run_policy(kdb, z, targets, None, None, advantages, weights, 1.0, 0.2, 0.2, 0.0)
    np.testing.assert_array_equal(np.isnan(losses), np.isin(np.arange(12), (2, 5, 6)))
    np.testing.assert_array_equal(losses[[7, 8, 11]], 0)
    np.testing.assert_array_equal(grad[[7, 8, 11]], 0)
    # a ratio beyond every number: held from above, free below
    old = np.full(12, -5000.0)
    for sign, loss in ((1, -1.2), (-1, np.inf)):
        losses, _, grad = run_policy(kdb, z, targets, old, None, advantages * dtype(sign), weights, 1.0, 0.2, 0.2, 0.0)
        np.testing.assert_allclose(losses[[0, 1, 3, 9]], loss, rtol=2 * np.finfo(dtype).eps)
        if sign == 1:
            assert (grad[[0, 1, 3, 9]] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [5000, 50257, 100003])
def test_rows_far_below_zero_behind_masked_ones(kdb, dtype, cols):
    """Nothing but -inf or the type's lowest value in a row's first thousands, and logits near -1e3 and -1e6 behind them."""
    rng = np.random.default_rng(cols)
    z, targets = logits_of(rng, 4, cols, dtype)
    targets[:] = rng.integers(cols - 100, cols, 4)
    z[:2, :cols - 100] = -np.inf
    z[2:, :cols - 100] = np.finfo(dtype).min
    z[0::2, cols - 100:] -= dtype(1e3)
    z[1::2, cols - 100:] -= dtype(1e6)
    logps, stats, _, _ = token_logps(kdb, z, targets, 1.0)
    with np.errstate(over="ignore"):
        same(logps.numpy(), answers.token_logps(z, targets, 1.0), logp_tolerance(z, 1.0))
    np.testing.assert_array_equal(stats.numpy()[:, 0], z.max(1))
    advantages = np.ones(4, dtype)
    check_policy(kdb, z, targets, None, None, advantages, advantages, 1.0, 0.2, 0.2, 0.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [5000, 50257])
def test_rows_that_rise(kdb, dtype, cols):
    """The largest logits at the end, far above or a little above what comes first, -inf and the type's lowest value ahead."""
    rng = np.random.default_rng(cols)
    z, targets = logits_of(rng, 6, cols, dtype)
    targets[:] = rng.integers(cols - 100, cols, 6)
    for r, rise in enumerate((30, 60, 1e4)):
        z[r, cols - 100:] += dtype(rise)
    z[3, :cols - 50], targets[3] = -np.inf, cols - 3
    z[4, :cols - 1], targets[4] = np.finfo(dtype).min, cols - 1
    z[5, cols - 1], targets[5] = np.finfo(dtype).max, cols - 1
    for temperature in (1.0, 0.05):
        logps, stats, _, _ = token_logps(kdb, z, targets, temperature)
        with np.errstate(over="ignore"):
            same(logps.numpy(), answers.token_logps(z, targets, temperature), logp_tolerance(z, temperature))
        np.testing.assert_array_equal(stats.numpy()[:, 0], z.max(1))


# ---- pairs ----------------------------------------------------------------------------------------


def run_pairs(kdb, dtype, logps, reference, targets, starts, weights, cols, beta, smoothing, rewards=True):
    rows, pairs = len(logps), len(weights)
    on = [kdb.to_device(a) if a is not None else None for a in (logps, reference, targets, starts, weights.astype(dtype))]
    losses, both, slopes = (kdb.to_device(np.full(s, 777, dtype)) for s in ((pairs,), (pairs, 2), (rows,)))
    kdb.call("preference_pairs", kd.DTYPE_OF[np.dtype(dtype)], losses.ptr, both.ptr if rewards else None, slopes.ptr,
             *(a.ptr if a is not None else None for a in on), pairs, rows, cols, beta, smoothing)
    return losses.numpy(), both.numpy(), slopes.numpy()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lengths", [[1, 1], [0, 3], [0, 0], [5, 0, 2, 7], [64, 65, 1, 300], [1000, 2000], [3, 4] * 40, [20000, 7, 0, 1]],
                         ids=lambda v: f"{len(v)}-{sum(v)}")
def test_pairs(kdb, lengths, dtype):
    """Empty answers, rows before the first sequence and behind the last, prompts; the sums' roundings are f64's, a step for
    each of a sum's terms, and beta's derivative is at most beta."""
    rng = np.random.default_rng(sum(lengths))
    ahead, behind = 3, 70
    starts = ahead + np.concatenate(([0], np.cumsum(lengths))).astype(np.int64)
    rows, pairs, cols, eps = int(starts[-1]) + behind, len(lengths) // 2, 11, np.finfo(dtype).eps
    logps = -10 * rng.random(rows)
    targets = rng.integers(-3, cols, rows)
    logps[targets < 0] = 0
    weights = rng.normal(size=pairs).astype(dtype)
    for beta, smoothing, reference in ((0.1, 0.0, logps + 0.3 * rng.normal(size=rows)), (2.0, 0.2, None)):
        got = run_pairs(kdb, dtype, logps, reference, targets, starts, weights, cols, beta, smoothing)
        want = answers.preference(logps, reference, targets, starts, weights.astype(np.float64), cols, beta, smoothing)
        off = beta * 2.0 ** -52 * max(lengths) * (10 if reference is None else 3) * max(max(lengths), 1)
        for g, w, by in zip(got, want, (1.0, 1.0, beta * np.abs(weights).max())):
            same(g, w, off * by + 8 * 2.0 ** -52 + eps / 2 * np.abs(w) * (1 + 1e-9))
    np.testing.assert_array_equal(got[2][:ahead], 0)
    np.testing.assert_array_equal(got[2][rows - behind:], 0)
    assert (run_pairs(kdb, dtype, logps, None, targets, starts, weights, cols, 1.0, 0.0, rewards=False)[1] == 777).all()


def test_pairs_at_the_ends_of_the_range(kdb):
    """Margins beyond the exponential's range, log-probabilities of -inf, starts outside the rows, no pairs."""
    targets, weights = np.zeros(4, np.int64), np.ones(2, np.float32)
    starts = np.array([0, 1, 2, 3, 4], np.int64)
    logps = np.array([-1e5, -1.0, -1.0, -1e5])
    for smoothing in (0.0, 0.25):
        losses, rewards, slopes = run_pairs(kdb, np.float32, logps, None, targets, starts, weights, 3, 1.0, smoothing)
        np.testing.assert_allclose(losses, [(1 - smoothing) * 99999, smoothing * 99999], rtol=1e-7)
        np.testing.assert_allclose(slopes, [smoothing - 1, 1 - smoothing, smoothing, -smoothing], rtol=1e-7)
    logps[0] = -np.inf
    losses, rewards, slopes = run_pairs(kdb, np.float32, logps, None, targets, starts, weights, 3, 1.0, 0.0)
    assert losses[0] == np.inf and rewards[0, 0] == -np.inf and (slopes[:2] == [-1, 1]).all() and losses[1] == 0
    starts = np.array([-7, 1, 2, 3, 2 ** 40], np.int64)
    got = run_pairs(kdb, np.float32, np.array([-1.0, -2, -3, -4]), None, targets, starts, weights, 3, 1.0, 0.0)
    want = answers.preference(np.array([-1.0, -2, -3, -4]), None, targets, starts, weights, 3, 1.0, 0.0)
    for g, w in zip(got, want):
        np.testing.assert_allclose(g, w, rtol=1e-6)
    slopes = kdb.to_device(np.full(1000, 777, np.float64))
    one = kdb.to_device(np.zeros(1000, np.int64))
    kdb.call("preference_pairs", kd.F64, None, None, slopes.ptr, slopes.ptr, None, one.ptr, None, None, 0, 1000, 5, 1.0, 0.0)
    assert (slopes.numpy() == 0).all()
    no_rows = run_pairs(kdb, np.float64, np.zeros(0), None, np.zeros(0, np.int64), np.zeros(3, np.int64), np.ones(1), 3, 1.0, 0.0)
    np.testing.assert_allclose(no_rows[0], np.log(2), rtol=1e-15)
