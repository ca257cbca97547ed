"""Log-probabilities by what their own terms can carry: an exponential's error counts by its share of the sum, so that a confident
target's log-probability is all but exact, whichever call gives it and wherever in the row the target stands."""
import numpy as np
import pytest

import answers
import kd
from test_gpu_answers import grad_tolerance, run_policy, same, token_logps

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]
IDS = ["f32", "f64"]


def by_shares(z, temperature):
    """The least errors of the rows' log-probabilities, from any base up to the row's largest logit. With D = (largest - z) / T,
    and u half a step: the term of D > 0 has D u of the difference's rounding, D u of the exponent's (in f64 two such, of
    1 / T and of the product), 2 u of a power good to one step; one of D = 0 is exactly 1. Of the rest all is f64: the sum over
    cols / 64 values of a lane, 16 waves and 6 steps of lanes; up to 16 + log2(cols) moves from one base to another, three
    steps each; the logarithm's step, and three of (z - largest) / T."""
    u, u64 = np.finfo(z.dtype).eps / 2, 2.0 ** -53
    z = z.astype(np.float64)
    below = (z.max(1, keepdims=True) - z) / temperature
    share = np.exp(-below)
    total = share.sum(1, keepdims=True)
    steps = np.where(below > 0, (2 if u > u64 else 3) * below + 2, 0)
    cols = z.shape[1]
    chain = (cols / 64 + 24 + 3 * (16 + np.log2(cols))) * u64
    return (share * steps).sum(1) / total[:, 0] * u * (1 + 1e-3) + chain + 2 * u64 * np.abs(np.log(total[:, 0])), below


def confident(rng, rows, cols, dtype, rise, temperature):
    """Targets past column 20000 that stand `rise` above the first 16384 columns."""
    z = (2 * rng.normal(size=(rows, cols))).astype(dtype)
    targets = rng.integers(20000, cols, rows)
    z[np.arange(rows), targets] = (z[:, :16384].max(1) + rise * temperature).astype(dtype)
    return z, targets


@pytest.mark.parametrize("rise", [4, 8, 12, 20, 39])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_confident_targets_far_into_a_row(kdb, dtype, rise):
    for rows, temperature in ((4, 1.0), (4, 0.7), (600, 1.0), (600, 0.7)):
        rng = np.random.default_rng(rows + rise)
        z, targets = confident(rng, min(rows, 40), 50257, dtype, rise, temperature)
        want = answers.token_logps(z, targets, temperature)
        off, below = by_shares(z, temperature)
        off = off + 3 * 2.0 ** -53 * below[np.arange(len(z)), targets]
        again = np.arange(rows) % len(z)
        z, targets, want, off = z[again], targets[again], want[again], off[again]
        logps, stats, _, _ = token_logps(kdb, z, targets, temperature)
        weights = np.ones(rows, dtype)
        for grad in (False, True):
            _, lp, _ = run_policy(kdb, z, targets, None, None, weights, weights, temperature, 0.2, 0.2, 0.0, grad=grad)
            same(lp, want, off)
            assert (lp <= 0).all()
        lp = logps.numpy()
        same(lp, want, off)
        assert (lp <= 0).all(), lp.max()
        assert (stats.numpy()[:, 1] >= 1).all()
        if rise >= 12:
            assert off.max() < 1e-7


@pytest.mark.parametrize("shape", [(4000, 90), (3000, 1100), (1000, 9000)], ids=lambda s: "x".join(map(str, s)))
def test_no_lean_over_many_rows(kdb, shape):
    """The mean error of many f32 rows at temperatures of which log2(e) / T is nearly half a step from an f32 number: a constant of one
    f32 alone would shift every logarithm the same way, by half a step times the mean distance from the largest logit.
    Errors that do not lean are a row's sqrt(sum (share steps u)^2) at most, over the rows' root; six of that, and a
    quarter of a step that the power of two may lean by."""
    rng = np.random.default_rng(shape[1])
    worst = []
    for temperature in rng.uniform(0.5, 2, 4000):
        c = np.log2(np.e) / temperature
        worst.append((abs(np.float64(np.float32(c)) - c) / c, temperature))
    for _, temperature in sorted(worst)[-2:]:
        rows, cols = shape
        z = (2 * rng.normal(size=shape)).astype(np.float32)
        targets = rng.integers(0, cols, rows)
        want = answers.token_logps(z, targets, temperature)
        below = (z.max(1, keepdims=True).astype(np.float64) - z) / temperature
        share = np.exp(-below)
        share /= share.sum(1, keepdims=True)
        u = 2.0 ** -24
        spread = np.sqrt((share ** 2 * np.where(below > 0, 2 * below + 2, 0) ** 2).sum()) * u / rows
        bound = 6 * spread + 2.0 ** -25
        # what half a step in all exponents would come to stands well above that
        assert 0.9 * u * (share * below).sum(1).mean() > 1.5 * bound
        weights = np.ones(rows, np.float32)
        for lp in (token_logps(kdb, z, targets, temperature)[0].numpy(),
                   run_policy(kdb, z, targets, None, None, weights, weights, temperature, 0.2, 0.2, 0.0)[1]):
            assert abs((lp - want).mean()) <= bound, ((lp - want).mean(), bound)


def held(kdb, z, targets, temperature, kl, advantages, moved, away):
    """A policy whose old and reference log-probabilities stand `moved` below and `away` above the ones that the call gives."""
    rows = len(z)
    weights = np.ones(rows, z.dtype)
    _, lp, _ = run_policy(kdb, z, targets, None, None, advantages, weights, temperature, 0.2, 0.3, 0.0)
    old, reference = lp - moved, lp + away
    losses, again, grad = run_policy(kdb, z, targets, old, reference, advantages, weights, temperature, 0.2, 0.3, kl)
    np.testing.assert_array_equal(again, lp)
    return losses, grad, lp - old, reference - lp


@pytest.mark.parametrize("shape", [(90, 40), (30, 700), (15, 3001), (15, 9000)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_model_that_is_still_close_to_its_reference(kdb, dtype, shape):
    """exp(d) - d - 1 is d^2 / 2 and its derivative d for small d. expm1 is good to one step; the difference, the weight and
    the result are half a step each."""
    rng = np.random.default_rng(shape[1])
    rows, cols = shape
    z = (2 * rng.normal(size=shape)).astype(dtype)
    targets = rng.integers(0, cols, rows)
    away = np.resize([1e-8, -1e-8, 3e-7, -1e-6, 1e-4, -1e-2, 0.3, -2, 20, -40, 0, 7e-9, -1.1e-8, 1e-7, 3e-3], rows)
    losses, grad, _, d = held(kdb, z, targets, 0.8, 0.3, np.zeros(rows, dtype), 0.0, away)
    e = np.expm1(d.astype(np.longdouble))
    want = 0.3 * (e - d)
    off = 0.3 * 2.0 ** -52 * np.abs(e) + (2.0 ** -52 + np.finfo(dtype).eps / 2) * np.abs(want) + np.finfo(dtype).tiny
    same(losses, want.astype(np.float64), off.astype(np.float64))
    slopes = (-0.3 * e).astype(np.float64)
    same(grad, answers.token_logps_grad(z, targets, slopes, 0.8), grad_tolerance(z, targets, slopes, 0.8))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_ratios_near_and_far_from_one_beside_a_reference(kdb, dtype):
    """A ratio is good to two steps (an exponential's one and two halves) however small or large it is; f32's one rounding more."""
    rng = np.random.default_rng(1)
    moved = np.array([-600, -80, -40, -3, -0.5, -1e-9, 0, 1e-9, 0.1, 0.5, 3, 40, 80])
    rows = len(moved)
    z = (2 * rng.normal(size=(rows, 50))).astype(dtype)
    targets = rng.integers(0, 50, rows)
    advantages = np.where(moved <= 0, 1, -1).astype(dtype)  # where no clip holds the ratio
    losses, _, moved, _ = held(kdb, z, targets, 1.0, 0.1, advantages, moved, 0.0)
    want = -np.exp(moved.astype(np.longdouble)) * advantages
    off = (2.0 ** -51 + np.finfo(dtype).eps / 2) * np.abs(want) + np.finfo(dtype).tiny * (dtype is np.float32)
    same(losses, want.astype(np.float64), off.astype(np.float64))
