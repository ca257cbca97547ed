"""kd_paged_attention at the ends of f32's range: values of tiny size, pages whose values are far larger than the others',
scores that f32 holds to no better than many units, key scales that are not finite. Against the definition in 64 bits
(tests/paged.py).
"""
import numpy as np
import pytest

import kd
import paged
from test_gpu_paged import batch_of, run_attention, workspace_for

pytestmark = pytest.mark.gpu

ROWS = [1, 3, 40]  # new tokens of a sequence, one kernel each


def sums_of_weights(cache, starts, lengths, q, scale):
    """Each row's sum of weights, in units of the largest, [tokens, heads, 1]."""
    total = np.ones((*q.shape[:2], 1))
    group = q.shape[1] // cache.kv_heads
    for s, length in enumerate(lengths):
        n = starts[s + 1] - starts[s]
        for h in range(q.shape[1]):
            k, _, there = paged.values_of(cache, s, h // group, length)
            for i in range(n):
                seen = there & (np.arange(length) <= length - n + i)
                score = k[seen] @ q[starts[s] + i, h].astype(np.float64) * scale
                total[starts[s] + i, h] = np.exp(score - score.max()).sum()
    return total


@pytest.mark.parametrize("split", [False, True], ids=["whole", "parts"])
@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e-27, 1e-30])
def test_attention_of_tiny_values(kdb, size, dim, new, split):
    """Every value scale around 2^-97 or 2^-107: within the definition's tolerance, which is relative to them."""
    rng = np.random.default_rng(21)
    keys = 3000 if split else 300
    starts, lengths, tokens = batch_of([new], [keys])
    cache = paged.Cache(rng, 1, -(-keys // 64), 1, 64, dim)
    cache.value_scales *= np.float32(size)
    q = rng.normal(0, 1, (tokens, 2, dim)).astype(np.float32)
    if new == 1:
        q = q[:, :1].copy()
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    got = run_attention(kdb, on, q, dim ** -0.5, keys, workspace_for(kdb, q.shape[1], 1, dim, 1, tokens, 1 << 20))
    off = np.abs(got - want)
    assert (off <= tolerance).all(), (off / tolerance).max()


@pytest.mark.parametrize("keys", [300, 3000])  # in one launch and in parts
@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e-33, 1e-35, 1e-37, 1e-39])
def test_attention_of_values_near_the_least(kdb, size, dim, new, keys):
    """Value scales around 2^-117, 2^-123, 2^-130 and 2^-137, the last two below the least normal number. A weight in
    units of 2^-149 is off by half a unit, so the sums of n keys by n * 127 * 2^-150, divided by the weights' sum, beside the
    definition's tolerance and 16 roundings to multiples of 2^-149."""
    rng = np.random.default_rng(22)
    starts, lengths, tokens = batch_of([new], [keys])
    cache = paged.Cache(rng, 1, -(-keys // 64), 1, 64, dim)
    cache.value_scales = (cache.value_scales * np.float64(size)).astype(np.float32)
    q = rng.normal(0, 1, (tokens, 1, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    tolerance = tolerance + keys * 127 * 2.0 ** -150 / sums_of_weights(cache, starts, lengths, q, dim ** -0.5) + 16 * 2.0 ** -150
    got = run_attention(kdb, on, q, dim ** -0.5, keys, workspace_for(kdb, 1, 1, dim, 1, tokens, 1 << 20))
    off = np.abs(got - want)
    assert (off <= tolerance).all(), (off / tolerance).max()
    assert (tolerance < 0.1 * np.abs(want).max()).all()  # a sum that is lost is seen


@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ratio", [24, 40, 60, 90])
def test_attention_beside_values_of_any_size(kdb, dim, new, ratio):
    """One page's values are 2^ratio times the others', its keys' weights 2^-ratio / 8000: the error follows what the rows sum
    up. The definition's tolerance, with the weighted mean of |v| in place of its largest. The page comes first, in the middle
    and last."""
    rng = np.random.default_rng(23)
    starts, lengths, tokens = batch_of([new], [500])
    for column in (0, 12, 29):
        cache = paged.Cache(rng, 1, 32, 1, 16, dim)
        far = cache.table[0, column]
        cache.keys[far] = -127
        cache.key_scales[far] = (np.log(2.0) * ratio + 9) / (127 * dim ** 0.5)
        cache.value_scales[far] = 0.0175 * 2.0 ** ratio
        q = (1 + 0.1 * rng.normal(0, 1, (tokens, 1, dim))).astype(np.float32)
        on = paged.Device(kdb, cache, starts, lengths, tokens)
        want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
        k, v, _ = paged.values_of(cache, 0, 0, 500)
        for i in range(tokens):
            seen = 500 - new + i + 1
            score = k[:seen] @ q[i, 0].astype(np.float64) * dim ** -0.5
            p = np.exp(score - score.max())
            tolerance[i] *= (p @ np.abs(v[:seen]) / p.sum()).max() / np.abs(v[:seen]).max()
        got = run_attention(kdb, on, q, dim ** -0.5, 500)
        off = np.abs(got - want)
        assert (off <= tolerance).all(), (column, (off / tolerance).max())


@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 21, 2.0 ** 25, 2.0 ** 33, -2.0 ** 33, 2.0 ** 60, 2.0 ** 110])
def test_attention_of_scores_far_from_zero(kdb, size, dim, new):
    """Scores of 2^21 to 2^110 in size: the largest has the whole weight, and the row is its key's values. Their weighted sum is exact
    but for the unit's pieces (2^-22) and the quotient, the joins of waves multiply by 1: 2^-20 of the value."""
    rng = np.random.default_rng(24)
    keys = 700
    starts, lengths, tokens = batch_of([new], [keys])
    cache = paged.Cache(rng, 1, 44, 1, 16, dim)
    q = rng.normal(0, 1, (tokens, 1, dim)).astype(np.float32)
    k, v, _ = paged.values_of(cache, 0, 0, keys)
    unit = np.abs(k @ q[:, 0].T.astype(np.float64)).max(0)  # scores of about 1 by it
    q = (q / unit[:, None, None] * np.sqrt(abs(size))).astype(np.float32)
    scale = float(np.sign(size) * np.sqrt(abs(size)))
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    got = run_attention(kdb, on, q, scale, keys)
    compared = 0
    for i in range(tokens):
        score = k[:keys - new + i + 1] @ q[i, 0].astype(np.float64) * scale
        order = np.argsort(score)
        if score[order[-1]] - score[order[-2]] < max(2.0 ** -16 * np.abs(score).max(), 40):
            continue  # the roundings of the scores decide between the two
        compared += 1
        want = v[order[-1]]
        assert (np.abs(got[i, 0] - want) <= 2.0 ** -20 * np.abs(want)).all(), (i, score[order[-1]])
    assert compared >= 0.8 * tokens


@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", [np.inf, np.nan])
def test_a_key_scale_that_is_not_finite_gives_nan(kdb, which, dim, new):
    """Also where the page's scores would all be -inf, whose weights are nothing."""
    rng = np.random.default_rng(25)
    starts, lengths, tokens = batch_of([new, new], [300, 300])
    cache = paged.Cache(rng, 2, 19, 1, 16, dim)
    cache.keys[cache.table[0, 4]] = -1
    cache.key_scales[cache.table[0, 4]] = which
    cache.key_scales[cache.table[1, 18]] = which
    lengths = [300, 280]  # the second sequence's page is not seen
    q = np.abs(rng.normal(0, 1, (tokens, 1, dim))).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    got = run_attention(kdb, on, q, dim ** -0.5, 300)
    assert np.isnan(got[:new]).all()
    with np.errstate(invalid="ignore"):
        want, tolerance = paged.attention(cache, starts, lengths, np.where(np.arange(tokens)[:, None, None] < new, 0, q), dim ** -0.5)
    assert (np.abs(got - want) <= tolerance)[new:].all()


@pytest.mark.parametrize("new", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", [np.inf, np.nan])
def test_a_value_scale_that_is_not_finite_gives_nan(kdb, which, dim, new):
    """Beside values near f32's largest, and of keys whose weight is next to nothing."""
    rng = np.random.default_rng(26)
    starts, lengths, tokens = batch_of([new], [300])
    cache = paged.Cache(rng, 1, 19, 1, 16, dim)
    cache.value_scales[:] = 2.0 ** 120
    far = cache.table[0, 9]
    cache.keys[far], cache.key_scales[far] = -1, 8 / dim ** 0.5  # scores of about -8 with queries of 1
    cache.value_scales[far] = which
    q = np.ones((tokens, 1, dim), np.float32)
    got = run_attention(kdb, paged.Device(kdb, cache, starts, lengths, tokens), q, dim ** -0.5, 300)
    assert np.isnan(got).all()
