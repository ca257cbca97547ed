"""kd_paged_attention at the ends of f32's range: values of tiny size. Against the definition in 64 bits
(tests/paged.py).
"""
import numpy as np
import pytest

import kd
import paged
from test_gpu_paged import batch_of, run_attention, workspace_for

pytestmark = pytest.mark.gpu

ROWS = [1, 3, 40]  # new tokens of a sequence, one kernel each


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
