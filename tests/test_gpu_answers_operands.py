"""Operands of the losses that stand elsewhere than a test's usually do: in each other's place, behind an odd element, in logits that
pass the caches or 32 bits of offsets. A row's bits depend on none of that."""
import numpy as np
import pytest

import answers
import kd
from test_gpu_answers import logits_of, policy_of, run_policy

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
