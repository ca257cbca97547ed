"""What kd_counter_dropout, kd_block_rows*, kd_token_logps*, kd_preference_pairs and kd_policy_rows refuse, on the host: no
device is needed, none is touched."""
import ctypes

import pytest

import kd

A = 1 << 30  # addresses that no check reads, a GiB apart
INVALID, UNSUPPORTED = -1, -4
NAN, INF = float("nan"), float("inf")


def at(n):
    return (n + 1) * A


@pytest.fixture(scope="module")
def lib():
    return kd.Backend()


def refused(lib, f, good, changes, name):
    for place, value, status in changes:
        args = list(good)
        args[place] = value
        assert f(*args) == status, (place, value)
        assert lib.error().startswith(name), lib.error()


def test_bad_dropouts(lib):
    c = kd.Counter(1, 2, 3, 0, None)
    refused(lib, lib.lib.kd_counter_dropout, [kd.F32, at(0), at(1), 10, 8, 0.5, c], (
        (0, kd.I64, UNSUPPORTED), (0, 9, UNSUPPORTED), (1, None, INVALID), (2, None, INVALID), (3, -1, INVALID), (4, -1, INVALID),
        (3, 1 << 62, INVALID), (5, 0.0, INVALID), (5, -0.5, INVALID), (5, 1.5, INVALID), (5, NAN, INVALID), (5, 2.0 ** -33, INVALID),
        (6, None, INVALID), (6, kd.Counter(1, 2, 3, -1, None), INVALID), (6, kd.Counter(1, 2, 3, 2 ** 32 - 9, None), INVALID),
        (6, kd.Counter(1, 2, 3, 2 ** 62, None), INVALID), (6, kd.Counter(1, 2, 3, 0, A + 4), INVALID), (2, at(0) + 4, INVALID),
        (2, at(0) - 4, INVALID), (4, 2 ** 34 + 1, INVALID)), "kd_counter_dropout")
    for rows, cols in ((0, 8), (8, 0)):
        assert lib.lib.kd_counter_dropout(kd.F64, None, None, rows, cols, 0.5, c) == 0


def block(**changes):
    given = dict(x=at(0), residual=at(1), gate=at(2), rows=10, cols=8, gate_rows=1, residual_scale=1.0, block_scale=1.0, keep=0.5,
                 after=kd.Norm(at(3), at(4), 1e-5, kd.NORM_LAYER), before=kd.Norm(at(5), at(6), 1e-5, kd.NORM_RMS),
                 counter=kd.Counter(1, 2, 3, 0, None))
    given.update(changes)
    return kd.Block(*given.values())


BLOCKS = [dict(rows=-1), dict(cols=-1), dict(rows=1 << 45, cols=1 << 20), dict(x=None), dict(gate_rows=0), dict(gate_rows=2),
          dict(gate_rows=-1), dict(gate=None), dict(residual_scale=NAN), dict(block_scale=INF), dict(keep=0.0), dict(keep=1.01),
          dict(after=kd.Norm(at(3), at(4), -1.0, kd.NORM_LAYER)), dict(before=kd.Norm(at(3), at(4), NAN, kd.NORM_RMS)),
          dict(before=kd.Norm(at(3), at(4), INF, kd.NORM_RMS)), dict(after=kd.Norm(at(3), at(4), 1.0, 3)),
          dict(after=kd.Norm(at(3), at(4), 1.0, -1)), dict(counter=kd.Counter(1, 2, 3, 2 ** 32 - 5, None))]


def backward(lib, b, grads=None, h=at(8), stats=at(9), grad_h=at(10), grad_y=at(11), room=at(12), size=1 << 20):
    grads = grads or kd.BlockGrads(at(13), at(14), at(15), at(16), at(17), at(18), at(19))
    return lib.lib.kd_block_rows_backward(kd.F32, grads, b, h, stats, grad_h, grad_y, room, size)


@pytest.mark.parametrize("changes", BLOCKS, ids=lambda c: "-".join(c))
def test_bad_blocks(lib, changes):
    assert lib.lib.kd_block_rows(kd.F32, at(8), at(9), at(10), block(**changes)) == INVALID
    assert lib.error().startswith("kd_block_rows:")
    assert backward(lib, block(**changes)) == INVALID
    assert lib.error().startswith("kd_block_rows_backward:")


def test_bad_forward_calls(lib):
    f = lib.lib.kd_block_rows
    size = 10 * 8 * 4
    refused(lib, f, [kd.F32, at(8), at(9), at(10), block()], (
        (0, kd.I64, UNSUPPORTED), (4, None, INVALID), (1, at(9), INVALID), (1, at(9) + size - 4, INVALID), (1, at(0) + 4, INVALID),
        (1, at(1) - 4, INVALID), (2, at(0) + 4, INVALID), (2, at(2), INVALID), (1, at(3), INVALID), (2, at(6) + 4, INVALID),
        (3, at(0), INVALID), (3, at(8) + 8, INVALID), (3, at(5), INVALID), (3, at(1), INVALID)), "kd_block_rows:")
    assert f(kd.F32, at(8), at(9), None, block(before=kd.Norm())) == INVALID  # y without a norm
    for changes in (dict(rows=0, gate_rows=0, gate=None), dict(rows=0, gate_rows=1), dict(cols=0)):
        assert f(kd.F32, None, None, None, block(**changes)) == 0


def test_bad_backward_calls(lib):
    for how in (dict(stats=None), dict(h=None), dict(room=None), dict(size=100), dict(room=at(12) + 8), dict(grad_h=at(14) + 4),
                dict(room=at(13)), dict(h=at(13)), dict(h=at(14)), dict(stats=at(13)), dict(grad_h=at(15)), dict(grad_y=at(16))):
        assert backward(lib, block(), **how) == INVALID, how
        assert lib.error().startswith("kd_block_rows_backward:")
    for grads in (kd.BlockGrads(at(13), at(13)), kd.BlockGrads(at(13), at(14), at(14)), kd.BlockGrads(residual=at(0) + 4, x=at(0)),
                  kd.BlockGrads(at(2)), kd.BlockGrads(after_weight=at(3)), kd.BlockGrads(before_bias=at(5)), kd.BlockGrads(residual=at(0))):
        assert backward(lib, block(), grads) == INVALID
    none = kd.Norm()
    assert backward(lib, block(before=none)) == INVALID  # grad_y without a norm
    assert backward(lib, block(before=none), kd.BlockGrads(before_weight=at(13)), grad_y=None) == INVALID
    assert backward(lib, block(after=none), kd.BlockGrads(after_bias=at(13))) == INVALID
    assert backward(lib, block(gate=None, gate_rows=0), kd.BlockGrads(gate=at(13))) == INVALID
    assert lib.lib.kd_block_rows_backward(kd.F32, None, block(), at(8), at(9), at(10), at(11), at(12), 1 << 20) == INVALID
    assert lib.lib.kd_block_rows_backward(kd.I64, kd.BlockGrads(), block(), at(8), at(9), at(10), at(11), at(12), 1 << 20) == UNSUPPORTED
    assert backward(lib, block(), kd.BlockGrads()) == 0 and backward(lib, block(cols=0)) == 0
    n = ctypes.c_int64()
    f = lib.lib.kd_block_rows_workspace
    assert f(None, kd.F32, 3, 3) == INVALID and f(ctypes.byref(n), kd.F32, -1, 3) == INVALID and f(ctypes.byref(n), kd.I64, 3, 3) == UNSUPPORTED
    assert f(ctypes.byref(n), kd.F32, 10, 8) == 0 and n.value > 0
    assert f(ctypes.byref(n), kd.F32, 0, 8) == 0 and n.value == 0


def test_bad_log_probabilities(lib):
    sizes = ((5, -1), (6, 0), (5, 1 << 22), (6, 1 << 31), (7, 0.0), (7, 1e7), (7, NAN))
    refused(lib, lib.lib.kd_token_logps, [kd.F32, at(0), at(1), at(2), at(3), 10, 8, 1.0],
            [(0, kd.BOOL, UNSUPPORTED)] + [(i, None, INVALID) for i in range(1, 5)] + [(i, v, INVALID) for i, v in sizes], "kd_token_logps:")
    refused(lib, lib.lib.kd_token_logps_grad, [kd.F32, at(0), at(1), at(2), at(3), at(4), 10, 8, 1.0],
            [(0, kd.BOOL, UNSUPPORTED), (1, at(1) + 4, INVALID)] + [(i, None, INVALID) for i in range(1, 6)] +
            [(i + 1, v, INVALID) for i, v in sizes], "kd_token_logps_grad:")
    assert lib.lib.kd_token_logps(kd.F32, None, None, None, None, 0, 8, 1.0) == 0
    assert lib.lib.kd_token_logps_grad(kd.F32, None, None, None, None, None, 0, 8, 1.0) == 0


def test_bad_pairs(lib):
    good = [kd.F32, at(0), at(1), at(2), at(3), at(4), at(5), at(6), at(7), 3, 10, 8, 0.1, 0.1]
    refused(lib, lib.lib.kd_preference_pairs, good, [(0, kd.I64, UNSUPPORTED)] + [(i, None, INVALID) for i in (1, 3, 4, 6, 7, 8)] + [
        (9, -1, INVALID), (9, 1 << 22, INVALID), (10, -1, INVALID), (10, 1 << 22, INVALID), (11, 0, INVALID), (12, 0.0, INVALID),
        (12, NAN, INVALID), (12, 1e7, INVALID), (13, -0.1, INVALID), (13, 0.5, INVALID), (13, NAN, INVALID)], "kd_preference_pairs:")
    assert lib.lib.kd_preference_pairs(kd.F32, *[None] * 8, 0, 0, 8, 0.1, 0.1) == 0


def test_bad_policies(lib):
    def policy(old=at(6), reference=at(7), advantages=at(8), temperature=1.0, low=0.2, high=0.2, kl=0.1):
        return kd.Policy(old, reference, advantages, temperature, low, high, kl)

    good = [kd.F32, at(0), at(1), at(2), at(3), at(4), policy(), at(5), 10, 8]
    refused(lib, lib.lib.kd_policy_rows, good, [(0, kd.I64, UNSUPPORTED)] + [(i, None, INVALID) for i in (1, 4, 5, 6, 7)] + [
        (3, at(3) + 4, INVALID), (8, -1, INVALID), (8, 1 << 22, INVALID), (9, 0, INVALID), (9, 1 << 31, INVALID)] + [
        (6, policy(**c), INVALID) for c in (dict(advantages=None), dict(temperature=0.0), dict(temperature=INF), dict(low=-0.1), dict(low=1.1),
                                            dict(low=NAN), dict(high=-0.1), dict(high=INF), dict(kl=-1.0), dict(kl=NAN))], "kd_policy_rows:")
    assert lib.lib.kd_policy_rows(kd.F32, None, None, None, None, None, policy(), None, 0, 8) == 0


def test_an_output_over_the_first_norms_bias(lib):
    assert backward(lib, block(), kd.BlockGrads(x=at(4), gate=at(15))) == INVALID
    assert backward(lib, block(), kd.BlockGrads(after_bias=at(4), gate=at(15))) == INVALID
    assert lib.error().startswith("kd_block_rows_backward:")
    assert lib.lib.kd_block_rows(kd.F32, at(8), at(9), at(10), block(cols=(1 << 28) + 4)) == INVALID


@pytest.mark.parametrize("dtype", [kd.F32, kd.F64])
@pytest.mark.parametrize("cols", [1, 30, 256, 1000, 1537, 2048, 4068, 4096, 5120, 20000])
def test_a_workspace_serves_fewer_rows(lib, cols, dtype):
    n = ctypes.c_int64()
    last = 0
    for rows in [*range(0, 1200), *range(1200, 70000, 37), 1 << 20, (1 << 20) + 1, 1 << 30]:
        assert lib.lib.kd_block_rows_workspace(ctypes.byref(n), dtype, rows, cols) == 0
        assert n.value >= last, rows
        last = n.value


def crossing(lib, f, good, rows, name):
    """`rows`: (argument, other argument, offset) triples of which one lies over the other's bytes."""
    for place, other, by in rows:
        args = list(good)
        args[place] = args[other] + by
        assert f(*args) == INVALID, (place, other, by)
        assert lib.error().startswith(name), lib.error()


def test_outputs_of_the_losses_over_their_operands(lib):
    """10 rows of 8 in f32: 320 bytes of logits, 80 of stats, targets and log-probabilities, 40 of a number a row."""
    crossing(lib, lib.lib.kd_token_logps, [kd.F32, at(0), at(1), at(2), at(3), 10, 8, 1.0],
             ((1, 2, 0), (1, 3, 0), (1, 3, 312), (2, 3, 76), (2, 3, 0), (2, 1, 76), (2, 4, -72), (1, 4, 72), (1, 2, -72)), "kd_token_logps:")
    crossing(lib, lib.lib.kd_token_logps_grad, [kd.F32, at(0), at(1), at(2), at(3), at(4), 10, 8, 1.0],
             ((1, 3, 0), (1, 3, 76), (1, 4, 0), (1, 4, -316), (1, 5, 36), (1, 5, 0)), "kd_token_logps_grad:")
    pairs = [kd.F32, at(0), at(1), at(2), at(3), at(4), at(5), at(6), at(7), 3, 10, 8, 0.1, 0.1]
    crossing(lib, lib.lib.kd_preference_pairs, pairs, [(1, 2, 0), (1, 3, 36), (2, 3, -20), (3, 2, 20)] + [
        (i, j, 0) for i in (1, 2, 3) for j in range(4, 9)], "kd_preference_pairs:")
    pairs[0] = kd.F64
    crossing(lib, lib.lib.kd_preference_pairs, pairs, ((3, 4, 8), (3, 5, -8), (3, 6, 0), (1, 4, 0)), "kd_preference_pairs:")

    def policy(lib, losses, logps, grad, logits, targets, old, reference, advantages, weights):
        return lib.lib.kd_policy_rows(kd.F32, losses, logps, grad, logits, targets, kd.Policy(old, reference, advantages, 1.0, 0.2, 0.2, 0.1),
                                      weights, 10, 8)

    good = [lib] + [at(i) for i in range(9)]
    crossing(lib, policy, good, ((1, 2, 0), (1, 2, 76), (2, 1, -76 + 4), (1, 3, 316), (3, 1, 36), (3, 2, 0), (1, 4, 0), (2, 4, 312), (3, 4, 4),
                                 (3, 5, 0), (1, 5, 0), (2, 5, 0), (3, 6, 0), (3, 7, 0), (3, 8, 0), (3, 9, 0), (2, 6, 8), (2, 7, -8), (2, 8, 0),
                                 (2, 9, 0), (1, 8, 4), (1, 9, -4), (1, 6, 0), (1, 7, 0)), "kd_policy_rows:")


def test_misaligned_operands_of_the_losses(lib):
    for f, good, places, name in (
            (lib.lib.kd_token_logps, [kd.F64, at(0), at(1), at(2), at(3), 10, 8, 1.0], (1, 2, 3, 4), "kd_token_logps:"),
            (lib.lib.kd_token_logps_grad, [kd.F64, at(0), at(1), at(2), at(3), at(4), 10, 8, 1.0], (1, 2, 3, 4, 5), "kd_token_logps_grad:"),
            (lib.lib.kd_preference_pairs, [kd.F64] + [at(i) for i in range(8)] + [3, 10, 8, 0.1, 0.1], range(1, 9), "kd_preference_pairs:")):
        refused(lib, f, good, [(i, good[i] + 4, INVALID) for i in places], name)
    assert lib.lib.kd_token_logps(kd.F32, at(0), at(1) + 2, at(2), at(3), 10, 8, 1.0) == INVALID


def test_misaligned_statistics_of_a_block(lib):
    assert lib.lib.kd_block_rows(kd.F32, at(8), at(9), at(10) + 4, block()) == INVALID
    assert lib.error().startswith("kd_block_rows:")
    assert backward(lib, block(), stats=at(9) + 4) == INVALID
    assert lib.error().startswith("kd_block_rows_backward:")


def test_outputs_over_a_masks_step(lib):
    """The step is read by every workgroup, while others write."""
    counter = kd.Counter(1, 2, 3, 0, at(20))
    for by in (-4, 0, 4):
        assert lib.lib.kd_counter_dropout(kd.F32, at(20) + by, at(1), 10, 8, 0.5, counter) == INVALID
        assert lib.error().startswith("kd_counter_dropout:")
        masked = block(counter=counter)
        for args in ((at(20) + by, at(9), at(10)), (at(8), at(20) - 316, at(10)), (at(8), at(9), at(20) - 312)):
            assert lib.lib.kd_block_rows(kd.F32, *args, masked) == INVALID
            assert lib.error().startswith("kd_block_rows:")
        for grads in (kd.BlockGrads(x=at(20) + by), kd.BlockGrads(residual=at(20) - 316), kd.BlockGrads(before_bias=at(20) + by)):
            assert backward(lib, masked, grads) == INVALID
            assert lib.error().startswith("kd_block_rows_backward:")
        assert backward(lib, masked, room=at(20) - 16) == INVALID
