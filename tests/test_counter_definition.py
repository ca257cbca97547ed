"""The counter's words against the published known answers of Philox4x32-10 (Random123's kat_vectors), and the definitions of
tests/block.py and tests/answers.py against differences: no device is needed."""
import numpy as np
import pytest

import answers
import block
import kd


@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_known_answers(counter, key, words):
    assert tuple(int(w) for w in block.philox(counter, key)) == words


def test_a_mask_keeps_its_share_and_changes_with_every_part_of_the_counter():
    n, keep = 400, 0.7
    masks = [block.kept(n, n, keep, **c) for c in (dict(), dict(seed=1), dict(seed=1 << 40), dict(stream=1), dict(step=1), dict(row=n))]
    for m in masks:  # within six deviations
        assert abs(m.mean() - keep) < 6 * np.sqrt(keep * (1 - keep) / n / n)
    for i in range(len(masks)):
        for j in range(i):
            same = keep ** 2 + (1 - keep) ** 2
            assert abs((masks[i] == masks[j]).mean() - same) < 6 * np.sqrt(same * (1 - same)) / n
    assert (block.kept(5, 9, keep, row=3) == block.kept(8, 9, keep)[3:]).all()
    assert (block.kept(3, 9, keep, step=7) == block.kept(3, 9, keep, step=2, more=5)).all()


@pytest.mark.parametrize("after", [None, kd.NORM_LAYER, kd.NORM_RMS])
@pytest.mark.parametrize("before", [None, kd.NORM_LAYER, kd.NORM_RMS])
@pytest.mark.parametrize("gate", [0, 1, 2])
def test_the_blocks_gradients_are_its_differences(after, before, gate):
    """Central differences of step 1e-5: their own error is 1e-10 of third derivatives and 1e-16 / 1e-5 of the values."""
    rng = np.random.default_rng(7)
    rows, cols = 3, 6
    norms = {n: kind and dict(kind=kind, eps=1e-3, weight=rng.normal(size=cols), bias=rng.normal(size=cols))
             for n, kind in (("after", after), ("before", before))}
    given = dict(x=rng.normal(size=(rows, cols)), residual=rng.normal(size=(rows, cols)),
                 gate=[None, rng.normal(size=cols), rng.normal(size=(rows, cols))][gate])
    grad_h, grad_y = rng.normal(size=(2, rows, cols))

    def case():
        return block.Case(**given, **{n: v or None for n, v in norms.items()}, residual_scale=0.7, block_scale=1.3, keep=0.8, seed=5)

    def value():
        h = case().sum()[0]
        return (grad_h * h).sum() + ((grad_y * case().next(h)[0]).sum() if before else 0)

    grads = case().backward(case().sum()[0], grad_h, grad_y if before else None)
    leaves = {"x": given["x"], "residual": given["residual"], "gate": given["gate"]}
    leaves.update({f"{n}_{p}": v[p] for n, v in norms.items() if v for p in ("weight", "bias")})
    for name, leaf in leaves.items():
        if leaf is None:
            continue
        for at in np.ndindex(leaf.shape):
            was, step = leaf[at], 1e-5
            leaf[at] = was + step
            up = value()
            leaf[at] = was - step
            down = value()
            leaf[at] = was
            assert abs((up - down) / (2 * step) - grads[name][0][at]) < 1e-7, (name, at)


def test_the_losses_gradients_are_their_differences():
    rng = np.random.default_rng(8)
    rows, cols = 9, 5
    z, targets = rng.normal(size=(rows, cols)), rng.integers(0, cols, rows)
    targets[[1, 4]] = -1
    starts, weights = np.array([0, 3, 5, 6, 8]), np.array([0.3, -1.1])
    reference, old, advantages = rng.normal(size=(3, rows)) - 1.5

    def pairs(z):
        losses, _, slopes = answers.preference(answers.token_logps(z, targets, 0.7), reference, targets, starts, weights, cols, 0.4, 0.1)
        return (weights * losses).sum(), slopes

    def policy(z):
        losses, slopes = answers.policy(answers.token_logps(z, targets, 0.7), targets, cols, old, reference, advantages, 0.2, 0.3, 0.5)
        return losses.sum(), slopes

    for loss in (pairs, policy):
        grad = answers.token_logps_grad(z, targets, loss(z)[1], 0.7)
        for at in np.ndindex(z.shape):
            up, down = z.copy(), z.copy()
            up[at] += 1e-5
            down[at] -= 1e-5
            assert abs((loss(up)[0] - loss(down)[0]) / 2e-5 - grad[at]) < 1e-7
