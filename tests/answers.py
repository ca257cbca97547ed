"""kd_token_logps*, kd_preference_pairs and kd_policy_rows restated in numpy from their definitions, in 64 bits."""
import numpy as np


def shares(logits, temperature):
    """log-softmax of the rows; NaN where a row has no distribution."""
    z = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        x = (z - z.max(1, keepdims=True)) / temperature
        return x - np.log(np.exp(x).sum(1, keepdims=True))


def counted(targets, cols):
    return (targets >= 0) & (targets < cols)


def token_logps(logits, targets, temperature):
    rows, cols = logits.shape
    there = counted(targets, cols)
    logs = shares(logits, temperature)
    return np.where(there, logs[np.arange(rows), np.where(there, targets, 0)], 0.0)


def token_logps_grad(logits, targets, slopes, temperature):
    rows, cols = logits.shape
    there = counted(targets, cols) & (slopes != 0)
    grad = np.zeros((rows, cols))
    soft = np.exp(shares(logits, temperature))
    for r in np.flatnonzero(there):
        grad[r] = -soft[r]
        grad[r, targets[r]] += 1
        grad[r] *= slopes[r] / temperature
    return grad


def log_sigmoid(m):
    with np.errstate(over="ignore"):
        return np.minimum(m, 0) - np.log1p(np.exp(-np.abs(m)))


def preference(logps, reference, targets, starts, weights, cols, beta, smoothing):
    rows, pairs = len(logps), len(weights)
    there = counted(targets, cols)
    apart = np.where(there, logps - (reference if reference is not None else 0.0), 0.0)
    at = np.clip(starts, 0, rows)
    rewards = np.zeros((pairs, 2))
    slopes = np.zeros(rows)
    losses = np.zeros(pairs)
    for p in range(pairs):
        rewards[p] = [beta * apart[at[2 * p + i]:at[2 * p + i + 1]].sum() for i in range(2)]
        m = rewards[p, 0] - rewards[p, 1]
        losses[p] = -(1 - smoothing) * log_sigmoid(m) - (smoothing * log_sigmoid(-m) if smoothing else 0)
        slope = beta * weights[p] * (smoothing * np.exp(log_sigmoid(m)) - (1 - smoothing) * np.exp(log_sigmoid(-m)))
        for i in range(2):
            rows_of = slice(at[2 * p + i], at[2 * p + i + 1])
            slopes[rows_of] = np.where(there[rows_of], slope if i == 0 else -slope, 0)
    return losses, rewards, slopes


def policy(lp, targets, cols, old, reference, advantages, low, high, kl_weight):
    """losses and slopes from the rows' log-probabilities."""
    there = counted(targets, cols)
    advantages = advantages.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        ratio = np.exp(lp - old) if old is not None else np.where(np.isnan(lp), np.nan, 1.0)
        free, held = ratio * advantages, np.clip(ratio, 1 - low, 1 + high) * advantages
        loss = np.where(held < free, -held, -free)
        slope = np.where(held < free, 0.0, -free)
        loss, slope = (np.where(advantages == 0, 0.0, v) for v in (loss, slope))
        if reference is not None and kl_weight:
            d = reference - lp
            loss, slope = loss + kl_weight * (np.expm1(d) - d), slope - kl_weight * np.expm1(d)
    return np.where(there, loss, 0.0), np.where(there, slope, 0.0)
