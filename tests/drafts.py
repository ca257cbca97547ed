"""kd_verify_drafts and kd_distill_* restated in numpy from their definitions, in 64 bits."""
import numpy as np


def verify(target, draft, drafted, counts, uniforms):
    sequences, drafts = drafted.shape
    vocab = target.shape[2]
    tokens = np.full((sequences, drafts + 1), -1, np.int64)
    accepted = np.zeros(sequences, np.int64)
    for s in range(sequences):
        count, kept = min(max(int(counts[s]), 0), drafts), 0
        while kept < count:
            x = int(drafted[s, kept])
            if not 0 <= x < vocab:
                break
            q = np.float64(draft[s, kept, x]) if draft is not None else 1.0
            if not uniforms[s, kept] * q < np.float64(target[s, kept, x]):
                break
            kept += 1
        p = target[s, kept].astype(np.float64)
        w = p
        if kept < count:
            q = np.zeros(vocab)
            if draft is not None:
                q = draft[s, kept].astype(np.float64)
            elif 0 <= drafted[s, kept] < vocab:
                q[drafted[s, kept]] = 1
            w = p - q
        w = np.where(w < 0, 0, w)
        if not w.sum() > 0:
            w = np.where(p < 0, 0, p)
        accepted[s] = kept
        tokens[s, :kept] = drafted[s, :kept]
        total = w.sum()
        if 0 < total < np.inf:
            over = np.cumsum(w) > uniforms[s, drafts] * total
            tokens[s, kept] = np.argmax(over) if over.any() else np.flatnonzero(w > 0)[-1]
    return tokens, accepted


def distill(logits, indices, teacher, temperature):
    """losses, the gradient for row weights of 1, and sum(pi) of each row."""
    z, t = logits.astype(np.float64), teacher.astype(np.float64)
    rows, cols = z.shape
    largest = z.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        x = (z - largest) / temperature
        e = np.exp(x)
        log_sigma = x - np.log(e.sum(1, keepdims=True))
        losses, grad = np.zeros(rows), np.zeros(z.shape)
        for r in range(rows):
            there = (indices[r] >= 0) & (indices[r] < cols)
            if not there.any() or (t[r, there] == -np.inf).all():
                continue
            y = (t[r, there] - t[r, there].max()) / temperature  # divided last: a far offset costs no bits
            log_pi = y - np.log(np.exp(y).sum())
            pi = np.exp(log_pi)
            terms = np.where(pi == 0, 0, pi * (log_pi - log_sigma[r, indices[r, there]]))
            losses[r] = temperature ** 2 * terms.sum()
            grad[r] = np.exp(log_sigma[r])
            np.subtract.at(grad[r], indices[r, there], pi)
            grad[r] *= temperature
    return losses, grad
