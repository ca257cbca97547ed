"""kd_counter_dropout and kd_block_rows* restated in numpy from their definitions, in 64 bits."""
import numpy as np

import kd

WORD = 0xFFFFFFFF


def philox(counter, key):
    """Philox4x32-10: four words from four counter words (arrays that broadcast) and a key of two."""
    c = [np.asarray(w, np.uint64) for w in np.broadcast_arrays(*counter)]
    k0, k1 = (int(k) for k in key)
    low = np.uint64(WORD)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [p1 >> np.uint64(32) ^ c[1] ^ np.uint64(k0), p1 & low, p0 >> np.uint64(32) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = k0 + 0x9E3779B9 & WORD, k1 + 0xBB67AE85 & WORD
    return c


def kept(rows, cols, keep, seed=0, stream=0, step=0, row=0, more=0):
    if keep == 1:
        return np.ones((rows, cols), bool)
    words = philox((np.arange(-(-cols // 4))[None, :], np.arange(row, row + rows)[:, None] & WORD, stream, step + more & WORD),
                   (seed & WORD, seed >> 32))
    words = np.stack(words, 2).reshape(rows, -(-cols // 4) * 4)[:, :cols]
    return words < np.uint64(round(keep * 2.0 ** 32))


def norm_stats(v, norm):
    """Mean and 1 / sqrt(mean square + eps) of each row; summed in 80 bits, since a constant row's mean that is a step of 64
    bits off has a mean square of its own beside a small eps."""
    if norm is None:
        return np.zeros(len(v)), np.ones(len(v))
    v = v.astype(np.longdouble)
    mean = v.mean(1) if norm["kind"] == kd.NORM_LAYER else np.zeros(len(v))
    with np.errstate(divide="ignore"):
        rate = 1 / np.sqrt(((v - mean[:, None]) ** 2).mean(1) + norm["eps"])
    return mean.astype(np.float64), rate.astype(np.float64)


def part(norm, name, otherwise):
    return norm[name].astype(np.float64) if norm is not None and norm[name] is not None else otherwise


class Case:
    """A block's operands; x, residual, gate, weights and biases in the element type, None where they are left out."""

    def __init__(self, x, residual=None, gate=None, after=None, before=None, residual_scale=1.0, block_scale=1.0, keep=1.0,
                 **counter):
        self.x, self.residual, self.gate, self.after, self.before = x, residual, gate, after, before
        self.residual_scale, self.block_scale, self.keep, self.counter = residual_scale, block_scale, keep, counter
        self.rows, self.cols = x.shape
        self.factor = kept(self.rows, self.cols, keep, **counter) / keep

    def branch(self):
        """a, and the size of the terms that its roundings go by."""
        x = self.x.astype(np.float64)
        mean, rate = norm_stats(x, self.after)
        u = (x - mean[:, None]) * rate[:, None]
        w, b = part(self.after, "weight", 1.0), part(self.after, "bias", 0.0)
        with np.errstate(invalid="ignore"):
            a = np.where(self.factor > 0, (u * w + b) * self.factor, 0)
            size = np.where(self.factor > 0, ((np.abs(x) + np.abs(mean)[:, None]) * rate[:, None] * np.abs(w) + np.abs(b)) * self.factor, 0)
        return a, size, u

    def sum(self):
        """h, and the size of its terms."""
        a, size, _ = self.branch()
        g = self.block_scale * (self.gate.astype(np.float64) if self.gate is not None else 1.0)
        h, size = g * a, np.abs(g) * size
        if self.residual is not None:
            r = self.residual_scale * self.residual.astype(np.float64)
            h, size = h + r, size + np.abs(r)
        return h, size

    def next(self, h):
        """y from h as it is stored, and the size of its terms."""
        h = h.astype(np.float64)
        mean, rate = norm_stats(h, self.before)
        w, b = part(self.before, "weight", 1.0), part(self.before, "bias", 0.0)
        y = (h - mean[:, None]) * rate[:, None] * w + b
        return y, (np.abs(h) + np.abs(mean)[:, None]) * rate[:, None] * np.abs(w) + np.abs(b)

    def norm_back(self, grad, unit, rate, norm):
        """The gradient through a norm from the gradient of its standardized rows, and the size of its terms."""
        mean = grad.mean(1, keepdims=True) if norm["kind"] == kd.NORM_LAYER else 0.0
        along = (grad * unit).mean(1, keepdims=True)
        size = np.abs(grad) + np.abs(grad).mean(1, keepdims=True) + np.abs(unit) * np.abs(grad * unit).mean(1, keepdims=True)
        return rate[:, None] * (grad - mean - unit * along), rate[:, None] * size

    def backward(self, h, grad_h, grad_y):
        """{name: (gradient, size of its terms)} from the stored h; summed gradients with the size of all rows' terms."""
        a, a_size, u = self.branch()
        out = {}
        total = grad_h.astype(np.float64) if grad_h is not None else np.zeros((self.rows, self.cols))
        size = np.abs(total)
        h = h.astype(np.float64)
        if self.before is not None:
            mean, rate = norm_stats(h, self.before)
            v = (h - mean[:, None]) * rate[:, None]
            v_size = (np.abs(h) + np.abs(mean)[:, None]) * rate[:, None]
            g = grad_y.astype(np.float64) if grad_y is not None else np.zeros(h.shape)
            back, back_size = self.norm_back(g * part(self.before, "weight", 1.0), v, rate, self.before)
            back_size = back_size * (1 + v_size)  # v's own roundings
            total, size = total + back, size + back_size
            out["before_weight"] = (g * v).sum(0), (np.abs(g) * v_size).sum(0)
            out["before_bias"] = g.sum(0), np.abs(g).sum(0)
        out["residual"] = self.residual_scale * total, np.abs(self.residual_scale) * size
        gate = self.block_scale * (self.gate.astype(np.float64) if self.gate is not None else 1.0)
        if self.gate is not None:
            one = self.block_scale * a * total, np.abs(self.block_scale) * (np.abs(a) + a_size) * size
            out["gate"] = one if self.gate.ndim == 2 else tuple(v.sum(0) for v in one)
        d, d_size = gate * total * self.factor, np.abs(gate) * size * self.factor
        if self.after is not None:
            x = self.x.astype(np.float64)
            mean, rate = norm_stats(x, self.after)
            u_size = (np.abs(x) + np.abs(mean)[:, None]) * rate[:, None]
            out["after_weight"] = (d * u).sum(0), (d_size * (np.abs(u) + u_size)).sum(0)
            out["after_bias"] = d.sum(0), d_size.sum(0)
            w = part(self.after, "weight", 1.0)
            back, _ = self.norm_back(d * w, u, rate, self.after)
            _, size = self.norm_back(d_size * np.abs(w), np.abs(u) + u_size, rate, self.after)
            d, d_size = back, size * (1 + u_size)
        out["x"] = d, d_size
        return out
