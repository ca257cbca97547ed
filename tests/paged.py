"""The paged 8-bit cache restated in numpy from its definition, in 64 bits, for the tests of kd_paged_*."""
import ctypes

import numpy as np

import kd


class Cache:
    """A cache of random codes and scales, its table handing out distinct pages, as host arrays."""

    def __init__(self, rng, sequences, columns, kv_heads, page, dim, spare=0):
        self.kv_heads, self.page, self.dim, self.columns = kv_heads, page, dim, columns
        self.pages = sequences * columns + spare
        self.keys = rng.integers(-127, 128, (self.pages, kv_heads, page, dim)).astype(np.int8)
        self.values = rng.integers(-127, 128, (self.pages, kv_heads, dim, page)).astype(np.int8)
        self.key_scales = rng.uniform(0.005, 0.03, (self.pages, kv_heads)).astype(np.float32)
        self.value_scales = rng.uniform(0.005, 0.03, (self.pages, kv_heads)).astype(np.float32)
        self.table = rng.permutation(self.pages)[:sequences * columns].reshape(sequences, columns).astype(np.int64)

    NAMES = ("keys", "values", "key_scales", "value_scales")

    def copy(self):
        other = object.__new__(Cache)
        other.__dict__.update(self.__dict__)
        for name in self.NAMES + ("table",):
            setattr(other, name, getattr(self, name).copy())
        return other

    def page_at(self, sequence, position):
        column = position // self.page
        if position < 0 or column >= self.columns:
            return -1
        page = int(self.table[sequence, column])
        return page if 0 <= page < self.pages else -1


class Device:
    """The cache and a batch on the device; `read_back` fetches the cache's arrays."""

    def __init__(self, kdb, cache, starts, lengths, tokens):
        self.cache, self.kdb = cache, kdb
        self.arrays = {n: kdb.to_device(getattr(cache, n)) for n in Cache.NAMES}
        self.table = kdb.to_device(cache.table)
        self.starts = kdb.to_device(np.asarray(starts, np.int64))
        self.lengths = kdb.to_device(np.asarray(lengths, np.int64))
        self.c = kd.PagedCache(*(self.arrays[n].ptr for n in Cache.NAMES), cache.pages, cache.kv_heads, cache.page, cache.dim)
        self.b = kd.PagedBatch(self.table.ptr, self.starts.ptr, self.lengths.ptr, len(lengths), cache.columns, tokens)

    def read_back(self):
        got = self.cache.copy()
        for n in Cache.NAMES:
            setattr(got, n, self.arrays[n].numpy())
        return got


def tables(positions, features, base=10000.0):
    half = features // 2
    angle = np.arange(positions)[:, None] * base ** (-np.arange(half) / max(half, 1))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def rotate(x, position, cosines, sines, features, interleaved):
    """One row x [heads, dim] in f64."""
    x = x.astype(np.float64)
    if not features:
        return x
    half = features // 2
    out = x.copy()
    if position < len(cosines):
        c, s = cosines[position].astype(np.float64), sines[position].astype(np.float64)
    else:
        c = s = np.full(half, np.nan)
    first, second = ((slice(0, features, 2), slice(1, features, 2)) if interleaved
                     else (slice(0, half), slice(half, features)))
    a, b = x[:, first], x[:, second]
    out[:, first], out[:, second] = a * c - b * s, b * c + a * s
    return out


def append(cache, starts, lengths, q, k, v, rotation=None):
    """The cache after the append, and the rotated queries (rows outside every sequence NaN-free copies of a marker)."""
    got = cache.copy()
    cosines, sines, features, interleaved = rotation or (None, None, 0, False)
    q_out = np.full(q.shape, -777.0, np.float32)
    for s, length in enumerate(lengths):
        rows = range(starts[s], starts[s + 1])
        first = length - len(rows)
        new = {}
        for i, row in enumerate(rows):
            position = first + i
            if position < 0:
                q_out[row] = np.nan
                continue
            q_out[row] = rotate(q[row], position, cosines, sines, features, interleaved).astype(np.float32)
            page = cache.page_at(s, position)
            if page >= 0:
                key = rotate(k[row], position, cosines, sines, features, interleaved)
                new.setdefault(page, []).append((position % cache.page, key, v[row].astype(np.float64)))
        for page, entries in new.items():
            slots = [e[0] for e in entries]
            held = slots[0]
            for n, name in ((1, "keys"), (2, "values")):
                x = np.stack([e[n] for e in entries], 1)  # [kv_heads, tokens, dim]
                codes, scales = getattr(got, name), getattr(got, name[:-1] + "_scales")
                for h in range(cache.kv_heads):
                    block = codes[page, h] if name == "keys" else codes[page, h].T
                    old = np.float32(scales[page, h]) if held else np.float32(0)
                    most = np.abs(x[h]).max()
                    scale = max(old, np.float32(most / 127)) if np.isfinite(most) and not np.isnan(old) else np.float32(np.nan)
                    if scale > old:
                        block[:held] = np.rint(block[:held].astype(np.float64) * (np.float64(old) / np.float64(scale)))
                    inverse = 1 / np.float64(scale) if scale > 0 else 0.0
                    with np.errstate(invalid="ignore"):
                        r = np.clip(np.rint(x[h] * inverse), -127, 127)
                    block[slots] = np.where(np.isnan(r), 0, r)
                    scales[page, h] = scale
    return got, q_out


def values_of(cache, sequence, head, length):
    """Keys and values [length, dim] in f64 and which positions have a page."""
    k, v = np.zeros((length, cache.dim)), np.zeros((length, cache.dim))
    there = np.zeros(length, bool)
    for j in range(length):
        page = cache.page_at(sequence, j)
        if page < 0:
            continue
        there[j] = True
        k[j] = cache.keys[page, head, j % cache.page] * np.float64(cache.key_scales[page, head])
        v[j] = cache.values[page, head, :, j % cache.page] * np.float64(cache.value_scales[page, head])
    return k, v, there


def attention(cache, starts, lengths, q, scale):
    """out [tokens, heads, dim] in f64 (-777 in rows outside every sequence), and each row's tolerance.

    With S a row's largest score in size and A the largest sum of its products' sizes: the query's pieces hold 2^-24 of it, and
    heads of 64 sum two products a piece per 32 features in f32 (2 dim / 32 roundings of at most A; the whole sums of heads of
    128 are exact); the score's factors, the exponent's argument and its base round 7 times at most S; the exponential adds 2
    steps and its pieces 2. Numerator and denominator carry that, every 64 keys add 4 roundings to the sums, the joining of waves
    and parts 32 altogether:
    2^-24 * max|v| * (2 * (A * (2 + dim / 16 or 0) + 7 S + 4) + 4 * keys / 64 + 32)."""
    tokens, heads, dim = q.shape
    out, tolerance = np.full(q.shape, -777.0), np.zeros(q.shape)
    group = heads // cache.kv_heads
    for s, length in enumerate(lengths):
        n = starts[s + 1] - starts[s]
        capacity = min(length, cache.columns * cache.page)
        for h in range(heads):
            k, v, there = values_of(cache, s, h // group, max(capacity, 0))
            for i in range(n):
                row = starts[s] + i
                seen = there & (np.arange(len(k)) <= length - n + i)
                if not seen.any():
                    out[row, h] = 0
                    continue
                score = k[seen] @ q[row, h].astype(np.float64) * scale
                size = np.abs(k[seen]) @ np.abs(q[row, h].astype(np.float64)) * abs(scale)
                p = np.exp(score - score.max())
                out[row, h] = p @ v[seen] / p.sum()
                tolerance[row, h] = 2.0 ** -24 * np.abs(v[seen]).max() * (
                    2 * (size.max() * (2 + (dim / 16 if dim == 64 else 0)) + 7 * np.abs(score).max() + 4)
                    + 4 * seen.sum() / 64 + 32)
    return out, tolerance


def byref(x):
    return ctypes.byref(x)
