"""The paged 8-bit cache (kd_paged_append, kd_paged_read, kd_paged_attention) against its definition in 64 bits
(tests/paged.py): codes, scales and rotated queries bit for bit, attention within a tolerance derived there.
"""
import ctypes

import numpy as np
import pytest

import kd
import paged

pytestmark = pytest.mark.gpu


def batch_of(new, lengths, first=0, after=0):
    starts = np.concatenate([[0], np.cumsum(new)]) + first
    return [int(x) for x in starts], list(lengths), int(starts[-1]) + after


def fused(rng, tokens, heads, kv_heads, dim):
    """q, k, v as views of one projection's rows."""
    x = rng.normal(0, 1, (tokens, heads + 2 * kv_heads, dim)).astype(np.float32)
    return x, x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]


def run_append(kdb, cache, starts, lengths, tokens, x, heads, rotation=None, with_q=True):
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    kv, dim = cache.kv_heads, cache.dim
    dx = kdb.to_device(x)
    rows = kd.strides(x.shape[1] * dim, dim)
    q_out = kdb.to_device(np.full((max(tokens, 1), heads, dim), -777.0, np.float32))
    turn, held = None, []
    if rotation is not None:
        held = [kdb.to_device(rotation[0]), kdb.to_device(rotation[1])]
        turn = kd.Rotation(held[0].ptr, held[1].ptr, len(rotation[0]), rotation[2], int(rotation[3]))
    size = 4 * dim
    kdb.call("paged_append", kd.F32, on.c, on.b, turn, q_out.ptr if with_q else None, dx.ptr if with_q else None, rows,
             heads, dx.ptr + heads * size, rows, dx.ptr + (heads + kv) * size, rows)
    return on, q_out.numpy()[:tokens]


def same_cache(got, want):
    for name in paged.Cache.NAMES:
        np.testing.assert_array_equal(getattr(got, name), getattr(want, name), err_msg=name)


# new tokens of each sequence, its length with them, kv heads, heads, page, dim
APPENDS = [
    ([1], [1], 1, 1, 16, 64), ([1], [16], 1, 2, 16, 64), ([1], [17], 2, 2, 16, 128), ([16], [16], 3, 3, 16, 64),
    ([17, 0, 5], [40, 7, 5], 2, 4, 16, 64), ([1] * 9, [1, 2, 15, 16, 17, 31, 32, 33, 48], 2, 6, 16, 64),
    ([70, 3], [133, 64], 1, 3, 64, 128), ([130], [260], 2, 2, 128, 64), ([1, 300, 2], [256, 300, 513], 1, 1, 256, 128),
    ([33, 31], [33, 63], 12, 12, 32, 64),
]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("case", APPENDS, ids=[f"{sum(a[0])}x{a[2]}p{a[4]}d{a[5]}" for a in APPENDS])
def test_append_is_its_definition(kdb, case, interleaved):
    new, lengths, kv, heads, page, dim = case
    rng = np.random.default_rng(hash((tuple(new), kv, page)) % 1000)
    starts, lengths, tokens = batch_of(new, lengths)
    cache = paged.Cache(rng, len(new), -(-max(lengths) // page) + 1, kv, page, dim, spare=2)
    x, q, k, v = fused(rng, tokens, heads, kv, dim)
    x[:, heads:] *= rng.choice([0.1, 1, 10], (tokens, 2 * kv, 1))  # scales that grow and that stay
    features = dim if not interleaved else dim // 2
    rotation = (*paged.tables(max(lengths), features), features, interleaved)
    on, q_out = run_append(kdb, cache, starts, lengths, tokens, x, heads, rotation)
    want, want_q = paged.append(cache, starts, lengths, q, k, v, rotation)
    np.testing.assert_array_equal(q_out, want_q)
    same_cache(on.read_back(), want)
    # once more with the same tokens: nothing changes
    again = paged.Device(kdb, on.read_back(), starts, lengths, tokens)
    same_cache(run_append(kdb, again.cache, starts, lengths, tokens, x, heads, rotation)[0].read_back(), want)


@pytest.mark.parametrize("features,interleaved,shift", [(2, False, 0), (6, True, 0), (50, False, 0), (64, False, 1), (64, True, 2),
                                                        (8, True, 0), (64, False, 0)])
def test_append_of_odd_views_and_rotations(kdb, features, interleaved, shift):
    """Rows that no 16-byte piece lies aligned in, heads outside the rows, rotations of a few features."""
    rng = np.random.default_rng(features + shift)
    starts, lengths, tokens = batch_of([21, 1, 7], [25, 40, 7])
    cache = paged.Cache(rng, 3, 3, 2, 16, 64)
    wide = rng.normal(0, 1, (8, tokens, 64 + 2 * shift)).astype(np.float32)  # [q 4, k 2, v 2][token][feature]
    q, k, v = (np.ascontiguousarray(wide[a:b, :, shift:shift + 64].transpose(1, 0, 2)) for a, b in ((0, 4), (4, 6), (6, 8)))
    rotation = (*paged.tables(40, features), features, interleaved)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    dx, c, s = kdb.to_device(wide), kdb.to_device(rotation[0]), kdb.to_device(rotation[1])
    out = kdb.to_device(np.full(q.shape, -777, np.float32))
    row = 64 + 2 * shift
    strides, head = kd.strides(row, tokens * row), tokens * row * 4
    at = dx.ptr + 4 * shift
    kdb.call("paged_append", kd.F32, on.c, on.b, kd.Rotation(c.ptr, s.ptr, 40, features, int(interleaved)), out.ptr, at, strides,
             4, at + 4 * head, strides, at + 6 * head, strides)
    want, want_q = paged.append(cache, starts, lengths, q, k, v, rotation)
    np.testing.assert_array_equal(out.numpy(), want_q)
    same_cache(on.read_back(), want)


def test_append_over_many_sequences(kdb):
    """More sequences than a wave has lanes, some of them without new tokens, rows before the first and behind the last."""
    rng = np.random.default_rng(8)
    new = [int(x) for x in rng.integers(0, 4, 200)]
    lengths = [n + int(x) for n, x in zip(new, rng.integers(0, 30, 200))]
    starts, lengths, tokens = batch_of(new, lengths, first=2, after=3)
    cache = paged.Cache(rng, 200, 3, 1, 16, 64)
    x, q, k, v = fused(rng, tokens, 2, 1, 64)
    rotation = (*paged.tables(40, 64), 64, False)
    on, q_out = run_append(kdb, cache, starts, lengths, tokens, x, 2, rotation)
    want, want_q = paged.append(cache, starts, lengths, q, k, v, rotation)
    np.testing.assert_array_equal(q_out, want_q)
    same_cache(on.read_back(), want)
    out, tolerance = paged.attention(want, starts, lengths, q_out, 0.125)
    got = run_attention(kdb, on, q_out, 0.125, 40)
    assert (np.abs(got - out) <= tolerance).all()


def test_append_without_rotation_queries_or_pages(kdb):
    """No rotation and no queries; positions without a page, before the first or past the table, are not written; rows
    before the first and behind the last sequence are left alone."""
    rng = np.random.default_rng(3)
    new, lengths = [5, 20, 4, 9], [3, 40, 70, 9]
    starts, lengths, tokens = batch_of(new, lengths, first=3, after=6)
    cache = paged.Cache(rng, 4, 3, 2, 16, 64)
    cache.table[1, 1] = -1
    cache.table[3, 0] = cache.pages + 5
    x, q, k, v = fused(rng, tokens, 4, 2, 64)
    on, q_out = run_append(kdb, cache, starts, lengths, tokens, x, 4, with_q=False)
    want, want_q = paged.append(cache, starts, lengths, q, k, v)
    same_cache(on.read_back(), want)
    assert (q_out == -777).all()
    on, q_out = run_append(kdb, cache, starts, lengths, tokens, x, 4)
    np.testing.assert_array_equal(q_out, want_q)
    same_cache(on.read_back(), want)


def test_append_of_what_is_not_finite_or_zero(kdb):
    rng = np.random.default_rng(4)
    starts, lengths, tokens = batch_of([20, 3, 2], [20, 19, 18])
    cache = paged.Cache(rng, 3, 2, 2, 16, 64)
    x, q, k, v = fused(rng, tokens, 2, 2, 64)
    x[3, 2, 5], x[17, 5, 0] = np.inf, np.nan  # a key of head 0's first page, a value of head 1's second
    x[20:23, 2:] = 0                          # zeros into a page that holds codes
    x[23:25] = 1e-42                          # below the least scale's reach
    on, _ = run_append(kdb, cache, starts, lengths, tokens, x, 2)
    want, _ = paged.append(cache, starts, lengths, q, k, v)
    same_cache(on.read_back(), want)
    assert np.isnan(want.key_scales).sum() == 1 and np.isnan(want.value_scales).sum() == 1


def test_a_position_past_the_rotation_tables_turns_into_nan(kdb):
    rng = np.random.default_rng(5)
    starts, lengths, tokens = batch_of([6], [20])
    cache = paged.Cache(rng, 1, 2, 1, 16, 64)
    x, q, k, v = fused(rng, tokens, 1, 1, 64)
    rotation = (*paged.tables(18, 32), 32, False)
    on, q_out = run_append(kdb, cache, starts, lengths, tokens, x, 1, rotation)
    want, want_q = paged.append(cache, starts, lengths, q, k, v, rotation)
    np.testing.assert_array_equal(q_out, want_q)
    same_cache(on.read_back(), want)
    assert np.isnan(q_out[4:, :, :32]).all() and np.isfinite(q_out[:4]).all()


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("shift", [0, 1])  # rows that 16-byte pieces lie aligned in, and rows that they do not
@pytest.mark.parametrize("positions", [0, 70])  # no tables, and tables
def test_append_of_rotated_rows_below_position_zero(kdb, interleaved, shift, positions):
    """More new rows than positions, with a rotation: there is no table row for them, the queries there are NaN, and the
    other rows and the cache are as ever."""
    rng = np.random.default_rng(19 + shift)
    starts, lengths, tokens = batch_of([40, 90, 7, 3], [11, 0, -5, 60], first=1, after=2)
    cache = paged.Cache(rng, 4, 4, 2, 16, 64)
    wide = rng.normal(0, 1, (tokens, 8, 64 + shift)).astype(np.float32)  # [token][q 4, k 2, v 2][feature]
    q, k, v = (np.ascontiguousarray(wide[:, a:b, shift:]) for a, b in ((0, 4), (4, 6), (6, 8)))
    cosines, sines = (t[:positions] for t in paged.tables(70, 48))
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    dx, c, s = kdb.to_device(wide), kdb.to_device(cosines), kdb.to_device(sines)
    turn = kd.Rotation(c.ptr if positions else None, s.ptr if positions else None, positions, 48, int(interleaved))
    out = kdb.to_device(np.full(q.shape, -777, np.float32))
    strides, head = kd.strides(8 * (64 + shift), 64 + shift), 4 * (64 + shift)
    at = dx.ptr + 4 * shift
    kdb.call("paged_append", kd.F32, on.c, on.b, turn, out.ptr, at, strides, 4, at + 4 * head, strides, at + 6 * head, strides)
    lengths = [max(n, 0) for n in lengths]  # a length below 0 counts as 0
    want, want_q = paged.append(cache, starts, lengths, q, k, v, (cosines, sines, 48, interleaved))
    got = out.numpy()
    np.testing.assert_array_equal(got, want_q)
    assert np.isnan(got[1:30]).all() and np.isnan(got[41:138]).all() and np.isfinite(got[138:141, :, 48:]).all()
    same_cache(on.read_back(), want)


@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (256, 64)])
def test_read_gives_the_values(kdb, page, dim):
    rng = np.random.default_rng(page)
    starts, lengths, tokens = batch_of([7, 0, 90, 4], [20, 5, 90, 2], first=1, after=3)
    cache = paged.Cache(rng, 4, -(-90 // page), 3, page, dim)
    cache.table[0, 0] = -1 if page == 16 else cache.table[0, 0]
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want = {n: np.full((tokens, 3, dim), -777, np.float32) for n in ("keys", "values")}
    for s, length in enumerate(lengths):
        n = starts[s + 1] - starts[s]
        for i in range(n):
            position = length - n + i
            at = cache.page_at(s, position)
            row, slot = starts[s] + i, position % page
            want["keys"][row] = cache.keys[at, :, slot] * cache.key_scales[at][:, None] if at >= 0 else 0
            want["values"][row] = cache.values[at, :, :, slot] * cache.value_scales[at][:, None] if at >= 0 else 0
    for skipped in (None, "keys", "values"):
        got = {n: kdb.to_device(np.full((tokens, 3, dim), -777, np.float32)) for n in want}
        ptr = {n: None if n == skipped else got[n].ptr for n in want}
        kdb.call("paged_read", kd.F32, ptr["keys"], ptr["values"], on.c, on.b)
        for n in want:
            np.testing.assert_array_equal(got[n].numpy(), np.full_like(want[n], -777) if n == skipped else want[n])


def test_read_of_more_rows_below_position_zero_than_31_bits_count(kdb):
    """2^27 rows without a position, 2^31 pieces of 16 bytes of keys (34 GB): all of them 0, and the rows behind them the values."""
    rng = np.random.default_rng(20)
    below, held = (1 << 27) + 3, 20
    cache = paged.Cache(rng, 1, 1, 1, 256, 64)
    on = paged.Device(kdb, cache, [0, below + held], [held], below + held)
    out = kdb.empty((below + held, 64), np.float32)
    kdb.call("fill", kd.F32, out.ptr, out.shape[0] * 64, ctypes.byref(ctypes.c_float(-777)))
    kdb.call("paged_read", kd.F32, out.ptr, None, on.c, on.b)
    for op in (kd.REDUCE_MIN, kd.REDUCE_MAX):  # of 1024 rows each, and of the last three
        ends = kdb.empty((1 << 17,), np.float32)
        kdb.call("reduce", op, kd.F32, kd.F32, ends.ptr, out.ptr, 64 << 10, 1 << 17)
        assert (ends.numpy() == 0).all()
        kdb.call("reduce", op, kd.F32, kd.F32, ends.ptr, out.ptr + (256 << 27), 3 * 64, 1)
        assert ends.numpy()[0] == 0
    rest = np.empty((held, 64), np.float32)
    kdb.check(kdb.lib.kd_copy_d2h(rest.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(out.ptr + below * 256), rest.nbytes), "kd_copy_d2h")
    at = cache.table[0, 0]
    np.testing.assert_array_equal(rest, cache.keys[at, 0, :held] * cache.key_scales[at, 0])


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_large_appends_and_reads_are_those_of_their_parts(kdb, dim, page):
    """Rows of more than 32 MiB, which go past the caches: the same bits as sequence by sequence."""
    rng = np.random.default_rng(dim)
    kv, heads, columns = 8, 16, 2400 // page + 1
    starts, lengths, tokens = batch_of([1900, 2300, 700 * 64 // dim, 2100, 2000 * 64 // dim], [1900, 2390, 1400, 2100, 2000])
    whole = paged.Cache(rng, 5, columns, kv, page, dim)
    rotation = (*paged.tables(2400, dim), dim, False)
    x, q, k, v = fused(rng, tokens, heads, kv, dim)
    on, q_out = run_append(kdb, whole, starts, lengths, tokens, x, heads, rotation)
    got = on.read_back()
    rows = [kdb.empty((tokens, kv, dim), np.float32) for _ in range(2)]
    kdb.call("paged_read", kd.F32, rows[0].ptr, rows[1].ptr, on.c, on.b)
    for s in range(5):
        part = slice(starts[s], starts[s + 1])
        count = starts[s + 1] - starts[s]
        cache = whole.copy()
        cache.table = whole.table[s:s + 1]
        alone, q_part = run_append(kdb, cache, [0, count], lengths[s:s + 1], count, np.ascontiguousarray(x[part]), heads, rotation)
        np.testing.assert_array_equal(q_out[part], q_part)
        own, used = alone.read_back(), whole.table[s][:-(-lengths[s] // page)]
        for name in paged.Cache.NAMES:
            np.testing.assert_array_equal(getattr(got, name)[used], getattr(own, name)[used])
        apart = [kdb.empty((count, kv, dim), np.float32) for _ in range(2)]
        for i in range(2):
            kdb.call("paged_read", kd.F32, *(a.ptr if j == i else None for j, a in enumerate(apart)), alone.c, alone.b)
            np.testing.assert_array_equal(rows[i].numpy()[part], apart[i].numpy())


# ---- attention ------------------------------------------------------------------------------------


def run_attention(kdb, on, q, scale, max_keys, workspace=None, strides=None, out=None):
    tokens, heads, dim = q.shape
    dq = kdb.to_device(q)
    out = out or kdb.to_device(np.full(q.shape, -777, np.float32))
    n = workspace.nbytes if workspace is not None else 0
    kdb.call("paged_attention", kd.F32, out.ptr, dq.ptr, strides or kd.strides(heads * dim, dim), heads, on.c, on.b,
             scale, max_keys, workspace.ptr if n else None, n)
    return out.numpy()


def workspace_for(kdb, heads, kv_heads, dim, sequences, tokens, max_keys):
    n = ctypes.c_int64()
    kdb.call("paged_attention_workspace", ctypes.byref(n), heads, kv_heads, dim, sequences, tokens, max_keys)
    return kdb.empty((max(n.value, 16),), np.uint8)


# new tokens, lengths, kv heads, heads, page, dim
ATTENTION = [
    ([1], [1], 1, 1, 16, 64), ([1], [64], 1, 1, 16, 64), ([1], [65], 2, 2, 32, 128), ([1], [1000], 3, 3, 16, 64),
    ([1], [2500], 1, 8, 64, 128), ([1] * 5, [1, 63, 200, 517, 1024], 2, 2, 16, 64), ([5, 3, 1], [5, 300, 77], 2, 6, 32, 64),
    ([16, 17], [16, 900], 1, 1, 16, 64), ([4, 4], [700, 4], 1, 4, 128, 128), ([5], [600], 1, 4, 64, 64),
    ([100, 1, 0, 65], [100, 500, 9, 130], 1, 2, 16, 64), ([33], [33], 2, 2, 256, 128), ([257], [300], 1, 1, 64, 64),
    ([80], [2600], 1, 1, 16, 64), ([40], [2100], 1, 2, 64, 128), ([33, 2], [3000, 1200], 1, 2, 32, 64), ([7], [2500], 2, 2, 16, 64),
    ([1] * 3, [5000, 20, 2100], 1, 2, 256, 128), ([1], [300], 1, 64, 16, 64), ([70, 64, 1, 128], [70, 64, 65, 200], 1, 1, 16, 128),
    ([9], [9], 1, 12, 16, 128), ([2] * 70, [2 + 7 * (s % 40) for s in range(70)], 1, 1, 16, 64),
]


@pytest.mark.parametrize("case", ATTENTION, ids=[f"{len(a[0])}s{sum(a[0])}t{max(a[1])}k{a[2]}of{a[3]}p{a[4]}d{a[5]}" for a in ATTENTION])
def test_attention_is_its_definition(kdb, case):
    new, lengths, kv, heads, page, dim = case
    rng = np.random.default_rng(len(new) + sum(lengths))
    starts, lengths, tokens = batch_of(new, lengths)
    cache = paged.Cache(rng, len(new), -(-max(lengths) // page), kv, page, dim, spare=1)
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    space = workspace_for(kdb, heads, kv, dim, len(new), tokens, max(lengths))
    # split as far as the call likes, on wrong hints, on less room, and not at all
    for hint, room in ((max(lengths), space), (1, space), (1 << 20, space), (max(lengths), None),
                       (max(lengths), kdb.empty((max(space.nbytes // 2 // 16 * 16, 16),), np.uint8))):
        got = run_attention(kdb, on, q, dim ** -0.5, hint, room)
        off = np.abs(got - want)
        assert (off <= tolerance).all(), (hint, off.max(), (off / np.maximum(tolerance, 1e-30)).max())
        # scores of at most about 6 whose dozen roundings of rms 2^-24 / sqrt(3) add up at random: 3.4e-8 * sqrt(12) * 6; a
        # piece that is lost makes 2^-12
        assert np.linalg.norm(off) <= 1e-6 * np.linalg.norm(want)
        np.testing.assert_array_equal(run_attention(kdb, on, q, dim ** -0.5, hint, room), got)


def test_attention_over_views_and_rows_of_no_sequence(kdb):
    rng = np.random.default_rng(11)
    starts, lengths, tokens = batch_of([3, 20], [30, 50], first=2, after=5)
    cache = paged.Cache(rng, 2, 4, 2, 16, 64)
    x = rng.normal(0, 1, (4, tokens, 3, 64)).astype(np.float32)  # heads outside the rows, a gap between rows
    q = np.ascontiguousarray(x[:, :, 1].transpose(1, 0, 2))
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, 0.3)
    dx, out = kdb.to_device(x), kdb.to_device(np.full(q.shape, -777, np.float32))
    kdb.call("paged_attention", kd.F32, out.ptr, dx.ptr + 64 * 4, kd.strides(3 * 64, tokens * 3 * 64), 4, on.c, on.b, 0.3,
             50, None, 0)
    got = out.numpy()
    assert (np.abs(got - want) <= tolerance).all()
    assert (got[:2] == -777).all() and (got[-5:] == -777).all()


# `times`: as few rows a sequence as share a workgroup's keys, or as many as take the prompts' kernel
@pytest.mark.parametrize("times", [1, 30])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_positions_without_a_page(kdb, dim, times):
    """Evicted pages, a sequence without any page, lengths past the table, more new tokens than positions."""
    rng = np.random.default_rng(12)
    starts, lengths, tokens = batch_of([times * n for n in (1, 2, 3, 9)], [100, 64, 500, 4])
    cache = paged.Cache(rng, 4, 8, 2, 16, dim)
    cache.table[0, [0, 2, 6]] = [-1, cache.pages, 1 << 40]
    cache.table[1] = -1
    q = rng.normal(0, 1, (tokens, 4, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, 0.125)
    got = run_attention(kdb, on, q, 0.125, 128, workspace_for(kdb, 4, 2, dim, 4, tokens, 128))
    assert (np.abs(got - want) <= tolerance).all()
    assert (got[times:3 * times] == 0).all() and (got[6 * times:15 * times - 4] == 0).all()


@pytest.mark.parametrize("heads", [1, 2])  # 20 and 40 rows a sequence: either kernel
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_takes_nan_from_what_it_sees_alone(kdb, dim, heads):
    """A NaN scale, of a page that one row sees and another does not; a query that is not finite."""
    rng = np.random.default_rng(13)
    starts, lengths, tokens = batch_of([20, 20], [40, 40])
    cache = paged.Cache(rng, 2, 3, 1, 16, dim)
    cache.key_scales[cache.table[0, 2], 0] = np.nan     # positions 32..47: rows 12.. of the first sequence
    cache.value_scales[cache.table[1, 2], 0] = np.nan
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    q[5, 0, 3], q[6, heads - 1, 63] = np.inf, np.nan
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    with np.errstate(invalid="ignore"):
        want, tolerance = paged.attention(cache, starts, lengths, np.where(np.isfinite(q), q, 0), 0.125)
    want[5, 0] = want[6, heads - 1] = np.nan
    want[12:20] = want[32:40] = np.nan
    got = run_attention(kdb, on, q, 0.125, 40)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= tolerance[fine]).all()


# new tokens, lengths, kv heads, heads: one, up to 4 and up to 8 rows a sequence on average, and some of them far more
FEW = [([1, 1, 0, 1, 0, 2], [300, 1, 9, 700, 5, 66], 2, 2), ([5, 0, 0, 0, 0], [333, 4, 4, 4, 4], 1, 1), ([1] * 9, [40 * s + 1 for s in range(9)], 1, 3),
       ([9, 1, 1, 0, 2], [300, 70, 1, 5, 900], 1, 1), ([20, 1, 1, 1, 1, 1], [400, 20, 64, 65, 63, 1], 2, 2), ([3], [1500], 2, 4),
       ([40, 1, 1, 1, 1, 1, 1, 1], [600, 9, 9, 9, 200, 9, 9, 1], 1, 1), ([4, 4, 1], [64, 1024, 3], 2, 4), ([1, 1], [5000, 2600], 1, 7)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", FEW, ids=[f"{len(a[0])}s{sum(a[0])}t{max(a[1])}k{a[2]}of{a[3]}" for a in FEW])
def test_attention_of_few_rows_is_its_definition(kdb, case, dim):
    new, lengths, kv, heads = case
    rng = np.random.default_rng(dim + sum(lengths))
    starts, lengths, tokens = batch_of(new, lengths)
    cache = paged.Cache(rng, len(new), -(-max(lengths) // 16), kv, 16, dim)
    cache.table[0, -(-int(lengths[0]) // 32)] = -1  # a page in the middle
    cache.value_scales[::3] *= 100
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    space = workspace_for(kdb, heads, kv, dim, len(new), tokens, max(lengths))
    for hint, room in ((max(lengths), space), (1, None)):
        got = run_attention(kdb, on, q, dim ** -0.5, hint, room)
        assert (np.abs(got - want) <= tolerance).all(), (np.abs(got - want) / np.maximum(tolerance, 1e-30)).max()
        np.testing.assert_array_equal(run_attention(kdb, on, q, dim ** -0.5, hint, room), got)


# prompts of few workgroups, whose teams of waves share a tile's keys, and of many; either in parts
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lengths,kv,heads", [([40], [40], 1, 1), ([150, 34], [170, 34], 2, 4), ([100], [3000], 1, 3), ([70], [64], 1, 1),
                                                  ([40] * 60, [40 + 3 * i for i in range(60)], 7, 14)],
                         ids=lambda x: str(len(x)) if isinstance(x, list) else str(x))
def test_attention_of_prompts_by_one_team_or_two(kdb, new, lengths, kv, heads, dim):
    rng = np.random.default_rng(dim + sum(lengths))
    starts, lengths, tokens = batch_of(new, lengths)
    cache = paged.Cache(rng, len(new), -(-max(lengths) // 32), kv, 32, dim)
    cache.table[0, -1] = -1
    cache.value_scales[::3] *= 100
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    for room in (workspace_for(kdb, heads, kv, dim, len(new), tokens, max(lengths)), None):
        got = run_attention(kdb, on, q, dim ** -0.5, max(lengths), room)
        assert (np.abs(got - want) <= tolerance).all(), (np.abs(got - want) / np.maximum(tolerance, 1e-30)).max()
        np.testing.assert_array_equal(run_attention(kdb, on, q, dim ** -0.5, max(lengths), room), got)


# single rows and few rows of more keys than one launch takes, split over the workspace that the call asks for
@pytest.mark.parametrize("heads", [2, 4, 10])
@pytest.mark.parametrize("dim", [64, 128])
def test_few_rows_of_many_keys_are_split(kdb, dim, heads):
    rng = np.random.default_rng(dim + heads)
    starts, lengths, tokens = batch_of([1, 0, 1], [5000, 7, 2222])
    cache = paged.Cache(rng, 3, 40, 2, 128, dim)
    cache.table[0, 20] = -1
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    space = workspace_for(kdb, heads, 2, dim, 3, tokens, 5000)
    assert space.nbytes >= 2 * tokens * heads * (dim + 2) * 4
    for hint, room in ((5000, space), (1 << 20, space), (5000, kdb.empty((space.nbytes // 2 // 16 * 16,), np.uint8)), (1 << 25, None)):
        got = run_attention(kdb, on, q, dim ** -0.5, hint, room)
        assert (np.abs(got - want) <= tolerance).all(), (np.abs(got - want) / np.maximum(tolerance, 1e-30)).max()
        np.testing.assert_array_equal(run_attention(kdb, on, q, dim ** -0.5, hint, room), got)


# as many workgroups as take eight waves at either width, and more: one, two and ten rows to a kv head, or five
@pytest.mark.parametrize("heads", [2, 4, 20])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sequences,new", [(110, 1), (150, 1), (110, 5)])
def test_attention_of_many_short_sequences(kdb, sequences, new, dim, heads):
    rng = np.random.default_rng(sequences + heads)
    starts, lengths, tokens = batch_of([new] * sequences, rng.integers(new, 40, sequences))
    cache = paged.Cache(rng, sequences, 3, 2, 16, dim)
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    want, tolerance = paged.attention(cache, starts, lengths, q, dim ** -0.5)
    got = run_attention(kdb, on, q, dim ** -0.5, 39)
    assert (np.abs(got - want) <= tolerance).all(), (np.abs(got - want) / np.maximum(tolerance, 1e-30)).max()


@pytest.mark.parametrize("heads", [1, 3, 6])
@pytest.mark.parametrize("dim", [64, 128])
def test_few_rows_take_nan_from_what_they_see_alone(kdb, dim, heads):
    """A sequence with a NaN key scale, one with a NaN value scale, one with queries that are not finite, one with neither."""
    rng = np.random.default_rng(18)
    starts, lengths, tokens = batch_of([1] * 5, [40, 200, 130, 300, 32])
    cache = paged.Cache(rng, 5, 20, 1, 16, dim)
    cache.key_scales[cache.table[0, 2], 0] = np.nan
    cache.value_scales[cache.table[1, 5], 0] = np.nan
    cache.key_scales[cache.table[4, 2], 0] = cache.value_scales[cache.table[4, 2], 0] = np.nan  # from position 32 on: not seen
    q = rng.normal(0, 1, (tokens, heads, dim)).astype(np.float32)
    q[2, 0, 3], q[3, heads - 1, 63] = np.inf, np.nan
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    with np.errstate(invalid="ignore"):
        want, tolerance = paged.attention(cache, starts, lengths, np.where(np.isfinite(q), q, 0), 0.125)
    want[:2] = want[2, 0] = want[3, heads - 1] = np.nan
    got = run_attention(kdb, on, q, 0.125, 300, workspace_for(kdb, heads, 1, dim, 5, tokens, 300))
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= tolerance[fine]).all()


@pytest.mark.parametrize("new", [3, 40])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 30.0, 1e30])
def test_attention_of_small_and_large_queries(kdb, size, dim, new):
    """One feature a thousand times the others', queries at both ends of the range, pages of zero and tiny scales."""
    rng = np.random.default_rng(14)
    starts, lengths, tokens = batch_of([new], [200])
    cache = paged.Cache(rng, 1, 13, 1, 16, dim)
    cache.value_scales[cache.table[0, 3]] = 0
    cache.key_scales[cache.table[0, 4]] = 0
    cache.value_scales[cache.table[0, 5]] = 1e-30
    q = rng.normal(0, 1, (tokens, 2, dim)).astype(np.float32)
    q[:, :, 7] *= 1000
    q *= np.float32(size)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    for scale in (1 / (1000 * size), -1 / (1000 * size), 0.0):
        want, tolerance = paged.attention(cache, starts, lengths, q, scale)
        got = run_attention(kdb, on, q, scale, 200)
        assert (np.abs(got - want) <= tolerance).all(), scale
    on.kdb.call("paged_attention", kd.F32, kdb.empty(q.shape, np.float32).ptr, kdb.to_device(q).ptr, kd.strides(2 * dim, dim), 2,
                on.c, kd.PagedBatch(on.table.ptr, on.starts.ptr, on.lengths.ptr, 1, 0, tokens), 1.0, 200, None, 0)


@pytest.mark.parametrize("new", [1, 3, 40])  # one kernel each
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_beside_pages_of_far_larger_values(kdb, dim, new):
    """A page whose values are 10^5 times the others' and whose keys get weights of about 10^-9: the error follows what the rows
    sum up, and not the largest value that they see. The definition's tolerance, with the weighted mean of |v| in place of
    its largest."""
    rng = np.random.default_rng(17)
    starts, lengths, tokens = batch_of([new], [500])
    cache = paged.Cache(rng, 1, 32, 1, 16, dim)
    far = cache.table[0, 3]
    cache.keys[far] = -127
    cache.key_scales[far] = 21 / (127 * dim ** 0.5)
    cache.value_scales[far] = 1500
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
    assert (off <= tolerance).all(), (off / tolerance).max()


def test_attention_of_more_keys_than_whole_sums_hold(kdb):
    """1.2 million keys of weight 1 to one row, whose lowest digits are all -128: some 2340 blocks of 64 to each of eight waves
    add up to more than 2^31. The weights and their sum are exact; a digit's sums round at most three times as they are turned
    into f32 and joined, the digits twice, the waves eight times, the quotient once, all within 2^-24 of the result."""
    pages, page, dim = 4688, 256, 64
    keys = pages * page
    scale = np.float32((2 ** 29 + 2 ** 23 + 2 ** 15 + 2 ** 7) / 2 ** 29)
    on = {n: kdb.to_device(a) for n, a in (
        ("keys", np.zeros((pages, 1, page, dim), np.int8)), ("values", np.full((pages, 1, dim, page), 127, np.int8)),
        ("key_scales", np.ones((pages, 1), np.float32)), ("value_scales", np.full((pages, 1), scale, np.float32)),
        ("table", np.arange(pages)[None]), ("starts", np.asarray([0, 1])), ("lengths", np.asarray([keys])),
        ("q", np.ones((1, 1, dim), np.float32)), ("out", np.zeros((1, 1, dim), np.float32)))}
    cache = kd.PagedCache(*(on[n].ptr for n in ("keys", "values", "key_scales", "value_scales")), pages, 1, page, dim)
    batch = kd.PagedBatch(on["table"].ptr, on["starts"].ptr, on["lengths"].ptr, 1, pages, 1)
    kdb.call("paged_attention", kd.F32, on["out"].ptr, on["q"].ptr, kd.strides(dim, dim), 1, cache, batch, 1.0, keys, None, 0)
    want = 127 * np.float64(scale)
    assert (np.abs(on["out"].numpy() - want) <= 14 * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("new", [1, 40])
def test_attention_without_any_page(kdb, new):
    """A cache of no pages, a table of no columns: nothing is visible and every row 0."""
    q = kdb.to_device(np.ones((new, 2, 64), np.float32))
    starts, lengths = kdb.to_device(np.asarray([0, new])), kdb.to_device(np.asarray([new]))
    table = kdb.to_device(np.zeros((1, 3), np.int64))
    for cache, columns in ((kd.PagedCache(None, None, None, None, 0, 1, 16, 64), 3), (kd.PagedCache(None, None, None, None, 0, 1, 16, 64), 0)):
        out = kdb.to_device(np.full((new, 2, 64), 7, np.float32))
        batch = kd.PagedBatch(table.ptr, starts.ptr, lengths.ptr, 1, columns, new)
        kdb.call("paged_attention", kd.F32, out.ptr, q.ptr, kd.strides(128, 64), 2, cache, batch, 1.0, 10, None, 0)
        assert (out.numpy() == 0).all()
        kdb.call("paged_append", kd.F32, cache, batch, None, None, None, None, 2, q.ptr, kd.strides(128, 64), q.ptr,
                 kd.strides(128, 64))
        got = kdb.to_device(np.full((new, 1, 64), 7, np.float32))
        kdb.call("paged_read", kd.F32, got.ptr, None, cache, batch)
        assert (got.numpy() == 0).all()


def test_a_prompt_drafts_and_single_tokens_in_turn(kdb):
    """A cache built by the calls themselves, as a server runs them: prompts, then drafted tokens, then single ones, each
    step's attention against the definition on the cache as the definition appends to it."""
    rng = np.random.default_rng(15)
    kv, heads, page, dim = 2, 4, 16, 64
    cache = paged.Cache(rng, 3, 5, kv, page, dim)
    lengths = [0, 0, 0]
    rotation = (*paged.tables(80, dim), dim, False)
    for new in ([37, 16, 1], [4, 4, 4], [1, 1, 1], [1, 0, 1], [5, 5, 0]):
        starts, lengths, tokens = batch_of(new, [a + b for a, b in zip(lengths, new)])
        x, q, k, v = fused(rng, tokens, heads, kv, dim)
        on, q_out = run_append(kdb, cache, starts, lengths, tokens, x, heads, rotation)
        cache, want_q = paged.append(cache, starts, lengths, q, k, v, rotation)
        same_cache(on.read_back(), cache)
        np.testing.assert_array_equal(q_out, want_q)
        want, tolerance = paged.attention(cache, starts, lengths, q_out, dim ** -0.5)
        got = run_attention(kdb, on, q_out, dim ** -0.5, max(lengths), workspace_for(kdb, heads, kv, dim, 3, tokens, 80))
        assert (np.abs(got - want) <= tolerance).all()
