"""The serving and training operators as a program runs them together: a decode step captured into a graph and replayed
over a growing cache, calls on two streams with workspaces of their own, a cache whose offsets pass 32 bits, a draft
trained by the distillation loss until the target takes its tokens.
"""
import contextlib
import ctypes

import numpy as np
import pytest

import drafts as draft_definition
import kd
import paged
from test_gpu_drafts import probabilities
from test_gpu_paged import batch_of, fused, same_cache, workspace_for

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def stream_of(kdb):
    """A HIP stream that the backend issues on meanwhile."""
    lib, stream = kdb.lib, ctypes.c_void_p()
    assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
    before = ctypes.c_void_p(lib.kd_get_stream())
    kdb.synchronize()
    lib.kd_set_stream(stream)
    try:
        yield stream
    finally:
        assert lib.hipStreamSynchronize(stream) == 0
        lib.kd_set_stream(before)
        lib.hipStreamDestroy(stream)


@contextlib.contextmanager
def graph_of(kdb, stream, calls):
    """The calls captured; yields a function that replays them and waits."""
    lib, graph, run = kdb.lib, ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0  # thread-local
    try:
        calls()
    finally:
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0

    def replay():
        assert lib.hipGraphLaunch(run, stream) == 0
        assert lib.hipStreamSynchronize(stream) == 0

    try:
        yield replay
    finally:
        lib.hipGraphExecDestroy(run)
        lib.hipGraphDestroy(graph)


@pytest.mark.parametrize("start", [20, 2500])
def test_a_captured_step_follows_the_cache(kdb, start):
    """Append and attention of one token a sequence in one graph, the longer caches split over a workspace: every replay
    sees the lengths and tokens as they stand then."""
    rng = np.random.default_rng(start)
    kv, heads, page, dim, sequences = 2, 4, 16, 64, 3
    columns = (start + 60) // page + 1
    cache = paged.Cache(rng, sequences, columns, kv, page, dim)
    lengths = [start, start - 7, start // 2]
    starts, _, tokens = batch_of([1] * sequences, lengths)
    rotation = (*paged.tables(start + 60, dim), dim, False)
    on = paged.Device(kdb, cache, starts, lengths, tokens)
    x, q, k, v = fused(rng, tokens, heads, kv, dim)
    dx, c, s = kdb.to_device(x), kdb.to_device(rotation[0]), kdb.to_device(rotation[1])
    q_out, out = kdb.empty(q.shape, np.float32), kdb.empty(q.shape, np.float32)
    turn = kd.Rotation(c.ptr, s.ptr, start + 60, dim, 0)
    row, size = kd.strides(x.shape[1] * dim, dim), 4 * dim
    room = workspace_for(kdb, heads, kv, dim, sequences, tokens, 60 + start)
    assert (room.nbytes > 16) == (start > 2048)

    def step():
        kdb.call("paged_append", kd.F32, on.c, on.b, turn, q_out.ptr, dx.ptr, row, heads, dx.ptr + heads * size, row,
                 dx.ptr + (heads + kv) * size, row)
        kdb.call("paged_attention", kd.F32, out.ptr, q_out.ptr, kd.strides(heads * dim, dim), heads, on.c, on.b, 0.125,
                 60 + start, room.ptr if room.nbytes > 16 else None, room.nbytes if room.nbytes > 16 else 0)

    def check():
        nonlocal cache
        cache, want_q = paged.append(cache, starts, lengths, q, k, v, rotation)
        same_cache(on.read_back(), cache)
        np.testing.assert_array_equal(q_out.numpy(), want_q)
        want, tolerance = paged.attention(cache, starts, lengths, want_q, 0.125)
        assert (np.abs(out.numpy() - want) <= tolerance).all()

    step()  # outside the capture first: the kernels are loaded
    check()
    with stream_of(kdb) as stream, graph_of(kdb, stream, step) as replay:
        for turn_at in range(5):
            lengths = [n + 1 for n in lengths]
            x, q, k, v = fused(rng, tokens, heads, kv, dim)
            dx.upload(x)
            on.lengths.upload(np.asarray(lengths, np.int64))
            if turn_at == 2:  # the program's own work between replays
                kdb.to_device(x).numpy()
                kdb.synchronize()
            replay()
            check()


def test_a_captured_verification_and_distillation(kdb):
    """Verification under capture is one launch, without the shared workspace; the loss and its gradient replay with it."""
    rng = np.random.default_rng(3)
    sequences, drafts, vocab = 4, 3, 40009  # eager calls of these sizes take two launches
    given = probabilities(rng, sequences, drafts, vocab, np.float32)
    on = [kdb.to_device(a) for a in given]
    tokens, accepted = kdb.empty((sequences, drafts + 1), np.int64), kdb.empty((sequences,), np.int64)
    rows, cols, kept = 6, 3000, 9
    z, t, w = (rng.normal(size=s) for s in ((rows, cols), (rows, kept), (rows,)))
    index = np.stack([rng.permutation(cols)[:kept] for _ in range(rows)]).astype(np.int64)
    dz, dt, dw, di = kdb.to_device(z), kdb.to_device(t), kdb.to_device(w), kdb.to_device(index)
    losses, stats, grad = (kdb.empty(s, np.float64) for s in ((rows,), (rows, 2), (rows, cols)))

    def step():
        kdb.call("verify_drafts", kd.F32, tokens.ptr, accepted.ptr, *(a.ptr for a in on), sequences, drafts, vocab)
        kdb.call("distill_rows", kd.F64, losses.ptr, stats.ptr, dz.ptr, di.ptr, dt.ptr, rows, cols, kept, 2.0)
        kdb.call("distill_grad", kd.F64, grad.ptr, dz.ptr, stats.ptr, di.ptr, dt.ptr, dw.ptr, rows, cols, kept, 2.0)

    step()
    with stream_of(kdb) as stream, graph_of(kdb, stream, step) as replay:
        for _ in range(4):
            given = probabilities(rng, sequences, drafts, vocab, np.float32)
            for a, b in zip(on, given):
                a.upload(b)
            z = rng.normal(size=z.shape)
            dz.upload(z)
            replay()
            want = draft_definition.verify(*given)
            np.testing.assert_array_equal(tokens.numpy(), want[0])
            np.testing.assert_array_equal(accepted.numpy(), want[1])
            want_losses, want_grad = draft_definition.distill(z, index, t, 2.0)
            # as in the tests of either: arguments of at most 10 / 2, a few steps more
            assert (np.abs(losses.numpy() - want_losses) <= 4 * 20 * 2.0 ** -52 * (1 + want_losses)).all()
            assert (np.abs(grad.numpy() - w[:, None] * want_grad) <= 2 * 20 * 2.0 ** -52 * np.abs(w).max()).all()
            step()  # eager between the replays, on the shared workspace


def test_two_streams_with_workspaces_of_their_own(kdb):
    """Split attention calls in flight on two streams at once give what they give alone."""
    rng = np.random.default_rng(4)
    shapes = [([1, 1], [3000, 2500], 2, 4), ([2], [4000], 1, 8)]
    runs = []
    for new, lengths, kv, heads in shapes:
        starts, lengths, tokens = batch_of(new, lengths)
        cache = paged.Cache(rng, len(new), -(-max(lengths) // 64), kv, 64, 64)
        q = rng.normal(size=(tokens, heads, 64)).astype(np.float32)
        on, dq = paged.Device(kdb, cache, starts, lengths, tokens), kdb.to_device(q)
        room = workspace_for(kdb, heads, kv, 64, len(new), tokens, max(lengths))
        assert room.nbytes > 16
        out = kdb.empty(q.shape, np.float32)
        args = (kd.F32, out.ptr, dq.ptr, kd.strides(heads * 64, 64), heads, on.c, on.b, 0.125, max(lengths), room.ptr, room.nbytes)
        kdb.call("paged_attention", *args)
        runs.append((args, out, out.numpy(), (on, dq, room)))
        want, tolerance = paged.attention(cache, starts, lengths, q, 0.125)
        assert (np.abs(runs[-1][2] - want) <= tolerance).all()
    with stream_of(kdb) as first, stream_of(kdb) as second:
        for stream, run in zip((first, second) * 10, runs * 10):
            kdb.lib.kd_set_stream(stream)
            kdb.call("paged_attention", *run[0])
        for stream in (first, second):
            assert kdb.lib.hipStreamSynchronize(stream) == 0
        kdb.lib.kd_set_stream(second)
    for _, out, alone, _ in runs:
        np.testing.assert_array_equal(out.numpy(), alone)


@pytest.mark.parametrize("new", [3, 50])
def test_a_cache_whose_offsets_pass_32_bits(kdb, new):
    """Pages at the far end of a cache of 5 GiB of keys and as much of values, against the same pages in a small one."""
    rng = np.random.default_rng(5)
    kv, heads, page, dim, pages = 4, 4, 256, 128, 41000
    assert pages * kv * page * dim > 2 ** 32
    starts, lengths, tokens = batch_of([new], [new + 300])
    small = paged.Cache(rng, 1, 2, kv, page, dim)
    x, q, k, v = fused(rng, tokens, heads, kv, dim)
    dx, q_out = kdb.to_device(x), kdb.empty(q.shape, np.float32)
    row, size = kd.strides(x.shape[1] * dim, dim), 4 * dim
    on = paged.Device(kdb, small, starts, lengths, tokens)
    far = {n: kdb.empty((pages, *getattr(small, n).shape[1:]), getattr(small, n).dtype) for n in paged.Cache.NAMES}
    places = [pages - 1, pages - 7]
    for n in paged.Cache.NAMES:  # the small cache's pages at their far places
        data = getattr(small, n)
        for column in range(2):
            one = np.ascontiguousarray(data[small.table[0, column]])
            kdb.check(kdb.lib.kd_copy_h2d(ctypes.c_void_p(far[n].ptr + places[column] * one.nbytes), one.ctypes.data_as(ctypes.c_void_p),
                                          one.nbytes), "kd_copy_h2d")
    table = kdb.to_device(np.asarray([places], np.int64))
    caches = [(on.c, on.b), (kd.PagedCache(*(far[n].ptr for n in paged.Cache.NAMES), pages, kv, page, dim),
                             kd.PagedBatch(table.ptr, on.starts.ptr, on.lengths.ptr, 1, 2, tokens))]
    results = []
    for c, b in caches:
        kdb.call("paged_append", kd.F32, c, b, None, None, None, row, heads, dx.ptr + heads * size, row,
                 dx.ptr + (heads + kv) * size, row)
        got = [kdb.empty((tokens, kv, dim), np.float32), kdb.empty((tokens, kv, dim), np.float32), kdb.empty(q.shape, np.float32)]
        kdb.call("paged_read", kd.F32, got[0].ptr, got[1].ptr, c, b)
        kdb.call("paged_attention", kd.F32, got[2].ptr, dx.ptr, row, heads, c, b, dim ** -0.5, new + 300, None, 0)
        results.append([a.numpy() for a in got])
    for near, there in zip(*results):
        np.testing.assert_array_equal(near, there)
    want, tolerance = paged.attention(on.read_back(), starts, lengths, q, dim ** -0.5)
    assert (np.abs(results[1][2] - want) <= tolerance).all()


def test_a_distilled_draft_is_accepted(kdb):
    """The loss's gradient moves a draft's logits towards the target's, and the verification then accepts its tokens: the
    operators from either end of the pair."""
    rng = np.random.default_rng(6)
    rows, vocab = 64, 40
    target_logits = 2 * rng.normal(size=(rows, vocab))
    index = np.argsort(-target_logits, 1).astype(np.int64)
    teacher = np.take_along_axis(target_logits, index, 1)  # every entry kept: the optimum is the target itself
    z = kdb.to_device(np.zeros((rows, vocab)))
    di, dt, w = kdb.to_device(index), kdb.to_device(teacher), kdb.to_device(np.ones(rows))
    losses, stats, grad = (kdb.empty(s, np.float64) for s in ((rows,), (rows, 2), (rows, vocab)))
    values = np.zeros((rows, vocab))
    for _ in range(3):
        z.upload(values)
        kdb.call("distill_rows", kd.F64, losses.ptr, stats.ptr, z.ptr, di.ptr, dt.ptr, rows, vocab, vocab, 1.0)
        kdb.call("distill_grad", kd.F64, grad.ptr, z.ptr, stats.ptr, di.ptr, dt.ptr, w.ptr, rows, vocab, vocab, 1.0)
        want_losses, want_grad = draft_definition.distill(values, index, teacher, 1.0)
        assert (np.abs(grad.numpy() - want_grad) <= 40 * 2.0 ** -52).all()
        assert (np.abs(losses.numpy() - want_losses) <= 40 * 2.0 ** -52 * (1 + np.abs(want_losses))).all()
        values = values - grad.numpy()
    # a draft with the target's own probabilities: u q < p holds for every draw below 1
    p = np.exp(target_logits - target_logits.max(1, keepdims=True))
    p = (p / p.sum(1, keepdims=True))[:, None].repeat(2, 1)
    drafted = rng.integers(0, vocab, (rows, 1))
    on = [kdb.to_device(a) for a in (p, p[:, :1].copy(), drafted, np.ones(rows, np.int64), rng.random((rows, 2)))]
    tokens, accepted = kdb.empty((rows, 2), np.int64), kdb.empty((rows,), np.int64)
    kdb.call("verify_drafts", kd.F64, tokens.ptr, accepted.ptr, *(a.ptr for a in on), rows, 1, vocab)
    assert (accepted.numpy() == 1).all() and (tokens.numpy()[:, 0] == drafted[:, 0]).all()


def test_a_draft_that_distillation_trains_is_taken_more_often(kdb):
    """A draft's logits follow the loss's gradient towards the target's largest ones; the tokens that the trained and the untrained draft
    draw are verified against the target, each as the definition does."""
    rng = np.random.default_rng(8)
    rows, vocab, kept, drafts = 300, 60, 30, 2
    target_logits = 2 * rng.normal(size=(rows, vocab))
    index = np.argsort(-target_logits, 1)[:, :kept].astype(np.int64)
    teacher = np.take_along_axis(target_logits, index, 1)
    values = np.zeros((rows, vocab))
    z, di, dt, w = (kdb.to_device(a) for a in (values, index, teacher, np.ones(rows)))
    losses, stats, grad = (kdb.empty(s, np.float64) for s in ((rows,), (rows, 2), (rows, vocab)))

    def softmax(x):
        e = np.exp(x - x.max(-1, keepdims=True))
        return e / e.sum(-1, keepdims=True)

    def taken():
        """The share of the draft's own tokens that the target takes."""
        p = softmax(target_logits)[:, None].repeat(drafts + 1, 1)
        q = softmax(values)[:, None].repeat(drafts, 1)
        over = np.cumsum(q, 2) > rng.random((rows, drafts))[..., None]
        drafted = np.where(over.any(2), over.argmax(2), vocab - 1).astype(np.int64)
        given = p, q, drafted, np.full(rows, drafts), rng.random((rows, drafts + 1))
        on = [kdb.to_device(a) for a in given]
        tokens, accepted = kdb.empty((rows, drafts + 1), np.int64), kdb.empty((rows,), np.int64)
        kdb.call("verify_drafts", kd.F64, tokens.ptr, accepted.ptr, *(a.ptr for a in on), rows, drafts, vocab)
        want = draft_definition.verify(*given)
        np.testing.assert_array_equal(tokens.numpy(), want[0])
        np.testing.assert_array_equal(accepted.numpy(), want[1])
        return want[1].sum() / (rows * drafts)

    untrained = taken()
    for _ in range(60):
        z.upload(values)
        kdb.call("distill_rows", kd.F64, losses.ptr, stats.ptr, z.ptr, di.ptr, dt.ptr, rows, vocab, kept, 1.0)
        kdb.call("distill_grad", kd.F64, grad.ptr, z.ptr, stats.ptr, di.ptr, dt.ptr, w.ptr, rows, vocab, kept, 1.0)
        want_losses, want_grad = draft_definition.distill(values, index, teacher, 1.0)
        assert (np.abs(grad.numpy() - want_grad) <= 40 * 2.0 ** -52).all()
        assert (np.abs(losses.numpy() - want_losses) <= 40 * 2.0 ** -52 * (1 + np.abs(want_losses))).all()
        values = values - 2 * grad.numpy()
    # of 600 tokens each a share of at most 1: deviations below 0.03
    assert taken() > untrained + 6 * 0.03
