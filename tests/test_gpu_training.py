"""Counter dropout, block ends and the losses together, as a program trains with them: a small model's step against the same
step in numpy, in 64 bits, and against differences of its own loss; captured steps that draw a new mask at every replay;
streams with workspaces of their own."""
import ctypes

import numpy as np
import pytest

import answers
import block
import kd
from test_gpu_serving import graph_of, stream_of

pytestmark = pytest.mark.gpu

L, R = kd.NORM_LAYER, kd.NORM_RMS


class Model:
    """Embedding dropout and a first norm, one linear block with its end (a norm, dropout, a gate, the residual, the next norm),
    logits; the policy loss of sampled tokens or the preference loss of pairs. f64, so that differences are exact enough."""

    def __init__(self, kdb, rng, rows=12, width=24, vocab=17, loss="policy"):
        self.kdb, self.rows, self.width, self.vocab, self.loss = kdb, rows, width, vocab, loss
        n = rng.normal
        self.values = {"x": n(size=(rows, width)), "first_w": 1 + 0.2 * n(size=width), "first_b": 0.1 * n(size=width),
                       "linear": n(size=(width, width)) / np.sqrt(width), "after_w": 1 + 0.2 * n(size=width),
                       "after_b": 0.1 * n(size=width), "gate": n(size=width), "before_w": 1 + 0.2 * n(size=width),
                       "before_b": 0.1 * n(size=width), "head": n(size=(width, vocab)) / np.sqrt(width)}
        self.targets = rng.integers(0, vocab, rows)
        self.targets[[1, 5]] = -1
        self.starts = np.array([0, 4, 6, 9, rows - 1])
        self.reference = -np.log(vocab) + 0.3 * n(size=rows)
        self.old, self.advantages = -np.log(vocab) + 0.3 * n(size=rows), n(size=rows)
        self.weights = rng.random(rows)
        self.on = {k: kdb.to_device(v) for k, v in self.values.items()}
        self.given = {k: kdb.to_device(np.asarray(getattr(self, k), np.int64 if k in ("targets", "starts") else np.float64))
                      for k in ("targets", "starts", "reference", "old", "advantages", "weights")}
        self.step = kdb.to_device(np.array([0], np.int64))
        shapes = {"h0": (rows, width), "y0": (rows, width), "z": (rows, width), "h": (rows, width), "y": (rows, width),
                  "logits": (rows, vocab), "losses": (rows,), "logps": (rows,), "slopes": (rows,), "rewards": (2, 2), "pairs": (2,),
                  "token_stats": (rows, 2), "stats0": (rows, 4), "stats": (rows, 4), "d_logits": (rows, vocab), "d_y": (rows, width),
                  "d_z": (rows, width), "d_h0": (rows, width), "d_y0": (rows, width), "d_x": (rows, width)}
        self.out = {k: kdb.empty(s, np.float64) for k, s in shapes.items()}
        self.grads = {k: kdb.empty(v.shape, np.float64) for k, v in self.values.items() if k not in ("x",)}
        size = ctypes.c_int64()
        kdb.call("block_rows_workspace", ctypes.byref(size), kd.F64, rows, width)
        self.room = kdb.to_device(np.zeros(max(size.value, 16), np.uint8))

    def blocks(self):
        o, v = self.out, self.on

        def counter(stream):
            return kd.Counter(77, stream, 3, 0, self.step.ptr)

        first = kd.Block(v["x"].ptr, None, None, self.rows, self.width, 0, 1.0, 1.0, 0.8, kd.Norm(),
                         kd.Norm(v["first_w"].ptr, v["first_b"].ptr, 1e-5, L), counter(0))
        end = kd.Block(o["z"].ptr, o["h0"].ptr, v["gate"].ptr, self.rows, self.width, 1, 0.9, 0.5, 0.7,
                       kd.Norm(v["after_w"].ptr, v["after_b"].ptr, 1e-5, R), kd.Norm(v["before_w"].ptr, v["before_b"].ptr, 1e-5, L),
                       counter(1))
        return first, end

    def product(self, out, a, b, rows, inner, columns, a_strides=None, b_strides=None):
        s = kd.MatmulStrides((ctypes.c_int64 * 3)(0, *(a_strides or (inner, 1))), (ctypes.c_int64 * 3)(0, *(b_strides or (columns, 1))),
                             (ctypes.c_int64 * 3)(0, columns, 1))
        self.kdb.call("matmul_strided", kd.F64, a.ptr, b.ptr, out.ptr, kd.MatmulSizes(1, rows, inner, columns), s)

    def run(self):
        """The whole step's calls; nothing is read back between them."""
        k, o, v, g, p = self.kdb, self.out, self.on, self.grads, self.given
        rows, width, vocab = self.rows, self.width, self.vocab
        first, end = self.blocks()
        k.call("block_rows", kd.F64, o["h0"].ptr, o["y0"].ptr, o["stats0"].ptr, first)
        self.product(o["z"], o["y0"], v["linear"], rows, width, width)
        k.call("block_rows", kd.F64, o["h"].ptr, o["y"].ptr, o["stats"].ptr, end)
        self.product(o["logits"], o["y"], v["head"], rows, width, vocab)
        if self.loss == "policy":
            policy = kd.Policy(p["old"].ptr, p["reference"].ptr, p["advantages"].ptr, 0.9, 0.2, 0.3, 0.2)
            k.call("policy_rows", kd.F64, o["losses"].ptr, o["logps"].ptr, o["d_logits"].ptr, o["logits"].ptr, p["targets"].ptr, policy,
                   p["weights"].ptr, rows, vocab)
        else:
            k.call("token_logps", kd.F64, o["logps"].ptr, o["token_stats"].ptr, o["logits"].ptr, p["targets"].ptr, rows, vocab, 0.9)
            k.call("preference_pairs", kd.F64, o["pairs"].ptr, o["rewards"].ptr, o["slopes"].ptr, o["logps"].ptr, p["reference"].ptr,
                   p["targets"].ptr, p["starts"].ptr, p["weights"].ptr, 2, rows, vocab, 0.3, 0.1)
            k.call("token_logps_grad", kd.F64, o["d_logits"].ptr, o["logits"].ptr, o["token_stats"].ptr, p["targets"].ptr, o["slopes"].ptr,
                   rows, vocab, 0.9)
        self.product(g["head"], o["y"], o["d_logits"], width, rows, vocab, a_strides=(1, width))
        self.product(o["d_y"], o["d_logits"], v["head"], rows, vocab, width, b_strides=(1, vocab))
        k.call("block_rows_backward", kd.F64,
               kd.BlockGrads(o["d_z"].ptr, o["d_h0"].ptr, g["gate"].ptr, g["after_w"].ptr, g["after_b"].ptr, g["before_w"].ptr,
                             g["before_b"].ptr), end, o["h"].ptr, o["stats"].ptr, None, o["d_y"].ptr, self.room.ptr, self.room.nbytes)
        self.product(g["linear"], o["y0"], o["d_z"], width, rows, width, a_strides=(1, width))
        self.product(o["d_y0"], o["d_z"], v["linear"], rows, width, width, b_strides=(1, width))
        k.call("block_rows_backward", kd.F64,
               kd.BlockGrads(x=o["d_x"].ptr, before_weight=g["first_w"].ptr, before_bias=g["first_b"].ptr), first, o["h0"].ptr,
               o["stats0"].ptr, o["d_h0"].ptr, o["d_y0"].ptr, self.room.ptr, self.room.nbytes)

    def results(self):
        return {**{"d_" + k: a.numpy() for k, a in self.grads.items()}, "d_x": self.out["d_x"].numpy(), "total": self.total()}

    def total(self):
        if self.loss == "policy":
            return (self.weights * self.out["losses"].numpy()).sum()
        return (self.weights[:2] * self.out["pairs"].numpy()).sum()

    def exact(self, step):
        """The same step in numpy from the definitions."""
        v = self.values
        first = block.Case(v["x"], None, None, None, dict(kind=L, eps=1e-5, weight=v["first_w"], bias=v["first_b"]), keep=0.8, seed=77,
                           stream=0, step=3, more=step)
        h0 = first.sum()[0]
        y0 = first.next(h0)[0]
        end = block.Case(y0 @ v["linear"], h0, v["gate"], dict(kind=R, eps=1e-5, weight=v["after_w"], bias=v["after_b"]),
                         dict(kind=L, eps=1e-5, weight=v["before_w"], bias=v["before_b"]), 0.9, 0.5, 0.7, seed=77, stream=1, step=3, more=step)
        h = end.sum()[0]
        y = end.next(h)[0]
        logits = y @ v["head"]
        lp = answers.token_logps(logits, self.targets, 0.9)
        if self.loss == "policy":
            losses, slopes = answers.policy(lp, self.targets, self.vocab, self.old, self.reference, self.advantages, 0.2, 0.3, 0.2)
            total, slopes = (self.weights * losses).sum(), self.weights * slopes
        else:
            losses, _, slopes = answers.preference(lp, self.reference, self.targets, self.starts, self.weights[:2], self.vocab, 0.3, 0.1)
            total = (self.weights[:2] * losses).sum()
        d_logits = answers.token_logps_grad(logits, self.targets, slopes, 0.9)
        back = {k: a[0] for k, a in end.backward(h, None, d_logits @ v["head"].T).items()}
        d_y0 = back["x"] @ v["linear"].T
        start = {k: a[0] for k, a in first.backward(h0, back["residual"], d_y0).items()}
        return {"d_head": y.T @ d_logits, "d_gate": back["gate"], "d_after_w": back["after_weight"], "d_after_b": back["after_bias"],
                "d_before_w": back["before_weight"], "d_before_b": back["before_bias"], "d_linear": y0.T @ back["x"],
                "d_first_w": start["before_weight"], "d_first_b": start["before_bias"], "d_x": start["x"], "total": total}


def near(got, want):
    """A dozen f64 operations in a row of at most 24 terms each, of values of size 10 at most: some thousand roundings."""
    for name, w in want.items():
        np.testing.assert_allclose(got[name], w, rtol=0, atol=4096 * 2.0 ** -53 * (1 + np.abs(w).max()), err_msg=name)


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_a_step_is_its_definition(kdb, loss):
    model = Model(kdb, np.random.default_rng(1), loss=loss)
    for step in (0, 1, 2 ** 32 - 1, -3):
        model.step.upload(np.array([step], np.int64))
        model.run()
        near(model.results(), model.exact(step))


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_a_steps_gradients_are_its_differences(kdb, loss):
    """Central differences of 1e-5: 1e-10 of the third derivative, 1e-16 / 1e-5 of the loss; the policy's borders are away."""
    model = Model(kdb, np.random.default_rng(2), loss=loss)
    model.run()
    grads = model.results()
    rng = np.random.default_rng(3)
    for name, value in model.values.items():
        for at in [tuple(rng.integers(0, n) for n in value.shape) for _ in range(3)]:
            sides = []
            for sign in (1, -1):
                moved = value.copy()
                moved[at] += sign * 1e-5
                model.on[name].upload(moved)
                model.run()
                sides.append(model.total())
            model.on[name].upload(value)
            assert abs((sides[0] - sides[1]) / 2e-5 - grads["d_" + name][at]) < 1e-6, (name, at)


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_a_captured_step_draws_a_new_mask_at_every_replay(kdb, loss):
    model = Model(kdb, np.random.default_rng(4), loss=loss)
    model.run()  # outside the capture first: the kernels are loaded
    kdb.synchronize()
    with stream_of(kdb) as stream, graph_of(kdb, stream, model.run) as replay:
        seen = []
        for step in (0, 1, 1, 5, 2 ** 31):
            model.step.upload(np.array([step], np.int64))
            replay()
            got = model.results()
            near(got, model.exact(step))
            seen.append(got["total"])
            model.run()  # eager between the replays, on the same buffers
            again = model.results()
            for name in got:
                np.testing.assert_array_equal(again[name], got[name])
        assert seen[1] == seen[2] and len(set(seen)) == 4


def test_a_captured_backward_of_every_kind(kdb):
    """Block ends of each plan (a wave, a team, a workgroup, long rows with their sums apart) and long rows of logits in one graph:
    replays on new contents give what eager calls give, bit for bit."""
    rng = np.random.default_rng(5)
    calls, held, outs = [], [], []
    for rows, cols, dtype in ((70, 200, np.float32), (40, 1000, np.float64), (30, 4096, np.float32), (9, 5000, np.float32), (3, 20001, np.float64)):
        x, r, gh, gy = (kdb.to_device(rng.normal(size=(rows, cols)).astype(dtype)) for _ in range(4))
        w = kdb.to_device((1 + 0.1 * rng.normal(size=cols)).astype(dtype))
        h, y, gx, gr = (kdb.empty((rows, cols), dtype) for _ in range(4))
        sums = [kdb.empty((cols,), dtype) for _ in range(5)]
        stats, n = kdb.empty((rows, 4), np.float64), ctypes.c_int64()
        d = kd.DTYPE_OF[np.dtype(dtype)]
        kdb.call("block_rows_workspace", ctypes.byref(n), d, rows, cols)
        room = kdb.empty((n.value,), np.uint8)
        b = kd.Block(x.ptr, r.ptr, w.ptr, rows, cols, 1, 1.0, 1.0, 0.9, kd.Norm(w.ptr, w.ptr, 1e-5, L), kd.Norm(w.ptr, w.ptr, 1e-5, R),
                     kd.Counter(1, 2, 3, 0, None))
        grads = kd.BlockGrads(gx.ptr, gr.ptr, *(s.ptr for s in sums))
        calls.append(("block_rows", d, h.ptr, y.ptr, stats.ptr, b))
        calls.append(("block_rows_backward", d, grads, b, h.ptr, stats.ptr, gh.ptr, gy.ptr, room.ptr, n.value))
        held += [x, r, gh, gy]
        outs += [h, y, gx, gr, *sums, stats, w, room]
    z = kdb.to_device(rng.normal(size=(40, 70001)).astype(np.float32))
    t = kdb.to_device(rng.integers(-1, 70001, 40))
    lp, st, g, s = kdb.empty((40,), np.float64), kdb.empty((40, 2), np.float32), kdb.empty((40, 70001), np.float32), kdb.to_device(np.ones(40, np.float32))
    calls.append(("token_logps", kd.F32, lp.ptr, st.ptr, z.ptr, t.ptr, 40, 70001, 1.0))
    calls.append(("token_logps_grad", kd.F32, g.ptr, z.ptr, st.ptr, t.ptr, s.ptr, 40, 70001, 1.0))
    held.append(z)
    results = [o for o in outs if o.dtype != np.uint8] + [lp, st, g]

    def run():
        for c in calls:
            kdb.call(*c)

    run()
    kdb.synchronize()
    with stream_of(kdb) as stream, graph_of(kdb, stream, run) as replay:
        for _ in range(3):
            for a in held:
                a.upload(rng.normal(size=a.shape).astype(a.dtype))
            replay()
            got = [o.numpy() for o in results]
            kdb.to_device(np.ones(1000)).numpy()
            run()
            for o, a in zip(results, got):
                np.testing.assert_array_equal(o.numpy(), a)
            replay()
            for o, a in zip(results, got):
                np.testing.assert_array_equal(o.numpy(), a)


def test_two_streams_with_workspaces_of_their_own(kdb):
    """Backward passes in flight on two streams at once give what they give alone."""
    models = [Model(kdb, np.random.default_rng(6 + i), rows=50 + 14 * i, loss=loss) for i, loss in enumerate(("policy", "preference"))]
    alone = []
    for m in models:
        m.run()
        alone.append(m.results())
    with stream_of(kdb) as first, stream_of(kdb) as second:
        for _ in range(10):
            for stream, m in zip((first, second), models):
                kdb.lib.kd_set_stream(stream)
                m.run()
        for stream in (first, second):
            assert kdb.lib.hipStreamSynchronize(stream) == 0
        kdb.lib.kd_set_stream(second)
    for m, want in zip(models, alone):
        got = m.results()
        for name in want:
            np.testing.assert_array_equal(got[name], want[name])


def test_dropout_inside_a_block_is_the_dropout_alone(kdb):
    """The mask of a block's dropout is kd_counter_dropout's for the same counter, whatever the kernel: an embedding's dropout as a
    block of nothing else, in rows of each kernel's length."""
    rng = np.random.default_rng(9)
    for cols in (3, 130, 700, 1023, 3000, 5000, 9001, 20000):
        x = kdb.to_device(rng.normal(size=(5, cols)))
        alone, inside = kdb.empty((5, cols), np.float64), kdb.empty((5, cols), np.float64)
        counter = kd.Counter(5, 6, 7, 8, None)
        kdb.call("counter_dropout", kd.F64, alone.ptr, x.ptr, 5, cols, 0.6, counter)
        kdb.call("block_rows", kd.F64, inside.ptr, None, None,
                 kd.Block(x.ptr, None, None, 5, cols, 0, 1.0, 1.0, 0.6, kd.Norm(), kd.Norm(), counter))
        np.testing.assert_array_equal(inside.numpy() == 0, alone.numpy() == 0)
        np.testing.assert_allclose(inside.numpy(), alone.numpy(), rtol=2.0 ** -52)
