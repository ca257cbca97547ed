"""The operators for training a transformer on sampled answers and on pairs of them, as cases that can be timed and compared.

Four kinds. `dropout`: a mask drawn from a counter, forward and backward, never stored. `block`: the end of a
transformer's block in one pass (a norm of the block's output, dropout, a gate, the residual sum) with the norm ahead of
the next block, and its backward pass. `policy`: the clipped policy loss of sampled tokens with a KL term, and its gradient with
respect to the logits. `preference`: the loss of chosen against rejected answers, and that gradient.

Sizes are those of the repository's configurations (the char-level GPT's 32 x 128 tokens of 256 features and 96
characters, GPT-2 small's 768 features and 50257 tokens) and generic ones (4096 features). `draw` spreads each kind over
its whole range.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "f64": torch.float64}
WORKSPACE = 128 << 20  # what a training program keeps for the block's column sums
WORD = 0xFFFFFFFF


def listed():
    return [
        # The char-level GPT's activations: a training step's dropout, many times a step. Latency.
        {"name": "dropout_char_4096x256", "kind": "dropout", "rows": 4096, "cols": 256, "keep": 0.9, "dtype": "f32"},
        # An odd width in f64.
        {"name": "dropout_1501x1537_f64", "kind": "dropout", "rows": 1501, "cols": 1537, "keep": 0.5, "dtype": "f64"},
        # A large model's activations: more than the caches hold.
        {"name": "dropout_16384x4096", "kind": "dropout", "rows": 16384, "cols": 4096, "keep": 0.9, "dtype": "f32"},
        # One decoding step of 16 GPT-2 small sequences: residual sum and the next norm, forward only. Latency.
        {"name": "block_decode_16x768", "kind": "block", "rows": 16, "cols": 768, "train": False, "after": "none",
         "before": "layer", "gate": "none", "keep": 1.0, "residual_scale": 1.0, "block_scale": 1.0, "dtype": "f32"},
        # A training step's block end of the char-level GPT with its dropout.
        {"name": "block_char_4096x256", "kind": "block", "rows": 4096, "cols": 256, "train": True, "after": "none",
         "before": "layer", "gate": "none", "keep": 0.9, "residual_scale": 1.0, "block_scale": 1.0, "dtype": "f32"},
        # A large model with norms on both sides, a learned gate for each feature and a scaled residual: the largest.
        {"name": "block_8192x4096", "kind": "block", "rows": 8192, "cols": 4096, "train": True, "after": "rms",
         "before": "rms", "gate": "shared", "keep": 0.9, "residual_scale": 0.8, "block_scale": 0.5, "dtype": "f32"},
        # A gate of its own for each token, an odd width, in f64.
        {"name": "block_1003x1537_f64", "kind": "block", "rows": 1003, "cols": 1537, "train": True, "after": "layer",
         "before": "rms", "gate": "rows", "keep": 0.8, "residual_scale": 1.0, "block_scale": 0.7, "dtype": "f64"},
        # The char-level GPT's step on sampled characters.
        {"name": "policy_4096x96", "kind": "policy", "rows": 4096, "vocab": 96, "masked": 0.25, "kl": True,
         "temperature": 1.0, "dtype": "f32"},
        # Sampled answers over GPT-2's vocabulary.
        {"name": "policy_2048x50257", "kind": "policy", "rows": 2048, "vocab": 50257, "masked": 0.1, "kl": True,
         "temperature": 0.8, "dtype": "f32"},
        # A few tokens without a reference model, an odd vocabulary, in f64.
        {"name": "policy_301x10007_f64", "kind": "policy", "rows": 301, "vocab": 10007, "masked": 0.3, "kl": False,
         "temperature": 1.0, "dtype": "f64"},
        # Pairs of the char-level GPT's context.
        {"name": "preference_16x128x96", "kind": "preference", "pairs": 16, "tokens": 128, "vocab": 96,
         "smoothing": 0.1, "beta": 0.1, "dtype": "f32"},
        # Pairs of answers over GPT-2's vocabulary.
        {"name": "preference_4x300x50257", "kind": "preference", "pairs": 4, "tokens": 300, "vocab": 50257,
         "smoothing": 0.0, "beta": 0.1, "dtype": "f32"},
    ]


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    largest = max(cost(c) for c in listed())
    while True:
        kind = rng.choice(("dropout", "block", "block", "policy", "preference"))
        case = {"kind": kind, "dtype": "f64" if rng.random() < 0.25 else "f32"}
        if kind == "dropout":
            case.update(rows=log_int(1, 65536), cols=log_int(1, 65536), keep=rng.choice((0.5, 0.9, 0.99)))
            if not 500 <= case["rows"] * case["cols"] <= 60e6:
                continue
        elif kind == "block":
            # from 16 features on: a norm's gradient over one or two is the difference of equal numbers
            case.update(rows=log_int(1, 32768), cols=log_int(16, 20000), train=rng.random() < 0.75,
                        after=rng.choice(("none", "layer", "rms")), before=rng.choice(("none", "layer", "rms")),
                        gate=rng.choice(("none", "shared", "rows")), keep=rng.choice((1.0, 0.9, 0.5)),
                        residual_scale=rng.choice((1.0, 0.9)), block_scale=rng.choice((1.0, 0.25)))
            if case["rows"] * case["cols"] > 30e6:
                continue
        elif kind == "policy":
            case.update(rows=log_int(1, 16384), vocab=log_int(2, 150000), masked=rng.choice((0.0, 0.1, 0.5)),
                        kl=rng.random() < 0.5, temperature=rng.choice((0.7, 1.0, 1.5)))
            if case["rows"] * case["vocab"] > 90e6:
                continue
        else:
            case.update(pairs=log_int(1, 64), tokens=log_int(1, 4000), vocab=log_int(2, 150000),
                        smoothing=rng.choice((0.0, 0.1)), beta=rng.choice((0.05, 0.1, 0.5)))
            if 2 * case["pairs"] * case["tokens"] * case["vocab"] > 90e6:
                continue
        if cost(case) <= largest:
            return case


def cost(case):
    done = work(case)
    return max(done["bytes"], done["flops"] / 50)


def lengths(case):
    """The answers' lengths, chosen and rejected in turn, between half of `tokens` and `tokens`."""
    most = case["tokens"]
    return [max(1, most - int(most * 0.5 * (s * 0.6180339887 % 1.0))) for s in range(2 * case["pairs"])]


def prompt(length):
    """How many of a sequence's first tokens are the prompt's, which no loss counts."""
    return length // 4


def masked(case):
    """Which rows of a policy case are padding or a prompt's."""
    return [(r + 1) * 0.6180339887 % 1.0 < case["masked"] for r in range(case["rows"])]


def work(case):
    size = 8 if case["dtype"] == "f64" else 4
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n * size, "flops": 2 * 26 * n}  # ten rounds for four elements, and the product
    if kind == "block":
        n, columns = case["rows"] * case["cols"], 0
        norms = (case["after"] != "none") + (case["before"] != "none")
        arrays = 3 + (case["gate"] == "rows") + (case["before"] != "none")
        columns = 2 * norms + (case["gate"] == "shared")
        if case["train"]:  # two gradients in (one without a norm ahead of the next block), two or three out
            arrays += 3 + (case["before"] != "none") + (case["gate"] == "rows")
            columns *= 2
        return {"bytes": (arrays * n + columns * case["cols"]) * size, "flops": (60 if case["train"] else 20) * n}
    if kind == "policy":
        rows, live = case["rows"], case["rows"] - sum(masked(case))
        return {"bytes": (rows + live) * case["vocab"] * size + rows * (8 + 8 + 8 * case["kl"] + 3 * size),
                "flops": 8 * live * case["vocab"]}
    rows = sum(lengths(case))
    live = rows - sum(prompt(n) for n in lengths(case))
    return {"bytes": (rows + live) * case["vocab"] * size + rows * 16 + case["pairs"] * (16 + 4 * size),
            "flops": 8 * live * case["vocab"]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPE[case["dtype"]]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"case": case}
    kind = case["kind"]
    if kind in ("dropout", "block"):
        rows, cols = case["rows"], case["cols"]
        # a program's seed, the number of this dropout within its step, and the step, counted on the device
        state.update(seed=(int(seed) * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 64), stream=7, step=1000,
                     more_steps=torch.tensor([int(seed) % 5000], device="cuda"))
        state["x"] = normal(rows, cols)
        if kind == "dropout":
            state["grad"] = normal(rows, cols)
            return state
        # a residual stream with an offset and features of unlike size, as trained models have them
        state["residual"] = normal(rows, cols) * torch.exp(0.5 * normal(1, cols)) + 0.3
        state["gate"] = {"none": lambda: None, "shared": lambda: 1 + 0.3 * normal(cols),
                         "rows": lambda: torch.sigmoid(normal(rows, cols))}[case["gate"]]()
        for name in ("after", "before"):
            state[name] = None
            if case[name] != "none":
                state[name] = {"weight": 1 + 0.2 * normal(cols), "bias": 0.1 * normal(cols), "eps": 1e-5}
        if case["train"]:
            state["grad_h"] = normal(rows, cols)
            state["grad_y"] = normal(rows, cols) if state["before"] else None
            state["workspace"] = torch.empty(WORKSPACE, device="cuda", dtype=torch.uint8)
        return state
    vocab = case["vocab"]
    hidden = masked(case) if kind == "policy" else [i < prompt(n) for n in lengths(case) for i in range(n)]
    hidden = torch.tensor(hidden, device="cuda")
    rows = hidden.numel()
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    # a trained model's logits: its own tokens are likely
    state["logits"] = 2 * normal(rows, vocab)
    state["logits"].scatter_add_(1, targets[:, None], 4 + normal(rows, 1))
    z = state["logits"].double() / case.get("temperature", 1.0)
    logps = z.gather(1, targets[:, None])[:, 0] - torch.logsumexp(z, 1)
    del z
    state["targets"] = torch.where(hidden, -1, targets)
    state["reference"] = logps + 0.2 * normal(rows, dtype=torch.float64)
    if kind == "policy":
        moved = 0.2 * normal(rows, dtype=torch.float64)
        # no ratio within rounding of the clip's borders, where the slope jumps and either side is right
        for border in (math.log(0.8), math.log(1.28)):
            moved = torch.where((moved - border).abs() < 1e-3, moved + 5e-3, moved)
        state["old"] = logps - moved
        state["advantages"] = normal(rows)
        state["weights"] = torch.full((rows,), 1.0 / rows, device="cuda", dtype=dtype)
        if not case["kl"]:
            state["reference"] = None
        return state
    starts = [0]
    for n in lengths(case):
        starts.append(starts[-1] + n)
    state["starts"] = torch.tensor(starts, device="cuda")
    state["weights"] = torch.full((case["pairs"],), 1.0 / case["pairs"], device="cuda", dtype=dtype)
    return state


CLIP_LOW, CLIP_HIGH, KL_WEIGHT = 0.2, 0.28, 0.05


def run(state):
    if own:
        return OWN[state["case"]["kind"]](state)
    return PLAIN[state["case"]["kind"]](state)


# ---- plain forms ----------------------------------------------------------------------------------


def kept(state):
    """Philox4x32-10: word c % 4 of the block (c / 4, r, stream, step) for row r and column c, below the keep share."""
    rows, cols = state["x"].shape
    c0 = torch.arange(-(-cols // 4), device="cuda").expand(rows, -1)
    c1 = torch.arange(rows, device="cuda")[:, None].expand_as(c0)
    c2 = torch.full_like(c0, state["stream"])
    c3 = ((state["step"] + state["more_steps"]) & WORD).expand_as(c0)
    k0, k1 = state["seed"] & WORD, state["seed"] >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & WORD) ^ c1 ^ k0, p1 & WORD, (p0 >> 32 & WORD) ^ c3 ^ k1, p0 & WORD
        k0, k1 = (k0 + 0x9E3779B9) & WORD, (k1 + 0xBB67AE85) & WORD
    words = torch.stack((c0, c1, c2, c3), 2).reshape(rows, -1)[:, :cols]
    return words < round(state["case"]["keep"] * 2 ** 32)


def plain_dropout(state):
    mask, keep = kept(state), state["case"]["keep"]
    return {"y": torch.where(mask, state["x"] / keep, 0), "grad": torch.where(mask, state["grad"] / keep, 0)}


def normed(x, norm, kind):
    """The norm's output, the standardized rows and the rows' reciprocal deviations."""
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    centred = x - mean
    rate = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + norm["eps"])
    unit = centred * rate
    return unit * norm["weight"] + norm["bias"], unit, rate


def norm_backward(grad, norm, kind, unit, rate):
    """The gradients of the norm's input, weight and bias."""
    g = grad * norm["weight"]
    back = g - unit * (g * unit).mean(1, keepdim=True)
    if kind == "layer":
        back = back - g.mean(1, keepdim=True)
    return back * rate, (grad * unit).sum(0), grad.sum(0)


def plain_block(state):
    case, x, after, before = state["case"], state["x"], state["after"], state["before"]
    out = {}
    factor = kept(state).to(x.dtype) / case["keep"] if case["keep"] < 1 else 1.0
    n, unit, rate = normed(x, after, case["after"]) if after else (x, None, None)
    gate = state["gate"] if state["gate"] is not None else 1.0
    a = n * factor
    out["h"] = h = case["residual_scale"] * state["residual"] + case["block_scale"] * (gate * a)
    if before:
        out["y"], next_unit, next_rate = normed(h, before, case["before"])
    if not case["train"]:
        return out
    total = state["grad_h"]
    if before:
        back, out["before_weight"], out["before_bias"] = norm_backward(state["grad_y"], before, case["before"],
                                                                       next_unit, next_rate)
        total = total + back
    out["grad_residual"] = case["residual_scale"] * total
    if state["gate"] is not None:
        by_row = case["block_scale"] * a * total
        out["grad_gate"] = by_row.sum(0) if case["gate"] == "shared" else by_row
    grad = case["block_scale"] * gate * total * factor
    if after:
        grad, out["after_weight"], out["after_bias"] = norm_backward(grad, after, case["after"], unit, rate)
    out["grad_x"] = grad
    return out


def logps_of(state):
    """The exponentials of the rows, their sums, and the targets' log-probabilities, the sums and those in 64 bits."""
    z, targets = state["logits"] / state["case"].get("temperature", 1.0), state["targets"].clamp(min=0)[:, None]
    largest = z.amax(1, keepdim=True)
    e = torch.exp(z - largest)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    # the quotient in 64 bits: its rounding would count in a long sum
    at = state["logits"].gather(1, targets).double() / state["case"].get("temperature", 1.0)
    return e, total, (at - largest.double() - torch.log(total))[:, 0]


def logits_grad(state, e, total, slopes):
    """The gradient from the loss's derivative with respect to each row's log-probability."""
    slopes = (slopes / state["case"].get("temperature", 1.0))[:, None]
    grad = e * (-slopes / total).to(e.dtype)
    grad.scatter_add_(1, state["targets"].clamp(min=0)[:, None], slopes.to(e.dtype))
    return grad


def plain_policy(state):
    counted = state["targets"] >= 0
    e, total, logps = logps_of(state)
    ratio = torch.exp(logps - state["old"])
    advantage = state["advantages"].double()
    free, held = ratio * advantage, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * advantage
    loss, slope = -torch.minimum(free, held), torch.where(free <= held, -free, 0.0)
    if state["reference"] is not None:
        apart = state["reference"] - logps
        loss = loss + KL_WEIGHT * (torch.exp(apart) - apart - 1)
        slope = slope + KL_WEIGHT * (1 - torch.exp(apart))
    slope = torch.where(counted, slope * state["weights"].double(), 0.0)
    return {"losses": torch.where(counted, loss, 0.0).to(e.dtype), "grad": logits_grad(state, e, total, slope)}


def plain_preference(state):
    case, starts = state["case"], state["starts"]
    counted = state["targets"] >= 0
    e, total, logps = logps_of(state)
    apart = torch.where(counted, logps - state["reference"], 0.0)
    sums = torch.cat((torch.zeros_like(apart[:1]), apart.cumsum(0)))
    rewards = (case["beta"] * (sums[starts[1:]] - sums[starts[:-1]])).reshape(-1, 2)
    margin = rewards[:, 0] - rewards[:, 1]
    smooth = case["smoothing"]

    def log_sigmoid(m):
        return m.clamp(max=0) - torch.log1p(torch.exp(-m.abs()))

    losses = -(1 - smooth) * log_sigmoid(margin) - smooth * log_sigmoid(-margin)
    slope = -(1 - smooth) * torch.exp(log_sigmoid(-margin)) + smooth * torch.exp(log_sigmoid(margin))
    slope = slope * case["beta"] * state["weights"].double()
    at = torch.arange(counted.numel(), device="cuda")
    sequence = (at[:, None] >= starts[None, 1:]).sum(1)
    slopes = torch.where(sequence % 2 == 0, 1.0, -1.0) * slope[sequence // 2]
    return {"losses": losses.to(e.dtype), "rewards": rewards.to(e.dtype),
            "grad": logits_grad(state, e, total, torch.where(counted, slopes, 0.0))}


PLAIN = {"dropout": plain_dropout, "block": plain_block, "policy": plain_policy, "preference": plain_preference}


# ---- the framework's calls ------------------------------------------------------------------------


def backend():
    package = str(Path(__file__).resolve().parents[1] / "kael.cpp_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kd
    return kd, kd.load()


def pointer(tensor):
    return tensor.data_ptr() if tensor is not None else None


def own_dropout(state):
    kd, b = backend()
    case, x = state["case"], state["x"]
    dtype = kd.F64 if case["dtype"] == "f64" else kd.F32
    counter = kd.Counter(state["seed"], state["stream"], state["step"], 0, state["more_steps"].data_ptr())
    y, grad = torch.empty_like(x), torch.empty_like(x)
    b.call("counter_dropout", dtype, y.data_ptr(), x.data_ptr(), case["rows"], case["cols"], case["keep"], counter)
    b.call("counter_dropout", dtype, grad.data_ptr(), state["grad"].data_ptr(), case["rows"], case["cols"], case["keep"],
           counter)
    return {"y": y, "grad": grad}


def own_block(state):
    kd, b = backend()
    case, x, gate = state["case"], state["x"], state["gate"]
    dtype = kd.F64 if case["dtype"] == "f64" else kd.F32
    rows, cols = x.shape
    kinds = {"none": kd.NORM_NONE, "layer": kd.NORM_LAYER, "rms": kd.NORM_RMS}
    norms = [kd.Norm(n["weight"].data_ptr(), n["bias"].data_ptr(), n["eps"], kinds[case[name]]) if n else kd.Norm()
             for name, n in (("after", state["after"]), ("before", state["before"]))]
    block = kd.Block(x.data_ptr(), state["residual"].data_ptr(), pointer(gate), rows, cols,
                     {"none": 0, "shared": 1, "rows": rows}[case["gate"]], case["residual_scale"], case["block_scale"],
                     case["keep"], *norms,
                     kd.Counter(state["seed"], state["stream"], state["step"], 0, state["more_steps"].data_ptr()))
    out = {"h": torch.empty_like(x)}
    if state["before"]:
        out["y"] = torch.empty_like(x)
    stats = torch.empty(rows, 4, device="cuda", dtype=torch.float64) if case["train"] else None
    b.call("block_rows", dtype, out["h"].data_ptr(), pointer(out.get("y")), pointer(stats), block)
    if not case["train"]:
        return out
    out["grad_x"], out["grad_residual"] = torch.empty_like(x), torch.empty_like(x)
    if gate is not None:
        out["grad_gate"] = torch.empty_like(gate)
    for name in ("after", "before"):
        if state[name]:
            out[name + "_weight"], out[name + "_bias"] = torch.empty_like(x[0]), torch.empty_like(x[0])
    grads = kd.BlockGrads(*(pointer(out.get(name)) for name in (
        "grad_x", "grad_residual", "grad_gate", "after_weight", "after_bias", "before_weight", "before_bias")))
    b.call("block_rows_backward", dtype, grads, block, out["h"].data_ptr(), stats.data_ptr(), state["grad_h"].data_ptr(),
           pointer(state["grad_y"]), state["workspace"].data_ptr(), WORKSPACE)
    return out


def own_policy(state):
    kd, b = backend()
    case, logits = state["case"], state["logits"]
    dtype = kd.F64 if case["dtype"] == "f64" else kd.F32
    losses, grad = torch.empty_like(state["advantages"]), torch.empty_like(logits)
    policy = kd.Policy(state["old"].data_ptr(), pointer(state["reference"]), state["advantages"].data_ptr(),
                       case["temperature"], CLIP_LOW, CLIP_HIGH, KL_WEIGHT)
    b.call("policy_rows", dtype, losses.data_ptr(), None, grad.data_ptr(), logits.data_ptr(),
           state["targets"].data_ptr(), policy, state["weights"].data_ptr(), case["rows"], case["vocab"])
    return {"losses": losses, "grad": grad}


def own_preference(state):
    kd, b = backend()
    case, logits = state["case"], state["logits"]
    dtype = kd.F64 if case["dtype"] == "f64" else kd.F32
    rows, pairs, vocab = logits.shape[0], case["pairs"], case["vocab"]
    logps = torch.empty(rows, device="cuda", dtype=torch.float64)
    stats = torch.empty(rows, 2, device="cuda", dtype=logits.dtype)
    slopes = torch.empty(rows, device="cuda", dtype=logits.dtype)
    losses, rewards = torch.empty_like(state["weights"]), torch.empty(pairs, 2, device="cuda", dtype=logits.dtype)
    grad = torch.empty_like(logits)
    b.call("token_logps", dtype, logps.data_ptr(), stats.data_ptr(), logits.data_ptr(), state["targets"].data_ptr(),
           rows, vocab, 1.0)
    b.call("preference_pairs", dtype, losses.data_ptr(), rewards.data_ptr(), slopes.data_ptr(), logps.data_ptr(),
           state["reference"].data_ptr(), state["targets"].data_ptr(), state["starts"].data_ptr(),
           state["weights"].data_ptr(), pairs, rows, vocab, case["beta"], case["smoothing"])
    b.call("token_logps_grad", dtype, grad.data_ptr(), logits.data_ptr(), stats.data_ptr(), state["targets"].data_ptr(),
           slopes.data_ptr(), rows, vocab, 1.0)
    return {"losses": losses, "rewards": rewards, "grad": grad}


OWN = {"dropout": own_dropout, "block": own_block, "policy": own_policy, "preference": own_preference}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"dropout": exact_dropout, "block": exact_block, "policy": exact_policy,
            "preference": exact_preference}[case["kind"]](state)


def drawn(state):
    """The mask's factors: 0 or 1 / keep. The words' products by halves of 16 bits."""
    (rows, cols), keep = state["x"].shape, state["case"]["keep"]
    blocks = (cols + 3) // 4
    counter = torch.zeros(4, rows, blocks, device="cuda", dtype=torch.int64)
    counter[0] += torch.arange(blocks, device="cuda")
    counter[1] += torch.arange(rows, device="cuda")[:, None]
    counter[2] += state["stream"]
    counter[3] += (state["step"] + int(state["more_steps"])) % 2 ** 32

    def wide(x, m):
        low = x * (m & 0xFFFF)
        high = x * (m >> 16) + (low >> 16)
        return high >> 16, (high & 0xFFFF) << 16 | low & 0xFFFF

    key = [state["seed"] % 2 ** 32, state["seed"] // 2 ** 32]
    for turn in range(10):
        (h0, l0), (h1, l1) = wide(counter[0], 0xD2511F53), wide(counter[2], 0xCD9E8D57)
        mixed = h1 ^ counter[1] ^ ((key[0] + turn * 0x9E3779B9) % 2 ** 32)
        other = h0 ^ counter[3] ^ ((key[1] + turn * 0xBB67AE85) % 2 ** 32)
        counter[0], counter[1], counter[2], counter[3] = mixed, l1, other, l0
    below = counter.permute(1, 2, 0).reshape(rows, -1)[:, :cols].double() / 2 ** 32 < round(keep * 2 ** 32) / 2 ** 32
    return below.double() / keep


def exact_dropout(state):
    factor = drawn(state)
    return {"y": state["x"].double() * factor, "grad": state["grad"].double() * factor}


def exact_block(state):
    """The forward pass from the definition, the gradients from its differentials by torch's autograd."""
    case = state["case"]
    leaves = {"grad_x": state["x"], "grad_residual": state["residual"]}
    if state["gate"] is not None:
        leaves["grad_gate"] = state["gate"]
    for name in ("after", "before"):
        if state[name]:
            leaves.update({name + "_" + part: state[name][part] for part in ("weight", "bias")})
    leaves = {name: t.double().requires_grad_(case["train"]) for name, t in leaves.items()}

    def apply(name, v):
        if case[name] == "none":
            return v
        if case[name] == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v * (v.pow(2).mean(1, keepdim=True) + state[name]["eps"]).rsqrt()
        return v * leaves[name + "_weight"] + leaves[name + "_bias"]

    a = apply("after", leaves["grad_x"])
    if case["keep"] < 1:
        a = a * drawn(state)
    h = case["residual_scale"] * leaves["grad_residual"] + case["block_scale"] * a * leaves.get("grad_gate", 1.0)
    out, given = {"h": h}, [state["grad_h"].double()] if case["train"] else None
    if state["before"]:
        out["y"] = apply("before", h)
    if case["train"]:
        if state["before"]:
            given.append(state["grad_y"].double())
        out.update(zip(leaves, torch.autograd.grad(list(out.values()), list(leaves.values()), given)))
    return {name: t.detach() for name, t in out.items()}


def shares(state):
    """Rows' log-softmax, and the rows that have a target with it."""
    logs = torch.log_softmax(state["logits"].double() / state["case"].get("temperature", 1.0), 1)
    return logs, torch.nonzero(state["targets"] >= 0)[:, 0]


def through(logs, rows, targets, slopes, temperature):
    """slopes (1 at the target - softmax) / temperature in the given rows, 0 in the others."""
    grad = torch.zeros_like(logs)
    grad[rows] = -logs[rows].exp()
    grad[rows, targets[rows]] += 1
    grad[rows] *= (slopes / temperature)[:, None]
    return grad


def exact_policy(state):
    logs, rows = shares(state)
    at = logs[rows, state["targets"][rows]]
    advantage = state["advantages"][rows].double()
    ratio = (at - state["old"][rows]).exp()
    clipped = ((advantage > 0) & (ratio > 1 + CLIP_HIGH)) | ((advantage < 0) & (ratio < 1 - CLIP_LOW))
    bounded = ratio.clone()
    bounded[clipped & (advantage > 0)], bounded[clipped & (advantage < 0)] = 1 + CLIP_HIGH, 1 - CLIP_LOW
    loss, slope = -bounded * advantage, torch.where(clipped, 0.0, -ratio * advantage)
    if state["reference"] is not None:
        apart = state["reference"][rows] - at
        loss, slope = loss + KL_WEIGHT * (apart.expm1() - apart), slope - KL_WEIGHT * apart.expm1()
    losses = torch.zeros(logs.shape[0], device="cuda", dtype=torch.float64)
    losses[rows] = loss
    return {"losses": losses, "grad": through(logs, rows, state["targets"], slope * state["weights"][rows].double(),
                                              state["case"]["temperature"])}


def exact_preference(state):
    case, starts = state["case"], state["starts"].tolist()
    logs, rows = shares(state)
    moved = torch.zeros(logs.shape[0], device="cuda", dtype=torch.float64)
    moved[rows] = logs[rows, state["targets"][rows]] - state["reference"][rows]
    rewards = case["beta"] * torch.stack([moved[a:b].sum() for a, b in zip(starts, starts[1:])]).reshape(-1, 2)
    margin, smooth = rewards[:, 0] - rewards[:, 1], case["smoothing"]
    losses = (1 - smooth) * torch.logaddexp(-margin, torch.zeros_like(margin))
    losses += smooth * torch.logaddexp(margin, torch.zeros_like(margin))
    by_margin = case["beta"] * state["weights"].double() * (torch.sigmoid(margin) - (1 - smooth))
    both = torch.stack((by_margin, -by_margin), 1).flatten()
    slopes = both.repeat_interleave(torch.tensor(starts[1:], device="cuda") - torch.tensor(starts[:-1], device="cuda"))
    return {"losses": losses, "rewards": rewards, "grad": through(logs, rows, state["targets"], slopes[rows], 1.0)}
