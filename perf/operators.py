"""The operators for serving with a draft model and for training one, as cases that can be timed and compared.

Four kinds. `append`: new keys and values rotated, quantised and appended to a paged 8-bit cache, then the pages that
they touch read back as the values they hold. `attention`: new queries of ragged sequences against that cache.
`verify`: drafted tokens accepted or replaced against the target's probabilities. `distill`: the loss against a
teacher's top logits and its gradient.

Sizes are those of the repository's configurations (GPT-2 small's 12 heads of 64 and 50257 tokens, the char-level GPT's
32 x 128 tokens of 96 characters) and generic ones (grouped heads of 128, long caches). `draw` spreads each kind over
its whole range.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "f64": torch.float64}
WORKSPACE = 64 << 20  # what a serving program keeps for the attention's partial sums


def listed():
    return [
        # One decode step of 64 GPT-2 small sequences: one token each. Latency.
        {"name": "append_decode_64", "kind": "append", "sequences": 64, "new": 1, "keys": 1000, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "rotated": 64, "interleaved": False},
        # Eight ragged prompts of a model with grouped heads, onto caches that already hold a prefix.
        {"name": "append_prompts_8", "kind": "append", "sequences": 8, "new": 1000, "keys": 1500, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "rotated": 128, "interleaved": True},
        # One sequence of GPT-2 small generating near the end of its context: the smallest launch.
        {"name": "attention_one_1000", "kind": "attention", "sequences": 1, "new": 1, "keys": 1000, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16},
        # A decode step of 64 such sequences, of ragged lengths.
        {"name": "attention_decode_64", "kind": "attention", "sequences": 64, "new": 1, "keys": 1024, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16},
        # A decode step over long caches with grouped heads: the cache's bytes decide.
        {"name": "attention_long_4x40000", "kind": "attention", "sequences": 4, "new": 1, "keys": 40000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64},
        # The target scoring 5 drafted positions of each of 32 sequences.
        {"name": "attention_drafted_32x5", "kind": "attention", "sequences": 32, "new": 5, "keys": 2000, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 32},
        # Whole GPT-2 prompts of ragged lengths.
        {"name": "attention_prompts_8x1000", "kind": "attention", "sequences": 8, "new": 1000, "keys": 1000,
         "heads": 12, "kv_heads": 12, "dim": 64, "page": 16},
        # Long prompts with grouped heads: the largest product.
        {"name": "attention_prompts_2x4096", "kind": "attention", "sequences": 2, "new": 4096, "keys": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # A few sequences' drafts against GPT-2's vocabulary, in f64.
        {"name": "verify_8x4_f64", "kind": "verify", "sequences": 8, "drafts": 4, "vocab": 50257, "dtype": "f64",
         "given": True},
        # A full batch's drafts.
        {"name": "verify_256x7", "kind": "verify", "sequences": 256, "drafts": 7, "vocab": 50257, "dtype": "f32",
         "given": True},
        # A training step's loss of the char-level GPT as the draft.
        {"name": "distill_4096x96", "kind": "distill", "rows": 4096, "vocab": 96, "kept": 8, "temperature": 2.0,
         "dtype": "f32"},
        # The same at GPT-2's vocabulary.
        {"name": "distill_2048x50257", "kind": "distill", "rows": 2048, "vocab": 50257, "kept": 64,
         "temperature": 1.5, "dtype": "f32"},
    ]


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    largest = max(cost(c) for c in listed())
    while True:
        kind = rng.choice(("append", "attention", "attention", "attention", "verify", "distill"))
        case = {"kind": kind}
        if kind in ("append", "attention"):
            sequences = log_int(1, 128)
            new = rng.choice((1, 1, log_int(2, 8), log_int(9, 4096)))
            keys = max(new, log_int(1, 40000))
            kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
            group = rng.choice((1, 1, 2, 3, 4, 8))
            dim = rng.choice((64, 128))
            case.update(sequences=sequences, new=new, keys=keys, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                        page=rng.choice((16, 32, 64, 128)))
            if kind == "append":
                case.update(rotated=rng.choice((0, dim // 2, dim)), interleaved=rng.random() < 0.5)
            pool = sequences * keys * kv_heads * dim
            scores = sequences * kv_heads * group * new * keys
            if pool > 170e6 or scores > 1.1e9 or sequences * new * case["heads"] * dim > 35e6:
                continue
        elif kind == "verify":
            case.update(sequences=log_int(1, 256), drafts=log_int(1, 8), vocab=log_int(2, 100000),
                        dtype="f64" if rng.random() < 0.3 else "f32", given=rng.random() < 0.75)
            if case["sequences"] * (case["drafts"] + 1) * case["vocab"] > 120e6:
                continue
        else:
            vocab = log_int(8, 100000)
            case.update(rows=log_int(1, 16384), vocab=vocab, kept=log_int(1, min(vocab, 128)),
                        temperature=rng.choice((0.7, 1.0, 2.0, 4.0)), dtype="f64" if rng.random() < 0.3 else "f32")
            if case["rows"] * vocab * (2 if case["dtype"] == "f64" else 1) > 2048 * 50257:
                continue
        if cost(case) <= largest:
            return case


def cost(case):
    done = work(case)
    return max(done["bytes"], done["flops"] / 50)


def ragged(most, least, count):
    """`count` lengths between half of `most` and `most`, the first of them `most`, none below `least`."""
    return [max(least, most - int(most * 0.5 * (s * 0.6180339887 % 1.0))) for s in range(count)]


def plan(case):
    """Each sequence's new tokens and its length with them."""
    new = ragged(case["new"], 1, case["sequences"]) if case["new"] > 8 else [case["new"]] * case["sequences"]
    return new, [max(n, length) for n, length in zip(new, ragged(case["keys"], 1, case["sequences"]))]


def touched(case):
    """The first position of each sequence's first touched page: from there on the append case reads back."""
    new, lengths = plan(case)
    return [(length - n) // case["page"] * case["page"] for n, length in zip(new, lengths)]


def work(case):
    kind = case["kind"]
    if kind in ("append", "attention"):
        new, lengths = plan(case)
        tokens, heads, kv_heads, dim = sum(new), case["heads"], case["kv_heads"], case["dim"]
        pages = sum(-(-length // case["page"]) for length in lengths)
        if kind == "append":
            values = sum(length - first for length, first in zip(lengths, touched(case)))
            # q and the new keys and values read, q and the codes written; then the touched codes read, their values written
            moved = tokens * dim * (heads * 8 + kv_heads * 2 * 5) + values * kv_heads * dim * 2 * 5
            return {"bytes": moved, "flops": 6 * tokens * heads * dim}
        cached = sum(lengths) * kv_heads * dim * 2 + pages * (kv_heads * 8 + 8)
        visible = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lengths))
        return {"bytes": cached + tokens * heads * dim * 8, "flops": 4 * dim * heads * visible}
    size = 8 if case["dtype"] == "f64" else 4
    if kind == "verify":
        # the row of the first rejected draft, or the last one: the target's, and the draft's where it is given
        rows = 2 if case["given"] else 1
        return {"bytes": case["sequences"] * (rows * case["vocab"] * size + case["drafts"] * (16 + 2 * size)),
                "flops": 3 * case["sequences"] * case["vocab"]}
    elements, kept = case["rows"] * case["vocab"], case["rows"] * case["kept"]
    # forward: the logits; backward: the logits again and the gradient
    return {"bytes": 3 * elements * size + 2 * kept * (8 + size), "flops": 8 * elements}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    def integers(values):
        return torch.tensor(values, device="cuda", dtype=torch.int64)

    state = {"case": case}
    kind = case["kind"]
    if kind in ("append", "attention"):
        new, lengths = plan(case)
        sequences, page, dim = case["sequences"], case["page"], case["dim"]
        heads, kv_heads = case["heads"], case["kv_heads"]
        columns = -(-max(lengths) // page)
        pages, tokens = sequences * columns, sum(new)
        starts = [sum(new[:s]) for s in range(sequences + 1)]
        state.update(pages=pages, columns=columns, tokens=tokens, longest=max(lengths), most_new=max(new),
                     table=torch.randperm(pages, generator=gen, device="cuda").reshape(sequences, columns),
                     starts=integers(starts), lengths=integers(lengths))
        # keys of features of unlike size, as trained models have them
        size = torch.exp(0.5 * normal(kv_heads, 1, dim))
        for name, by in (("keys", size), ("values", torch.ones_like(size))):
            values = normal(pages, kv_heads, page, dim) * by
            scales = values.abs().amax((2, 3)) / 127
            codes = torch.round(values / scales[:, :, None, None]).to(torch.int8)
            state[name] = codes if name == "keys" else codes.transpose(2, 3).contiguous()
            state[name[:-1] + "_scales"] = scales
        # the fused projection's rows: queries, keys and values side by side
        fused = normal(tokens, heads + 2 * kv_heads, dim)
        state.update(q=fused[:, :heads], k=fused[:, heads:heads + kv_heads], v=fused[:, heads + kv_heads:])
        if kind == "append":
            first = touched(case)
            state.update(first=integers(first), read=sum(lengths) - sum(first), read_starts=integers(
                [sum(lengths[:s]) - sum(first[:s]) for s in range(sequences + 1)]))
            half = max(case["rotated"] // 2, 1)
            angle = (torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None]
                     * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
            state.update(cosines=angle.cos().float(), sines=angle.sin().float())
        else:
            state["workspace"] = torch.empty(WORKSPACE, device="cuda", dtype=torch.uint8)
        return state
    dtype = DTYPE[case["dtype"]]
    if kind == "verify":
        sequences, drafts, vocab = case["sequences"], case["drafts"], case["vocab"]
        logits = 2 * normal(sequences, drafts + 1, vocab, dtype=dtype)
        state["target"] = torch.softmax(logits, -1)
        if case["given"]:  # a draft that is near its target: most of its tokens are accepted
            state["draft"] = torch.softmax(logits[:, :drafts] + 0.5 * normal(sequences, drafts, vocab, dtype=dtype), -1)
            picked = state["draft"]
        else:
            state["draft"], picked = None, state["target"][:, :drafts]
        state["drafted"] = torch.multinomial(picked.reshape(-1, vocab), 1, generator=gen).reshape(sequences, drafts)
        state["counts"] = integers([drafts - (s % 3 if drafts > 3 else 0) for s in range(sequences)])
        state["uniforms"] = torch.rand((sequences, drafts + 1), generator=gen, device="cuda", dtype=torch.float64)
        return state
    rows, vocab, kept = case["rows"], case["vocab"], case["kept"]
    state["logits"] = 2 * normal(rows, vocab, dtype=dtype)
    # a teacher near the student, its largest logits of each row
    teacher, indices = torch.topk(state["logits"] + normal(rows, vocab, dtype=dtype), kept, dim=1)
    state.update(teacher=teacher.contiguous(), indices=indices.contiguous(),
                 weights=torch.full((rows,), 1.0 / rows, device="cuda", dtype=dtype))
    return state


def run(state):
    if own:
        return OWN[state["case"]["kind"]](state)
    return PLAIN[state["case"]["kind"]](state)


# ---- plain forms ----------------------------------------------------------------------------------


def rows_of(starts, tokens):
    """Each token's sequence, and its place among the sequence's tokens."""
    at = torch.arange(tokens, device=starts.device)
    sequence = (at[:, None] >= starts[None, 1:]).sum(1)
    return sequence, at - starts[sequence]


def rotated(x, state, position):
    """x [tokens, heads, dim] in f64, its first `rotated` features turned by the position's angles."""
    x, features = x.double(), state["case"]["rotated"]
    if not features:
        return x
    c = state["cosines"].double()[position][:, None, :]
    s = state["sines"].double()[position][:, None, :]
    turned, rest = x[..., :features], x[..., features:]
    if state["case"]["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        both = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = turned[..., :features // 2], turned[..., features // 2:]
        both = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((both, rest), -1)


def append_codes(state, x, name, sequence, position):
    """The values x [tokens, kv_heads, dim] quantised into their pages of the cache `name`, in place."""
    page_size, codes, scales = state["case"]["page"], state[name], state[name[:-1] + "_scales"]
    turned = name == "values"  # the values' pages hold a feature's tokens side by side
    page = state["table"][sequence, position // page_size]
    slot = position % page_size
    largest = torch.zeros(scales.shape, device=x.device, dtype=torch.float64)
    largest.index_reduce_(0, page, x.abs().amax(2), "amax")
    begun = torch.zeros(scales.shape[0], device=x.device, dtype=torch.bool)
    begun[page] = True
    # the page that a sequence's first new token falls in may hold tokens already
    added = state["starts"][1:] - state["starts"][:-1]
    from_ = state["lengths"] - added
    sequences = torch.arange(from_.numel(), device=x.device)
    open_page = state["table"][sequences, from_ // page_size]
    held = from_ % page_size
    old = torch.zeros_like(scales)
    old[open_page] = torch.where(held[:, None] > 0, scales[open_page], torch.zeros_like(scales[open_page]))
    fresh = torch.maximum(old, (largest / 127).float())
    scales.copy_(torch.where(begun[:, None], fresh, scales))
    open_codes = codes[open_page]
    ratio = old[open_page].double() / torch.where(fresh[open_page] > 0, fresh[open_page], 1.0).double()
    again = torch.round(open_codes.double() * ratio[:, :, None, None]).to(torch.int8)
    slots = torch.arange(page_size, device=x.device)
    kept = slots[None, :] < held[:, None]
    kept = kept[:, None, None, :] if turned else kept[:, None, :, None]
    codes[open_page] = torch.where(kept, again, open_codes)
    scale = fresh[page].double()
    inverse = torch.where(scale > 0, 1 / scale, 0.0)
    quantised = torch.round(x * inverse[:, :, None]).clamp(-127, 127).to(torch.int8)
    if turned:
        codes[page, :, :, slot] = quantised
    else:
        codes[page, :, slot] = quantised


def plain_append(state):
    sequence, at = rows_of(state["starts"], state["tokens"])
    added = state["starts"][1:] - state["starts"][:-1]
    position = (state["lengths"] - added)[sequence] + at
    q = rotated(state["q"], state, position).float()
    append_codes(state, rotated(state["k"], state, position), "keys", sequence, position)
    append_codes(state, state["v"].double(), "values", sequence, position)
    # the pages that were touched, read back
    sequence, at = rows_of(state["read_starts"], state["read"])
    position = state["first"][sequence] + at
    page_size = state["case"]["page"]
    page, slot = state["table"][sequence, position // page_size], position % page_size
    keys = state["keys"][page, :, slot].float() * state["key_scales"][page][:, :, None]
    values = state["values"][page, :, :, slot].float() * state["value_scales"][page][:, :, None]
    return {"q": q, "keys": keys, "values": values}


def plain_attention(state):
    case = state["case"]
    sequences, heads, kv_heads, dim = case["sequences"], case["heads"], case["kv_heads"], case["dim"]
    new, keys = state["most_new"], state["columns"] * case["page"]
    sequence, at = rows_of(state["starts"], state["tokens"])
    added = state["starts"][1:] - state["starts"][:-1]
    q = torch.zeros(sequences, new, heads, dim, device="cuda")
    q[sequence, at] = state["q"]
    q = q.reshape(sequences, new, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(sequences, kv_heads, -1, dim)
    k = state["keys"][state["table"]].float() * state["key_scales"][state["table"]][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(sequences, kv_heads, keys, dim)
    v = state["values"][state["table"]].float() * state["value_scales"][state["table"]][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(sequences, kv_heads, keys, dim)
    scores = (q @ k.transpose(2, 3)) * dim ** -0.5
    last = (state["lengths"] - added)[:, None] + torch.arange(new, device="cuda")
    hidden = torch.arange(keys, device="cuda") > last[..., None]
    scores = scores.view(sequences, kv_heads, -1, new, keys).masked_fill_(hidden[:, None, None], -math.inf)
    weights = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(sequences, kv_heads, -1, keys) @ v).view(sequences, kv_heads, -1, new, dim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(sequences, new, heads, dim)[sequence, at]


def plain_verify(state):
    case, target, draft, drafted = state["case"], state["target"], state["draft"], state["drafted"]
    sequences, drafts, vocab = case["sequences"], case["drafts"], case["vocab"]
    counts, uniforms = state["counts"], state["uniforms"]
    place = torch.arange(drafts, device="cuda")
    p = target[:, :drafts].gather(2, drafted[..., None])[..., 0].double()
    q = draft.gather(2, drafted[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    kept = (uniforms[:, :drafts] * q < p) & (place < counts[:, None])
    accepted = kept.long().cumprod(1).sum(1)
    sequence = torch.arange(sequences, device="cuda")
    row = target[sequence, accepted].double()
    failed = torch.minimum(accepted, torch.full_like(accepted, drafts - 1))
    if draft is not None:
        other = draft[sequence, failed].double()
    else:
        other = (torch.arange(vocab, device="cuda") == drafted[sequence, failed][:, None]).double()
    rest = torch.where((accepted < counts)[:, None], (row - other).clamp(min=0.0), row)
    weights = torch.where((rest.sum(1) > 0)[:, None], rest, row)
    sums = weights.cumsum(1)
    # the draws that follow the accepted ones decide the sampled token
    point = uniforms[:, drafts] * sums[:, -1]
    token = torch.minimum((sums <= point[:, None]).sum(1), torch.full_like(accepted, vocab - 1))
    tokens = torch.full((sequences, drafts + 1), -1, device="cuda", dtype=torch.int64)
    tokens[:, :drafts] = torch.where(place < accepted[:, None], drafted, -1)
    tokens[sequence, accepted] = token
    return {"tokens": tokens, "accepted": accepted}


def plain_distill(state):
    case, logits, indices = state["case"], state["logits"], state["indices"]
    temperature = case["temperature"]
    x = logits / temperature
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    y = state["teacher"].double() / temperature
    y = y - y.amax(1, keepdim=True)
    log_teacher = y - torch.log(torch.exp(y).sum(1, keepdim=True))
    share = torch.exp(log_teacher)
    log_student = x.gather(1, indices).double() - torch.log(total)
    losses = temperature ** 2 * (share * (log_teacher - log_student)).sum(1)
    weights = (state["weights"] * temperature)[:, None]
    grad = e * (weights / total.to(e.dtype))
    grad.scatter_add_(1, indices, -weights * share.to(e.dtype))
    return {"losses": losses.to(logits.dtype), "grad": grad}


PLAIN = {"append": plain_append, "attention": plain_attention, "verify": plain_verify, "distill": plain_distill}


# ---- the framework's calls ------------------------------------------------------------------------


def backend():
    package = str(Path(__file__).resolve().parents[1] / "kael.cpp_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kd
    return kd, kd.load()


def cache_and_batch(kd, state, starts, tokens):
    case = state["case"]
    cache = kd.PagedCache(state["keys"].data_ptr(), state["values"].data_ptr(), state["key_scales"].data_ptr(),
                          state["value_scales"].data_ptr(), state["pages"], case["kv_heads"], case["page"], case["dim"])
    return cache, kd.PagedBatch(state["table"].data_ptr(), starts.data_ptr(), state["lengths"].data_ptr(),
                                case["sequences"], state["columns"], tokens)


def own_append(state):
    kd, b = backend()
    case = state["case"]
    cache, batch = cache_and_batch(kd, state, state["starts"], state["tokens"])
    q, k, v = state["q"], state["k"], state["v"]
    out = torch.empty(q.shape, device="cuda")
    rotation = kd.Rotation(state["cosines"].data_ptr(), state["sines"].data_ptr(), state["cosines"].shape[0],
                           case["rotated"], case["interleaved"])
    b.call("paged_append", kd.F32, cache, batch, rotation, out.data_ptr(), q.data_ptr(), kd.strides(*q.stride()[:2]),
           case["heads"], k.data_ptr(), kd.strides(*k.stride()[:2]), v.data_ptr(), kd.strides(*v.stride()[:2]))
    batch = kd.PagedBatch(state["table"].data_ptr(), state["read_starts"].data_ptr(), state["lengths"].data_ptr(),
                          case["sequences"], state["columns"], state["read"])
    keys = torch.empty(state["read"], case["kv_heads"], case["dim"], device="cuda")
    values = torch.empty_like(keys)
    b.call("paged_read", kd.F32, keys.data_ptr(), values.data_ptr(), cache, batch)
    return {"q": out, "keys": keys, "values": values}


def own_attention(state):
    kd, b = backend()
    case, q = state["case"], state["q"]
    cache, batch = cache_and_batch(kd, state, state["starts"], state["tokens"])
    out = torch.empty(q.shape, device="cuda")
    b.call("paged_attention", kd.F32, out.data_ptr(), q.data_ptr(), kd.strides(*q.stride()[:2]), case["heads"], cache,
           batch, case["dim"] ** -0.5, state["longest"], state["workspace"].data_ptr(), WORKSPACE)
    return out


def own_verify(state):
    kd, b = backend()
    case, draft = state["case"], state["draft"]
    tokens = torch.empty(case["sequences"], case["drafts"] + 1, device="cuda", dtype=torch.int64)
    accepted = torch.empty(case["sequences"], device="cuda", dtype=torch.int64)
    b.call("verify_drafts", kd.F64 if case["dtype"] == "f64" else kd.F32, tokens.data_ptr(), accepted.data_ptr(),
           state["target"].data_ptr(), draft.data_ptr() if draft is not None else None, state["drafted"].data_ptr(),
           state["counts"].data_ptr(), state["uniforms"].data_ptr(), case["sequences"], case["drafts"], case["vocab"])
    return {"tokens": tokens, "accepted": accepted}


def own_distill(state):
    kd, b = backend()
    case, logits = state["case"], state["logits"]
    dtype = kd.F64 if case["dtype"] == "f64" else kd.F32
    rows, vocab, kept, temperature = case["rows"], case["vocab"], case["kept"], case["temperature"]
    losses = torch.empty(rows, device="cuda", dtype=logits.dtype)
    stats = torch.empty(rows, 2, device="cuda", dtype=logits.dtype)
    grad = torch.empty_like(logits)
    b.call("distill_rows", dtype, losses.data_ptr(), stats.data_ptr(), logits.data_ptr(), state["indices"].data_ptr(),
           state["teacher"].data_ptr(), rows, vocab, kept, temperature)
    b.call("distill_grad", dtype, grad.data_ptr(), logits.data_ptr(), stats.data_ptr(), state["indices"].data_ptr(),
           state["teacher"].data_ptr(), state["weights"].data_ptr(), rows, vocab, kept, temperature)
    return {"losses": losses, "grad": grad}


OWN = {"append": own_append, "attention": own_attention, "verify": own_verify, "distill": own_distill}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": exact_append, "attention": exact_attention, "verify": lambda s: None,
            "distill": exact_distill}[case["kind"]](state)


def exact_append(state):
    case = state["case"]
    page_size, half = case["page"], case["rotated"] // 2
    new, lengths = plan(case)
    q_out = state["q"].double().clone()
    read = {"keys": [], "values": []}
    row = 0
    for s, (n, length) in enumerate(zip(new, lengths)):
        begin, rows = length - n, slice(row, row + n)
        row += n
        given = {"keys": state["k"][rows].double().clone(), "values": state["v"][rows].double()}
        if half:
            c, d = (state[t][begin:length].double()[:, None] for t in ("cosines", "sines"))
            for x in (q_out[rows], given["keys"]):
                lower, upper = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"]
                                else (slice(0, half), slice(half, 2 * half)))
                a, b = x[..., lower].clone(), x[..., upper].clone()
                x[..., lower], x[..., upper] = a * c - b * d, a * d + b * c
        first = begin // page_size
        for name in ("keys", "values"):
            pages = state["table"][s, first:-(-length // page_size)]
            codes, scales = state[name][pages].double(), state[name[:-1] + "_scales"][pages].double()
            if name == "values":
                codes = codes.transpose(2, 3)
            codes = codes.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])  # one row a position
            held = begin - first * page_size
            added = torch.zeros_like(codes)
            added[held:held + n] = given[name]
            old = scales.clone()
            old[1:] = 0
            if not held:
                old[0] = 0
            most = added.abs().view(len(pages), page_size, *added.shape[1:]).amax((1, 3))
            scale = torch.maximum(old, (most / 127).float().double())
            by_row = scale.repeat_interleave(page_size, 0)[..., None]
            result = torch.round(added * (1 / by_row)).clamp(-127, 127)
            result[:held] = torch.round(codes[:held] * (old[0] / scale[0])[None, :, None])
            read[name].append((result * by_row)[:held + n])
    return {"q": q_out, "keys": torch.cat(read["keys"]), "values": torch.cat(read["values"])}


def exact_attention(state):
    case = state["case"]
    new, lengths = plan(case)
    group, page_size = case["heads"] // case["kv_heads"], case["page"]
    out = torch.empty(state["q"].shape, device="cuda", dtype=torch.float64)
    row = 0
    for s, (n, length) in enumerate(zip(new, lengths)):
        pages = state["table"][s, :-(-length // page_size)]
        seen = torch.arange(length, device="cuda")[None, :] <= torch.arange(length - n, length, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            k = state["keys"][pages, h].double() * state["key_scales"][pages, h].double()[:, None, None]
            v = state["values"][pages, h].double() * state["value_scales"][pages, h].double()[:, None, None]
            k, v = k.reshape(-1, case["dim"])[:length], v.transpose(1, 2).reshape(-1, case["dim"])[:length]
            for g in range(h * group, (h + 1) * group):
                score = torch.mm(state["q"][row:row + n, g].double(), k.t().contiguous()) / math.sqrt(case["dim"])
                share = torch.softmax(score.masked_fill(~seen, -math.inf), 1)
                out[row:row + n, g] = torch.mm(share, v)
        row += n
    return out


def exact_distill(state):
    temperature = state["case"]["temperature"]
    log_student = torch.log_softmax(state["logits"].double() / temperature, 1)
    log_teacher = torch.log_softmax(state["teacher"].double() / temperature, 1)
    teacher = log_teacher.exp()
    losses = (teacher * (log_teacher - log_student.gather(1, state["indices"]))).sum(1) * temperature ** 2
    grad = log_student.exp_()
    grad[torch.arange(grad.shape[0], device="cuda")[:, None], state["indices"]] -= teacher
    return {"losses": losses, "grad": grad * (temperature * state["weights"].double())[:, None]}
