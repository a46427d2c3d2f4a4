"""What a decoding step does around its cache and attention, as cases to time and compare.

A case is one pass of one operator:

* "rope": the query and key heads of the fused projection's rows are normed (or
  not) and rotated by their tokens' positions, before the keys enter the cache;
* "mass": the weight that the step's queries give each cached token, summed over
  the queries and the heads that share a key/value head, added to what the tokens
  had gathered before;
* "evict": of each sequence the first and last tokens stay, and the heaviest of
  the others, up to a number of tokens; they move to other pages, and are read back;
* "logprobs": log probabilities of given tokens, the entropy and the likeliest
  tokens of rows of logits.

Rows are f32, as the projections give and take them.  A cache holds f16 values, or
8-bit codes with one f32 scale per token and head: scale = max |x| / 127, code =
x / scale rounded to nearest, ties to even.

`own` chooses the framework's calls; otherwise run() computes the same in
elementary torch operations in 32 bits (angles and the codes' borders in 64).
"""
import math

import torch

own = False

# heads, key/value heads and width of a head
HEADS = {"mixtral": (32, 8, 128), "qwen3": (32, 4, 128), "small": (16, 2, 64),
         "wide": (16, 8, 256), "full": (12, 12, 96), "single": (24, 1, 128)}


def _rope(shape, tokens, start, norm, style="halves", rotary=0):
    heads, kv_heads, dim = HEADS[shape]
    return dict(kind="rope", heads=heads, kv_heads=kv_heads, dim=dim, tokens=tokens, start=start, norm=norm,
                style=style, rotary=rotary or dim)


def _mass(fmt, shape, seqs, tokens, ctx, page=64, mixed=False):
    heads, kv_heads, dim = HEADS[shape]
    return dict(kind="mass", fmt=fmt, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, tokens=tokens, ctx=ctx,
                page=page, mixed=mixed)


def _evict(fmt, shape, seqs, ctx, keep, sinks, recent, page=64):
    heads, kv_heads, dim = HEADS[shape]
    return dict(kind="evict", fmt=fmt, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, ctx=ctx, keep=keep,
                sinks=sinks, recent=recent, page=page, tokens=0, mixed=False)


def _logprobs(tokens, vocab, given, top):
    return dict(kind="logprobs", tokens=tokens, vocab=vocab, given=given, top=top)


def listed():
    cases = {
        # one sequence's next token, no norm: latency
        "rope_1": _rope("mixtral", 1, 516, norm=False),
        # a long prompt's chunk, heads normed
        "rope_norm_prompt": _rope("qwen3", 8191, 122880, norm=True),
        # heads of which a part is rotated, in neighbouring pairs
        "rope_pairs_part": _rope("full", 2039, 77, norm=True, style="pairs", rotary=32),
        # one decode step of one short sequence: latency
        "mass_f16_1": _mass("f16", "mixtral", 1, 1, 517),
        # a decode step of a serving batch, contexts of all lengths
        "mass_f16_batch": _mass("f16", "mixtral", 61, 1, 8191),
        # the last queries of two long prompts say what of them to keep
        "mass_int8_last": _mass("int8", "qwen3", 2, 37, 32003, page=32),
        # every query of a prompt does
        "mass_f16_prompt": _mass("f16", "mixtral", 1, 4093, 4093),
        # a long prompt is cut to its heaviest tokens once
        "evict_f16_prompt": _evict("f16", "mixtral", 1, 16381, 4096, sinks=4, recent=509),
        # sequences of a serving batch that have outgrown their budget
        "evict_int8_batch": _evict("int8", "qwen3", 23, 5003, 3001, sinks=4, recent=64, page=32),
        # the next token of one sequence, with alternatives: latency
        "logprobs_1": _logprobs(1, 32000, 1, 20),
        # the next tokens of a running batch
        "logprobs_batch": _logprobs(61, 131072, 1, 5),
        # a prompt's (or an evaluation's) tokens are scored; rows of an odd length
        "logprobs_prompt": _logprobs(2039, 100003, 1, 1),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """A step of any kind, shape and format, within the largest listed cases' work and memory."""
    while True:
        kind, shape = rng.choice(("rope", "mass", "mass", "evict", "logprobs")), rng.choice(sorted(HEADS))
        fmt, page = rng.choice(("f16", "int8")), rng.choice((32, 64, 128, 256))
        heads, kv_heads, dim = HEADS[shape]
        if kind == "rope":
            rotary = rng.choice((dim, dim, dim // 2, dim // 4))
            case = _rope(shape, _log_int(rng, 1, 16384), rng.randint(0, 1 << 20), rng.random() < 0.6,
                         rng.choice(("halves", "pairs")), rotary)
        elif kind == "mass":
            step = rng.random() < 0.5
            tokens = rng.choice((1, 1, 2, 3, 5)) if step else _log_int(rng, 6, 4096)
            seqs = _log_int(rng, 1, 96) if step else _log_int(rng, 1, 4)
            case = _mass(fmt, shape, seqs, tokens, max(tokens, _log_int(rng, 1, 100000)), page)
            if tokens > 8 and rng.random() < 0.3:
                case.update(seqs=rng.randint(2, 24), mixed=True)
            scores = case["seqs"] * tokens * heads * case["ctx"]
            if scores > 6e8 or case["seqs"] * (case["ctx"] + 256) * kv_heads * dim > 5e8:
                continue
        elif kind == "evict":
            ctx = _log_int(rng, 1, 100000)
            keep = _log_int(rng, 1, 16384)
            sinks = min(rng.choice((0, 1, 4, 64)), keep)
            recent = rng.randint(0, (keep - sinks) // 2)
            case = _evict(fmt, shape, _log_int(rng, 1, 48), ctx, keep, sinks, recent, page)
            if case["seqs"] * (ctx + 256) * kv_heads * dim > 1.5e8:
                continue
        else:
            case = _logprobs(_log_int(rng, 1, 4096), _log_int(rng, 100, 200000), rng.choice((0, 1, 1, 3)),
                             rng.choice((0, 1, 5, 20)))
        cost = work(case)
        if cost["bytes"] <= 8e8 and cost["flops"] <= 6.5e10:
            return case


# ---------------------------------------------------------------- what a case says
def _new(case):
    """New tokens of each sequence: `tokens`, or one in all but the first."""
    n = case["tokens"]
    return [n] + [1 if case["mixed"] else n] * (case["seqs"] - 1)


def _lengths(case):
    """Tokens of each sequence, the new ones among them: from ctx down to about a quarter of it."""
    S, ctx = case["seqs"], case["ctx"]
    return [max(n, ctx - (s * 37 % S) * (3 * ctx // 4) // S) for s, n in enumerate(_new(case))]


def _kept(case):
    return [min(n, case["keep"]) for n in _lengths(case)]


def work(case):
    if case["kind"] == "logprobs":
        T, V = case["tokens"], case["vocab"]
        return {"bytes": 4 * T * V + T * (8 * case["given"] + 4 + 8 * case["top"]), "flops": 6 * T * V}
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        values = case["tokens"] * (H + G) * D
        return {"bytes": 8 * values + 4 * case["tokens"], "flops": (4 * case["norm"] + 3) * values}
    stored = G * (2 * D if case["fmt"] == "f16" else D + 4)  # bytes of one token's keys
    lengths = _lengths(case)
    if case["kind"] == "mass":
        pairs = sum(n * length - n * (n - 1) // 2 for n, length in zip(_new(case), lengths))
        return {"bytes": sum(lengths) * (stored + 8 * G) + 4 * sum(_new(case)) * H * D, "flops": 2 * pairs * H * D}
    kept = sum(_kept(case))
    # keys and values out of their pages, into others, out of those as f32; the weights, which
    # tokens stay, and their weights
    return {"bytes": kept * (6 * stored + 8 * G * D + 8 * G) + 4 * G * sum(lengths), "flops": kept * G * D}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(case, seed):
    """The fused projection's rows: q, then k, then v."""
    width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    count = case["tokens"] if case["kind"] == "rope" else sum(_new(case))
    return torch.randn((count, width), generator=_generator(seed * 8 + 3), device="cuda")


def _norms(case, seed):
    return 1 + torch.randn((2, case["dim"]), generator=_generator(seed * 8 + 4), device="cuda") / 8


def _angles(case, seed):
    """Each token's position (a prompt's follow each other) and the angles of one position."""
    start = case["start"] + seed % 61
    positions = torch.arange(start, start + case["tokens"], dtype=torch.int32, device="cuda")
    pair = torch.arange(0, case["rotary"], 2, dtype=torch.float64, device="cuda")
    return positions, torch.exp(pair / case["rotary"] * -math.log(1e6)).float()


def _tables(case, seed):
    """First row, length and pages of each sequence: its pages, and those that it moves to, are
    anywhere in the pool."""
    lengths, rows = _lengths(case), [0]
    for n in _new(case):
        rows.append(rows[-1] + n)
    width, to_width = -(-max(lengths) // case["page"]), 0
    if case["kind"] == "evict":
        to_width = -(-max(_kept(case)) // case["page"])
    S = case["seqs"]
    order = torch.randperm(S * (width + to_width) + 3, generator=_generator(seed * 8 + 1), device="cuda")
    order = order.to(torch.int32)
    return {"row_start": torch.tensor(rows, dtype=torch.int32, device="cuda"),
            "kv_len": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            "pages": order[:S * width].reshape(S, width),
            "to_pages": order[S * width:S * (width + to_width)].reshape(S, to_width), "pool": order.numel()}


def _context(case, seed):
    """Keys and values of every token of the sequences, one sequence behind the other: a few
    channels of the keys are larger than the others."""
    g = _generator(seed * 8 + 2)
    shape = (sum(_lengths(case)), case["kv_heads"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda")
    k[:, :, ::29] *= 3.0
    return k, torch.randn(shape, generator=g, device="cuda")


def _weights(case, seed):
    """What the tokens have gathered [seqs, kv_heads, tokens]: a few have most of it, and some
    nothing that 32 bits hold.  Where a step adds to it, not much more than a step gives."""
    shape = (case["seqs"], case["kv_heads"], max(_lengths(case)))
    g = _generator(seed * 8 + 5)
    w = torch.exp(2.5 * torch.randn(shape, generator=g, device="cuda") - (11 if case["kind"] == "mass" else 6))
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.02, torch.zeros_like(w), w)


def _logits(case, seed):
    """Rows of logits with a few likely tokens, and the tokens that are asked for."""
    T, V, g = case["tokens"], case["vocab"], _generator(seed * 8 + 6)
    x = torch.randn((T, V), generator=g, device="cuda") * 2.5
    likely = torch.randint(0, V, (T, 8), generator=g, device="cuda")
    x.scatter_add_(1, likely, 8 * torch.rand((T, 8), generator=g, device="cuda"))
    given = torch.randint(0, V, (T, case["given"]), generator=g, device="cuda")
    if case["given"]:
        given[:, 0] = torch.where(torch.arange(T, device="cuda") % 3 == 0, given[:, 0], likely[:, 0])
    return x, given.to(torch.int32)


_shared = {}


def _framework():
    """One context on one stream that torch uses too, as a program keeps it."""
    import nexus_amd as nx

    if not _shared:
        stream = torch.cuda.Stream()
        torch.cuda.set_stream(stream)
        ctx = nx.Context(0)
        ctx.set_stream(stream.cuda_stream)
        _shared.update(ctx=ctx, stream=stream)
    return nx, _shared["ctx"]


def prepare(case, seed):
    framework = _framework() if own else None
    kind = case["kind"]
    if kind == "logprobs":
        T, n, top = case["tokens"], case["given"], case["top"]
        logits, given = _logits(case, seed)
        state = {"case": case, "logits": logits, "given": given}
        if framework:
            state.update(ctx=framework[1], logprobs=torch.empty((T, n), device="cuda"),
                         entropy=torch.empty(T, device="cuda"),
                         top_ids=torch.empty((T, top), dtype=torch.int32, device="cuda"),
                         top_logprobs=torch.empty((T, top), device="cuda"))
        return state
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if kind == "rope":
        positions, freq = _angles(case, seed)
        state = {"case": case, "rows": _rows(case, seed), "positions": positions, "freq": freq}
        state["norms"] = _norms(case, seed) if case["norm"] else None
        if framework:
            nx, ctx = framework
            norms = [n.data_ptr() for n in state["norms"]] if case["norm"] else [0, 0]
            style = nx.ROPE_HALVES if case["style"] == "halves" else nx.ROPE_PAIRS
            state.update(ctx=ctx, rope=nx.Rope(D, case["rotary"], freq.data_ptr(), style, *norms, eps=1e-6),
                         q=torch.empty((case["tokens"], H * D), device="cuda"),
                         k=torch.empty((case["tokens"], G * D), device="cuda"))
        return state
    state = dict(_tables(case, seed), case=case, weights=_weights(case, seed))
    k, v = _context(case, seed)
    starts = torch.cat([state["kv_len"].new_zeros(1), state["kv_len"].cumsum(0)]).to(torch.int32)
    if kind == "mass":
        state["rows"] = _rows(case, seed)
    else:
        ends = [0]
        for n in _kept(case):
            ends.append(ends[-1] + n)
        state["to_start"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        state["count"] = ends[-1]
    if framework:
        nx, ctx = framework
        fmt = nx.KV_F16 if case["fmt"] == "f16" else nx.KV_INT8
        state["cache"] = cache = nx.KvCache(ctx, fmt, state["pool"], case["page"], G, D)

        def batch(rows, starts, lengths, pages):
            return nx.KvBatch(case["seqs"], rows, pages.shape[1], starts.data_ptr(), lengths.data_ptr(),
                              pages.data_ptr())

        cache.write_dev(batch(len(k), starts, state["kv_len"], state["pages"]), k.data_ptr(), v.data_ptr(), G * D)
        state["batch"] = batch(sum(_new(case)), state["row_start"], state["kv_len"], state["pages"])
        if kind == "mass":
            state["mass"] = torch.zeros_like(state["weights"])
        else:
            shape = (case["seqs"], G, case["keep"])
            state.update(kept=torch.empty(shape, dtype=torch.int32, device="cuda"),
                         new_len=torch.empty_like(state["kv_len"]), mass=torch.zeros(shape, device="cuda"),
                         k=torch.empty((state["count"], G * D), device="cuda"),
                         v=torch.empty((state["count"], G * D), device="cuda"))
            state["to"] = batch(state["count"], state["to_start"], state["new_len"], state["to_pages"])
        torch.cuda.synchronize()
        return state
    for name in "kv":
        dtype = torch.float16 if case["fmt"] == "f16" else torch.int8
        state["pool_" + name] = torch.zeros((state["pool"] * case["page"], G, D), dtype=dtype, device="cuda")
        state["scale_" + name] = torch.zeros((state["pool"] * case["page"], G, 1), device="cuda")
    seq, place = _sequence_of(starts, len(k))
    at = _slot(state, state["pages"], seq, place)
    _store(state, "k", at, k)
    _store(state, "v", at, v)
    return state


# ---------------------------------------------------------------- the plain form
def _sequence_of(starts, count):
    """The sequence of each row, and the row's place among its sequence's rows."""
    row = torch.arange(count, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row.to(starts.dtype), right=True)
    return seq, row - starts[seq]


def _slot(state, pages, seq, at):
    page = state["case"]["page"]
    return pages[seq, at // page].long() * page + at % page


def _store(state, name, at, x):
    if state["case"]["fmt"] == "f16":
        state["pool_" + name][at] = x.to(torch.float16)
        return
    scale = (x.abs().amax(-1, keepdim=True).double() / 127.0).float()
    codes = torch.round(x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double())
    state["pool_" + name][at] = codes.to(torch.int8)
    state["scale_" + name][at] = scale


def _load(state, name, at):
    x = state["pool_" + name][at].float()
    return x if state["case"]["fmt"] == "f16" else x * state["scale_" + name][at]


def _rotate(state, x, norm):
    """Rows of heads [T, heads, D], normed and rotated."""
    case = state["case"]
    if norm is not None:
        x = x * (1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)) * norm
    R = case["rotary"]
    angle = state["positions"].double()[:, None, None] * state["freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    y = x.clone()
    first, second = ((slice(0, R // 2), slice(R // 2, R)) if case["style"] == "halves" else
                     (slice(0, R, 2), slice(1, R, 2)))
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., first] * sin + x[..., second] * cos
    return y


def _plain_rope(state):
    case, rows = state["case"], state["rows"]
    H, G, D, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    norms = state["norms"] if case["norm"] else (None, None)
    q = _rotate(state, rows[:, :H * D].reshape(T, H, D), norms[0])
    k = _rotate(state, rows[:, H * D:(H + G) * D].reshape(T, G, D), norms[1])
    return {"q": q.reshape(T, H * D), "k": k.reshape(T, G * D)}


def _plain_mass(state):
    case = state["case"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    S, n, T = case["seqs"], case["tokens"], state["rows"].shape[0]
    starts, length = state["row_start"], state["kv_len"][:, None]
    new = (starts[1:] - starts[:-1])[:, None]
    key = torch.arange(state["weights"].shape[2], device="cuda").expand(S, -1)
    at = _slot(state, state["pages"], torch.arange(S, device="cuda")[:, None], torch.minimum(key, length - 1))
    k = _load(state, "k", at).permute(0, 2, 3, 1).contiguous()
    place = torch.arange(n, device="cuda")[None, :]
    row = torch.minimum(starts[:-1, None] + place, starts[1:, None] - 1)
    q = state["rows"][:, :H * D].reshape(T, G, H // G, D)[row] / math.sqrt(D)
    q = q.permute(0, 2, 1, 3, 4).reshape(S, G, n * (H // G), D).contiguous()
    scores = torch.matmul(q, k).reshape(S, G, n, H // G, -1)
    query = (length - new + place)[:, :, None]
    seen = (key[:, None, :] <= query) & (place[:, :, None] < new[:, :, None])
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    p = p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    before = torch.where((key < length - new)[:, None, :], state["weights"], torch.zeros_like(state["weights"]))
    return before + p.sum((2, 3))


def _plain_evict(state):
    case, w, length = state["case"], state["weights"], state["kv_len"]
    S, G, L = w.shape
    keep, key = case["keep"], torch.arange(L, device="cuda")
    last = torch.minimum(length, length.new_full((), keep))[:, None]
    always = (key < case["sinks"]) | (key >= length[:, None] - case["recent"])
    w = w.masked_fill(always[:, None], math.inf).masked_fill((key >= length[:, None])[:, None], -math.inf)
    # the heaviest first, of equal ones the lower; then in their own order
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    place = torch.arange(order.shape[-1], device="cuda")
    behind = (place >= last)[:, None]
    kept = torch.sort(order.masked_fill(behind, L), dim=-1).values
    full = torch.full((S, G, keep), -1, dtype=torch.int32, device="cuda")
    full[..., :order.shape[-1]] = kept.masked_fill(behind, -1)
    mass = torch.zeros((S, G, keep), device="cuda")
    picked = torch.gather(state["weights"], 2, kept.clamp(max=L - 1))
    mass[..., :order.shape[-1]] = picked.masked_fill(behind, 0.0)
    # the kept tokens in their new pages, and back
    seq, place = _sequence_of(state["to_start"], state["count"])
    head = torch.arange(G, device="cuda")
    old = _slot(state, state["pages"], seq[:, None], kept[seq[:, None], head, place[:, None]])
    new = _slot(state, state["to_pages"], seq, place)
    out = {"kept": full, "new_len": last[:, 0], "mass": mass}
    for name in "kv":
        for pool in ("pool_", "scale_")[:1 if case["fmt"] == "f16" else 2]:
            state[pool + name][new] = state[pool + name][old, head]
        out[name] = _load(state, name, new).reshape(state["count"], -1)
    return out


def _plain_logprobs(state):
    case, x = state["case"], state["logits"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    norm = top + torch.log(total)
    entropy = torch.log(total[:, 0]) - (e * (x - top)).sum(-1) / total[:, 0]
    ids = given = state["given"].long()
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ids = ids[:, :case["top"]]
    return {"logprobs": torch.gather(x, 1, given) - norm, "entropy": entropy,
            "top_ids": ids.to(torch.int32), "top_logprobs": torch.gather(x, 1, ids) - norm}


# ---------------------------------------------------------------- the call
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"rope": _plain_rope, "mass": _plain_mass, "evict": _plain_evict,
                "logprobs": _plain_logprobs}[kind](state)
    if kind == "logprobs":
        state["ctx"].logprobs_dev(state["logits"].data_ptr(), state["logits"].stride(0), case["tokens"], case["vocab"],
                                  state["given"].data_ptr(), case["given"], state["logprobs"].data_ptr(),
                                  state["entropy"].data_ptr(), case["top"], state["top_ids"].data_ptr(),
                                  state["top_logprobs"].data_ptr())
        return {name: state[name] for name in ("logprobs", "entropy", "top_ids", "top_logprobs")}
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if kind == "rope":
        rows = state["rows"]
        q, k = rows[:, :H * D], rows[:, H * D:(H + G) * D]
        state["ctx"].qk_rope_dev(state["rope"], state["positions"].data_ptr(), case["tokens"], H, G, q.data_ptr(),
                                 q.stride(0), k.data_ptr(), k.stride(0), state["q"].data_ptr(), H * D,
                                 state["k"].data_ptr(), G * D)
        return {"q": state["q"], "k": state["k"]}
    w, cache = state["weights"], state["cache"]
    if kind == "mass":
        rows = state["rows"]
        cache.attention_mass_dev(state["batch"], rows.data_ptr(), rows.stride(0), H, w.data_ptr(),
                                 state["mass"].data_ptr(), w.shape[2], 1.0 / math.sqrt(D))
        return state["mass"]
    cache.evict_dev(state["batch"], state["to_pages"].data_ptr(), state["to_pages"].shape[1], case["keep"],
                    case["sinks"], case["recent"], w.data_ptr(), w.shape[2], state["kept"].data_ptr(),
                    state["new_len"].data_ptr(), state["mass"].data_ptr(), case["keep"])
    cache.read_dev(state["to"], state["k"].data_ptr(), state["v"].data_ptr(), G * D)
    return {name: state[name] for name in ("kept", "new_len", "mass", "k", "v")}


# ---------------------------------------------------------------- in 64 bits
def _stored(case, x):
    """What the cache holds of x, in 64 bits."""
    if case["fmt"] == "f16":
        return x.half().double()
    x = x.double()
    scale = (x.abs().max(-1, keepdim=True).values / 127).float().double()
    return torch.round(x / scale) * scale


def _exact_rope(case, seed):
    H, G, D, T, R = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["rotary"]
    positions, freq = _angles(case, seed)
    rows = _rows(case, seed)[:, :(H + G) * D].double().reshape(T, H + G, D)
    if case["norm"]:
        norms = _norms(case, seed).double()
        weight = torch.cat([norms[:1].expand(H, D), norms[1:].expand(G, D)])
        rows = rows / (rows.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * weight
    turn = torch.polar(torch.ones((T, R // 2), dtype=torch.float64, device="cuda"),
                       torch.outer(positions.double(), freq.double()))[:, None, :]
    part = rows[..., :R]
    if case["style"] == "pairs":
        turned = torch.view_as_real(torch.view_as_complex(part.reshape(T, H + G, R // 2, 2).contiguous()) * turn)
    else:
        turned = torch.view_as_real(torch.complex(part[..., :R // 2].contiguous(),
                                                  part[..., R // 2:].contiguous()) * turn).transpose(-1, -2)
    out = torch.cat([turned.reshape(T, H + G, R), rows[..., R:]], -1)
    return {"q": out[:, :H].reshape(T, H * D), "k": out[:, H:].reshape(T, G * D)}


def _exact_mass(case, seed):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    k, _ = _context(case, seed)
    rows, out = _rows(case, seed), torch.zeros_like(_weights(case, seed), dtype=torch.float64)
    before, row, at = _weights(case, seed).double(), 0, 0
    for s, (n, length) in enumerate(zip(_new(case), _lengths(case))):
        position = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = torch.arange(length, device="cuda")[None, :] > position
        out[s, :, :length - n] = before[s, :, :length - n]
        for h in range(H):
            ks = _stored(case, k[at:at + length, h * G // H]).t().contiguous()
            x = torch.mm(rows[row:row + n, h * D:(h + 1) * D].double().contiguous(), ks) / math.sqrt(D)
            x[hidden] = -math.inf
            out[s, h * G // H, :length] += torch.softmax(x, 1).sum(0)
        row, at = row + n, at + length
    return out


def _exact_evict(case, seed):
    k, v = _context(case, seed)
    w, lengths, keep = _weights(case, seed), _lengths(case), case["keep"]
    S, G = w.shape[:2]
    kept = torch.full((S, G, keep), -1, dtype=torch.int32, device="cuda")
    mass, rows, at = torch.zeros((S, G, keep), dtype=torch.float64, device="cuda"), {"k": [], "v": []}, 0
    for s, length in enumerate(lengths):
        n, sinks = min(length, keep), min(case["sinks"], length)
        recent = min(case["recent"], length - sinks)
        middle = torch.arange(sinks, length - recent, device="cuda")
        for g in range(G):
            # the heaviest of the middle, of equal ones the lower
            value, index = w[s, g, middle].cpu().numpy(), middle.cpu().numpy()
            chosen = index[(-value).argsort(kind="stable")][:max(n - sinks - recent, 0)]
            ids = torch.cat([torch.arange(sinks), torch.from_numpy(chosen).sort().values,
                             torch.arange(length - recent, length)])[:n].cuda()
            kept[s, g, :n] = ids.to(torch.int32)
            mass[s, g, :n] = w[s, g, ids].double()
        ids = kept[s, :, :n].long()
        for name, x in (("k", k), ("v", v)):
            own_rows = torch.stack([x[at + ids[g], g] for g in range(G)], 1)
            rows[name].append(_stored(case, own_rows).reshape(n, -1))
        at += length
    new_len = torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device="cuda")
    return {"kept": kept, "new_len": new_len, "mass": mass, "k": torch.cat(rows["k"]), "v": torch.cat(rows["v"])}


def _exact_logprobs(case, seed):
    x, given = _logits(case, seed)
    T, top = case["tokens"], min(case["top"], case["vocab"])
    out = {"logprobs": torch.empty((T, case["given"]), dtype=torch.float64, device="cuda"),
           "entropy": torch.empty(T, dtype=torch.float64, device="cuda"),
           "top_ids": torch.empty((T, top), dtype=torch.int32, device="cuda"),
           "top_logprobs": torch.empty((T, top), dtype=torch.float64, device="cuda")}
    step = max(1, (1 << 26) // case["vocab"])
    for t in range(0, T, step):
        rows = slice(t, min(t + step, T))
        logp = torch.log_softmax(x[rows].double(), -1)
        out["logprobs"][rows] = logp.gather(1, given[rows].long())
        out["entropy"][rows] = -(logp.exp() * logp).sum(-1)
        left, ids = x[rows].clone(), torch.arange(case["vocab"], device="cuda")
        for i in range(top):  # the largest, of equal ones the lowest
            best = torch.where(left == left.amax(-1, keepdim=True), ids, case["vocab"]).amin(-1, keepdim=True)
            out["top_ids"][rows, i] = best[:, 0].to(torch.int32)
            out["top_logprobs"][rows, i] = logp.gather(1, best)[:, 0]
            left.scatter_(1, best, -math.inf)
    return out


def exact(case, seed):
    return {"rope": _exact_rope, "mass": _exact_mass, "evict": _exact_evict,
            "logprobs": _exact_logprobs}[case["kind"]](case, seed)
