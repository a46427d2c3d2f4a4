"""The paged key/value cache and the attention that reads it, as cases to time
and compare.

A case is one pass of one operator, as a decoder layer makes it between its
q/k/v and its output projections:

* "cache": the new tokens' keys and values are written into the pages of their
  sequences, quantised to the cache's format, and read back (a prefix that is
  checked, moved or swapped out);
* "attention": the new tokens attend over their sequences' pages, causally;
* "window": the same with a sliding window and a few first tokens that stay
  visible.

Rows are f32, as the projections give and take them; q, k and v lie side by
side in the rows of one fused projection.  A cache holds f16 values, or 8-bit
codes with one f32 scale per token and head: scale = max |x| / 127, code = x /
scale rounded to nearest, ties to even.

`own` chooses the framework's calls; otherwise run() computes the same in
elementary torch operations in 32 bits (the codes' borders in 64).
"""
import math

import torch

own = False

# heads, key/value heads and width of a head: the attention shapes of the
# repository's model configurations, and generic ones
HEADS = {"mixtral": (32, 8, 128), "qwen3": (32, 4, 128), "small": (16, 2, 64),
         "wide": (16, 8, 256), "full": (12, 12, 96), "single": (24, 1, 128)}


def _case(kind, fmt, shape, seqs, tokens, ctx, page=64, window=0, sinks=0, mixed=False):
    heads, kv_heads, dim = HEADS[shape]
    return dict(kind=kind, fmt=fmt, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, tokens=tokens,
                ctx=ctx, page=page, window=window, sinks=sinks, mixed=mixed)


def listed():
    cases = {
        # one sequence's next token: latency
        "cache_f16_1": _case("cache", "f16", "mixtral", 1, 1, 517),
        # the next tokens of a running batch
        "cache_int8_batch": _case("cache", "int8", "mixtral", 61, 1, 3001),
        # a long prompt's chunk enters the cache behind an earlier one
        "cache_int8_prompt": _case("cache", "int8", "qwen3", 2, 8191, 12287, page=32),
        # one decode step of one short sequence: latency
        "attn_f16_1": _case("attention", "f16", "mixtral", 1, 1, 517),
        # a decode step of a serving batch, contexts of all lengths
        "attn_f16_batch": _case("attention", "f16", "mixtral", 61, 1, 8191),
        # a few long documents
        "attn_int8_long": _case("attention", "int8", "mixtral", 3, 1, 131071, page=128),
        # a prompt from its first token on
        "attn_f16_prompt": _case("attention", "f16", "mixtral", 1, 4093, 4093),
        # a chunk of a prompt whose earlier chunks are in the cache
        "attn_int8_chunk": _case("attention", "int8", "qwen3", 2, 509, 16127, page=32),
        # decoding sequences and one prompt's chunk in the same step
        "attn_f16_mixed": _case("attention", "f16", "mixtral", 17, 257, 2047, mixed=True),
        # a decode step of long sequences that see their last 1024 tokens
        "window_int8_batch": _case("window", "int8", "mixtral", 29, 1, 32749, window=1024, sinks=4),
        # one sequence of narrow heads and a short window: latency
        "window_f16_1": _case("window", "f16", "small", 1, 1, 5003, window=128, sinks=4),
        # a chunk of a long prompt
        "window_f16_chunk": _case("window", "f16", "mixtral", 1, 2039, 20011, window=4096, sinks=8),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """A decode step or a prompt's chunk of any of the shapes, kinds and formats,
    within the largest listed cases' work and memory."""
    while True:
        kind = rng.choice(("cache", "attention", "attention", "window"))
        step = rng.random() < 0.5
        seqs = _log_int(rng, 1, 96) if step else _log_int(rng, 1, 4)
        tokens = rng.choice((1, 1, 2, 3, 5)) if step else _log_int(rng, 6, 4096)
        case = _case(kind, rng.choice(("f16", "int8")), rng.choice(sorted(HEADS)), seqs, tokens,
                     max(tokens, _log_int(rng, 1, 100000)), page=rng.choice((32, 64, 128, 256)))
        if kind == "window":
            case.update(window=_log_int(rng, 1, 8192), sinks=rng.choice((0, 1, 4, 7, 64)))
        if kind == "attention" and tokens > 8 and rng.random() < 0.3:
            case.update(seqs=rng.randint(2, 24), mixed=True)
        scores = case["seqs"] * tokens * case["heads"] * _span(case)
        values = case["seqs"] * max(_span(case), tokens) * case["kv_heads"] * case["dim"]
        pool = case["seqs"] * (case["ctx"] + 256) * case["kv_heads"] * case["dim"]
        if scores > 6e8 or values > 5e8 or pool > 5e8:
            continue
        cost = work(case)
        if cost["bytes"] <= 1.2e9 and cost["flops"] <= 2e11:
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


def _span(case):
    """The most keys that one sequence's new tokens see."""
    if not case["window"]:
        return case["ctx"]
    return min(case["ctx"], case["window"] + case["tokens"] - 1 + case["sinks"])


def _pairs_and_keys(case):
    """(query, key) pairs that are visible, and keys that are read, over all sequences."""
    pairs = keys = 0
    for n, length in zip(_new(case), _lengths(case)):
        w, f = case["window"] or length, case["sinks"] if case["window"] else 0
        for p in range(length - n, length):
            pairs += min(p + 1, w + min(f, max(0, p + 1 - w)))
        first = max(0, length - n - w + 1)
        keys += length - first + min(f, first)
    return pairs, keys


def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    T = sum(_new(case))
    stored = G * (2 * D if case["fmt"] == "f16" else D + 4)  # bytes of one token's keys
    if case["kind"] == "cache":
        return {"bytes": 2 * T * (4 * G * D + 2 * stored + 4 * G * D), "flops": 4 * T * G * D}
    pairs, keys = _pairs_and_keys(case)
    return {"bytes": 2 * keys * stored + 8 * T * H * D, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(case, seed):
    """First row, length and pages of each sequence: its pages are anywhere in the pool."""
    lengths, rows = _lengths(case), [0]
    for n in _new(case):
        rows.append(rows[-1] + n)
    width = -(-max(lengths) // case["page"])
    order = torch.randperm(case["seqs"] * width + 3, generator=_generator(seed * 8 + 1), device="cuda")
    return {"row_start": torch.tensor(rows, dtype=torch.int32, device="cuda"),
            "kv_len": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            "pages": order[:case["seqs"] * width].to(torch.int32).reshape(case["seqs"], width)}


def _context(case, seed):
    """Keys and values of every token of the sequences, one sequence behind the
    other: a few channels of the keys are larger than the others."""
    g = _generator(seed * 8 + 2)
    total = sum(_lengths(case)) if case["kind"] != "cache" else sum(_new(case))
    shape = (total, case["kv_heads"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda")
    k[:, :, ::29] *= 3.0
    return k, torch.randn(shape, generator=g, device="cuda")


def _rows(case, seed):
    """The fused projection's rows: q, then k, then v."""
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    T = sum(_new(case))
    rows = torch.randn((T, (H + 2 * G) * D), generator=_generator(seed * 8 + 3), device="cuda")
    if case["kind"] == "cache":
        k, v = _context(case, seed)
        rows[:, H * D:(H + G) * D] = k.reshape(T, G * D)
        rows[:, (H + G) * D:] = v.reshape(T, G * D)
    return rows


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
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    framework = _framework() if own else None
    state = dict(_tables(case, seed), case=case, rows=_rows(case, seed))
    T = state["rows"].shape[0]
    if case["kind"] == "cache":
        state["k"] = torch.empty((T, G * D), device="cuda")
        state["v"] = torch.empty((T, G * D), device="cuda")
    else:
        state["out"] = torch.empty((T, H * D), device="cuda")
    pool = state["pages"].numel() + 3
    filled = case["kind"] != "cache"
    if filled:  # the whole sequences are in the cache when the step attends
        k, v = _context(case, seed)
        starts = torch.cat([state["kv_len"].new_zeros(1), state["kv_len"].cumsum(0)]).to(torch.int32)
    if framework:
        nx, ctx = framework
        fmt = nx.KV_F16 if case["fmt"] == "f16" else nx.KV_INT8
        state["cache"] = cache = nx.KvCache(ctx, fmt, pool, case["page"], G, D)
        state["batch"] = nx.KvBatch(case["seqs"], T, state["pages"].shape[1], state["row_start"].data_ptr(),
                                    state["kv_len"].data_ptr(), state["pages"].data_ptr())
        if filled:
            whole = nx.KvBatch(case["seqs"], len(k), state["pages"].shape[1], starts.data_ptr(),
                               state["kv_len"].data_ptr(), state["pages"].data_ptr())
            cache.write_dev(whole, k.data_ptr(), v.data_ptr(), G * D)
            torch.cuda.synchronize()
        return state
    for name in "kv":
        dtype = torch.float16 if case["fmt"] == "f16" else torch.int8
        state["pool_" + name] = torch.zeros((pool * case["page"], G, D), dtype=dtype, device="cuda")
        state["scale_" + name] = torch.zeros((pool * case["page"], G, 1), device="cuda")
    if filled:
        at = _slots(state, starts, len(k))
        _store(state, "k", at, k)
        _store(state, "v", at, v)
    return state


# ---------------------------------------------------------------- the plain form
def _sequence_of(starts, count):
    """The sequence of each row, and the row's place among its sequence's rows."""
    row = torch.arange(count, device="cuda")
    seq = (row[:, None] >= starts[None, 1:]).sum(1)
    return seq, row - starts[seq]


def _slots(state, starts, count):
    """The pool slot of each row: the rows are their sequences' last tokens."""
    seq, place = _sequence_of(starts, count)
    at = state["kv_len"][seq] - (starts[seq + 1] - starts[seq]) + place
    return _slot(state, seq, at)


def _slot(state, seq, at):
    page = state["case"]["page"]
    return state["pages"][seq, at // page].long() * page + at % page


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


def _attend(state):
    case = state["case"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    S, n, T = case["seqs"], case["tokens"], state["rows"].shape[0]
    starts, length = state["row_start"], state["kv_len"][:, None]
    new = (starts[1:] - starts[:-1])[:, None]
    # keys that may be seen: everything, or the first ones and what the windows span
    if case["window"]:
        first = torch.clamp(length - new - case["window"] + 1, min=case["sinks"])
        spans = first + torch.arange(_span(case), device="cuda")
        sinks = torch.arange(case["sinks"], device="cuda").expand(S, -1)
        key = torch.cat([sinks, spans], 1)
    else:
        key = torch.arange(_span(case), device="cuda").expand(S, -1)
    at = _slot(state, torch.arange(S, device="cuda")[:, None], torch.minimum(key, length - 1))
    k = _load(state, "k", at).permute(0, 2, 3, 1).contiguous()
    v = _load(state, "v", at).permute(0, 2, 1, 3).contiguous()
    place = torch.arange(n, device="cuda")[None, :]
    row = torch.minimum(starts[:-1, None] + place, starts[1:, None] - 1)
    q = state["rows"][:, :H * D].reshape(T, G, H // G, D)[row] / math.sqrt(D)
    q = q.permute(0, 2, 1, 3, 4).reshape(S, G, n * (H // G), D).contiguous()
    scores = torch.matmul(q, k).reshape(S, G, n, H // G, -1)
    query = (length - new + place)[:, :, None]
    seen = (key[:, None, :] <= query) & (key[:, None, :] < length[:, :, None])
    if case["window"]:
        seen &= (key[:, None, :] > query - case["window"]) | (key[:, None, :] < case["sinks"])
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1).reshape(S, G, n * (H // G), 1)
    out = torch.matmul(p.reshape(S, G, n * (H // G), -1), v) / total
    out = out.reshape(S, G, n, H // G, D).permute(0, 2, 1, 3, 4).reshape(S, n, H * D)
    return out[_sequence_of(starts, T)]


# ---------------------------------------------------------------- the call
def run(state):
    case, rows = state["case"], state["rows"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "cache":
        k, v = rows[:, H * D:(H + G) * D], rows[:, (H + G) * D:]
        if own:
            state["cache"].write_dev(state["batch"], k.data_ptr(), v.data_ptr(), rows.stride(0))
            state["cache"].read_dev(state["batch"], state["k"].data_ptr(), state["v"].data_ptr(), G * D)
            return {"k": state["k"], "v": state["v"]}
        at = _slots(state, state["row_start"], len(rows))
        _store(state, "k", at, k.reshape(-1, G, D))
        _store(state, "v", at, v.reshape(-1, G, D))
        return {"k": _load(state, "k", at).reshape(-1, G * D), "v": _load(state, "v", at).reshape(-1, G * D)}
    if own:
        state["cache"].attention_dev(state["batch"], rows.data_ptr(), rows.stride(0), H, state["out"].data_ptr(),
                                     H * D, 1.0 / math.sqrt(D), window=case["window"], sinks=case["sinks"])
        return state["out"]
    return _attend(state)


# ---------------------------------------------------------------- in 64 bits
def _stored(case, x):
    """What the cache holds of x, in 64 bits."""
    if case["fmt"] == "f16":
        return x.half().double()
    x = x.double()
    scale = (x.abs().max(-1, keepdim=True).values / 127).float().double()
    return torch.round(x / scale) * scale


def exact(case, seed):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    k, v = _context(case, seed)
    if case["kind"] == "cache":
        return {"k": _stored(case, k).reshape(-1, G * D), "v": _stored(case, v).reshape(-1, G * D)}
    rows, outs, row, at = _rows(case, seed), [], 0, 0
    for n, length in zip(_new(case), _lengths(case)):
        q = rows[row:row + n, :H * D].double().reshape(n, H, D)
        position = torch.arange(length - n, length, device="cuda")[:, None]
        # only the keys that some query sees
        keep = torch.arange(length, device="cuda")
        if case["window"]:
            keep = keep[(keep < case["sinks"]) | (keep > length - n - case["window"])]
        seen = keep[None, :] <= position
        if case["window"]:
            seen &= (position - keep[None, :] < case["window"]) | (keep[None, :] < case["sinks"])
        out = torch.empty_like(q)
        for g in range(G):
            ks, vs = _stored(case, k[at + keep, g]), _stored(case, v[at + keep, g])
            for h in range(g * (H // G), (g + 1) * (H // G)):
                s = torch.mm(q[:, h].contiguous(), ks.t().contiguous()) / math.sqrt(D)
                s[~seen] = -math.inf
                out[:, h] = torch.mm(torch.softmax(s, 1), vs)
        outs.append(out.reshape(n, H * D))
        row, at = row + n, at + length
    return torch.cat(outs)
