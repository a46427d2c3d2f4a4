"""The calls around the cache (nx_kv_evict, nx_attention_mass, nx_logprobs, nx_qk_rope) at the edges of
what they accept, against formulas in 64 bits."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, INT8, Batch, random_kv, stored
from moe_cases import DeviceArray, assert_same_bits
from step_cases import HALVES, PAIRS, rope
from test_gpu_evict import Case
from test_gpu_kv import device_batch
from test_gpu_step import Hip

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


# ---------------------------------------------------------------- eviction
@pytest.mark.parametrize("fmt", FORMATS)
def test_first_kept_tokens_of_a_group(ctx, fmt):
    """The first two tokens of a new group out of one chunk of eight, the first chunk and later
    ones, or out of two."""
    pairs = [(0, 1), (0, 7), (7, 8), (0, 8), (8, 9), (9, 15), (15, 16), (3, 17), (24, 31), (31, 32), (40, 47), (40, 48),
             (32, 33), (47, 90), (200, 201), (207, 208)]
    G, keep = len(pairs), 40
    c = Case(ctx, np.random.default_rng(21), fmt, [300], 32, G, 64, keep)
    c.mass[:] /= c.mass.max() * 2
    for g, (a, b) in enumerate(pairs):
        # the pair, and 38 tokens that follow it; in every other head as the second group's first
        first = [a, b] + [b + 1 + i + i // 3 for i in range(38)]
        if g % 2:
            first = [a, b] + list(range(260, 298))
        c.mass[0, g, first] += 1
    got = c.cache.evict(c.b.kv_len, c.b.pages, c.to, keep, c.mass)
    for g, pair in enumerate(pairs):
        assert tuple(got[0][0, g, :2]) == pair
    c.check(got, 0, 0)
    # and with 32 tokens before them
    lead = np.full((1, G, 332), 1, np.float32)
    lead[0, :, 32:] = c.mass[0] * np.float32(0.25)
    c.cache.close()
    c = Case(ctx, np.random.default_rng(22), fmt, [332], 32, G, 64, 72)
    c.mass = lead
    got = c.cache.evict(c.b.kv_len, c.b.pages, c.to, 72, c.mass, 32, 0)
    for g, (a, b) in enumerate(pairs):
        assert tuple(got[0][0, g, 32:34]) == (a + 32, b + 32)
    c.check(got, 32, 0)
    c.cache.close()


@pytest.mark.parametrize("lens", [[300, 40], [300, 40, 0], [60, 300]])
@pytest.mark.parametrize("fmt", FORMATS)
def test_host_weights_that_end_with_the_last_token(ctx, fmt, lens):
    """Rows of weights as far apart as the longest sequence is long, in memory that ends with the last
    sequence's last weight: the host calls' results are those of whole rows.  What lies behind may be
    the same call's new weights."""
    G, heads, D, keep, stride = 2, 4, 64, 37, 311
    rng = np.random.default_rng(23)
    c = Case(ctx, rng, fmt, lens, 32, G, D, keep)
    S, last = len(lens), max(s for s, n in enumerate(lens) if n)
    end = (last * G + G - 1) * stride + lens[last]
    rows = np.full((S, G, stride), np.nan, np.float32)
    rows[:, :, :max(lens)] = c.mass
    whole = c.cache.evict(c.b.kv_len, c.b.pages, c.to, keep, c.mass, 2, 3)
    memory = np.full(end + S * G * keep, 7, np.float32)
    exact, moved = memory[:end], memory[end:].reshape(S, G, keep)
    exact[:] = rows.ravel()[:end]
    L, kept, new_len = nx.lib(), np.zeros((S, G, keep), np.int32), np.zeros(S, np.int32)
    b, hold = c.cache._host_batch(np.zeros(S + 1), c.b.kv_len, c.b.pages, 0)
    nx.check(L.nx_kv_evict(ctx.h, c.cache.h, b.ref, c.to.ctypes.data, c.to.shape[1], keep, 2, 3, exact.ctypes.data, stride,
                           kept.ctypes.data, new_len.ctypes.data, moved.ctypes.data, keep))
    assert np.array_equal(kept, whole[0]) and np.array_equal(new_len, whole[1])
    for s in range(S):
        assert_same_bits(moved[s, :, :new_len[s]], whole[2][s, :, :new_len[s]])
    # a new token of each sequence that has any
    starts = np.concatenate([[0], np.cumsum(np.minimum(lens, 1))]).astype(np.int32)
    q = rng.standard_normal((starts[-1], heads, D), dtype=np.float32)
    want = c.cache.attention_mass(starts, c.b.kv_len, c.b.pages, q, heads, before=np.nan_to_num(rows, nan=7))
    b, hold = c.cache._host_batch(starts, c.b.kv_len, c.b.pages, len(q))
    got = exact.copy()
    nx.check(L.nx_attention_mass(ctx.h, c.cache.h, b.ref, q.ctypes.data, heads * D, heads, D ** -0.5, got.ctypes.data,
                                 got.ctypes.data, stride))
    got = np.append(got, np.full(rows.size - end, 7, np.float32)).reshape(rows.shape)
    for s, n in enumerate(lens):
        assert_same_bits(got[s, :, :n], want[s, :, :n])
    c.cache.close()


# ---------------------------------------------------------------- gathered weights
def mass_by_rows(b, keys, q, heads, scale, before=None):
    """mass [seqs x G x width], a bound, and which tokens get NaNs, of keys and queries that may hold
    anything: the formula in 64 bits row by row.  A row with a NaN or +infinity among its scores gives
    NaNs to the tokens that it sees; a score of -infinity is a token of no weight.

    The bound is step_cases.attention_mass's, whose magnitudes are those of finite terms: a score that is
    an infinity has no rounding."""
    G, D = keys.shape[1:]
    width = max(max(b.lens), 1)
    out = np.zeros((len(b.ns), G, width)) if before is None else before.astype(np.float64)
    bound, nan, at = np.zeros_like(out), np.zeros(out.shape, bool), 0
    U = 2.0 ** -24
    for s, (n, length) in enumerate(zip(b.ns, b.lens)):
        if n:
            out[s, :, length - n:length] = 0
        for i in range(n):
            p = length - n + i
            for h in range(heads):
                g = h * G // heads
                k = keys[at:at + p + 1, g].astype(np.float64)
                r = q[b.row_start[s] + i, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    terms = scale * (r * k)
                    x = terms.sum(1)
                    mag = np.where(np.isfinite(terms), np.abs(terms), 0).sum(1).max()
                if np.isnan(x).any() or (x == np.inf).any():
                    nan[s, g, :p + 1] = True
                    continue
                if (x == -np.inf).all():
                    continue
                w = np.exp(x - x.max())
                w /= w.sum()
                e = 2 * ((2.0 ** -21 + D * U) * mag + 2.0 ** -21)
                out[s, g, :p + 1] += w
                bound[s, g, :p + 1] += (2 * e + (length + 64) * U + 2 * U * (1.5 * mag + np.log2(length + 1))) * w
        bound[s] += (n * heads // G + 8) * U * out[s] + 2.0 ** -120
        at += length
    return out, bound, nan


def mass_of(ctx, b, fmt, k, q, heads, scale, before=None):
    """What the call gives, and the keys that its cache holds."""
    cache = nx.KvCache(ctx, fmt, b.num_pages, b.page_tokens, *k.shape[1:])
    cache.write(b.whole(), b.kv_len, b.pages, k, np.zeros_like(k))
    got = cache.attention_mass(*b.args(), q, heads, scale=scale, before=before)
    cache.close()
    return got, stored(fmt, k)


def check_mass(b, got, ref, bound, nan):
    for s, (n, length) in enumerate(zip(b.ns, b.lens)):
        if not n:
            continue
        g, r, o, bad = (a[s, :, :length] for a in (got, ref, bound, nan))
        assert np.array_equal(np.isnan(g), bad), (s, np.isnan(g).sum(1), bad.sum(1))
        off = np.abs(g.astype(np.float64) - r)[~bad]
        assert (off <= o[~bad]).all(), float((off / o[~bad]).max())


SHAPES = [
    (4, 1, 64, [1], [70]),
    (8, 2, 128, [3, 1, 0], [133, 40, 9]),
    (16, 2, 96, [1, 2], [500, 33]),
    (4, 2, 256, [2], [65]),
    (8, 2, 64, [40], [100]),          # tiles of many rows
    (24, 1, 128, [33, 1], [64, 300]),
    (4, 2, 96, [150], [300]),
    (4, 4, 256, [70, 2], [90, 80]),
]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_infinite_keys_that_no_row_gives_weight(ctx, heads, G, D, ns, lens, sign):
    """F16 keys above 65520 are infinities.  Where a query's element has the other sign the score is
    -infinity: the token has no weight, and the others what they have without it."""
    rng = np.random.default_rng(31 + D)
    b = Batch(rng, ns, lens, 32)
    k, _ = random_kv(rng, sum(lens), G, D)
    q = rng.standard_normal((b.rows, heads, D), dtype=np.float32)
    # elements whose halves differ in sign or not, of a short one and of one with no second half, and one
    # that is next to nothing beside the others
    q[..., 5] = -sign * np.abs(q[..., 5])
    q[..., 17] = -sign * np.float32(0.25)
    q[..., 40] = -sign * np.abs(q[..., 40]) * np.float32(1e-20)
    for at, d in ((0, 5), (3, 17), (7, 40), (20, 5), (31, 17)):
        k[at, :, d] = sign * np.float32(1e6)
    k[25, :, 5], k[25, :, 17], k[26, 0, 40] = sign * np.inf, sign * np.float32(65536), sign * np.inf
    before = rng.random((len(ns), G, max(lens)), dtype=np.float32) / 50
    got, keys = mass_of(ctx, b, F16, k, q, heads, D ** -0.5, before)
    assert np.isinf(keys).any()
    ref, bound, nan = mass_by_rows(b, keys, q, heads, D ** -0.5, before)
    assert not nan.any()
    check_mass(b, got, ref, bound, nan)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_keys_that_are_not_finite_under_any_query(ctx, fmt, heads, G, D, ns, lens):
    """Rows with a NaN or +infinity among their scores give NaNs to all tokens that they see, and
    only to those; the heads beside them, and rows before the token, are as ever."""
    rng = np.random.default_rng(32 + D)
    b = Batch(rng, ns, lens, 32)
    for bad in (np.inf, -np.inf, np.nan):
        k, _ = random_kv(rng, sum(lens), G, D)
        q = rng.standard_normal((b.rows, heads, D), dtype=np.float32)
        end = np.cumsum(lens)
        for s, n in enumerate(ns):  # among the step's own tokens, and before them
            k[end[s] - max(n, 1) // 2 - 1, G - 1, 9] = bad
        k[2, 0, 11] = bad
        q[0, 0, 11] = 0  # an infinity by nothing
        got, keys = mass_of(ctx, b, fmt, k, q, heads, 0.1)
        check_mass(b, got, *mass_by_rows(b, keys, q, heads, 0.1))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_queries_that_are_not_finite(ctx, fmt, heads, G, D, ns, lens):
    """A row's own NaN or infinity spoils all tokens that it sees, and no other row's; a row whose
    scores are all -infinity gives nothing."""
    rng = np.random.default_rng(33 + D)
    b = Batch(rng, ns, lens, 32)
    for bad in (np.inf, -np.inf, np.nan):
        k, _ = random_kv(rng, sum(lens), G, D)
        q = rng.standard_normal((b.rows, heads, D), dtype=np.float32)
        q[b.rows // 2, heads - 1, 3] = bad
        got, keys = mass_of(ctx, b, fmt, k, q, heads, 0.1)
        check_mass(b, got, *mass_by_rows(b, keys, q, heads, 0.1))
    k[..., 3] = np.abs(k[..., 3]) + 1
    q[b.rows // 2, heads - 1, 3] = -np.inf
    got, keys = mass_of(ctx, b, fmt, k, q, heads, 0.1)
    ref = mass_by_rows(b, keys, q, heads, 0.1)
    assert not ref[2].any()
    check_mass(b, got, *ref)


@pytest.mark.parametrize("heads,G,D,n,length,first", [
    (256, 32, 256, 1300, 1300, 268),  # slices of 508 rows, of which the first has 240
    (32, 8, 128, 2000, 2000, 0),
    (32, 4, 128, 37, 20000, 0),       # the keys shared out
    (32, 4, 128, 1, 20000, 0),
])
def test_infinite_keys_of_long_calls(ctx, heads, G, D, n, length, first):
    """Scores of 0, and -infinity for every 97th token: a row gives each of the others that it sees the
    same weight, whatever parts and slices it is worked out in.

    The bound is step_cases.attention_mass's with scores of no magnitude."""
    rng = np.random.default_rng(36)
    b = Batch(rng, [n], [length], 64, first_row=first)
    k, _ = random_kv(rng, length, G, D)
    k[:, :, 3] = 0
    k[5::97, :, 3] = np.inf
    q = np.zeros((b.rows, heads, D), np.float32)
    q[:, :, 3] = -rng.random((b.rows, heads), dtype=np.float32) - np.float32(1e-3)
    got, _ = mass_of(ctx, b, F16, k, q, heads, 0.1)
    finite = np.ones(length)
    finite[5::97] = 0
    sees = np.cumsum(finite)[length - n:]  # of each row
    group = heads // G
    each = np.zeros(length)
    each[length - n:] = group / sees
    total = np.cumsum(each[::-1])[::-1] * finite
    bound = (4 * 2.0 ** -21 + (length + 64 + 2 * np.log2(length + 1) + group * n + 8) * 2.0 ** -24) * total
    assert (np.abs(got[0] - total) <= bound).all()


@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_products_past_the_range_under_scores_within(ctx, heads, G, D, ns, lens):
    """INT8: a key's scale and a query's size whose product f32 does not hold, at elements that do not
    meet: the score is 0."""
    rng = np.random.default_rng(37 + D)
    b = Batch(rng, ns, lens, 32)
    k = np.zeros((sum(lens), G, D), np.float32)
    k[..., 0] = rng.standard_normal(k.shape[:2]) * 1e-20
    k[2::9, :, 0] = 0
    k[2::9, :, 1] = 3e38
    q = np.zeros((b.rows, heads, D), np.float32)
    q[..., 0] = rng.standard_normal(q.shape[:2]) * 1e20
    got, keys = mass_of(ctx, b, INT8, k, q, heads, 1.0)
    ref = mass_by_rows(b, keys, q, heads, 1.0)
    assert not ref[2].any()
    check_mass(b, got, *ref)


@pytest.mark.parametrize("up", [1e36, 1e33, 1e-33])
@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_sizes_that_meet_in_ordinary_scores(ctx, heads, G, D, ns, lens, up):
    """INT8 keys next to f32's largest under queries next to nothing, and the other way round; tokens of
    ordinary size among them."""
    rng = np.random.default_rng(39 + D)
    b = Batch(rng, ns, lens, 32)
    k, _ = random_kv(rng, sum(lens), G, D)
    k *= np.float32(up)
    k[4::11] *= np.float32(1 / up)
    q = rng.standard_normal((b.rows, heads, D), dtype=np.float32) * np.float32(1 / up)
    if up < 1:
        k[4::11] = 0  # (ordinary keys would leave the range)
    got, keys = mass_of(ctx, b, INT8, k, q, heads, 0.125)
    ref = mass_by_rows(b, keys, q, heads, 0.125)
    assert not ref[2].any()
    check_mass(b, got, *ref)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e29, 3e30, 1e33, 1e37])
@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_scores_far_below_zero(ctx, fmt, heads, G, D, ns, lens, size):
    """Rows whose scores are all of that size below 0: the highest takes all, and the only token of a
    row takes it, as with any other scores.

    Tokens differ by a thousandth or more, far above any rounding, so a weight is 0 or 1 and their sums
    are whole numbers, which f32 holds."""
    rng = np.random.default_rng(34 + D)
    b = Batch(rng, ns, lens, 32)
    # D terms of q k scale / D, q of one size and k of another
    k_size = 100.0 if fmt == F16 else 1e18
    k = np.empty((sum(lens), G, D), np.float32)
    at = 0
    for n in lens:
        for g in range(G):
            k[at:at + n, g] = (k_size * (1 + rng.permutation(n) / 50))[:, None]
        at += n
    q = np.full((b.rows, heads, D), -size / k_size * (1 / D), np.float32) * (1 + rng.random((b.rows, heads, 1), dtype=np.float32))
    got, keys = mass_of(ctx, b, fmt, k, q, heads, 1.0)
    want, at = np.zeros_like(got), 0
    for s, (n, length) in enumerate(zip(ns, lens)):
        for p in range(length - n, length):
            for g in range(G):
                want[s, g, keys[at:at + p + 1, g, 0].argmin()] += heads // G
        at += length
    assert np.array_equal(got, want)


@pytest.mark.parametrize("heads,G,D,ns,lens", SHAPES)
def test_low_scores_beside_infinite_ones(ctx, heads, G, D, ns, lens):
    """A finite score of any size has weight beside those of -infinity."""
    rng = np.random.default_rng(35 + D)
    b = Batch(rng, ns, lens, 32)
    k = np.full((sum(lens), G, D), np.inf, np.float32)
    at = 0
    for n in lens:
        k[at + n // 3] = 1
        at += n
    q = np.full((b.rows, heads, D), -1e32, np.float32)
    got, _ = mass_of(ctx, b, F16, k, q, heads, 1.0)
    want = np.zeros_like(got)
    for s, (n, length) in enumerate(zip(ns, lens)):
        want[s, :, length // 3] = heads // G * min(n, length - length // 3)
    assert np.array_equal(got, want)


# ---------------------------------------------------------------- rotation
@pytest.mark.parametrize("D", [64, 62, 256, 512])
@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-30])
def test_norm_of_heads_next_to_nothing(ctx, D, eps):
    """Heads of subnormal values, one of them even of the least, with an eps that does not cover them;
    heads of zeros, whose norm without eps is 0 / 0."""
    rng = np.random.default_rng(51)
    x = rng.standard_normal((7, 2, D)).astype(np.float32)
    for i, size in enumerate((1e-38, 1e-40, 1e-43, 1e-30, 1e-20, 1.0)):
        x[i] *= np.float32(size)
    x[2, 1] = 0
    x[2, 1, D // 2 + 1] = 2.0 ** -149
    x[6] = 0
    w, freq = (1 + rng.random(D)).astype(np.float32), np.linspace(1, 0.01, D // 2).astype(np.float32)
    for style in (HALVES, PAIRS):
        got, _ = ctx.qk_rope(np.arange(7), x, None, freq, style, w, None, eps)
        ref, bound = rope(np.arange(7), x, freq, style, w, eps)
        assert (np.abs(got[:6] - ref[:6]) <= bound[:6]).all()
        assert np.isnan(got[6]).all() if eps == 0 else not got[6].any()


# ---------------------------------------------------------------- log probabilities
def promised(value, spread):
    """What a log probability or an entropy may be off."""
    return 2.0 ** -20 * (1 + np.abs(value) + spread)


def on_rows(ctx, x, tokens):
    """logprobs_dev of device rows: the log probabilities of one token each, and the entropy."""
    T, V = x.shape
    d = DeviceArray(x.size)
    d.upload(x)
    dt, lp, ent = DeviceArray(T), DeviceArray(T), DeviceArray(T)
    dt.upload(np.asarray(tokens, np.int32).view(np.float32))
    ctx.logprobs_dev(d.ptr, V, T, V, dt.ptr, 1, lp.ptr, ent.ptr, 0, 0, 0)
    ctx.sync()
    return lp.download().astype(np.float64), ent.download().astype(np.float64)


@pytest.mark.parametrize("T,V", [(1, 1 << 26), (5, 1 << 23), (513, 262144)])
def test_flat_rows_of_many_logits(ctx, T, V):
    """One logit above V - 1 equal ones: every term rounds the same way, so a sum of many of them in
    f32 would be further off the more there are."""
    for low in np.linspace(-14, -0.25, 4) if T == 1 else [None]:
        c = np.float32([low] if T == 1 else np.linspace(-14, -0.25, T))
        x = np.empty((T, V), np.float32)
        x[:] = c[:, None]
        peak = (np.arange(T) * 7919) % V
        x[np.arange(T), peak] = 0
        lp, ent = on_rows(ctx, x, (peak + 1) % V)
        d = c.astype(np.float64)
        p = np.exp(d)
        S = 1 + (V - 1) * p
        want = d - np.log(S)
        spread = (V - 1) * p / S * -d
        for name, got, ref in (("logprobs", lp, want), ("entropy", ent, np.log(S) + spread)):
            off = np.abs(got - ref) / promised(ref, spread)
            assert (off <= 1).all(), (name, off.max(), c[off.argmax()])


@pytest.mark.parametrize("T,V", [(1, 1 << 24), (513, 100003)])
@pytest.mark.parametrize("rise", [0.75, 40.0])
def test_rising_rows_of_many_logits(ctx, T, V, rise):
    """The largest logit so far moves on with every step."""
    row = np.linspace(-rise, 0, V).astype(np.float32)
    lp, ent = on_rows(ctx, np.broadcast_to(row, (T, V)), np.arange(T))
    d = row.astype(np.float64)
    p = np.exp(d)
    S, spread = p.sum(), (p * -d).sum() / p.sum()
    for got, ref in ((lp, d[:T] - np.log(S)), (ent, np.log(S) + spread)):
        off = np.abs(got - ref) / promised(ref, spread)
        assert (off <= 1).all(), off.max()


def test_workspace_of_few_long_rows_under_capture():
    """Calls of more or shorter rows do not allocate what few long rows take: the first of those is
    refused while the stream is captured, the others are not, and after one outside it is taken."""
    hip = Hip()
    rng = np.random.default_rng(41)
    shapes = [(600, 4097), (512, 4096), (512, 4097), (3, 9000)]
    with nx.Context(0) as ctx:
        stream = hip.stream()
        ctx.set_stream(stream.value)
        x = rng.standard_normal(600 * 4097).astype(np.float32)
        d, ent = DeviceArray(x.size), DeviceArray(600)
        d.upload(x)

        def call(T, V):
            ctx.logprobs_dev(d.ptr, V, T, V, 0, 0, 0, ent.ptr, 0, 0, 0)

        for warm in (False, True):
            for T, V in shapes[:2] + shapes[2:] * warm:
                call(T, V)
            ctx.sync()
            refused = []

            def calls():
                for shape in shapes[:2] + shapes[2:] * (not warm):
                    try:
                        call(*shape)
                    except nx.NexusError as e:
                        refused.append((shape, e.code))
                if warm:
                    call(*shapes[3])

            g, graph = hip.graph(stream, calls)
            assert refused == ([] if warm else [(s, nx.NX_ERR_UNSUPPORTED) for s in shapes[2:]])
            for _ in range(3):
                ent.upload(np.zeros(600))
                hip.hipGraphLaunch(graph, stream)
                ctx.sync()
                T, V = shapes[3] if warm else shapes[1]
                rows = x[:T * V].reshape(T, V).astype(np.float64)
                p = np.exp(rows - rows.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                ref, spread = -(p * np.log(p)).sum(1), (p * (rows.max(1, keepdims=True) - rows)).sum(1)
                assert (np.abs(ent.download()[:T] - ref) <= promised(ref, spread)).all()
            hip.hipGraphExecDestroy(graph)
            hip.hipGraphDestroy(g)
        ctx.set_stream(None)
        hip.hipStreamDestroy(stream)


@pytest.mark.parametrize("ns,lens", [([2, 1], [70, 40]), ([60, 1], [300, 40])])
def test_infinite_keys_in_a_graph(ns, lens):
    """What is done by the formula is replayed with the rest, whatever eager calls come between."""
    hip = Hip()
    rng = np.random.default_rng(38)
    heads, G, D = 8, 2, 64
    b = Batch(rng, ns, lens, 32)
    k, v = random_kv(rng, sum(lens), G, D)
    k[9, :, 7] = np.inf
    q = rng.standard_normal((2, b.rows, heads, D), dtype=np.float32)
    q[..., 7] = -np.abs(q[..., 7])
    with nx.Context(0) as ctx:
        cache = nx.KvCache(ctx, F16, b.num_pages, 32, G, D)
        cache.write(b.whole(), b.kv_len, b.pages, k, v)
        want = [cache.attention_mass(*b.args(), x, heads) for x in q]
        assert all(np.isfinite(w).all() for w in want)
        stream, d, dq = hip.stream(), device_batch(b), DeviceArray(q[0].size)
        mass = DeviceArray(want[0].size)
        ctx.sync()
        ctx.set_stream(stream.value)
        g, graph = hip.graph(stream, lambda: cache.attention_mass_dev(d, dq.ptr, heads * D, heads, 0, mass.ptr, max(lens),
                                                                      D ** -0.5))
        for x, w in zip(q[[0, 1, 0]], [want[0], want[1], want[0]]):
            dq.upload(x), mass.upload(np.zeros(w.size))
            hip.hipGraphLaunch(graph, stream)
            ctx.sync()
            got = mass.download().reshape(w.shape)
            for s, n in enumerate(lens):
                assert_same_bits(got[s, :, :n], w[s, :, :n])
            cache.attention_mass(*b.args(), q[1], heads)
        hip.hipGraphExecDestroy(graph)
        hip.hipGraphDestroy(g)
        cache.close()
        ctx.set_stream(None)
        hip.hipStreamDestroy(stream)
