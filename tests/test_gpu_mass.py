"""The weight that a step's queries give each cached token (nx_attention_mass), against the
formula in 64 bits."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, INT8, Batch, random_kv, stored
from moe_cases import DeviceArray, assert_same_bits
from step_cases import attention_mass
from test_gpu_kv import device_batch, ints

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


def filled(ctx, rng, b, fmt, G, D, k=None):
    """A cache of the batch's sequences, and the keys that it holds."""
    keys, v = random_kv(rng, sum(b.lens), G, D)
    k = keys if k is None else k
    cache = nx.KvCache(ctx, fmt, b.num_pages, b.page_tokens, G, D)
    if sum(b.lens):
        cache.write(b.whole(), b.kv_len, b.pages, k, v)
    return cache, stored(fmt, k)


def check(got, ref, bound):
    err = np.abs(got.astype(np.float64) - ref)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,G,D,page,ns,lens", [
    (4, 1, 64, 32, [1], [1]),
    (32, 8, 128, 64, [1], [517]),
    (32, 4, 128, 32, [1, 1, 1], [1, 33, 700]),
    (16, 8, 256, 128, [2, 1], [300, 129]),
    (12, 12, 96, 64, [5, 3, 1], [5, 1000, 64]),       # one head of each
    (24, 1, 128, 64, [1, 1], [600, 95]),              # more heads than a tile has rows
    (8, 2, 64, 32, [40], [40]),                       # a prompt
    (16, 2, 64, 32, [37, 1], [1300, 20]),
    (12, 12, 96, 32, [129], [400]),
    (6, 3, 256, 64, [70], [200]),
    (32, 4, 128, 256, [33, 1, 0, 250], [2000, 513, 99, 250]),  # prompts and steps
    (5, 1, 128, 1024, [700], [1500]),                 # a group that is no power of two
])
def test_against_formula(ctx, fmt, heads, G, D, page, ns, lens):
    print(f"mass fmt={fmt} heads={heads} G={G} D={D} page={page} ns={ns} lens={lens}", flush=True)
    rng = np.random.default_rng(sum(lens) + D + heads)
    b = Batch(rng, ns, lens, page)
    cache, keys = filled(ctx, rng, b, fmt, G, D)
    q = rng.standard_normal((b.rows, heads, D), dtype=np.float32)
    before = rng.random((len(ns), G, max(lens)), dtype=np.float32) / 50
    ref, bound = attention_mass(b, keys, q, heads, D ** -0.5, before)
    check(cache.attention_mass(*b.args(), q, heads, before=before), ref, bound)
    # nothing before, a scale of its own
    ref, bound = attention_mass(b, keys, q, heads, 0.3)
    check(cache.attention_mass(*b.args(), q, heads, scale=0.3), ref, bound)
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_many_sequences(ctx, fmt):
    """More than a wave finds by itself, with and without prompts among them."""
    rng = np.random.default_rng(3)
    for ns in ([1] * 150, [1, 0, 2] * 40 + [60, 1, 200]):
        lens = [int(n + rng.integers(0, 90)) for n in ns]
        b = Batch(rng, ns, lens, 32)
        cache, keys = filled(ctx, rng, b, fmt, 2, 64)
        q = rng.standard_normal((b.rows, 6, 64), dtype=np.float32)
        ref, bound = attention_mass(b, keys, q, 6, 0.125)
        check(cache.attention_mass(*b.args(), q, 6), ref, bound)
        cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_one_sequence_has_the_rows_of_many(ctx, fmt):
    """A batch of the shape of single tokens whose rows are one sequence's."""
    rng = np.random.default_rng(4)
    for ns in ([0, 0, 0, 7, 0, 0, 0], [0, 90, 0] + [0] * 87, [2, 0, 3, 0, 2]):
        lens = [n + 100 for n in ns]
        b = Batch(rng, ns, lens, 32)
        cache, keys = filled(ctx, rng, b, fmt, 2, 64)
        q = rng.standard_normal((b.rows, 8, 64), dtype=np.float32)
        ref, bound = attention_mass(b, keys, q, 8, 0.125)
        check(cache.attention_mass(*b.args(), q, 8), ref, bound)
        cache.close()


def on_device(cache, b, q, heads, before, stride=None, where="other", scale=None, **arrays):
    """attention_mass_dev with guards around the weights; before: None, or [S x G x stride]."""
    S, G, D = len(b.ns), cache.kv_heads, cache.head_dim
    stride = stride or max(b.lens)
    dq = DeviceArray(q.size)
    dq.upload(q)
    d = device_batch(b)
    for name, a in arrays.items():
        keep = ints(a)
        setattr(d.c, name, keep.ptr)
        d.keep += (keep,)
    m = DeviceArray(S * G * stride + 1, fill=7.0)
    old = DeviceArray(S * G * stride + 1, fill=7.0) if where == "other" else m
    if before is not None:
        old.upload(before)
    cache.attention_mass_dev(d, dq.ptr, heads * D, heads, 0 if before is None else old.ptr, m.ptr, stride,
                             D ** -0.5 if scale is None else scale)
    cache.ctx.sync()
    got = m.download()
    assert got[-1] == 7.0
    return got[:-1].reshape(S, G, stride)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ns,lens", [([1, 0, 2], [70, 50, 33]), ([40, 0, 1, 60], [300, 50, 31, 60])])
@pytest.mark.parametrize("where", ["other", "same"])
def test_device_call(ctx, fmt, ns, lens, where):
    """In place or not; what is behind a sequence's tokens, and sequences without rows, stay."""
    rng = np.random.default_rng(5)
    b = Batch(rng, ns, lens, 32, first_row=2, padding=3)
    cache, keys = filled(ctx, rng, b, fmt, 2, 96)
    q = rng.standard_normal((b.rows, 8, 96), dtype=np.float32)
    width = max(lens) + 9
    before = rng.random((len(ns), 2, width), dtype=np.float32)
    ref, bound = attention_mass(b, keys, q, 8, 96 ** -0.5, before, width)
    got = on_device(cache, b, q, 8, before, width, where)
    for s, (n, length) in enumerate(zip(ns, lens)):
        length = length if n else 0
        check(got[s, :, :length], ref[s, :, :length], bound[s, :, :length])
        rest = before[s, :, length:] if where == "same" else np.full_like(before[s, :, length:], 7.0)
        assert np.array_equal(got[s, :, length:], rest)
    # rows of fewer weights than tokens
    ref, bound = attention_mass(b, keys, q, 8, 96 ** -0.5, None)
    got = on_device(cache, b, q, 8, None, 30)
    for s, n in enumerate(ns):
        if n:
            check(got[s], ref[s, :, :30], bound[s, :, :30])
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (0, 3), (2, 1)])
@pytest.mark.parametrize("ns", [[3, 1], [50, 1]])
def test_strided_and_unaligned_queries(ctx, fmt, shift, extra, ns):
    rng = np.random.default_rng(6)
    lens, heads, D = [n + 60 for n in ns], 4, 64
    b = Batch(rng, ns, lens, 64)
    cache, keys = filled(ctx, rng, b, fmt, 2, D)
    stride = heads * D + extra
    rows = rng.standard_normal((b.rows, stride)).astype(np.float32)
    dq, d = DeviceArray(rows.size + 8, fill=np.nan), device_batch(b)
    dq.upload(rows, shift)
    m = DeviceArray(2 * 2 * max(lens), fill=0.0)
    cache.attention_mass_dev(d, dq.ptr + 4 * shift, stride, heads, 0, m.ptr, max(lens), 0.2)
    ctx.sync()
    q = rows[:, :heads * D].reshape(b.rows, heads, D)
    ref, bound = attention_mass(b, keys, q, heads, 0.2)
    check(m.download().reshape(ref.shape), ref, bound)
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ns,lens", [([1, 1], [200, 100]), ([50, 1], [200, 100])])
def test_tables_that_name_no_page(ctx, fmt, ns, lens):
    """Tokens of missing pages have no part in the softmax; lengths are cut to the table; rows
    before the first token see nothing."""
    rng = np.random.default_rng(7)
    b = Batch(rng, ns, lens, 32)
    cache, keys = filled(ctx, rng, b, fmt, 1, 64)
    q = rng.standard_normal((b.rows, 4, 64), dtype=np.float32)
    pages = b.pages.copy()
    pages[0, 2], pages[1, 0] = -1, b.num_pages
    got = on_device(cache, b, q, 4, None, pages=pages)
    gone = np.zeros((2, 200), bool)
    gone[0, 64:96], gone[1, :32] = True, True
    assert not got[gone[:, None]].any()
    for s in range(2):  # as if the other tokens were the sequence
        n, length, at = ns[s], lens[s], [0, lens[0]][s]
        stay = np.flatnonzero(~gone[s, :length])
        one = Batch(rng, [n], [len(stay)], 32)
        rows = slice(b.row_start[s], b.row_start[s] + n)
        ref, bound = attention_mass(one, keys[at + stay], q[rows], 4, 0.125)
        check(got[s, :, stay].T[None], ref, bound)
    # longer than the table, and shorter than its rows
    got = on_device(cache, b, q, 4, None, kv_len=[10 ** 9, -3])
    assert (got[1] == 7.0).all() and np.isfinite(got[0]).all()
    # (24 of the table's 224 tokens have no weight to gather, and keys of zeros)
    assert 2 * ns[0] < got[0].sum() < 4 * ns[0]
    if ns[0] > 4:
        got = on_device(cache, b, q, 4, None, kv_len=[4, 100])
        one = Batch(rng, [4], [4], 32)
        ref, bound = attention_mass(one, keys[:4], q[ns[0] - 4:ns[0]], 4, 0.125)
        check(got[:1, :, :4], ref, bound)
        assert (got[0, :, 4:] == 7.0).all()
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ns,lens", [([2], [70]), ([40], [100])])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_non_finite_values_reach_no_further_than_their_rows(ctx, fmt, ns, lens, bad):
    """A NaN in a late token's keys spoils the rows that see it, in its head; in places that no
    row sees it spoils nothing; neither does a row's own NaN reach another row's tokens."""
    rng = np.random.default_rng(8)
    n, length = ns[0], lens[0]
    b = Batch(rng, ns, lens, 32)
    k, _ = random_kv(rng, length, 2, 64)
    late = length - 1
    k[late, 1, 3] = bad
    cache, keys = filled(ctx, rng, b, fmt, 2, 64, k)
    q = np.abs(rng.standard_normal((b.rows, 4, 64), dtype=np.float32)) + np.float32(0.1)
    got = on_device(cache, b, q, 4, None)
    clean = keys.copy()
    clean[late] = 0
    ref, bound = attention_mass(b, clean, q, 4, 0.125)
    # the last row sees every token, the others do not see the last
    assert np.isnan(got[0, 1]).all() or (fmt == F16 and bad == np.inf and np.isnan(got[0, 1, late]))
    assert np.isfinite(got[0, 0]).all()
    # without its last row the batch does not see it: stale values behind the end
    short = Batch(rng, [n - 1], [length - 1], 32)
    short.pages = b.pages
    short.max_pages = b.max_pages
    ref, bound = attention_mass(short, keys[:late], q[:n - 1], 4, 0.125)
    check(on_device(cache, short, q[:n - 1], 4, None), ref, bound)
    # a row that is not finite itself: the tokens that it sees
    q[0, 2] = bad
    k[late] = 1
    cache.write(b.whole(), b.kv_len, b.pages, k, k)
    got = on_device(cache, b, q, 4, None)
    sees = length - n + 1
    assert np.isnan(got[0, 1, :sees]).any() and np.isfinite(got[0, 1, sees:]).all() and np.isfinite(got[0, 0]).all()
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", [1, 60])
def test_scores_of_any_size(ctx, fmt, n):
    """One token takes all; queries and keys next to nothing; queries of zeros."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [n], [150], 64)
    for up, down in ((100.0, 1.0), (1e-30, 1.0), (1e18, 1e-18), (1e-12, 1e-3)):
        k = rng.standard_normal((150, 1, 64), dtype=np.float32) * np.float32(down)
        if fmt == F16 and down < 1e-4:
            continue
        cache, keys = filled(ctx, rng, b, fmt, 1, 64, k)
        q = rng.standard_normal((n, 2, 64), dtype=np.float32) * np.float32(up)
        q[0, 0] = 0
        ref, bound = attention_mass(b, keys, q, 2, 0.125)
        check(on_device(cache, b, q, 2, None), ref, bound)
        cache.close()


def check_sequences(b, got, ref, bound):
    """What on_device gives: behind a sequence's tokens nothing is written."""
    for s, length in enumerate(b.lens):
        check(got[s, :, :length], ref[s, :, :length], bound[s, :, :length])
        assert (got[s, :, length:] == 7.0).all()


def test_wide_tables(ctx):
    """Tables so wide that the batch's scores are stored in turns, or not at all."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [1] * 40, [5 + s for s in range(40)], 32, max_pages=4096)
    cache, keys = filled(ctx, rng, b, F16, 1, 64)
    q = rng.standard_normal((40, 16, 64), dtype=np.float32)
    ref, bound = attention_mass(b, keys, q, 16, 0.125)
    check_sequences(b, on_device(cache, b, q, 16, None), ref, bound)
    cache.close()
    # single tokens beside longer ones, more sequences than rows / 16
    b = Batch(rng, [1] * 255 + [40], [3 + s % 50 for s in range(255)] + [60], 32, max_pages=600)
    cache, keys = filled(ctx, rng, b, F16, 1, 64)
    q = rng.standard_normal((b.rows, 1, 64), dtype=np.float32)
    ref, bound = attention_mass(b, keys, q, 1, 0.125)
    check_sequences(b, on_device(cache, b, q, 1, None), ref, bound)
    cache.close()
    b = Batch(rng, [1, 2], [1500, 7], 1024, max_pages=5000)
    cache, keys = filled(ctx, rng, b, F16, 1, 64)
    q = rng.standard_normal((3, 16, 64), dtype=np.float32)
    ref, bound = attention_mass(b, keys, q, 16, 0.125)
    check_sequences(b, on_device(cache, b, q, 16, None), ref, bound)
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_runs_are_alike(ctx, fmt):
    rng = np.random.default_rng(11)
    b = Batch(rng, [200, 1, 3], [700, 2000, 90], 64)
    cache, _ = filled(ctx, rng, b, fmt, 2, 128)
    q = rng.standard_normal((b.rows, 8, 128), dtype=np.float32)
    first = on_device(cache, b, q, 8, None)
    for _ in range(5):
        assert_same_bits(on_device(cache, b, q, 8, None), first)
    cache.close()


def test_rows_that_decrease_touch_nothing_else(ctx):
    """Sequences that share rows: what they give is not defined, but the call ends and stays
    within its buffers."""
    rng = np.random.default_rng(12)
    b = Batch(rng, [8] * 6, [40] * 6, 32)
    cache, _ = filled(ctx, rng, b, F16, 1, 64)
    q = rng.standard_normal((48, 4, 64), dtype=np.float32)
    on_device(cache, b, q, 4, None, row_start=[0, 48, 0, 48, 0, 48, 0])
    b2 = Batch(rng, [1] * 6, [40] * 6, 32)
    b2.pages, b2.num_pages, b2.max_pages = b.pages, b.num_pages, b.max_pages
    on_device(cache, b2, q[:6], 4, None, row_start=[0, 6, 0, 6, 0, 6, 0])
    cache.close()


def test_refusals(ctx):
    rng = np.random.default_rng(13)
    b = Batch(rng, [2, 1], [40, 20], 32)
    cache, _ = filled(ctx, rng, b, F16, 2, 64)
    d, a = device_batch(b), DeviceArray(8192)

    def code(q=a.ptr, qs=256, heads=4, before=0, mass=a.ptr + 4096, ms=40, scale=0.1):
        with pytest.raises(nx.NexusError) as e:
            cache.attention_mass_dev(d, q, qs, heads, before, mass, ms, scale)
        return e.value.code

    assert code(q=0) == code(mass=0) == code(heads=0) == code(scale=np.nan) == nx.NX_ERR_INVALID_ARG
    assert code(before=a.ptr + 4100) == code(before=a.ptr + 4096 - 160) == nx.NX_ERR_INVALID_ARG
    assert code(qs=255) == code(heads=5) == code(ms=0) == nx.NX_ERR_SHAPE
    d.c.num_tokens = 1 << 24
    assert code(heads=256, qs=256 * 64) == nx.NX_ERR_UNSUPPORTED
    q = np.zeros((3, 4, 64), np.float32)
    for kw in (dict(kv_len=[1, 20]), dict(kv_len=[400, 20]), dict(row_start=[0, 2, 4])):
        args = dict(row_start=b.row_start, kv_len=b.kv_len, pages=b.pages)
        args.update(kw)
        with pytest.raises(nx.NexusError) as e:
            cache.attention_mass(q=q, heads=4, **args)
        assert e.value.code == nx.NX_ERR_SHAPE
    cache.close()


def test_calls_in_slices_of_rows(ctx):
    """More query rows than the workspace holds at once: the first slice sets what the later ones add
    to, for sequences that begin in either."""
    rng = np.random.default_rng(14)
    heads, G, D = 256, 2, 256  # 508 rows at once
    for ns, lens in (([600], [640]), ([300, 1, 400], [300, 50, 411])):
        b = Batch(rng, ns, lens, 64)
        cache, keys = filled(ctx, rng, b, F16, G, D)
        q = rng.standard_normal((b.rows, heads, D), dtype=np.float32)
        before = rng.random((len(ns), G, max(lens)), dtype=np.float32)
        ref, bound = attention_mass(b, keys, q, heads, D ** -0.5, before)
        got = on_device(cache, b, q, heads, before)
        for s, n in enumerate(lens):
            check(got[s, :, :n], ref[s, :, :n], bound[s, :, :n])
        cache.close()


def test_slices_that_end_before_a_tile_of_keys(ctx):
    """A slice's last rows see nothing of the keys behind them, though its last part would reach them
    by its size: what an earlier call left there is no part of the sum.

    Scores of nothing: each of a token's 8 rows gives 1 / (p + 1) to the p + 1 tokens that it sees.
    The bound is attention_mass's with scores of no magnitude."""
    rng = np.random.default_rng(15)
    heads, G, D, n, first = 256, 32, 256, 1300, 268  # 508 rows at once, 240 of them the sequence's
    b = Batch(rng, [n], [n], 64, first_row=first)
    cache, _ = filled(ctx, rng, b, F16, G, D)
    q = np.zeros((b.rows, heads, D), np.float32)
    on_device(cache, b, q, heads, None, row_start=[0, n])  # writes what the second call must not read
    got = on_device(cache, b, q, heads, None)[0]
    total = np.cumsum((8.0 / np.arange(1, n + 1))[::-1])[::-1]
    bound = (4 * 2.0 ** -21 + (n + 64 + 2 * np.log2(n + 1) + 8 * n + 8) * 2.0 ** -24) * total
    check(got, np.tile(total, (G, 1)), np.tile(bound, (G, 1)))
    cache.close()
