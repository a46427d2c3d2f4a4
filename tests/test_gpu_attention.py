"""Attention over the paged cache against its formula in 64 bits, on the values
that the cache holds (kv_cases.attention, with its bound)."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, INT8, Batch, assert_close, attention, random_kv, stored
from kv_cases import attention_dense
from moe_cases import DeviceArray, assert_same_bits
from test_gpu_kv import device_batch, ints

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]
# (token, head) rows of a step from which sequences of several are taken 128 rows at a time
MANY = 4096


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


def filled(ctx, rng, b, fmt, G, D):
    """A cache with the batch's sequences in it, and what it holds of them."""
    k, v = random_kv(rng, sum(b.lens), G, D)
    cache = nx.KvCache(ctx, fmt, b.num_pages, b.page_tokens, G, D)
    cache.write(b.whole(), b.kv_len, b.pages, k, v)
    return cache, stored(fmt, k), stored(fmt, v)


def check(ctx, fmt, H, G, D, page, ns, lens, window=0, sinks=0, seed=0, factor=1.0, beside=False):
    """beside: with one sequence more, whose rows make the step one of many."""
    if beside:
        n = MANY // H + 1
        ns, lens = [*ns, n], [*lens, n + 5]
    rng = np.random.default_rng([seed, D, page, len(ns), sum(lens)])
    b = Batch(rng, ns, lens, page)
    cache, k, v = filled(ctx, rng, b, fmt, G, D)
    q = rng.standard_normal((b.rows, H, D)).astype(np.float32) * np.float32(factor)
    got = cache.attention(*b.args(), q, H, window=window, sinks=sinks)
    ref, bound = attention(b, k, v, q, H, np.float32(D ** -0.5), window, sinks)
    assert_close(got, ref, bound, scores=8 * factor)
    again = cache.attention(*b.args(), q, H, window=window, sinks=sinks)
    assert_same_bits(again, got)
    cache.close()


SHAPES = [(32, 8, 128), (4, 1, 64), (6, 6, 96), (4, 2, 256), (20, 1, 128), (3, 3, 64), (40, 2, 128)]
BATCHES = [
    ([1], [1]),
    ([1], [33]),
    ([1, 1, 1], [2, 700, 64]),
    ([3, 1, 0, 2], [3, 129, 77, 1000]),
    ([1] * 9, [31, 32, 33, 63, 64, 65, 127, 128, 129]),
    ([40], [40]),
    ([33, 1, 70], [97, 300, 70]),
]


@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,G,D", SHAPES)
@pytest.mark.parametrize("ns,lens", BATCHES, ids=lambda v: "-".join(map(str, v))[:24])
def test_parity(ctx, fmt, H, G, D, ns, lens, beside):
    print(f"attention fmt={fmt} H={H} G={G} D={D} ns={ns} lens={lens}", flush=True)
    check(ctx, fmt, H, G, D, 64, ns, lens, beside=beside)


@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", [32, 128, 1024])
def test_pages(ctx, fmt, page, beside):
    check(ctx, fmt, 8, 2, 128, page, [1, 50, 2], [1500, 65, 320], beside=beside)


@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (7, 1), (32, 33), (100, 0), (128, 4), (300, 64),
                                          (4096, 4), (2 ** 31 - 1, 2 ** 31 - 1), (5, 2000)])
@pytest.mark.parametrize("ns,lens", [([1, 1, 1], [5, 130, 1100]), ([200, 3], [900, 40]), ([65], [65])],
                         ids=["step", "chunk", "prompt"])
def test_window(ctx, fmt, window, sinks, ns, lens, beside):
    print(f"window fmt={fmt} window={window} sinks={sinks} ns={ns} lens={lens}", flush=True)
    check(ctx, fmt, 8, 2, 64, 32, ns, lens, window, sinks, beside=beside)


@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,G,D", [(32, 8, 128), (8, 1, 64), (6, 6, 96), (4, 2, 256)])
def test_chunks(ctx, fmt, H, G, D, beside):
    """Chunks of several hundred tokens, behind a context and from the first token on."""
    print(f"chunk fmt={fmt} H={H} G={G} D={D}", flush=True)
    check(ctx, fmt, H, G, D, 64, [517, 1, 130], [1203, 700, 130], beside=beside)
    check(ctx, fmt, H, G, D, 32, [300], [2500], window=257, sinks=5, beside=beside)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_wide_tables(ctx, fmt, window, sinks):
    """Tables far wider than the sequences: only the lengths say how much there is to do."""
    rng = np.random.default_rng(23)
    H, G, D, page = 16, 2, 64, 32
    for ns, lens in (([200], [900]), ([90, 1, 40], [700, 50, 40]), ([120], [21000])):
        b = Batch(rng, ns, lens, page)
        cache, k, v = filled(ctx, rng, b, fmt, G, D)
        q = rng.standard_normal((b.rows, H, D)).astype(np.float32)
        got = cache.attention(*b.args(), q, H, window=window, sinks=sinks)
        ref, bound = attention(b, k, v, q, H, np.float32(D ** -0.5), window, sinks)
        assert_close(got, ref, bound)
        pages = np.full((len(ns), 8000), -1, np.int32)
        pages[:, :b.max_pages] = b.pages
        assert_same_bits(cache.attention(b.row_start, b.kv_len, pages, q, H, window=window, sinks=sinks), got)
        cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_context(ctx, fmt):
    """Few rows and many tokens: the axis that is split and joined."""
    check(ctx, fmt, 8, 1, 64, 256, [1], [40013])
    check(ctx, fmt, 4, 2, 128, 128, [2, 1], [9001, 17])
    check(ctx, fmt, 4, 2, 128, 128, [1], [20000], window=5000, sinks=70)


@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("factor", [1e-30, 30.0, 1e-5])
def test_score_ranges(ctx, fmt, factor, beside):
    """Scores of all but nothing, and a softmax that one token takes."""
    check(ctx, fmt, 8, 2, 128, 64, [1, 40], [500, 300], factor=factor, beside=beside)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H", [8, 104])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 4.0])
def test_scales_of_the_scores(ctx, fmt, H, scale):
    """No scale (all tokens alike), a negative one, and the extremes of a softmax."""
    rng = np.random.default_rng(22)
    b = Batch(rng, [1, 40], [70, 300], 32)
    cache, k, v = filled(ctx, rng, b, fmt, 2, 64)
    q = rng.standard_normal((b.rows, H, 64)).astype(np.float32)
    ref, bound = attention(b, k, v, q, H, np.float32(scale))
    # q k: a standard deviation of sqrt(61 + 3 * 9) = 9.4, up to some four of them
    assert_close(cache.attention(*b.args(), q, H, scale=scale), ref, bound, scores=40 * abs(scale))
    cache.close()


def test_value_scales_of_all_sizes(ctx):
    """INT8: neighbouring tokens' scales many powers of two apart."""
    rng = np.random.default_rng(3)
    for n, length, H in ((1, 700, 4), (150, 300, 4), (150, 300, 28)):
        b = Batch(rng, [n], [length], 32)
        k, v = random_kv(rng, length, 2, 128)
        v *= (10.0 ** rng.integers(-20, 5, (length, 2, 1))).astype(np.float32)
        k *= (10.0 ** rng.integers(-3, 1, (length, 2, 1))).astype(np.float32)
        cache = nx.KvCache(ctx, INT8, b.num_pages, 32, 2, 128)
        cache.write(b.whole(), b.kv_len, b.pages, k, v)
        q = rng.standard_normal((n, H, 128)).astype(np.float32)
        ref, bound = attention(b, stored(INT8, k), stored(INT8, v), q, H, np.float32(128 ** -0.5))
        assert_close(cache.attention(*b.args(), q, H), ref, bound)
        cache.close()


def close_int8(ctx, k, v, q, n, scale, scores=8.0):
    """INT8 attention of the last n of the tokens k, v against its formula."""
    length, G, D = k.shape
    b = Batch(np.random.default_rng(25), [n], [length], 32)
    cache = nx.KvCache(ctx, INT8, b.num_pages, 32, G, D)
    cache.write(b.whole(), b.kv_len, b.pages, k, v)
    H = q.shape[1]
    ref, bound = attention(b, stored(INT8, k), stored(INT8, v), q, H, np.float32(scale))
    assert_close(cache.attention(*b.args(), q, H, scale=scale), ref, bound, scores)
    cache.close()


# one workgroup of 16-row tiles, several, and 128-row tiles whole and in parts
INT8_STEPS = [(1, 4, 700), (2, 2, 9000), (150, 28, 300), (150, 28, 1500)]


@pytest.mark.parametrize("n,H,length", INT8_STEPS)
@pytest.mark.parametrize("small,large", [(0.0, 1e25), (1e-24, 1e29), (0.0, 1.0)])
@pytest.mark.parametrize("order", ["first", "last", "groups", "tokens"])
def test_value_scales_far_apart(ctx, n, H, length, small, large, order):
    """INT8: tokens of next to no value count in the denominator, wherever the large ones are."""
    rng = np.random.default_rng(26)
    j = np.arange(length)
    is_large = {"first": j < length // 2, "last": j >= length // 2, "groups": j // 32 % 2 == 1,
                "tokens": rng.random(length) < 0.5}[order]
    k, v = random_kv(rng, length, 2, 128)
    v *= np.where(is_large, large, small).astype(np.float32)[:, None, None]
    close_int8(ctx, k, v, rng.standard_normal((n, H, 128)).astype(np.float32), n, 128 ** -0.5)


@pytest.mark.parametrize("n,H,length", INT8_STEPS)
@pytest.mark.parametrize("large", [1.0, 1e20, 1e30, 1e36])
def test_many_small_weights_beside_a_large_value(ctx, n, H, length, large):
    """INT8: one token's value decides the reference, the others' weights the denominator."""
    rng = np.random.default_rng(27)
    u = rng.choice([-1.0, 1.0], 128)
    k = np.repeat((-6.0 / 128 * u).astype(np.float32)[None, None], length, 0).repeat(2, 1)
    _, v = random_kv(rng, length, 2, 128)
    k[7], v[7] = 0, v[7] * np.float32(large)
    close_int8(ctx, k, v, np.tile(u.astype(np.float32), (n, H, 1)), n, 1.0)


@pytest.mark.parametrize("n,H,length", INT8_STEPS)
@pytest.mark.parametrize("low,high", [(-33, -33), (-36, -28), (31, 31), (36, 37), (-36, 37)])
def test_values_of_any_size(ctx, n, H, length, low, high):
    """INT8: values from next to f32's smallest to next to its largest, alone and mixed."""
    rng = np.random.default_rng(28)
    k, v = random_kv(rng, length, 2, 128)
    v *= (10.0 ** rng.integers(low, high + 1, (length, 2, 1))).astype(np.float32)
    close_int8(ctx, k, v, rng.standard_normal((n, H, 128)).astype(np.float32), n, 128 ** -0.5)


@pytest.mark.parametrize("n,H,length", INT8_STEPS)
def test_keys_next_to_the_largest(ctx, n, H, length):
    """INT8: keys of 1.4e35 to 1.9e35 under queries of 2^-112: scores of -13.6 to -18.3."""
    rng = np.random.default_rng(29)
    u = rng.choice([-1.0, 1.0], 128)
    _, v = random_kv(rng, length, 2, 128)
    k = (-rng.uniform(1.4e35, 1.9e35, (length, 2, 1)) * u).astype(np.float32)
    q = np.tile((2.0 ** -112 * u).astype(np.float32), (n, H, 1))
    close_int8(ctx, k, v, q, n, 2.0 ** -8, scores=20)


@pytest.mark.parametrize("H", [4, 204])
def test_zeros(ctx, H):
    """Zero queries average, zero keys and values give what the formula gives."""
    rng = np.random.default_rng(4)
    for fmt in FORMATS:
        b = Batch(rng, [1, 20], [90, 50], 32)
        k, v = random_kv(rng, sum(b.lens), 2, 64)
        k[:30] = 0
        v[10:40] = 0
        cache = nx.KvCache(ctx, fmt, b.num_pages, 32, 2, 64)
        cache.write(b.whole(), b.kv_len, b.pages, k, v)
        q = rng.standard_normal((21, H, 64)).astype(np.float32)
        q[0] = 0
        q[5] = -0.0
        ref, bound = attention(b, stored(fmt, k), stored(fmt, v), q, H, np.float32(0.125))
        assert_close(cache.attention(*b.args(), q, H), ref, bound)
        cache.close()


@pytest.mark.parametrize("H", [4, 80])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_non_finite_where_no_row_looks(ctx, fmt, n, bad, H):
    """Keys and values between the first tokens and the windows, and behind the
    last token of a sequence, change nothing."""
    rng = np.random.default_rng(11)
    G, D, page, length = 2, 128, 64, 400
    b = Batch(rng, [n], [length], page, max_pages=8)
    k, v = random_kv(rng, length, G, D)
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    window, sinks = 50, 3
    for where in ("between", "behind"):
        cache = nx.KvCache(ctx, fmt, b.num_pages, page, G, D)
        if where == "between":
            k2, v2 = k.copy(), v.copy()
            k2[3:length - n - window + 1] = bad
            v2[3:length - n - window + 1] = bad
            cache.write(b.whole(), b.kv_len, b.pages, k2, v2)
        else:  # an older sequence's tokens in the same page
            old = 448 - length
            cache.write([0, old], [448], b.pages, np.full((old, G, D), bad), np.full((old, G, D), bad))
            cache.write(b.whole(), b.kv_len, b.pages, k, v)
        ref, bound = attention(b, stored(fmt, k), stored(fmt, v), q, H, np.float32(D ** -0.5), window, sinks)
        assert_close(cache.attention(*b.args(), q, H, window=window, sinks=sinks), ref, bound)
        cache.close()


@pytest.mark.parametrize("H", [4, 60])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_non_finite_future(ctx, fmt, bad, H):
    """A chunk's later tokens hold infinities or NaNs: earlier rows are what they
    are without them, rows that see them what the formula gives."""
    rng = np.random.default_rng(12)
    G, D, n, length = 2, 64, 70, 200
    b = Batch(rng, [n], [length], 32)
    k, v = random_kv(rng, length, G, D)
    k[170, 0, 5] = bad
    v[185, 1, 9] = bad
    cache = nx.KvCache(ctx, fmt, b.num_pages, 32, G, D)
    cache.write(b.whole(), b.kv_len, b.pages, k, v)
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    got = cache.attention(*b.args(), q, H)
    ref, bound = attention(b, stored(fmt, k), stored(fmt, v), q, H, np.float32(0.125))
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
    assert fine[:40].all() and not fine[60:].all()
    assert np.all(np.abs(got[fine] - ref[fine]) <= bound[fine])
    cache.close()


@pytest.mark.parametrize("H", [8, 104])
@pytest.mark.parametrize("fmt", FORMATS)
def test_non_finite_query(ctx, fmt, H):
    """A NaN or infinite query spoils its own head's row and no other."""
    rng = np.random.default_rng(13)
    for n, length in ((1, 100), (40, 140)):
        b = Batch(rng, [n], [length], 32)
        cache, k, v = filled(ctx, rng, b, fmt, 2, 64)
        q = rng.standard_normal((n, H, 64)).astype(np.float32)
        clean = cache.attention(*b.args(), q, H)
        q[n - 1, 3, 7] = np.nan
        q[0, 6, 0] = np.inf
        got = cache.attention(*b.args(), q, H)
        spoiled = np.zeros((n, H), bool)
        spoiled[n - 1, 3] = spoiled[0, 6] = True
        assert np.all(np.isnan(got[spoiled]))
        assert_same_bits(got[~spoiled], clean[~spoiled])
        cache.close()


@pytest.mark.parametrize("H", [4, 46])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shift,extra", [(0, 0), (0, 16), (1, 3)])
def test_strided_and_unaligned_rows(ctx, fmt, shift, extra, H):
    rng = np.random.default_rng(14)
    G, D = 2, 128
    for ns in ([1, 1], [3, 90]):
        b = Batch(rng, ns, [77, 210], 64, first_row=1, padding=2)
        cache, k, v = filled(ctx, rng, b, fmt, G, D)
        stride = H * D + extra
        rows = rng.standard_normal((b.rows, stride)).astype(np.float32)
        src, dst = DeviceArray(rows.size + 4), DeviceArray(rows.size + 4, fill=7.0)
        src.upload(rows, shift)
        cache.attention_dev(device_batch(b), src.ptr + 4 * shift, stride, H, dst.ptr + 4 * shift, stride, 0.1)
        ctx.sync()
        raw = dst.download()
        got = raw[shift:shift + rows.size].reshape(b.rows, stride)
        ref, bound = attention(b, k, v, rows[:, :H * D].reshape(b.rows, H, D), H, np.float32(0.1))
        own = slice(1, b.rows - 2)
        assert_close(got[own, :H * D].reshape(-1, H, D), ref[own], bound[own])
        left = np.ones_like(got, bool)
        left[own, :H * D] = False
        assert np.all(got[left] == 7.0)
        assert np.all(raw[:shift] == 7.0) and np.all(raw[shift + rows.size:] == 7.0)
        cache.close()


@pytest.mark.parametrize("H", [4, 28])
@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_see_nothing(ctx, fmt, H):
    """Device batches whose lengths and tables leave rows without a token give zeros."""
    rng = np.random.default_rng(15)
    G, D, page = 2, 64, 32
    for n in (2, 50):
        b = Batch(rng, [n, n, n], [n + 40, n + 40, n + 40], page, max_pages=3)
        cache, k, v = filled(ctx, rng, b, fmt, G, D)
        q = rng.standard_normal((b.rows, H, D)).astype(np.float32)
        b.kv_len[0] = n - 1  # its first row is before the first token
        b.pages[1, :] = [-1, b.num_pages, 1 << 30]
        dq, do = DeviceArray(q.size), DeviceArray(q.size, fill=7.0)
        dq.upload(q)
        cache.attention_dev(device_batch(b), dq.ptr, H * D, H, do.ptr, H * D, 0.125)
        ctx.sync()
        got = do.download().reshape(q.shape)
        assert np.all(got[0] == 0) and np.all(got[n:2 * n] == 0)
        # the others: sequence 0 with a row fewer, sequence 2 as it was
        at = n + 40
        short = Batch.__new__(Batch)
        short.ns, short.lens, short.row_start, short.rows = [n - 1, n], [n - 1, at], [1, 2 * n], 3 * n
        kk = np.concatenate([k[:n - 1], k[2 * at:]])
        vv = np.concatenate([v[:n - 1], v[2 * at:]])
        ref, bound = attention(short, kk, vv, q, H, np.float32(0.125))
        assert_close(got, ref, bound)
        cache.close()


@pytest.mark.parametrize("H", [4, 138])
@pytest.mark.parametrize("window", [1, 9, 2 ** 31 - 1])
def test_rows_before_the_first_token_in_a_window(ctx, window, H):
    """A tile whose first rows are before the first token: the others' windows count."""
    rng = np.random.default_rng(20)
    G, D, n, length = 2, 64, 30, 12
    b = Batch(rng, [n], [n], 32)
    cache, k, v = filled(ctx, rng, b, F16, G, D)
    b.kv_len[0] = length  # rows 0 .. 17 are tokens -18 .. -1
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    dq, do = DeviceArray(q.size), DeviceArray(q.size, fill=7.0)
    dq.upload(q)
    cache.attention_dev(device_batch(b), dq.ptr, H * D, H, do.ptr, H * D, 0.125, window=window)
    ctx.sync()
    got = do.download().reshape(q.shape)
    assert np.all(got[:n - length] == 0)
    short = Batch(rng, [length], [length], 32)
    ref, bound = attention(short, k[:length], v[:length], q[n - length:], H, np.float32(0.125), window)
    assert_close(got[n - length:], ref, bound)
    cache.close()


@pytest.mark.parametrize("H", [4, 70])
@pytest.mark.parametrize("fmt", FORMATS)
def test_missing_page_in_the_middle(ctx, fmt, H):
    """Tokens on a page that the cache does not have are not attended to."""
    rng = np.random.default_rng(16)
    G, D = 2, 64
    for n in (1, 60):
        b = Batch(rng, [n], [200], 32)
        cache, k, v = filled(ctx, rng, b, fmt, G, D)
        b.pages[0, 2] = b.num_pages
        q = rng.standard_normal((n, H, D)).astype(np.float32)
        dq, do = DeviceArray(q.size), DeviceArray(q.size)
        dq.upload(q)
        cache.attention_dev(device_batch(b), dq.ptr, H * D, H, do.ptr, H * D, 0.125)
        ctx.sync()
        # without tokens 64 .. 95 the others' order and causality are the same
        keep = np.r_[0:64, 96:200]
        c = Batch(rng, [n], [168], 32)
        ref, bound = attention(c, k[keep], v[keep], q, H, np.float32(0.125))
        assert_close(do.download().reshape(q.shape), ref, bound)
        cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H", [4, 46])
def test_pages_behind_a_window(ctx, fmt, H):
    """A window's caller may give back the pages that no row sees any more."""
    rng = np.random.default_rng(24)
    G, D, page = 2, 96, 64
    for n in (1, 90):
        b = Batch(rng, [n], [900], page)
        cache, k, v = filled(ctx, rng, b, fmt, G, D)
        q = rng.standard_normal((n, H, D)).astype(np.float32)
        want = cache.attention(*b.args(), q, H, window=130, sinks=3)
        first = (900 - n - 129) // page
        other = [np.full((64, G, D), np.nan)] * 2
        for p in range(1, first):  # the next owners write to them
            cache.write([0, 64], [64], b.pages[:, p:p + 1], *other)
        b.pages[0, 1:first] = -1
        assert_same_bits(cache.attention(*b.args(), q, H, window=130, sinks=3), want)
        with pytest.raises(nx.NexusError):
            cache.attention(*b.args(), q, H, window=130 + page, sinks=3)
        cache.close()


def test_shared_pages(ctx):
    """Two sequences with one prefix in the same pages."""
    rng = np.random.default_rng(17)
    G, D, page = 2, 64, 32
    b = Batch(rng, [1, 30], [80, 110], page)
    b.pages[1, :2] = b.pages[0, :2]  # 64 tokens
    k, v = random_kv(rng, 190, G, D)
    k[80:144], v[80:144] = k[:64], v[:64]
    cache = nx.KvCache(ctx, F16, b.num_pages, page, G, D)
    with pytest.raises(nx.NexusError):
        cache.write(b.whole(), b.kv_len, b.pages, k, v)  # both write the prefix
    cache.write([0, 80, 80], b.kv_len, b.pages, k[:80], v[:80])
    cache.write([0, 0, 46], b.kv_len, b.pages, k[144:], v[144:])
    q = rng.standard_normal((31, 4, D)).astype(np.float32)
    ref, bound = attention(b, stored(F16, k), stored(F16, v), q, 4, np.float32(0.125))
    assert_close(cache.attention(*b.args(), q, 4), ref, bound)
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(ctx, fmt):
    G, D, page = 16, 256, 1024
    pages = (1 << 32) // (page * G * D) + 3
    rng = np.random.default_rng(18)
    cache = nx.KvCache(ctx, fmt, pages, page, G, D)
    for n, H in ((1, G), (40, G), (40, 7 * G)):
        b = Batch(rng, [n], [1100], page)
        b.pages = np.array([[pages - 1, pages - 2]], np.int32)
        k, v = random_kv(rng, 1100, G, D)
        cache.write(b.whole(), b.kv_len, b.pages, k, v)
        q = rng.standard_normal((n, H, D)).astype(np.float32)
        ref, bound = attention(b, stored(fmt, k), stored(fmt, v), q, H, np.float32(0.0625))
        assert_close(cache.attention(*b.args(), q, H), ref, bound)
    cache.close()


def test_many_sequences(ctx):
    """More sequences than a workgroup has threads, some without rows."""
    rng = np.random.default_rng(19)
    ns = [int(n) for n in rng.integers(0, 3, 600)]
    lens = [n + int(x) for n, x in zip(ns, rng.integers(0, 90, 600))]
    check(ctx, F16, 2, 1, 64, 32, ns, lens)


# Steps with more tiles than workgroups, or with more than 64 sequences: workgroups that take
# equal runs of units, over tiles, heads and sequences.  `heads` key/value heads of narrow width,
# and of 256 (half as many workgroups).
RUNS = {
    # long tiles of one sequence, the workgroup's scan over more than eight of them
    "prompt": dict(heads=(64, 32), ns=[1040], lens=[1077]),
    "window": dict(heads=(64, 32), ns=[1040], lens=[1500], window=100, sinks=5),
    # up to four tiles of a sequence, a wave's plan
    "prompts": dict(heads=(64, 32), ns=[400, 290, 3, 333], lens=[400, 500, 700, 340]),
    # 16-row tiles
    "decode": dict(heads=(8, 8), group=2, ns=[1 + s % 3 for s in range(40)], lens=[9 + 37 * s % 300 for s in range(40)]),
    # more than 64 sequences, a long one among them, in both kernels
    "many": dict(heads=(3, 3), group=2, ns=[s % 3 for s in range(70)] + [1300] + [1, 40] * 15,
                 lens=[2 + 61 * s % 400 for s in range(70)] + [1500] + [333, 90] * 15),
    "many-window": dict(heads=(3, 3), group=2, ns=[1] * 90 + [1300], lens=[1 + 53 * s % 500 for s in range(90)] + [1300],
                        window=77, sinks=3),
}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("name", RUNS)
def test_equal_runs(ctx, fmt, D, name):
    print(f"runs fmt={fmt} D={D} {name}", flush=True)
    case = dict(group=1, window=0, sinks=0) | RUNS[name]
    G = case["heads"][D == 256]
    H, rng = G * case["group"], np.random.default_rng([D, len(name)])
    b = Batch(rng, case["ns"], case["lens"], 64)
    cache, k, v = filled(ctx, rng, b, fmt, G, D)
    q = rng.standard_normal((b.rows, H, D)).astype(np.float32)
    seen = dict(window=case["window"], sinks=case["sinks"])
    got = cache.attention(*b.args(), q, H, **seen)
    ref, bound = attention_dense(b, k, v, q, H, np.float32(D ** -0.5), **seen)
    assert_close(got, ref, bound)
    assert_same_bits(cache.attention(*b.args(), q, H, **seen), got)
    cache.close()


def test_refusals(ctx):
    cache = nx.KvCache(ctx, F16, 4, 64, 2, 64)
    q = np.zeros((1, 4 * 64), np.float32)

    def refused(code, **kw):
        a = dict(row_start=[0, 1], kv_len=[1], pages=[[0]], q=q, heads=4) | kw
        with pytest.raises(nx.NexusError) as e:
            cache.attention(**a)
        assert e.value.code == code, str(e.value)

    refused(nx.NX_ERR_SHAPE, heads=1)
    refused(nx.NX_ERR_INVALID_ARG, scale=float("nan"))
    refused(nx.NX_ERR_INVALID_ARG, window=-1)
    refused(nx.NX_ERR_INVALID_ARG, window=4, sinks=-1)
    refused(nx.NX_ERR_INVALID_ARG, pages=[[4]])
    refused(nx.NX_ERR_SHAPE, kv_len=[0])
    refused(nx.NX_ERR_SHAPE, kv_len=[65])
    L, b = nx.lib(), nx.KvBatch(1, 1, 1, 8, 8, 8)
    call = lambda q, qs, H, o, os: L.nx_attention_dev(ctx.h, cache.h, b.ref, q, qs, H, 1.0, 0, 0, o, os)  # noqa: E731
    assert call(8, 255, 4, 8, 256) == nx.NX_ERR_SHAPE
    assert call(8, 256, 4, 8, 255) == nx.NX_ERR_SHAPE
    assert call(None, 256, 4, 8, 256) == nx.NX_ERR_INVALID_ARG
    assert call(8, 256, 4, None, 256) == nx.NX_ERR_INVALID_ARG
    assert call(8, 256, 0, 8, 256) == nx.NX_ERR_INVALID_ARG
    assert cache.attention([0, 0], [0], [[0]], np.zeros((0, 256), np.float32), 4).shape == (0, 4, 64)
    cache.close()
