"""The paged cache on the device: what is written is read back as the format
holds it, bit for bit, wherever the pages are."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, INT8, Batch, random_kv, stored
from moe_cases import DeviceArray, assert_same_bits

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


def ints(a):
    """An int32 array on the device."""
    a = np.ascontiguousarray(a, np.int32).ravel()
    d = DeviceArray(a.size)
    d.upload(a.view(np.float32))
    return d


def device_batch(b):
    """The batch's arrays on the device, and its descriptor (which keeps them)."""
    rs, ln, pg = ints(b.row_start), ints(b.kv_len), ints(b.pages)
    d = nx.KvBatch(len(b.lens), b.rows, b.max_pages, rs.ptr, ln.ptr, pg.ptr)
    d.keep = rs, ln, pg
    return d


def special_rows(rng, rows, D):
    """Rows whose largest values, borders and signs are unusual."""
    x = rng.standard_normal((rows, D)).astype(np.float32)
    scales = [1e-38, 1e-42, 3e-45, 1e-30, 1e30, 3e38, 6e-8, 65504.0, 1.0]
    for i in range(rows):
        x[i] = np.clip(x[i] / 4, -1, 1) * np.float32(scales[i % len(scales)])
    x[0] = 0
    x[1 % rows] = -0.0
    # ties: with a largest value of 127 the scale is 1, and n + 1/2 is halfway
    t = 2 % rows
    x[t] = np.arange(D, dtype=np.float32) % 100 - 50 + 0.5
    x[t, 0] = 127
    # just beside them
    t = 3 % rows
    x[t] = np.nextafter(np.arange(D, dtype=np.float32) % 100 - 50 + 0.5, np.float32(1e9), dtype=np.float32)
    x[t, 1] = -127
    return x


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("G,D,page,ns,lens", [
    (1, 64, 32, [1], [1]),
    (8, 128, 64, [1, 1, 1], [1, 64, 517]),
    (3, 96, 32, [5, 0, 33, 32], [5, 40, 70, 32]),
    (2, 256, 128, [130, 1], [300, 129]),
    (4, 128, 256, [257, 31], [700, 31]),
    (5, 64, 1024, [7, 40], [1030, 1024]),
])
def test_write_and_read_back(ctx, fmt, G, D, page, ns, lens):
    print(f"kv fmt={fmt} G={G} D={D} page={page} ns={ns} lens={lens}", flush=True)
    rng = np.random.default_rng(D + page + sum(lens))
    b = Batch(rng, ns, lens, page)
    cache = nx.KvCache(ctx, fmt, b.num_pages, page, G, D)
    # the whole sequences first, then other values in their last tokens
    k0, v0 = random_kv(rng, sum(lens), G, D)
    whole = b.whole()
    cache.write(whole, b.kv_len, b.pages, k0, v0)
    k1 = special_rows(rng, b.rows * G, D).reshape(b.rows, G, D)
    v1 = special_rows(rng, b.rows * G, D)[::-1].reshape(b.rows, G, D)
    cache.write(*b.args(), k1, v1)
    k, v = cache.read(*b.args())
    assert_same_bits(k, stored(fmt, k1))
    assert_same_bits(v, stored(fmt, v1))
    # the other tokens are what they were
    at = np.concatenate([whole[s] + lens[s] - n + np.arange(n) for s, n in enumerate(ns)])
    k0[at], v0[at] = k1, v1
    k, v = cache.read(whole, b.kv_len, b.pages)
    assert_same_bits(k, stored(fmt, k0))
    assert_same_bits(v, stored(fmt, v0))
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_token_by_token(ctx, fmt):
    """Appending one token at a time fills a cache as writing them together."""
    rng = np.random.default_rng(5)
    G, D, page, n = 2, 64, 32, 75
    b = Batch(rng, [n], [n], page)
    k, v = random_kv(rng, n, G, D)
    cache = nx.KvCache(ctx, fmt, b.num_pages, page, G, D)
    for t in range(n):
        cache.write([0, 1], [t + 1], b.pages, k[t], v[t])
    gk, gv = cache.read(*b.args())
    assert_same_bits(gk, stored(fmt, k))
    assert_same_bits(gv, stored(fmt, v))
    cache.close()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_non_finite_rows(ctx, bad):
    """INT8: the token's row of that head is NaN, no other; F16 holds the value."""
    rng = np.random.default_rng(6)
    G, D = 3, 128
    b = Batch(rng, [9], [41], 32)
    k, v = random_kv(rng, 9, G, D)
    k[4, 1, 77] = bad
    v[8, 2, 0] = bad
    v[0, 0, 5] = 70000.0  # past half's range
    for fmt in FORMATS:
        cache = nx.KvCache(ctx, fmt, b.num_pages, 32, G, D)
        cache.write(*b.args(), k, v)
        gk, gv = cache.read(*b.args())
        assert_same_bits(gk, stored(fmt, k))
        assert_same_bits(gv, stored(fmt, v))
        cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shift,extra", [(0, 0), (0, 12), (1, 0), (2, 5)])
def test_strided_and_unaligned_rows(ctx, fmt, shift, extra):
    """k and v as columns of wider rows, at any float address; padding rows and
    the columns between are left alone."""
    rng = np.random.default_rng(7)
    G, D, page = 2, 96, 64
    b = Batch(rng, [3, 40], [35, 100], page, first_row=2, padding=3)
    width, stride = G * D, 2 * G * D + extra
    rows = rng.standard_normal((b.rows, stride)).astype(np.float32)
    src = DeviceArray(rows.size + 8)
    src.upload(rows, shift)
    dst = DeviceArray(rows.size + 8, fill=7.0)
    cache = nx.KvCache(ctx, fmt, b.num_pages, page, G, D)
    d = device_batch(b)
    for buf, call in ((src, cache.write_dev), (dst, cache.read_dev)):
        call(d, buf.ptr + 4 * shift, buf.ptr + 4 * (shift + width), stride)
    ctx.sync()
    raw = dst.download()
    got = raw[shift:shift + rows.size].reshape(rows.shape)
    want = np.full_like(rows, 7.0)
    own = slice(2, 45)
    want[own, :width] = stored(fmt, rows[own, :width].reshape(-1, G, D)).reshape(-1, width)
    want[own, width:2 * width] = stored(fmt, rows[own, width:2 * width].reshape(-1, G, D)).reshape(-1, width)
    assert_same_bits(got, want)
    assert np.all(raw[:shift] == 7.0) and np.all(raw[shift + rows.size:] == 7.0)
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_device_tables_that_name_no_page(ctx, fmt):
    """Tokens without a page in the cache are not written and read as zeros."""
    rng = np.random.default_rng(8)
    G, D, page = 2, 64, 32
    b = Batch(rng, [70, 4, 40], [70, 70, 40], page, max_pages=3)
    k, v = random_kv(rng, b.rows, G, D)
    cache = nx.KvCache(ctx, fmt, b.num_pages, page, G, D)
    cache.write(*b.args(), k, v)
    pages, lens = b.pages.copy(), b.kv_len.copy()
    b.pages[0, 1], b.pages[2, 0] = -1, b.num_pages  # tokens 32 .. 63, and 0 .. 31
    b.kv_len[1] = 2  # rows 70, 71 before the first token; 72, 73 are tokens 0, 1
    b.kv_len[2] = 100  # rows: tokens 60 .. 99, the last four behind three pages
    k2, v2 = random_kv(rng, b.rows, G, D)
    dk, dv = DeviceArray(k2.size), DeviceArray(v2.size)
    dk.upload(k2), dv.upload(v2)
    d = device_batch(b)
    cache.write_dev(d, dk.ptr, dv.ptr, G * D)
    ok, ov = DeviceArray(k2.size, fill=7.0), DeviceArray(k2.size, fill=7.0)
    cache.read_dev(d, ok.ptr, ov.ptr, G * D)
    ctx.sync()
    there = np.ones(b.rows, bool)
    there[32:64] = False
    there[70:72] = False
    # sequence 2, tokens 60 .. 99: page 1 holds 60 .. 63; page 2 of its table is -1
    there[74:114] = False
    there[74:78] = True
    for got, x in ((ok, k2), (ov, v2)):
        want = np.where(there[:, None, None], stored(fmt, x), 0)
        assert_same_bits(got.download(), want)
    # nothing else changed: sequence 0's middle page by the good table
    gk, gv = cache.read([0, 70, 70, 70], lens, pages)
    assert_same_bits(gk[32:64], stored(fmt, k[32:64]))
    assert_same_bits(gv[32:64], stored(fmt, v[32:64]))
    cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(ctx, fmt):
    """Pages whose bytes and elements lie behind 2^32."""
    G, D, page = 16, 256, 1024
    per_page = page * G * D
    pages = (1 << 32) // per_page + 3
    cache = nx.KvCache(ctx, fmt, pages, page, G, D)
    assert cache.device_bytes() > 2 << 32
    rng = np.random.default_rng(9)
    k, v = random_kv(rng, 37, G, D)
    tables = {"high": [[pages - 1, pages - 2]], "low": [[0, 1]], "middle": [[(1 << 31) // per_page, 2]]}
    for i, t in enumerate(tables.values()):
        cache.write([0, 37], [1030], t, k + i, v - i)
    for i, t in enumerate(tables.values()):
        gk, gv = cache.read([0, 37], [1030], t)
        assert_same_bits(gk, stored(fmt, k + i))
        assert_same_bits(gv, stored(fmt, v - i))
    cache.close()


def test_many_sequences(ctx):
    """More sequences than a workgroup has threads, most of one token."""
    rng = np.random.default_rng(10)
    G, D, page = 1, 64, 32
    ns = [int(n) for n in rng.integers(0, 3, 700)]
    lens = [n + int(x) for n, x in zip(ns, rng.integers(0, 40, 700))]
    b = Batch(rng, ns, lens, page)
    k, v = random_kv(rng, b.rows, G, D)
    cache = nx.KvCache(ctx, F16, b.num_pages, page, G, D)
    cache.write(*b.args(), k, v)
    gk, gv = cache.read(*b.args())
    assert_same_bits(gk, stored(F16, k))
    assert_same_bits(gv, stored(F16, v))
    cache.close()


def test_more_tokens_than_one_launch_takes(ctx):
    """2100 single tokens on 4096 heads: more than 2^32 threads.  Each page has 32 sequences'
    tokens, and a row's values are the next row's keys."""
    G, D, page, S = 4096, 64, 32, 2100
    x = np.add.outer((np.arange(S + 1) % 1021).astype(np.float32), (np.arange(G * D) % 1024).astype(np.float32))
    src, out = DeviceArray(x.size), DeviceArray(2 * S * G * D)
    src.upload(x)
    s = np.arange(S)
    rs, ln, pg = ints(np.arange(S + 1)), ints(s % page + 1), ints(s // page)
    d = nx.KvBatch(S, S, 1, rs.ptr, ln.ptr, pg.ptr)
    cache = nx.KvCache(ctx, F16, -(-S // page), page, G, D)
    print(f"kv S={S} G={G} D={D}", flush=True)
    cache.write_dev(d, src.ptr, src.ptr + 4 * G * D, G * D)
    cache.read_dev(d, out.ptr, out.ptr + 4 * G * D, 2 * G * D)
    ctx.sync()
    got = out.download().reshape(S, 2, G * D)
    assert np.array_equal(got[:, 0], x[:-1])
    assert np.array_equal(got[:, 1], x[1:])
    cache.close()


def test_steps_without_sequences(ctx):
    cache = nx.KvCache(ctx, F16, 4, 64, 2, 64)
    none = np.zeros((0, 128), np.float32)
    cache.write([0], [], np.zeros((0, 4)), none, none)
    k, v = cache.read([0], [], [])
    assert k.shape == v.shape == (0, 2, 64)
    assert cache.attention([0], [], [], none, 4).shape == (0, 4, 64)
    cache.close()


def test_refusals(ctx):
    def refused(code, f, *a, **kw):
        with pytest.raises(nx.NexusError) as e:
            f(*a, **kw)
        assert e.value.code == code, str(e.value)

    refused(nx.NX_ERR_INVALID_ARG, nx.KvCache, ctx, 7, 4, 64, 2, 64)
    refused(nx.NX_ERR_UNSUPPORTED, nx.KvCache, ctx, F16, 4, 48, 2, 64)
    refused(nx.NX_ERR_UNSUPPORTED, nx.KvCache, ctx, F16, 4, 64, 2, 80)
    refused(nx.NX_ERR_INVALID_ARG, nx.KvCache, ctx, F16, 0, 64, 2, 64)
    refused(nx.NX_ERR_OOM, nx.KvCache, ctx, F16, 1 << 30, 1024, 16, 256)
    cache = nx.KvCache(ctx, F16, 4, 64, 2, 64)
    x = np.zeros((2, 128), np.float32)
    refused(nx.NX_ERR_INVALID_ARG, cache.write, [0, 2], [2], [[4]], x, x)
    refused(nx.NX_ERR_SHAPE, cache.write, [0, 2], [1], [[0]], x, x)
    refused(nx.NX_ERR_SHAPE, cache.write, [0, 3], [3], [[0]], x, x)
    refused(nx.NX_ERR_SHAPE, cache.write, [0, 2], [65], [[0]], x, x)
    refused(nx.NX_ERR_INVALID_ARG, cache.write, [0, 1, 2], [9, 9], [[3], [3]], x, x)
    refused(nx.NX_ERR_INVALID_ARG, cache.read, [0, 2], [2], [[-1]])
    L, b = nx.lib(), nx.KvBatch(1, 2, 1, 8, 8, 8)
    assert L.nx_kv_write_dev(ctx.h, cache.h, b.ref, None, None, 128) == nx.NX_ERR_INVALID_ARG
    assert L.nx_kv_write_dev(ctx.h, cache.h, b.ref, 8, 8, 127) == nx.NX_ERR_SHAPE
    assert L.nx_kv_read_dev(ctx.h, None, b.ref, 8, 8, 128) == nx.NX_ERR_INVALID_ARG
    assert L.nx_kv_read_dev(ctx.h, cache.h, None, 8, 8, 128) == nx.NX_ERR_INVALID_ARG
    # nothing to do
    none = nx.KvBatch(0, 0, 0, 0, 0, 0)
    assert L.nx_kv_write_dev(ctx.h, cache.h, none.ref, None, None, 128) == nx.NX_OK
    k, _ = cache.read([0, 0], [0], [[0]])
    assert k.shape == (0, 2, 64)
    cache.close()
