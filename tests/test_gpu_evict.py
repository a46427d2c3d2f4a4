"""Giving up cached tokens (nx_kv_evict): which ones stay, and that they move as they are stored."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, INT8, Batch, random_kv, stored
from moe_cases import DeviceArray, assert_same_bits
from step_cases import evicted
from test_gpu_kv import ints

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


class Case:
    """Sequences in a cache, new pages for `keep` tokens of each, and weights."""

    def __init__(self, ctx, rng, fmt, lens, page, G, D, keep, spare=2):
        need = [-(-min(n, keep) // page) for n in lens]
        self.b = Batch(rng, [0] * len(lens), lens, page, spare=sum(need) + spare)
        self.to = np.full((len(lens), max(max(need), 1)), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.to[s, :n] = self.b.unused[at:at + n]
            at += n
        self.lens, self.fmt, self.G, self.keep, self.page = lens, fmt, G, keep, page
        self.k, self.v = random_kv(rng, sum(lens), G, D)
        self.cache = nx.KvCache(ctx, fmt, self.b.num_pages, page, G, D)
        if sum(lens):
            self.cache.write(self.b.whole(), self.b.kv_len, self.b.pages, self.k, self.v)
        self.mass = np.exp(2 * rng.standard_normal((len(lens), G, max(max(lens), 1)))).astype(np.float32)

    def check(self, got, sinks, recent, mass=None):
        kept, new_len, moved = got
        mass = self.mass if mass is None else mass
        starts = self.b.whole()
        assert np.array_equal(new_len, np.minimum(self.lens, self.keep))
        want_k, want_v = [], []
        for s, n in enumerate(self.lens):
            at = np.empty((self.G, new_len[s]), int)
            for g in range(self.G):
                at[g] = evicted(mass[s, g], n, self.keep, sinks, recent)
                assert np.array_equal(kept[s, g, :new_len[s]], at[g]), (s, g)
                assert (kept[s, g, new_len[s]:] == -1).all()
                if moved is not None:
                    assert_same_bits(moved[s, g, :new_len[s]], mass[s, g, at[g]])
            for want, x in ((want_k, self.k), (want_v, self.v)):
                want += [np.stack([x[starts[s] + at[g], g] for g in range(self.G)], 1)]
        ends = np.concatenate([[0], np.cumsum(new_len)])
        if ends[-1]:
            k, v = self.cache.read(ends, new_len, self.to)
            assert_same_bits(k, stored(self.fmt, np.concatenate(want_k)))
            assert_same_bits(v, stored(self.fmt, np.concatenate(want_v)))
        # the old pages are what they were
        if sum(self.lens):
            k, v = self.cache.read(starts, self.b.kv_len, self.b.pages)
            assert_same_bits(k, stored(self.fmt, self.k))
            assert_same_bits(v, stored(self.fmt, self.v))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens,page,G,D,keep,sinks,recent", [
    ([100], 32, 2, 64, 40, 4, 10),
    ([517, 1, 0, 64, 63, 2000], 64, 8, 128, 64, 4, 20),
    ([33, 70], 32, 3, 96, 33, 0, 0),
    ([300], 128, 2, 256, 1, 0, 0),           # one token
    ([300], 128, 1, 64, 1, 1, 0),
    ([300, 5], 128, 1, 64, 1, 0, 1),
    ([1025], 1024, 2, 64, 1024, 1000, 24),   # nothing is chosen
    ([5003, 3001], 32, 4, 128, 3001, 4, 64),
    ([20011], 256, 1, 64, 9973, 0, 4096),
])
def test_kept_tokens(ctx, fmt, lens, page, G, D, keep, sinks, recent):
    print(f"evict fmt={fmt} lens={lens} page={page} G={G} D={D} keep={keep} {sinks} {recent}", flush=True)
    c = Case(ctx, np.random.default_rng(sum(lens) + D), fmt, lens, page, G, D, keep)
    c.check(c.cache.evict(c.b.kv_len, c.b.pages, c.to, keep, c.mass, sinks, recent), sinks, recent)
    c.cache.close()


@pytest.mark.parametrize("kind", ["one value", "few values", "zeros", "special", "nan", "falling", "rising", "near"])
def test_weights_that_are_alike_or_unusual(ctx, kind):
    rng = np.random.default_rng(2)
    c = Case(ctx, rng, F16, [3000, 2050], 64, 2, 64, 999)
    m = c.mass
    if kind == "one value":
        m[:] = 0.5
    elif kind == "few values":
        m[:] = rng.integers(0, 3, m.shape)
    elif kind == "zeros":
        m[:] = np.where(rng.random(m.shape) < 0.5, np.float32(0), np.float32(-0.0))
        m[:, :, 1500] = 1e-45
        m[:, :, 3] = -1e-45
    elif kind == "special":
        m *= np.where(rng.random(m.shape) < 0.3, -1, 1)
        for i, v in enumerate([np.inf, -np.inf, 3e38, -3e38, 1e-40, -1e-40]):
            m[:, :, 100 + 7 * i] = v
            m[:, :, 1400 + i] = v
    elif kind == "nan":
        m[:, :, ::2] = np.nan
        m[0, 0, 1::4] = -np.nan
        m[1, 1] = np.nan
    elif kind == "falling":
        m[:] = -np.arange(3000)
    elif kind == "rising":
        m[:] = np.arange(3000)
    else:  # values that differ in their last bits alone
        m[:] = (np.float32(1).view(np.int32) + rng.integers(0, 900, m.shape)).astype(np.int32).view(np.float32)
    c.check(c.cache.evict(c.b.kv_len, c.b.pages, c.to, 999, m, 5, 40), 5, 40)
    c.cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_special_values_move_as_they_are(ctx, fmt):
    """Infinities and NaNs, and INT8 scales next to nothing, keep their bits."""
    rng = np.random.default_rng(3)
    c = Case(ctx, rng, fmt, [70], 32, 2, 64, 50)
    c.k[3, 0, 5], c.k[60, 1, 0], c.v[61, 0, 1] = np.inf, np.nan, -np.inf
    c.k[2] *= 1e-41
    c.v[4] = 0
    c.cache.write(c.b.whole(), c.b.kv_len, c.b.pages, c.k, c.v)
    c.check(c.cache.evict(c.b.kv_len, c.b.pages, c.to, 50, c.mass, 5, 12), 5, 12)
    c.cache.close()


def on_device(c, kv_len=None, pages=None, to=None, mass=None, stride=None, moved=True, sinks=3, recent=9):
    """evict_dev on the case's arrays, with guards behind every output."""
    S, G, keep = len(c.lens), c.G, c.keep
    ln, pg = ints(c.b.kv_len if kv_len is None else kv_len), ints(c.b.pages if pages is None else pages)
    tp = ints(c.to if to is None else to)
    mass = c.mass if mass is None else mass
    stride = stride or mass.shape[2]
    m = DeviceArray(S * G * stride)
    whole = np.full((S, G, stride), np.nan, np.float32)
    whole[:, :, :mass.shape[2]] = mass[:, :, :stride]
    m.upload(whole)
    kept, new_len = DeviceArray(S * G * keep + 1, fill=7.0), DeviceArray(S + 1, fill=7.0)
    mo = DeviceArray(S * G * (keep + 5) + 1, fill=7.0)
    b = nx.KvBatch(S, 0, c.b.max_pages, 0, ln.ptr, pg.ptr)
    c.cache.evict_dev(b, tp.ptr, c.to.shape[1], keep, sinks, recent, m.ptr, stride, kept.ptr, new_len.ptr,
                      mo.ptr if moved else 0, keep + 5 if moved else 0)
    c.cache.ctx.sync()
    k, n, w = kept.download(), new_len.download(), mo.download()
    assert k[-1] == n[-1] == w[-1] == 7.0
    w = w[:-1].reshape(S, G, keep + 5)
    n = n[:-1].view(np.int32)
    for s in range(S):
        assert (w[s, :, n[s] if moved else 0:] == 7.0).all()
    return k[:-1].view(np.int32).reshape(S, G, keep), n, w[:, :, :keep] if moved else None


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("moved", [True, False])
def test_device_call(ctx, fmt, moved):
    c = Case(ctx, np.random.default_rng(4), fmt, [300, 40, 0, 129], 32, 3, 96, 77)
    c.check(on_device(c, stride=311, moved=moved), 3, 9)
    c.cache.close()


def test_weights_of_fewer_tokens(ctx):
    """Tokens behind the rows of weights count as NaN."""
    c = Case(ctx, np.random.default_rng(5), F16, [300, 90], 32, 2, 64, 77)
    got = on_device(c, stride=100)
    short = np.full_like(c.mass, np.nan)
    short[:, :, :100] = c.mass[:, :, :100]
    for s in range(2):
        for g in range(2):
            assert np.array_equal(got[0][s, g], evicted(short[s, g], c.lens[s], 77, 3, 9))
            assert not got[2][s, g][got[0][s, g] >= 100].any()
    c.cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_tables_that_name_no_page(ctx, fmt):
    """Missing old pages move as zeros, missing new ones are left out, and lengths are cut to
    the table; nothing else is written."""
    rng = np.random.default_rng(6)
    c = Case(ctx, rng, fmt, [200, 160], 32, 2, 64, 64)
    pages, to = c.b.pages.copy(), c.to.copy()
    pages[0, 2], pages[1, 1] = -1, c.b.num_pages
    lost, to[1, 1] = to[1, 1], 1 << 30
    kept, new_len, _ = on_device(c, kv_len=[10 ** 9, -5], pages=pages, to=to)
    assert new_len.tolist() == [64, 0] and (kept[1] == -1).all()
    # the table holds 224 tokens of the first sequence, of which 24 are what an empty page has
    mass = np.full((2, 224), np.nan, np.float32)
    mass[:, :200] = c.mass[0]
    k, v = c.cache.read([0, 64], [64], c.to[:1])
    for g in range(2):
        at = evicted(mass[g], 224, 64, 3, 9)
        assert np.array_equal(kept[0, g], at)
        there = (at // 32 != 2) & (at < 200)
        for got, x in ((k, c.k), (v, c.v)):
            want = np.where(there[:, None], stored(fmt, x[np.minimum(at, 199), g]), 0)
            assert_same_bits(got[:, g], want.astype(np.float32))
    k, v = c.cache.read([0, 32], [32], [[lost]])
    assert not k.any() and not v.any()  # as it was
    c.cache.close()


def test_rest_of_the_last_group_is_cleared(ctx):
    """Also where the page held something that is not finite."""
    rng = np.random.default_rng(7)
    c = Case(ctx, rng, F16, [100], 64, 1, 64, 37)
    bad = np.full((64, 1, 64), np.inf, np.float32)
    c.cache.write([0, 64], [64], c.to, bad, bad)
    c.check(c.cache.evict(c.b.kv_len, c.b.pages, c.to, 37, c.mass), 0, 0)
    k, v = c.cache.read([0, 64], [64], c.to)
    assert not k[37:].any() and not v[37:].any()
    c.cache.close()


def test_refusals(ctx):
    c = Case(ctx, np.random.default_rng(8), F16, [100, 50], 32, 2, 64, 40)
    a = DeviceArray(4096)

    def code(S=2, mp=c.b.max_pages, ln=a.ptr, pg=a.ptr, to=a.ptr, tmp=2, keep=40, sinks=1, recent=2, m=a.ptr,
             ms=200, kept=a.ptr, nl=a.ptr + 64, nm=a.ptr + 4000, nms=40):
        with pytest.raises(nx.NexusError) as e:
            c.cache.evict_dev(nx.KvBatch(S, 0, mp, 0, ln, pg), to, tmp, keep, sinks, recent, m, ms, kept, nl, nm, nms)
        return e.value.code

    assert code(S=-1) == code(keep=0) == code(keep=-3) == code(sinks=-1) == code(recent=-1) == nx.NX_ERR_INVALID_ARG
    assert code(ln=0) == code(pg=0) == code(to=0) == code(m=0) == code(kept=0) == code(nl=0) == nx.NX_ERR_INVALID_ARG
    assert code(sinks=30, recent=11) == code(mp=0) == code(tmp=0) == code(ms=0) == code(nms=39) == nx.NX_ERR_SHAPE
    assert code(nm=a.ptr) == code(nm=a.ptr + 16) == nx.NX_ERR_INVALID_ARG  # new weights over old ones
    assert code(nl=a.ptr) == code(nl=a.ptr + 4) == nx.NX_ERR_INVALID_ARG  # new lengths over old ones
    # host arrays are looked at
    good = (c.b.kv_len, c.b.pages, c.to)

    def host(kv_len=good[0], pages=good[1], to=good[2], keep=40, mass=c.mass):
        with pytest.raises(nx.NexusError) as e:
            c.cache.evict(kv_len, pages, to, keep, mass)
        return e.value.code

    twice, old, off = c.to.copy(), c.to.copy(), c.to.copy()
    twice[1, 0], old[0, 0], off[1, 1] = c.to[0, 0], c.b.pages[1, 0], c.b.num_pages
    assert host(to=twice) == host(to=old) == host(to=off) == nx.NX_ERR_INVALID_ARG
    bad = c.b.pages.copy()
    bad[0, 1] = -1
    assert host(pages=bad) == nx.NX_ERR_INVALID_ARG
    assert host(kv_len=[-1, 50]) == host(kv_len=[1000, 50]) == host(mass=c.mass[:, :, :99]) == nx.NX_ERR_SHAPE
    assert host(to=c.to[:, :1]) == nx.NX_ERR_SHAPE
    c.check(c.cache.evict(*good, 40, c.mass), 0, 0)
    none = nx.KvBatch(0, 0, 0, 0, 0, 0)
    c.cache.evict_dev(none, 0, 0, 5, 0, 0, 0, 0, 0, 0)
    c.cache.close()
