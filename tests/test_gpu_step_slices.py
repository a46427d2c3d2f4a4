"""Calls around the cache that are so large that they go in several launches (a launch has fewer than
2^32 threads): rotations and log probabilities of more than 2^22 rows, evictions of more than 2^20
sequences' heads and 2^23 groups of kept tokens.  The formulas in 64 bits, all rows at once."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, stored
from moe_cases import DeviceArray, assert_same_bits
from step_cases import HALVES, U, rope
from test_gpu_kv import ints

pytestmark = pytest.mark.gpu
ROWS = (1 << 22) + 77


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("D", [8, 2])  # whole float4, and not
def test_rotation_of_more_rows_than_a_launch_takes(ctx, D):
    rng = np.random.default_rng(61)
    x = rng.standard_normal((ROWS, 1, D), dtype=np.float32)
    positions, freq = rng.integers(0, 100000, ROWS), np.linspace(0.5, 1, D // 2).astype(np.float32)
    w = (1 + rng.random(D)).astype(np.float32)
    d, p, df, dw = DeviceArray(x.size + 1, fill=7.0), ints(positions), DeviceArray(D // 2), DeviceArray(D)
    d.upload(x), df.upload(freq), dw.upload(w)
    ctx.qk_rope_dev(nx.Rope(D, D, df.ptr, HALVES, dw.ptr, 0, eps=1e-6), p.ptr, ROWS, 1, 0, d.ptr, D, 0, 0, d.ptr, D, 0, 0)
    ctx.sync()
    got = d.download()
    assert got[-1] == 7.0
    ref, bound = rope(positions, x, freq, HALVES, w, 1e-6)
    assert (np.abs(got[:-1].reshape(x.shape) - ref) <= bound).all()


def test_log_probabilities_of_more_rows_than_a_launch_takes(ctx):
    rng = np.random.default_rng(62)
    V = 5
    x = (2 * rng.standard_normal((ROWS, V))).astype(np.float32)
    tokens = rng.integers(0, V, ROWS)
    d, t, lp, ent = DeviceArray(x.size), ints(tokens), DeviceArray(ROWS + 1, fill=7.0), DeviceArray(ROWS + 1, fill=7.0)
    ids, tlp = DeviceArray(2 * ROWS + 1, fill=7.0), DeviceArray(2 * ROWS + 1, fill=7.0)
    d.upload(x)
    ctx.logprobs_dev(d.ptr, V, ROWS, V, t.ptr, 1, lp.ptr, ent.ptr, 2, ids.ptr, tlp.ptr)
    ctx.sync()
    lp, ent, ids, tlp = (a.download() for a in (lp, ent, ids, tlp))
    assert lp[-1] == ent[-1] == ids[-1] == tlp[-1] == 7.0
    r = x.astype(np.float64)
    m = r.max(1, keepdims=True)
    e = np.exp(r - m)
    p = e / e.sum(1, keepdims=True)
    logp = r - m - np.log(e.sum(1, keepdims=True))
    spread = (p * (m - r)).sum(1)
    order = np.argsort(-x, axis=1, kind="stable")[:, :2]
    assert np.array_equal(ids[:-1].view(np.int32).reshape(ROWS, 2), order)
    rows = np.arange(ROWS)
    for got, ref, wide in ((lp[:-1], logp[rows, tokens], spread), (ent[:-1], -(p * logp).sum(1), spread),
                           (tlp[:-1].reshape(ROWS, 2), np.take_along_axis(logp, order, 1), spread[:, None])):
        assert (np.abs(got - ref) <= 16 * U * (1 + np.abs(ref) + wide)).all()


def test_eviction_of_more_heads_than_a_launch_takes(ctx):
    """1100 sequences of 4096 heads, of which seven have tokens: at the ends, and where a launch begins
    (256 sequences of the choice, 1024 of the move)."""
    rng = np.random.default_rng(63)
    S, G, D, page, n, keep = 1100, 4096, 64, 32, 40, 33
    there = [0, 255, 256, 511, 1023, 1024, 1099]
    order = rng.permutation(4 * len(there) + 1).astype(np.int32)
    pages, to = np.full((S, 2), -1, np.int32), np.full((S, 2), -1, np.int32)
    pages[there], to[there] = order[:14].reshape(-1, 2), order[14:28].reshape(-1, 2)
    lens = np.zeros(S, np.int32)
    lens[there] = n
    cache = nx.KvCache(ctx, F16, len(order), page, G, D)
    starts = (n * np.arange(len(there) + 1)).astype(np.int32)
    k = rng.standard_normal((n * len(there), G, D), dtype=np.float32)
    cache.write(starts, lens[there], pages[there], k, -k)
    weights = rng.integers(0, 1000, (len(there), G, n)).astype(np.float32)  # some are alike
    mass, new_mass = DeviceArray(S * G * n), DeviceArray(S * G * keep + 1)
    kept, new_len = DeviceArray(S * G * keep + 1), DeviceArray(S + 1, fill=7.0)
    for i, s in enumerate(there):
        mass.upload(weights[i], s * G * n)
    for d in (kept, new_mass):
        d.upload([7.0], S * G * keep)
    ln, pg, tp = ints(lens), ints(pages), ints(to)
    cache.evict_dev(nx.KvBatch(S, 0, 2, 0, ln.ptr, pg.ptr), tp.ptr, 2, keep, 1, 2, mass.ptr, n, kept.ptr, new_len.ptr,
                    new_mass.ptr, keep)
    ctx.sync()
    kept, new_mass, got_len = (d.download() for d in (kept, new_mass, new_len))
    assert kept[-1] == new_mass[-1] == got_len[-1] == 7.0
    assert np.array_equal(got_len[:-1].view(np.int32), np.minimum(lens, keep))
    kept, new_mass = kept[:-1].view(np.int32).reshape(S, G, keep), new_mass[:-1].reshape(S, G, keep)
    for s in (1, 254, 257, 1022, 1025, 1098):
        assert (kept[s] == -1).all()
    w = weights.copy()
    w[:, :, 0] = w[:, :, -2:] = 2000
    want = np.sort(np.argsort(-w, axis=2, kind="stable")[:, :, :keep], axis=2)
    assert np.array_equal(kept[there], want)
    assert np.array_equal(new_mass[there], np.take_along_axis(weights, want, 2))
    gk, gv = cache.read((keep * np.arange(len(there) + 1)).astype(np.int32), np.full(len(there), keep, np.int32), to[there])
    for i in range(len(there)):
        x = np.take_along_axis(k[n * i:n * i + n], want[i].T[:, :, None], 0)
        assert_same_bits(gk[keep * i:keep * i + keep], stored(F16, x))
        assert_same_bits(gv[keep * i:keep * i + keep], stored(F16, -x))
    cache.close()
