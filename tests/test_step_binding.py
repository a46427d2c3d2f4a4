"""What the Python binding of the calls around the cache makes of host arrays (no device)."""
import numpy as np
import pytest

import nexus_amd as nx


@pytest.fixture
def ctx():
    c = object.__new__(nx.Context)
    c.h = None
    return c


@pytest.fixture
def cache():
    c = object.__new__(nx.KvCache)
    c.h, c.kv_heads, c.head_dim = None, 2, 64
    c.ctx = object.__new__(nx.Context)
    c.ctx.h = None
    return c


def test_heads_of_other_shapes_are_refused(ctx):
    q, k, freq = np.zeros((3, 4, 64)), np.zeros((3, 2, 64)), np.zeros(32)
    for bad in ((q[:2], k), (q, k[:, :, :32]), (q[0], k), (q.reshape(3, 256), k)):
        with pytest.raises(ValueError):
            ctx.qk_rope(np.arange(3), *bad, freq)
    for norms in (dict(q_norm=np.ones(63)), dict(k_norm=np.ones((2, 64)))):
        with pytest.raises(ValueError):
            ctx.qk_rope(np.arange(3), q, k, freq, **norms)


def test_rows_of_other_shapes_are_refused(ctx):
    for x, t, top in ((np.zeros(5), None, 0), (np.zeros((3, 0)), None, 0), (np.zeros((3, 5)), np.zeros(3), 0),
                      (np.zeros((3, 5)), np.zeros((2, 1)), 0), (np.zeros((3, 5)), None, -1)):
        with pytest.raises(ValueError):
            ctx.logprobs(x, t, top)


def test_weights_of_other_shapes_are_refused(cache):
    good = dict(kv_len=[5, 6], pages=np.zeros((2, 4)), to_pages=np.zeros((2, 1)), keep=3, mass=np.zeros((2, 2, 8)))
    for name, bad in (("mass", np.zeros((2, 8))), ("mass", np.zeros((1, 2, 8))), ("mass", np.zeros((2, 3, 8))),
                      ("to_pages", np.zeros(2)), ("to_pages", np.zeros((3, 1))), ("pages", np.zeros((3, 4))),
                      ("keep", -1)):
        with pytest.raises(ValueError):
            cache.evict(**{**good, name: bad})
    q = np.zeros((2, 4 * 64))
    for before in (np.zeros((2, 8)), np.zeros((2, 1, 8)), np.zeros((3, 2, 8))):
        with pytest.raises(ValueError):
            cache.attention_mass([0, 1, 2], [5, 6], np.zeros((2, 4)), q, 4, before=before)
    with pytest.raises(ValueError):
        cache.attention_mass([0, 1, 2], [5, 6], np.zeros((2, 4)), np.zeros((2, 65)), 4)


def test_a_null_context_is_an_error(ctx, cache):
    """The C entries look at the context first."""
    for call in (lambda: ctx.qk_rope(np.arange(1), np.zeros((1, 2, 64)), None, np.zeros(32)),
                 lambda: ctx.logprobs(np.zeros((1, 5))),
                 lambda: cache.evict([5], np.zeros((1, 4)), np.zeros((1, 1)), 3, np.zeros((1, 2, 8))),
                 lambda: cache.attention_mass([0, 1], [5], np.zeros((1, 4)), np.zeros((1, 256)), 4)):
        with pytest.raises(nx.NexusError) as e:
            call()
        assert e.value.code == nx.NX_ERR_INVALID_ARG and "null context" in str(e.value)
