"""The calls around the cache (nx_kv_evict, nx_attention_mass, nx_logprobs, nx_qk_rope) at the edges of
what they accept, against formulas in 64 bits."""
import numpy as np
import pytest

import nexus_amd as nx
from kv_cases import F16, INT8, Batch, random_kv, stored
from moe_cases import DeviceArray, assert_same_bits
from test_gpu_evict import Case

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
