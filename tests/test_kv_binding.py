"""What the Python binding of the cache makes of host arrays (no device)."""
import numpy as np
import pytest

import nexus_amd as nx


@pytest.fixture
def cache():
    c = object.__new__(nx.KvCache)
    c.h, c.kv_heads, c.head_dim = None, 2, 64
    return c


def test_page_tables_of_other_sequences_are_refused(cache):
    """A row of pages for each sequence: tables of more or fewer are not cut up anew."""
    for pages in (np.zeros((4, 8)), np.zeros((1, 8)), np.zeros((2, 4, 2)), np.zeros((0, 8))):
        with pytest.raises(ValueError):
            cache._host_batch([0, 1, 2], [3, 4], pages, 2)
    with pytest.raises(ValueError):
        cache._host_batch([0, 1, 2], [3, 4], np.arange(5), 2)
    with pytest.raises(ValueError):
        cache._host_batch([0, 1], [3, 4], np.zeros((2, 8)), 2)
    for pages in (np.arange(16).reshape(2, 8), np.arange(16), np.arange(32).reshape(2, 16)[:, ::2] // 2):
        b, (_, _, kept) = cache._host_batch([0, 1, 2], [3, 4], pages, 2)
        assert (b.c.num_seqs, b.c.max_pages) == (2, 8)
        assert np.array_equal(kept, np.arange(16).reshape(2, 8))


def test_no_sequences(cache):
    """A step without sequences is one that the library takes (and does nothing for)."""
    for pages in (np.zeros((0, 8)), np.zeros((0, 0)), []):
        b, _ = cache._host_batch([0], [], pages, 0)
        assert (b.c.num_seqs, b.c.num_tokens) == (0, 0)


def test_rows_of_no_width(cache):
    for width in (0, -64):
        with pytest.raises(ValueError):
            cache._rows(np.zeros((2, 64)), width)
    with pytest.raises(ValueError):
        cache.read([], [], [])
    with pytest.raises(ValueError):
        cache.attention([0, 1], [1], [[0]], np.zeros((1, 64)), 0)
