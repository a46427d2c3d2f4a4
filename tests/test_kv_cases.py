"""The references of the cache and attention tests against each other (CPU only)."""
import numpy as np
import pytest

from kv_cases import Batch, attention, attention_dense, random_kv


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (40, 100)])
def test_both_forms_agree(window, sinks):
    rng = np.random.default_rng(1)
    b = Batch(rng, [5, 0, 1, 30], [40, 3, 1, 30], 32, first_row=2, padding=1)
    k, v = random_kv(rng, sum(b.lens), 2, 64)
    q = rng.standard_normal((b.rows, 6, 64)).astype(np.float32)
    for one, other in zip(attention(b, k, v, q, 6, 0.125, window, sinks),
                          attention_dense(b, k, v, q, 6, 0.125, window, sinks)):
        assert np.allclose(one, other, rtol=1e-12, atol=1e-14)
