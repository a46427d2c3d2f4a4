"""Log probabilities, entropy and the likeliest tokens (nx_logprobs), against the formulas in 64 bits."""
import numpy as np
import pytest

import nexus_amd as nx
from moe_cases import DeviceArray
from step_cases import check_logprobs
from test_gpu_kv import ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


def logits(rng, T, V):
    x = (2.5 * rng.standard_normal((T, V))).astype(np.float32)
    x[np.arange(T), rng.integers(0, V, T)] += np.float32(7)
    return x


@pytest.mark.parametrize("T,V,given,top", [
    (1, 32000, 1, 20),
    (1, 1, 1, 1),
    (3, 2, 2, 5),            # fewer tokens than alternatives
    (2, 63, 1, 64),
    (5, 65, 0, 64),
    (7, 1021, 3, 20),
    (1, 200003, 1, 64),
    (61, 4099, 1, 5),
    (300, 1500, 1, 1),
    (2500, 130, 1, 3),       # more rows than are split
    (1100, 4097, 1, 20),
    (9, 100003, 1, 0),
])
def test_against_formula(ctx, T, V, given, top):
    print(f"logprobs T={T} V={V} given={given} top={top}", flush=True)
    rng = np.random.default_rng(T + V)
    x = logits(rng, T, V)
    tokens = rng.integers(0, V, (T, given)).astype(np.int32)
    check_logprobs(ctx.logprobs(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("V", [7, 300, 5000, 70001])
def test_ties_go_to_the_lower_id(ctx, V):
    """Rows of few different values, of one value, and of zeros of both signs."""
    rng = np.random.default_rng(V)
    x = rng.integers(-2, 3, (6, V)).astype(np.float32)
    x[1] = 3.25
    x[2] = np.where(rng.random(V) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[3, V // 2:] = x[3, 0] = 9
    tokens = np.zeros((6, 1), np.int32)
    for top in (1, 5, 64):
        check_logprobs(ctx.logprobs(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(ctx, order):
    """Every logit passes what came before it, or none does."""
    x = np.sort(logits(np.random.default_rng(8), 3, 30011), axis=1)[:, ::order].copy()
    tokens = np.full((3, 1), 5, np.int32)
    check_logprobs(ctx.logprobs(x, tokens, 33), x, tokens, 33)


@pytest.mark.parametrize("V", [9, 2048, 33333])
def test_masked_tokens(ctx, V):
    """Tokens taken out by -infinity, all but a few and all; masks of the lowest value."""
    rng = np.random.default_rng(V)
    x = logits(rng, 7, V)
    x[0, rng.random(V) < 0.5] = -np.inf
    x[1, 1:] = -np.inf
    x[2, :-3] = -np.inf
    x[3] = -np.inf
    x[4] = np.finfo(np.float32).min
    x[5, 2:] = np.finfo(np.float32).min
    x[6, :2] = np.finfo(np.float32).max
    tokens = rng.integers(0, V, (7, 2)).astype(np.int32)
    tokens[:, 0] = 0
    tokens[5, 1] = 1
    got = ctx.logprobs(x, tokens, 6)
    check_logprobs(got, x, tokens, 6)
    assert got[0][3, 0] == -np.inf and got[1][3] == 0 and (got[2][3] == -1).all() and (got[3][3] == -np.inf).all()
    assert got[2][1, 1] == -1 and got[3][1, 1] == -np.inf and got[0][1, 0] == 0


@pytest.mark.parametrize("V", [50, 20000])
@pytest.mark.parametrize("bad", [np.nan, -np.nan, np.inf])
def test_non_finite_rows(ctx, V, bad):
    """A row with a NaN or +infinity, and its neighbours."""
    rng = np.random.default_rng(9)
    x = logits(rng, 4, V)
    x[1, V // 3] = bad
    x[2, :] = bad
    x[2, 7] = -np.inf
    tokens = rng.integers(0, V, (4, 1)).astype(np.int32)
    check_logprobs(ctx.logprobs(x, tokens, 4), x, tokens, 4)


def test_tokens_that_are_none(ctx):
    x = logits(np.random.default_rng(10), 3, 100)
    tokens = np.array([[-1, 5, 100], [-100, 99, 0], [2 ** 31 - 1, -2 ** 31, 1]], np.int32)
    check_logprobs(ctx.logprobs(x, tokens, 2), x, tokens, 2)


def test_certain_rows(ctx):
    """One token has all but nothing of the probability: entropy is next to 0, never below."""
    x = np.zeros((5, 3000), np.float32)
    x[np.arange(5), [0, 1, 1500, 2998, 2999]] = [10, 20, 40, 80, 3e38]
    tokens = np.array([[0], [1], [0], [2], [0]], np.int32)
    got = ctx.logprobs(x, tokens, 2)
    check_logprobs(got, x, tokens, 2)
    assert (got[1] >= 0).all()


def test_far_apart_logits(ctx):
    """Differences beyond f32's range."""
    x = np.full((2, 4100), -3e38, np.float32)
    x[0, [5, 4099]] = 3e38
    x[1, 4000] = 1e38
    tokens = np.array([[5, 0], [4000, 1]], np.int32)
    got = ctx.logprobs(x, tokens, 3)
    assert np.allclose(got[0], [[-np.log(2), -np.inf], [0, -np.inf]], atol=1e-6, rtol=0) or \
        np.allclose(got[0], [[-np.log(2), -6e38], [0, -4e38]])
    assert np.allclose(got[1], [np.log(2), 0], atol=1e-6)
    assert got[2].tolist() == [[5, 4099, 0], [4000, 0, 1]]


@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (2, 3), (3, 1), (0, 4)])
@pytest.mark.parametrize("T,V", [(3, 5003), (2100, 66)])
def test_strided_and_unaligned_rows(ctx, T, V, shift, extra):
    """Rows at any float address; what lies between them is not looked at, and optional
    outputs are left out."""
    rng = np.random.default_rng(11)
    x = logits(rng, T, V)
    rows = np.full((T, V + extra), np.nan, np.float32)
    rows[:, :V] = x
    d = DeviceArray(rows.size + 8, fill=np.nan)
    d.upload(rows, shift)
    tokens = rng.integers(0, V, (T, 1)).astype(np.int32)
    dt, lp, ent = ints(tokens), DeviceArray(T + 1, fill=7.0), DeviceArray(T + 1, fill=7.0)
    ids, tlp = DeviceArray(4 * T + 1, fill=7.0), DeviceArray(4 * T + 1, fill=7.0)
    ctx.logprobs_dev(d.ptr + 4 * shift, V + extra, T, V, dt.ptr, 1, lp.ptr, ent.ptr, 4, ids.ptr, tlp.ptr)
    ctx.sync()
    out = [lp.download(), ent.download(), ids.download(), tlp.download()]
    assert [float(a[-1]) for a in out] == [7.0] * 4
    got = (out[0][:-1].reshape(T, 1), out[1][:-1], out[2][:-1].view(np.int32).reshape(T, 4), out[3][:-1].reshape(T, 4))
    check_logprobs(got, x, tokens, 4)
    # nothing but alternatives, then nothing but the entropy, then nothing
    ent.upload(np.full(T + 1, 7.0)), tlp.upload(np.full(4 * T + 1, 7.0))
    ctx.logprobs_dev(d.ptr + 4 * shift, V + extra, T, V, 0, 0, 0, 0, 4, ids.ptr, tlp.ptr)
    ctx.logprobs_dev(d.ptr + 4 * shift, V + extra, T, V, 0, 0, 0, ent.ptr, 0, 0, 0)
    ctx.logprobs_dev(d.ptr + 4 * shift, V + extra, T, V, 0, 0, 0, 0, 0, 0, 0)
    ctx.sync()
    check_logprobs((np.zeros((T, 0)), ent.download()[:-1], ids.download()[:-1].view(np.int32).reshape(T, 4),
                    tlp.download()[:-1].reshape(T, 4)), x, np.zeros((T, 0), int), 4)


def test_runs_are_alike(ctx):
    """The last workgroup of a row joins the parts in their order, whichever it is."""
    x = logits(np.random.default_rng(12), 5, 150001)
    tokens = np.arange(5, dtype=np.int32)[:, None]
    first = ctx.logprobs(x, tokens, 20)
    for _ in range(5):
        for a, b in zip(first, ctx.logprobs(x, tokens, 20)):
            assert np.array_equal(a, b)


def test_refusals(ctx):
    a, i = DeviceArray(256), DeviceArray(256)

    def code(x=a.ptr, stride=64, T=2, V=64, t=i.ptr, given=1, lp=a.ptr, top=2, ids=i.ptr, tlp=a.ptr):
        with pytest.raises(nx.NexusError) as e:
            ctx.logprobs_dev(x, stride, T, V, t, given, lp, a.ptr, top, ids, tlp)
        return e.value.code

    assert code(T=-1) == code(V=0) == code(V=-5) == code(given=-1) == code(top=-1) == nx.NX_ERR_INVALID_ARG
    assert code(x=0) == code(t=0) == code(lp=0) == code(ids=0) == code(tlp=0) == nx.NX_ERR_INVALID_ARG
    assert code(stride=63) == nx.NX_ERR_SHAPE
    assert code(top=65) == code(T=(1 << 24) + 1) == code(given=(1 << 20) + 1) == nx.NX_ERR_UNSUPPORTED
    ctx.logprobs_dev(0, 64, 0, 64, 0, 1, 0, 0, 1, 0, 0)  # no rows
