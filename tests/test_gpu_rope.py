"""Query and key heads, normed and rotated (nx_qk_rope), against the formula in 64 bits."""
import numpy as np
import pytest

import nexus_amd as nx
from moe_cases import DeviceArray
from step_cases import HALVES, PAIRS, rope
from test_gpu_kv import ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


def angles(R, base=1e4):
    return (base ** (-np.arange(0, R, 2) / max(R, 1))).astype(np.float32)


def check(got, positions, x, freq, style, weight, eps):
    ref, bound = rope(positions, x, freq, style, weight, eps)
    err = np.abs(got.astype(np.float64) - ref)
    assert np.all(err <= bound), float((err / bound).max())


@pytest.mark.parametrize("style", [HALVES, PAIRS])
@pytest.mark.parametrize("T,H,G,D,R,norm", [
    (1, 32, 8, 128, 128, True),
    (1, 1, 0, 64, 64, False),
    (5, 0, 3, 96, 96, True),
    (61, 16, 8, 256, 256, True),
    (33, 12, 12, 96, 32, True),
    (7, 4, 2, 128, 40, False),
    (3, 130, 1, 64, 16, True),     # more heads than one workgroup takes
    (2, 3, 1, 512, 512, True),     # the widest
    (9, 5, 2, 512, 0, True),       # a norm alone
    (4, 2, 1, 2, 2, True),         # the narrowest
    (6, 7, 3, 80, 20, True),       # R no multiple of 8
    (5, 3, 1, 90, 90, True),       # nor D
    (3, 9, 2, 130, 62, False),
    (1021, 24, 1, 128, 64, True),
])
def test_against_formula(ctx, style, T, H, G, D, R, norm):
    print(f"rope style={style} T={T} H={H} G={G} D={D} R={R} norm={norm}", flush=True)
    rng = np.random.default_rng(T + H + D + R)
    q, k = (rng.standard_normal((T, n, D), dtype=np.float32) for n in (H, G))
    wq, wk = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in "qk")
    positions = rng.integers(0, 1 << 17, T)
    freq = angles(R)
    gq, gk = ctx.qk_rope(positions, q, k, freq, style, wq, wk, 1e-5)
    check(gq, positions, q, freq, style, wq, 1e-5)
    check(gk, positions, k, freq, style, wk, 1e-5)


def test_one_side_normed(ctx):
    rng = np.random.default_rng(3)
    q, k = (rng.standard_normal((9, n, 128), dtype=np.float32) for n in (8, 2))
    w, positions, freq = rng.standard_normal(128).astype(np.float32), np.arange(9), angles(128)
    for wq, wk in ((w, None), (None, w)):
        gq, gk = ctx.qk_rope(positions, q, k, freq, HALVES, wq, wk)
        check(gq, positions, q, freq, HALVES, wq, 1e-6)
        check(gk, positions, k, freq, HALVES, wk, 1e-6)


@pytest.mark.parametrize("D", [128, 90])
def test_far_positions(ctx, D):
    """Angles of up to 2^31 radians, either sign, and a freq that is no power of two."""
    rng = np.random.default_rng(4)
    positions = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 10 ** 9, 77777777])
    q = rng.standard_normal((len(positions), 2, D), dtype=np.float32)
    freq = np.linspace(0.1, 1, D // 2).astype(np.float32)
    gq, _ = ctx.qk_rope(positions, q, None, freq, HALVES)
    check(gq, positions, q, freq, HALVES, None, 0)


@pytest.mark.parametrize("D", [64, 62])
def test_magnitudes(ctx, D):
    """Squares past f32's range either way, rows of zeros, eps 0."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 1, D), dtype=np.float32)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3] *= 1e-40  # subnormal
    w, freq = np.ones(D, np.float32), angles(D)
    gq, _ = ctx.qk_rope(np.arange(6), x, None, freq, PAIRS, w, None, 1e-6)
    check(gq, np.arange(6), x, freq, PAIRS, w, 1e-6)
    assert not gq[2].any()
    keep = [0, 1, 4, 5]
    gq, _ = ctx.qk_rope(np.arange(6)[keep], x[keep], None, freq, PAIRS, w, None, 0.0)
    check(gq, np.arange(6)[keep], x[keep], freq, PAIRS, w, 0.0)


@pytest.mark.parametrize("D", [128, 66])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_non_finite_values_stay_in_their_head(ctx, D, bad):
    rng = np.random.default_rng(6)
    q = rng.standard_normal((4, 3, D), dtype=np.float32)
    clean, _ = ctx.qk_rope(np.arange(4), q, None, angles(D), HALVES, np.ones(D, np.float32))
    q[2, 1, 5] = bad
    got, _ = ctx.qk_rope(np.arange(4), q, None, angles(D), HALVES, np.ones(D, np.float32))
    got[2, 1] = clean[2, 1] = 0
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("shift,extra", [(0, 0), (0, 12), (0, 2), (1, 0), (3, 5)])
@pytest.mark.parametrize("in_place", [True, False])
def test_rows_of_a_fused_projection(ctx, shift, extra, in_place):
    """q and k as columns of wider rows at any float address, in place or not; the other
    columns, and rows behind the last, are left as they were."""
    rng = np.random.default_rng(7)
    T, H, G, D = 13, 6, 2, 64
    width, stride = (H + 2 * G) * D, (H + 2 * G) * D + extra
    rows = rng.standard_normal((T + 2, stride)).astype(np.float32)
    w, freq, positions = (1 + rng.random(D)).astype(np.float32), angles(32), np.arange(T) * 37
    src = DeviceArray(rows.size + 8)
    src.upload(rows, shift)
    out = src if in_place else DeviceArray(rows.size + 8, fill=7.0)
    dw, df, dp = DeviceArray(D), DeviceArray(16), ints(positions)
    dw.upload(w), df.upload(freq)
    r = nx.Rope(D, 32, df.ptr, HALVES, dw.ptr, 0, eps=1e-6)
    a, b = src.ptr + 4 * shift, out.ptr + 4 * shift
    ctx.qk_rope_dev(r, dp.ptr, T, H, G, a, stride, a + 4 * H * D, stride, b, stride, b + 4 * H * D, stride)
    ctx.sync()
    got = out.download()[shift:shift + rows.size].reshape(rows.shape)
    q, k = rows[:T, :H * D].reshape(T, H, D), rows[:T, H * D:(H + G) * D].reshape(T, G, D)
    check(got[:T, :H * D].reshape(q.shape), positions, q, freq, HALVES, w, 1e-6)
    check(got[:T, H * D:(H + G) * D].reshape(k.shape), positions, k, freq, HALVES, None, 0)
    rest = rows if in_place else np.full_like(rows, 7.0)
    assert np.array_equal(got[:T, (H + G) * D:], rest[:T, (H + G) * D:])
    assert np.array_equal(got[T:], rest[T:])
    assert width <= stride


def test_nothing_to_do(ctx):
    r = nx.Rope(64, 64, 0, HALVES)
    ctx.qk_rope_dev(r, 0, 0, 4, 1, 0, 0, 0, 0, 0, 0, 0, 0)
    ctx.qk_rope_dev(r, 0, 5, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def test_refusals(ctx):
    a, f, p = DeviceArray(4096), DeviceArray(32), DeviceArray(16)

    def code(D=64, R=64, style=HALVES, eps=1e-6, T=4, H=2, G=1, freq=f.ptr, pos=p.ptr, q=a.ptr, qs=256,
             k=a.ptr + 512, ks=256, qo=a.ptr, qos=256, ko=a.ptr + 512, kos=256):
        with pytest.raises(nx.NexusError) as e:
            ctx.qk_rope_dev(nx.Rope(D, R, freq, style, eps=eps), pos, T, H, G, q, qs, k, ks, qo, qos, ko, kos)
        return e.value.code

    assert code(T=-1) == code(H=-1) == code(D=0) == code(R=-2) == code(style=2) == nx.NX_ERR_INVALID_ARG
    assert code(eps=-1.0) == code(eps=np.inf) == code(eps=np.nan) == nx.NX_ERR_INVALID_ARG
    assert code(R=66) == code(qs=100) == code(kos=63) == nx.NX_ERR_SHAPE
    assert code(D=65, R=64) == code(R=63) == code(D=514, R=2) == code(H=65537) == nx.NX_ERR_UNSUPPORTED
    assert code(freq=0) == code(pos=0) == code(q=0) == code(ko=0) == nx.NX_ERR_INVALID_ARG
    # outputs that overlap other rows than their own
    assert code(qo=a.ptr + 4) == code(qos=260) == code(ko=a.ptr + 256) == code(qo=a.ptr + 512) == nx.NX_ERR_INVALID_ARG
