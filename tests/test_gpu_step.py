"""The calls around the cache and the attention as a decoder uses them together: heads normed and
rotated, weights gathered, tokens given up, log probabilities; in a layer's steps, in graphs, and on
contexts of their own."""
import ctypes as C

import numpy as np
import pytest

import nexus_amd as nx
import oracle
from kv_cases import F16, INT8, Batch, attention, random_kv, rel_l2, stored
from moe_cases import DeviceArray, assert_same_bits
from step_cases import HALVES, attention_mass, check_logprobs, evicted, rope
from test_gpu_attention_step import Hip
from test_gpu_kv import device_batch, ints

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]
EPS = 1e-5


class Decoder:
    """One layer without its FFN, and an output head: RMSNorm, q/k/v, heads normed and rotated, cache,
    attention, output projection, residual, RMSNorm, logits."""

    H, heads, G, D, V = 256, 4, 2, 64, 500

    def __init__(self, ctx, rng):
        self.ctx = ctx
        near = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
        self.norm1, self.norm2, self.wq, self.wk = near(self.H), near(self.H), near(self.D), near(self.D)
        self.width = (self.heads + 2 * self.G) * self.D
        self.mats = [self.matrix(rng, r, c) for r, c in ((self.width, self.H), (self.H, self.heads * self.D),
                                                         (self.V, self.H))]
        self.freq = (1e4 ** (-np.arange(0, self.D, 2) / self.D)).astype(np.float32)
        self.keep = []
        self.rope = nx.Rope(self.D, self.D, self.up(self.freq), HALVES, self.up(self.wq), self.up(self.wk), eps=EPS)
        self.n1, self.n2 = self.up(self.norm1), self.up(self.norm2)

    def up(self, a):
        d = DeviceArray(a.size)
        d.upload(a)
        self.keep.append(d)
        return d.ptr

    def matrix(self, rng, rows, cols):
        q = oracle.quantize(nx.Q8_0, (0.1 * rng.standard_normal((rows, cols))).astype(np.float32))
        m = nx.Matrix(self.ctx, nx.Q8_0, rows, cols)
        m.load(q)
        return m, oracle.dequantize(nx.Q8_0, q, rows * cols).reshape(rows, cols).astype(np.float64)

    def step(self, cache, batch, positions, x, mass, stride, tokens, top):
        """The device's calls of a step on hidden rows x: logits, what they say, and mass in place."""
        T, HD, GD = len(x), self.heads * self.D, self.G * self.D
        dx, dn, rows = DeviceArray(x.size), DeviceArray(x.size), DeviceArray(T * self.width)
        att, logits = DeviceArray(T * HD), DeviceArray(T * self.V)
        dx.upload(x)
        d, pos, dt = device_batch(batch), ints(positions), ints(tokens)
        qkv, o, head = (m for m, _ in self.mats)
        self.ctx.rms_norm_dev(dx.ptr, x.size, self.n1, self.H, EPS, T, self.H, dn.ptr)
        qkv.matvec_dev(dn.ptr, x.size, T, rows.ptr)
        k = rows.ptr + 4 * HD
        self.ctx.qk_rope_dev(self.rope, pos.ptr, T, self.heads, self.G, rows.ptr, self.width, k, self.width, rows.ptr,
                             self.width, k, self.width)
        cache.write_dev(d, k, k + 4 * GD, self.width)
        cache.attention_dev(d, rows.ptr, self.width, self.heads, att.ptr, HD, self.D ** -0.5)
        cache.attention_mass_dev(d, rows.ptr, self.width, self.heads, mass.ptr, mass.ptr, stride, self.D ** -0.5)
        out = DeviceArray(x.size)
        o.matvec_dev(att.ptr, T * HD, T, out.ptr)
        self.ctx.sync()
        dx.upload(x + out.download().reshape(x.shape))
        self.ctx.rms_norm_dev(dx.ptr, x.size, self.n2, self.H, EPS, T, self.H, dn.ptr)
        head.matvec_dev(dn.ptr, x.size, T, logits.ptr)
        lp, ent, ids, tlp = DeviceArray(T), DeviceArray(T), DeviceArray(T * top), DeviceArray(T * top)
        self.ctx.logprobs_dev(logits.ptr, self.V, T, self.V, dt.ptr, 1, lp.ptr, ent.ptr, top, ids.ptr, tlp.ptr)
        self.ctx.sync()
        said = (lp.download().reshape(T, 1), ent.download(), ids.download().view(np.int32).reshape(T, top),
                tlp.download().reshape(T, top))
        return logits.download().reshape(T, self.V), said

    def exact(self, state, batch, positions, x, fmt, mass):
        """The same in 64 bits; state: the sequences' keys and values so far."""
        norm = lambda y, w: y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * w  # noqa: E731
        x = x.astype(np.float64)
        rows = norm(x, self.norm1) @ self.mats[0][1].T
        q, k, v = np.split(rows, [self.heads * self.D, (self.heads + self.G) * self.D], axis=1)
        q = rope(positions, q.reshape(-1, self.heads, self.D), self.freq, HALVES, self.wq, EPS)[0]
        k = rope(positions, k.reshape(-1, self.G, self.D), self.freq, HALVES, self.wk, EPS)[0]
        v = v.reshape(-1, self.G, self.D)
        for s, nt in enumerate(batch.ns):
            r = slice(batch.row_start[s], batch.row_start[s] + nt)
            for i, new in enumerate((k[r], v[r])):
                state[s][i] = np.concatenate([state[s][i], stored(fmt, new)])
        ks, vs = (np.concatenate([state[s][i] for s in range(len(batch.ns))]) for i in (0, 1))
        att, _ = attention(batch, ks, vs, q, self.heads, self.D ** -0.5)
        gathered, _ = attention_mass(batch, ks, q, self.heads, self.D ** -0.5, mass, mass.shape[2])
        h = x + att.reshape(len(x), -1) @ self.mats[1][1].T
        return norm(h, self.norm2) @ self.mats[2][1].T, gathered


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_decoding_with_a_budget(ctx, fmt):
    """Prompts, steps, eviction to a budget onto other pages, and steps behind it.  Logits and gathered
    weights are held to the GEMV path's relative error, 1e-4 (keys and values 1e-7 off, of which some 2^-11 are
    rounded to the cache's other neighbour); which tokens stay is held to the device's own weights, bit for
    bit, and log probabilities to its own logits."""
    rng = np.random.default_rng(41)
    dec = Decoder(ctx, rng)
    page, keep, sinks, recent, stride = 32, 40, 4, 8, 192
    lens, behind = [0, 0, 0], [0, 0, 0]  # cached tokens, and positions
    pool = Batch(rng, [0, 0, 0], [160, 160, 160], page, spare=16)
    cache = nx.KvCache(ctx, fmt, pool.num_pages, page, dec.G, dec.D)
    empty = np.zeros((0, dec.G, dec.D))
    state = [[empty, empty] for _ in lens]
    mass = DeviceArray(3 * dec.G * stride, fill=0.0)
    tables, spare = pool.pages, [int(p) for p in pool.unused]
    for ns in ([70, 33, 1], [1, 1, 1], [1, 1, 1], None, [1, 1, 1], [2, 0, 30], [1, 1, 1]):
        before = mass.download().reshape(3, dec.G, stride)
        if ns is None:
            to = np.full_like(tables, -1)
            to[:, :2] = np.array(spare[:6]).reshape(3, 2)
            kept, new_len, moved = cache.evict(lens, tables, to, keep, before, sinks, recent)
            for s in range(3):
                for g in range(dec.G):
                    want = evicted(before[s, g], lens[s], keep, sinks, recent)
                    assert np.array_equal(kept[s, g, :len(want)], want)
                at = kept[s, :, :new_len[s]]
                state[s] = [np.stack([a[at[g], g] for g in range(dec.G)], 1) for a in state[s]]
            again = np.zeros((3, dec.G, stride), np.float32)
            again[:, :, :keep] = moved
            mass.upload(again)
            lens, tables = [int(n) for n in new_len], to
            # a table grows by pages that nobody uses
            free = [p for p in range(pool.num_pages) if p not in to]
            tables[:, 2:] = np.array(free[:3 * (tables.shape[1] - 2)]).reshape(3, -1)
            continue
        lens = [a + n for a, n in zip(lens, ns)]
        b = Batch(rng, ns, lens, page)
        b.pages, b.max_pages = tables, tables.shape[1]
        positions = np.concatenate([behind[s] + np.arange(n) for s, n in enumerate(ns)])
        behind = [p + n for p, n in zip(behind, ns)]
        x = rng.standard_normal((b.rows, dec.H)).astype(np.float32)
        tokens = rng.integers(0, dec.V, b.rows)
        logits, said = dec.step(cache, b, positions, x, mass, stride, tokens, 5)
        ref, gathered = dec.exact(state, b, positions, x, fmt, before)
        assert rel_l2(logits, ref) < 1e-4, (ns, rel_l2(logits, ref))
        got = mass.download().reshape(before.shape)
        for s, n in enumerate(ns):
            if n:
                assert rel_l2(got[s, :, :lens[s]], gathered[s, :, :lens[s]]) < 1e-4
            assert np.array_equal(got[s, :, lens[s]:], before[s, :, lens[s]:])
        check_logprobs(said, logits, tokens[:, None], 5)
    cache.close()


# ---------------------------------------------------------------- graphs
class Calls:
    """The device buffers of a step's calls, and the calls."""

    heads, G, D, V, top, keep = 8, 2, 64, 9001, 5, 50

    def __init__(self, b, to):
        T, S = b.rows, len(b.ns)
        HD, GD = self.heads * self.D, self.G * self.D
        self.b, self.width, self.stride = b, HD + 2 * GD, 1300
        self.rows = DeviceArray(T * self.width, fill=0.0)
        self.logits = DeviceArray(T * self.V, fill=0.0)
        self.freq, self.norm = DeviceArray(self.D // 2), DeviceArray(self.D, fill=1.25)
        self.freq.upload(1e4 ** (-np.arange(0, self.D, 2) / self.D))
        self.rope = nx.Rope(self.D, self.D, self.freq.ptr, HALVES, self.norm.ptr, self.norm.ptr)
        self.pos, self.tok, self.to, self.to_width = ints(np.arange(T)), ints(np.arange(T)), ints(to), to.shape[1]
        self.d = device_batch(b)
        self.ln = self.d.keep[1]
        self.outs = {"q": DeviceArray(T * HD), "k": DeviceArray(T * GD),
                     "mass": DeviceArray(S * self.G * self.stride, fill=0.5),
                     "kept": DeviceArray(S * self.G * self.keep), "new_len": DeviceArray(S),
                     "moved": DeviceArray(S * self.G * self.keep, fill=0.0), "lp": DeviceArray(T),
                     "ent": DeviceArray(T), "ids": DeviceArray(T * self.top), "tlp": DeviceArray(T * self.top)}

    def calls(self, ctx, cache):
        o, T = self.outs, self.b.rows
        HD, GD = self.heads * self.D, self.G * self.D
        k = self.rows.ptr + 4 * HD
        ctx.qk_rope_dev(self.rope, self.pos.ptr, T, self.heads, self.G, self.rows.ptr, self.width, k, self.width,
                        o["q"].ptr, HD, o["k"].ptr, GD)
        # (values of another stride: written with the keys' rows, out of the fused ones)
        cache.write_dev(self.d, k, k + 4 * GD, self.width)
        cache.attention_mass_dev(self.d, o["q"].ptr, HD, self.heads, o["mass"].ptr, o["mass"].ptr, self.stride, 0.125)
        cache.evict_dev(self.d, self.to.ptr, self.to_width, self.keep, 2, 5, o["mass"].ptr, self.stride, o["kept"].ptr,
                        o["new_len"].ptr, o["moved"].ptr, self.keep)
        ctx.logprobs_dev(self.logits.ptr, self.V, T, self.V, self.tok.ptr, 1, o["lp"].ptr, o["ent"].ptr, self.top,
                         o["ids"].ptr, o["tlp"].ptr)

    def got(self):
        return {name: a.download() for name, a in self.outs.items()}


def set_up(ctx, rng, fmt, ns, extra):
    lens = [n + e for n, e in zip(ns, extra)]
    b = Batch(rng, ns, lens, 32, max_pages=40)
    total = Batch(rng, ns, [1200] * len(ns), 32, max_pages=40, spare=2 * len(ns))
    b.pages, b.num_pages = total.pages, total.num_pages
    to = np.array(total.unused, np.int32).reshape(len(ns), 2)
    caches = [nx.KvCache(ctx, fmt, b.num_pages, 32, Calls.G, Calls.D) for _ in range(2)]
    for c in caches:
        k, v = random_kv(np.random.default_rng(1), sum(lens), Calls.G, Calls.D)
        c.write(b.whole(), b.kv_len, b.pages, k, v)
    return b, to, lens, caches


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ns", [[1, 1, 1], [90, 1, 3]], ids=["decode", "mixed"])
def test_captured_calls_follow_their_arrays(fmt, ns):
    """A graph of all the calls, replayed while lengths, rows and logits change, with other work of the
    context in between: every replay equals the eager calls bit for bit."""
    hip = Hip()
    rng = np.random.default_rng(42)
    with nx.Context(0) as ctx:
        stream = hip.stream()
        ctx.set_stream(stream.value)
        b, to, lens, (cache, eager) = set_up(ctx, rng, fmt, ns, (30, 500, 0))
        step, same = Calls(b, to), Calls(b, to)
        for s in (step, same):
            s.calls(ctx, cache if s is step else eager)  # (workspaces and kernels come outside the capture)
        ctx.sync()
        g, x = hip.graph(stream, lambda: step.calls(ctx, cache))
        for t in range(4):
            lens = [a + n for a, n in zip(lens, ns)]
            rows, logits = (rng.standard_normal(a.n).astype(np.float32) for a in (step.rows, step.logits))
            for s in (step, same):
                s.rows.upload(rows), s.logits.upload(logits)
                s.ln.upload(np.array(lens, np.int32).view(np.float32))
            hip.hipGraphLaunch(x, stream)
            ctx.sync()
            same.calls(ctx, eager)
            ctx.sync()
            want = same.got()
            for name, a in step.got().items():
                assert_same_bits(a, want[name])
            ctx.logprobs(rng.standard_normal((3 << t, 5000)).astype(np.float32), None, 3)
            cache.read([0] + [lens[0]] * 3, lens, b.pages)
        hip.hipGraphExecDestroy(x)
        hip.hipGraphDestroy(g)
        cache.close(), eager.close()
        ctx.set_stream(None)
        hip.hipStreamDestroy(stream)


def test_two_graphs_of_a_context_in_turn(ctx):
    """Two graphs that share the context's workspaces, one after the other, over and over."""

    hip = Hip()
    rng = np.random.default_rng(43)
    stream = C.c_void_p()
    nx.check(nx.lib().nx_ctx_get_stream(ctx.h, C.byref(stream)))
    made = []
    for ns, extra in (([1, 1], (700, 40)), ([120, 1], (300, 5))):
        b, to, _, (cache, other) = set_up(ctx, rng, F16, ns, extra)
        other.close()
        s = Calls(b, to)
        s.rows.upload(rng.standard_normal(s.rows.n)), s.logits.upload(rng.standard_normal(s.logits.n))

        def again(s=s):
            s.outs["mass"].upload(np.full(s.outs["mass"].n, 0.5, np.float32))

        again()
        s.calls(ctx, cache)
        ctx.sync()
        made.append((s, cache, s.got(), again, hip.graph(stream, lambda: s.calls(ctx, cache))))
    for _ in range(10):
        for s, _cache, _want, again, (_, x) in made:
            again()
            hip.hipGraphLaunch(x, stream)
            ctx.sync()
        for s, _cache, want, _, _ in made:
            for name, a in s.got().items():
                assert_same_bits(a, want[name])
    for _s, cache, _, _, (g, x) in made:
        hip.hipGraphExecDestroy(x)
        hip.hipGraphDestroy(g)
        cache.close()


def test_first_calls_are_refused_under_capture():
    """What allocates a workspace is refused while the stream is captured, and the capture goes on."""

    hip = Hip()
    rng = np.random.default_rng(44)
    with nx.Context(0) as ctx:
        stream = hip.stream()
        b, to, _, (cache, other) = set_up(ctx, rng, F16, [1, 1], (50, 60))
        other.close()
        s = Calls(b, to)
        ctx.sync()
        ctx.set_stream(stream.value)
        codes = []

        def calls():
            for f in (lambda: cache.attention_mass_dev(s.d, s.rows.ptr, s.width, 8, 0, s.outs["mass"].ptr, s.stride, 0.1),
                      lambda: ctx.logprobs_dev(s.logits.ptr, s.V, 2, s.V, 0, 0, 0, s.outs["ent"].ptr, 0, 0, 0)):
                with pytest.raises(nx.NexusError) as e:
                    f()
                codes.append(e.value.code)
            ctx.qk_rope_dev(s.rope, s.pos.ptr, 2, 8, 2, s.rows.ptr, s.width, s.rows.ptr + 2048, s.width, s.outs["q"].ptr,
                            512, s.outs["k"].ptr, 128)

        g, x = hip.graph(stream, calls)
        assert codes == [nx.NX_ERR_UNSUPPORTED] * 2
        rows = rng.standard_normal(s.rows.n).astype(np.float32)
        s.rows.upload(rows)
        for _ in range(3):
            s.outs["q"].upload(np.zeros(s.outs["q"].n, np.float32))
            hip.hipGraphLaunch(x, stream)
            ctx.sync()
            ref, bound = rope(np.arange(2), rows.reshape(2, -1)[:, :512].reshape(2, 8, 64), s.freq.download(), HALVES,
                              s.norm.download(), 1e-6)
            assert (np.abs(s.outs["q"].download().reshape(ref.shape) - ref) <= bound).all()
        # outside of the capture they are taken
        s.calls(ctx, cache)
        ctx.sync()
        hip.hipGraphExecDestroy(x)
        hip.hipGraphDestroy(g)
        cache.close()
        ctx.set_stream(None)
        hip.hipStreamDestroy(stream)


def test_contexts_on_streams_of_their_own():
    """Two contexts at once on one cache: each has its own workspaces."""
    rng = np.random.default_rng(45)
    with nx.Context(0) as one, nx.Context(0) as two:
        b, to, lens, (cache, other) = set_up(one, rng, F16, [60, 1], (900, 400))
        other.close()
        k, _ = random_kv(np.random.default_rng(1), sum(lens), Calls.G, Calls.D)
        keys = stored(F16, k)
        L, steps = nx.lib(), [Calls(b, to) for _ in range(2)]
        q = rng.standard_normal((2, b.rows, 8, 64)).astype(np.float32)
        x = (2 * rng.standard_normal((2, b.rows, Calls.V))).astype(np.float32)
        for s, a, y in zip(steps, q, x):
            s.outs["q"].upload(a), s.logits.upload(y)
        for _ in range(20):
            for c, s in zip((one, two), steps):
                o = s.outs
                nx.check(L.nx_attention_mass_dev(c.h, cache.h, s.d.ref, o["q"].ptr, 512, 8, 0.125, 0, o["mass"].ptr,
                                                 s.stride))
                c.logprobs_dev(s.logits.ptr, s.V, b.rows, s.V, s.tok.ptr, 1, o["lp"].ptr, o["ent"].ptr, 5, o["ids"].ptr,
                               o["tlp"].ptr)
        one.sync(), two.sync()
        for s, a, y in zip(steps, q, x):
            ref, bound = attention_mass(b, keys, a, 8, 0.125)
            got = s.outs["mass"].download().reshape(2, 2, s.stride)
            for i, n in enumerate(lens):
                assert (np.abs(got[i, :, :n] - ref[i, :, :n]) <= bound[i, :, :n]).all()
            T = b.rows
            o = {name: d.download() for name, d in s.outs.items()}
            check_logprobs((o["lp"].reshape(T, 1), o["ent"], o["ids"].view(np.int32).reshape(T, 5), o["tlp"].reshape(T, 5)),
                           y, np.arange(T)[:, None], 5)
        cache.close()


# ---------------------------------------------------------------- far places
def test_places_past_32_bits():
    """Pages whose keys lie beyond 4 GiB, and rows as far apart: the same as near ones."""
    rng = np.random.default_rng(46)
    G, D, page, pages = 8, 128, 1024, 2300  # 2 MiB of keys a page
    with nx.Context(0) as ctx:
        cache = nx.KvCache(ctx, F16, pages, page, G, D)
        b = Batch(rng, [3, 40], [1500, 2048], page)
        b.pages = np.array([[2298, 2199], [2201, 2299]], np.int32)
        b.num_pages = pages
        k, v = random_kv(rng, 3548, G, D)
        cache.write(b.whole(), b.kv_len, b.pages, k, v)
        q = rng.standard_normal((43, 8, D), dtype=np.float32)
        ref, bound = attention_mass(b, stored(F16, k), q, 8, 0.1)
        got = cache.attention_mass(*b.args(), q, 8, scale=0.1)
        assert (np.abs(got - ref) <= bound).all()
        to = np.array([[2200], [2297]], np.int32)
        kept, new_len, _ = cache.evict(b.kv_len, b.pages, to, 700, got, 4, 30)
        gk, gv = cache.read([0, 700, 1400], new_len, to)
        at = 0
        for s, n in enumerate(b.lens):
            for g in range(G):
                i = evicted(got[s, g], n, 700, 4, 30)
                assert np.array_equal(kept[s, g], i)
                assert_same_bits(gk[700 * s:700 * s + 700, g], stored(F16, k[at + i, g]))
                assert_same_bits(gv[700 * s:700 * s + 700, g], stored(F16, v[at + i, g]))
            at += n
        cache.close()
        # two rows 4.8 GB apart
        stride, V = 1_200_000_001, 4000
        far = DeviceArray(stride + V)
        x = rng.standard_normal((2, V)).astype(np.float32)
        for r in range(2):
            far.upload(x[r], r * stride)
        ent, ids, tlp = DeviceArray(2), DeviceArray(6), DeviceArray(6)
        ctx.logprobs_dev(far.ptr, stride, 2, V, 0, 0, 0, ent.ptr, 3, ids.ptr, tlp.ptr)
        ctx.sync()
        check_logprobs((np.zeros((2, 0)), ent.download(), ids.download().view(np.int32).reshape(2, 3),
                        tlp.download().reshape(2, 3)), x, np.zeros((2, 0), int), 3)
        freq, pos, out = DeviceArray(32), ints([7, 123456]), DeviceArray(2 * V)
        freq.upload(np.linspace(0.1, 1, 32))
        ctx.qk_rope_dev(nx.Rope(64, 64, freq.ptr, HALVES), pos.ptr, 2, 8, 0, far.ptr, stride, 0, 0, out.ptr, V, 0, 0)
        ctx.sync()
        ref, bound = rope([7, 123456], x[:, :512].reshape(2, 8, 64), np.linspace(0.1, 1, 32).astype(np.float32), HALVES)
        assert (np.abs(out.download().reshape(2, V)[:, :512].reshape(ref.shape) - ref) <= bound).all()
