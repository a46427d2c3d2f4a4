"""The cache and the attention as a decoder layer uses them: between its projections
and the MoE block, under graph capture, on other streams, and many times over."""
import ctypes as C

import numpy as np
import pytest

import nexus_amd as nx
import oracle
from kv_cases import F16, INT8, Batch, assert_close, attention, random_kv, rel_l2, stored
from moe_cases import DeviceArray, assert_same_bits
from test_gpu_attention import filled
from test_gpu_kv import device_batch, ints

pytestmark = pytest.mark.gpu
FORMATS = [F16, INT8]


@pytest.fixture(scope="module")
def ctx():
    c = nx.Context(0)
    yield c
    c.close()


# ---------------------------------------------------------------- a layer's steps
EPS = 1e-5


class Layer:
    """One decoder layer without position encoding: RMSNorm, q/k/v, attention,
    output projection, residual, MoE block."""

    H, heads, G, D, E, F, k = 256, 4, 2, 64, 4, 256, 2

    def __init__(self, ctx, rng):
        self.ctx = ctx
        width = (self.heads + 2 * self.G) * self.D
        self.norm1 = (1 + 0.1 * rng.standard_normal(self.H)).astype(np.float32)
        self.norm2 = (1 + 0.1 * rng.standard_normal(self.H)).astype(np.float32)
        self.router = (0.05 * rng.standard_normal((self.E, self.H))).astype(np.float32)
        self.dqkv, self.qkv = self.matrix(rng, width, self.H)
        self.do, self.o = self.matrix(rng, self.H, self.heads * self.D)
        self.experts = nx.Experts(ctx, nx.Q8_0, self.E, self.H, self.F)
        self.dense = {}
        for e in range(self.E):
            for role, shape in ((nx.ROLE_GATE, (self.F, self.H)), (nx.ROLE_UP, (self.F, self.H)),
                                (nx.ROLE_DOWN, (self.H, self.F))):
                q = oracle.quantize(nx.Q8_0, (0.05 * rng.standard_normal(shape)).astype(np.float32))
                self.experts.load(e, role, q)
                self.dense[e, role] = oracle.dequantize(nx.Q8_0, q, shape[0] * shape[1])

    def matrix(self, rng, rows, cols):
        q = oracle.quantize(nx.Q8_0, (0.08 * rng.standard_normal((rows, cols))).astype(np.float32))
        m = nx.Matrix(self.ctx, nx.Q8_0, rows, cols)
        m.load(q)
        return m, oracle.dequantize(nx.Q8_0, q, rows * cols).reshape(rows, cols).astype(np.float64)

    def step(self, cache, batch, x, window, sinks):
        """The device's step on hidden rows x: the calls of a serving loop."""
        T, width = len(x), self.dqkv.rows
        dx, dn, dw = DeviceArray(x.size), DeviceArray(x.size), DeviceArray(self.H)
        rows, att = DeviceArray(T * width), DeviceArray(T * self.heads * self.D)
        out, nw, rw = DeviceArray(x.size), DeviceArray(self.H), DeviceArray(self.router.size)
        dx.upload(x), dw.upload(self.norm1), nw.upload(self.norm2), rw.upload(self.router)
        d = device_batch(batch)
        self.ctx.rms_norm_dev(dx.ptr, x.size, dw.ptr, self.H, EPS, T, self.H, dn.ptr)
        self.dqkv.matvec_dev(dn.ptr, x.size, T, rows.ptr)
        k = rows.ptr + 4 * self.heads * self.D
        cache.write_dev(d, k, k + 4 * self.G * self.D, width)
        cache.attention_dev(d, rows.ptr, width, self.heads, att.ptr, self.heads * self.D, self.D ** -0.5,
                            window=window, sinks=sinks)
        self.do.matvec_dev(att.ptr, T * self.heads * self.D, T, out.ptr)
        self.ctx.sync()
        hidden = x + out.download().reshape(x.shape)
        return self.experts.block(hidden, self.norm2, EPS, self.router, self.k, path=nx.PATH_GEMV)

    def exact(self, state, batch, x, fmt, window, sinks):
        """The same in 64 bits; state: the sequences' keys and values so far."""
        x = x.astype(np.float64)
        n = x / np.sqrt((x * x).mean(1, keepdims=True) + EPS) * self.norm1
        rows = n @ self.qkv.T
        q, k, v = np.split(rows, [self.heads * self.D, (self.heads + self.G) * self.D], axis=1)
        shape = (-1, self.G, self.D)
        for s, nt in enumerate(batch.ns):
            r = slice(batch.row_start[s], batch.row_start[s] + nt)
            for i, new in enumerate((k[r], v[r])):
                state[s][i] = np.concatenate([state[s][i], stored(fmt, new.reshape(shape))])
        ks, vs = (np.concatenate([state[s][i] for s in range(len(batch.ns))]) for i in (0, 1))
        att, _ = attention(batch, ks, vs, q.reshape(-1, self.heads, self.D), self.heads, self.D ** -0.5, window,
                           sinks)
        h = x + att.reshape(len(x), -1) @ self.o.T
        n = h / np.sqrt((h * h).mean(1, keepdims=True) + EPS) * self.norm2
        logits = (n @ self.router.T).astype(np.float32)
        mats = [[self.dense[e, r] for e in range(self.E)] for r in (0, 1, 2)]
        return h + oracle.moe_layer(n.astype(np.float32), logits, *mats, self.k)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_layer_steps(ctx, fmt, window, sinks):
    """Two prompts, then steps in which the sequences grow by one, several and no
    tokens.  Each step is held to the GEMV path's relative error (1e-4) against 64
    bits: of k and v, 1e-7 off, some 2^-11 of the values are rounded to the cache's
    other neighbour, which adds less than 1e-5."""
    rng = np.random.default_rng(21)
    layer = Layer(ctx, rng)
    page, lens = 32, [0, 0, 0]
    steps = [[40, 97, 1], [1, 1, 1], [3, 1, 0], [1, 70, 1]]
    pool = Batch(rng, [0, 0, 0], [128, 192, 64], page)
    cache = nx.KvCache(ctx, fmt, pool.num_pages, page, layer.G, layer.D)
    empty = np.zeros((0, layer.G, layer.D))
    state = [[empty, empty] for _ in lens]
    for ns in steps:
        lens = [a + n for a, n in zip(lens, ns)]
        b = Batch(rng, ns, lens, page)
        b.pages, b.max_pages = pool.pages, pool.max_pages
        x = rng.standard_normal((b.rows, layer.H)).astype(np.float32)
        got = layer.step(cache, b, x, window, sinks)
        ref = layer.exact(state, b, x, fmt, window, sinks)
        assert rel_l2(got, ref) < 1e-4, (ns, rel_l2(got, ref))
    cache.close()


# ---------------------------------------------------------------- streams and graphs
class Hip:
    """The runtime that the library links, for streams and graphs."""

    def __init__(self):
        self.h = DeviceArray.hip()
        self.vp = C.c_void_p

    def __getattr__(self, name):
        f = getattr(self.h, name)

        def call(*args):
            rc = f(*args)
            assert rc == 0, f"{name}: {rc}"

        return call

    def stream(self):
        s = self.vp()
        self.hipStreamCreateWithFlags(C.byref(s), C.c_uint(1))
        return s

    def graph(self, stream, calls):
        """An executable graph of what `calls` enqueues on `stream`."""
        g, x = self.vp(), self.vp()
        self.hipStreamBeginCapture(stream, C.c_int(2))
        calls()
        self.hipStreamEndCapture(stream, C.byref(g))
        self.hipGraphInstantiate(C.byref(x), g, None, None, C.c_size_t(0))
        return g, x


class Step:
    """The device buffers of one captured step."""

    def __init__(self, b, heads, G, D):
        self.b, self.heads, self.G, self.D = b, heads, G, D
        self.q, self.out = (DeviceArray(b.rows * heads * D, fill=0.0) for _ in range(2))
        self.k, self.v = (DeviceArray(b.rows * G * D, fill=0.0) for _ in range(2))
        self.d = device_batch(b)
        self.rs, self.ln, self.pg = self.d.keep

    def calls(self, cache, window=0, sinks=0):
        cache.write_dev(self.d, self.k.ptr, self.v.ptr, self.G * self.D)
        cache.attention_dev(self.d, self.q.ptr, self.heads * self.D, self.heads, self.out.ptr,
                            self.heads * self.D, self.D ** -0.5, window=window, sinks=sinks)

    def got(self):
        return self.out.download().reshape(self.b.rows, self.heads, self.D)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ns,heads", [([1, 1, 1], 8), ([40, 1, 3], 8), ([150, 1, 3], 32)],
                         ids=["decode", "mixed", "chunk"])
def test_captured_step_follows_the_lengths(fmt, ns, heads):
    """A graph of a write and its attention, replayed while the sequences grow, with
    other work of the context (that enlarges its workspace) in between: every replay
    equals the eager calls bit for bit."""
    hip = Hip()
    rng = np.random.default_rng(31)
    G, D, page = 2, 128, 32
    with nx.Context(0) as ctx:
        stream = hip.stream()
        ctx.set_stream(stream.value)
        lens = [n + e for n, e in zip(ns, (30, 500, 0))]
        b = Batch(rng, ns, lens, page, max_pages=40)
        total = Batch(rng, ns, [900, 900, 900], page, max_pages=40)
        b.pages, b.num_pages = total.pages, total.num_pages
        cache, eager = (nx.KvCache(ctx, fmt, b.num_pages, page, G, D) for _ in range(2))
        for c in (cache, eager):
            k, v = random_kv(np.random.default_rng(1), sum(lens), G, D)
            c.write(b.whole(), b.kv_len, b.pages, k, v)
        step, same = Step(b, heads, G, D), Step(b, heads, G, D)
        for s in (step, same):
            s.calls(cache if s is step else eager)  # (kernels load outside the capture)
        ctx.sync()
        g, x = hip.graph(stream, lambda: step.calls(cache))
        for t in range(4):
            lens = [a + n for a, n in zip(lens, ns)]
            new = [rng.standard_normal(a.n).astype(np.float32) for a in (step.q, step.k, step.v)]
            for s in (step, same):
                for a, values in zip((s.q, s.k, s.v), new):
                    a.upload(values)
                s.ln.upload(np.array(lens, np.int32).view(np.float32))
            hip.hipGraphLaunch(x, stream)
            ctx.sync()
            same.calls(eager)
            ctx.sync()
            assert_same_bits(step.got(), same.got())
            # other work on the context between the replays, more of it each time
            ctx.rms_norm(rng.standard_normal((64 << t, 256)).astype(np.float32), np.ones(256, np.float32), EPS)
            cache.read([0, lens[0], lens[0], lens[0]], lens, b.pages)
        hip.hipGraphExecDestroy(x)
        hip.hipGraphDestroy(g)
        cache.close(), eager.close()
        ctx.set_stream(None)
        hip.hipStreamDestroy(stream)


def test_two_graphs_of_a_context_in_turn(ctx):
    """Two graphs that share the context's workspace, replayed one after the other
    on its stream, over and over."""
    hip = Hip()
    rng = np.random.default_rng(32)
    heads, G, D = 4, 1, 64
    stream = C.c_void_p()
    nx.check(nx.lib().nx_ctx_get_stream(ctx.h, C.byref(stream)))
    cases = []
    for ns, lens in (([1, 1], [3000, 40]), ([1], [5000]), ([90], [400]), ([700, 1, 400], [900, 5000, 400])):
        b = Batch(rng, ns, lens, 64)
        cache, k, v = filled(ctx, rng, b, F16, G, D)
        s = Step(b, heads, G, D)
        q = rng.standard_normal((b.rows, heads, D)).astype(np.float32)
        s.q.upload(q)
        at = np.concatenate([b.whole()[i] + lens[i] - n + np.arange(n) for i, n in enumerate(ns)])
        s.k.upload(k[at]), s.v.upload(v[at])
        s.calls(cache)
        ctx.sync()
        want = s.got()
        ref, bound = attention(b, k, v, q, heads, np.float32(D ** -0.5))
        assert_close(want, ref, bound)
        cases.append((s, cache, want, hip.graph(stream, lambda: s.calls(cache))))
    for _ in range(20):
        for s, _cache, _want, (_, x) in cases:
            s.out.upload(np.zeros(s.out.n, np.float32))
            hip.hipGraphLaunch(x, stream)
        ctx.sync()
        for s, _cache, want, _ in cases:
            assert_same_bits(s.got(), want)
    for s, cache, _, (g, x) in cases:
        hip.hipGraphExecDestroy(x)
        hip.hipGraphDestroy(g)
        cache.close()


def test_contexts_on_streams_of_their_own():
    """One cache read by two contexts at once: each has its own workspace."""
    rng = np.random.default_rng(33)
    heads, G, D = 8, 2, 64
    with nx.Context(0) as one, nx.Context(0) as two:
        b = Batch(rng, [1, 1, 1], [4000, 900, 77], 64)
        cache, k, v = filled(one, rng, b, F16, G, D)
        q = rng.standard_normal((2, b.rows, heads, D)).astype(np.float32)
        d, L = device_batch(b), nx.lib()
        qs, outs = [DeviceArray(q[0].size) for _ in q], [DeviceArray(q[0].size) for _ in q]
        for a, values in zip(qs, q):
            a.upload(values)
        for _ in range(50):
            for c, a, o in zip((one, two), qs, outs):
                nx.check(L.nx_attention_dev(c.h, cache.h, d.ref, a.ptr, heads * D, heads, D ** -0.5, 0, 0, o.ptr,
                                            heads * D))
        one.sync(), two.sync()
        for values, o in zip(q, outs):
            ref, bound = attention(b, k, v, values, heads, np.float32(D ** -0.5))
            assert_close(o.download().reshape(values.shape), ref, bound)
        cache.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ns,lens", [([1], [9000]), ([1] * 20, [700 + 37 * i for i in range(20)]),
                                     ([200], [5000]), ([3, 80, 1], [2000, 300, 4000]),
                                     ([300], [5000]), ([3, 280, 1], [2000, 300, 4000])],
                         ids=["long", "batch", "chunk", "mixed", "chunk-of-many", "mixed-of-many"])
def test_many_runs_agree(ctx, fmt, ns, lens):
    """Split tiles are joined in the order of their parts, whoever ends last: 200
    calls in a row give the same bits."""
    rng = np.random.default_rng(34)
    heads, G, D = 16, 4, 128
    b = Batch(rng, ns, lens, 64)
    cache, k, v = filled(ctx, rng, b, fmt, G, D)
    q = rng.standard_normal((b.rows, heads, D)).astype(np.float32)
    ref, bound = attention(b, k, v, q, heads, np.float32(D ** -0.5))
    dq = DeviceArray(q.size)
    dq.upload(q)
    d = device_batch(b)
    outs = [DeviceArray(q.size) for _ in range(4)]
    first = None
    for _ in range(50):
        for o in outs:
            cache.attention_dev(d, dq.ptr, heads * D, heads, o.ptr, heads * D, D ** -0.5)
        ctx.sync()
        for o in outs:
            got = o.download().reshape(q.shape)
            if first is None:
                assert_close(got, ref, bound)
                first = got
            assert_same_bits(got, first)
    cache.close()


@pytest.mark.parametrize("long", [1, 150, 1000])
def test_very_many_sequences(ctx, long):
    """Several rounds of a workgroup's threads of sequences, a long one among them,
    in both kernels."""
    rng = np.random.default_rng(35)
    ns = [int(n) for n in rng.integers(0, 3, 1300)]
    ns[1201] = long
    lens = [n + int(x) for n, x in zip(ns, rng.integers(0, 70, 1300))]
    lens[1201] = 2000 + long
    b = Batch(rng, ns, lens, 32)
    heads, G, D = 2, 1, 64
    cache, k, v = filled(ctx, rng, b, F16, G, D)
    q = rng.standard_normal((b.rows, heads, D)).astype(np.float32)
    ref, bound = attention(b, k, v, q, heads, np.float32(D ** -0.5))
    assert_close(cache.attention(*b.args(), q, heads), ref, bound)
    cache.close()


def test_first_calls_under_capture_are_refused():
    """What allocates and clears memory is refused while the context's stream is captured, and
    leaves the capture whole; the same calls outside of it, and captured ones behind them, run."""
    hip = Hip()
    rng = np.random.default_rng(37)
    heads, G, D = 8, 2, 64
    with nx.Context(0) as one, nx.Context(0) as two:
        b = Batch(rng, [1, 1], [4000, 77], 64)
        cache, k, v = filled(one, rng, b, F16, G, D)
        q = rng.standard_normal((b.rows, heads, D)).astype(np.float32)
        ref, bound = attention(b, k, v, q, heads, np.float32(D ** -0.5))
        s = Step(b, heads, G, D)
        s.q.upload(q)
        stream = hip.stream()
        two.set_stream(stream.value)
        cache.ctx = two
        attend = lambda: cache.attention_dev(s.d, s.q.ptr, heads * D, heads, s.out.ptr,  # noqa: E731
                                             heads * D, D ** -0.5)

        def refused():
            for f in (attend, lambda: nx.KvCache(two, F16, 1, 32, 1, 64)):
                with pytest.raises(nx.NexusError) as e:
                    f()
                assert e.value.code == nx.NX_ERR_UNSUPPORTED and "capture" in str(e.value)

        graphs = [hip.graph(stream, refused)]
        attend()
        two.sync()
        assert_close(s.got(), ref, bound)
        want = s.got()
        graphs.append(hip.graph(stream, attend))
        for _ in range(3):
            s.out.upload(np.zeros(s.out.n, np.float32))
            for _, x in graphs:
                hip.hipGraphLaunch(x, stream)
            two.sync()
            assert_same_bits(s.got(), want)
            attend()
            two.sync()
            assert_same_bits(s.got(), want)
        for g, x in graphs:
            hip.hipGraphExecDestroy(x)
            hip.hipGraphDestroy(g)
        cache.close()
        two.set_stream(None)
        hip.hipStreamDestroy(stream)


def test_size_of_the_workspace():
    """A context's attention takes the memory that the header states, and nothing for growth."""
    with nx.Context(0) as ctx:
        ctx.sync()
        free, _ = ctx.mem_info()
        cache = nx.KvCache(ctx, F16, 1, 32, 1, 64)
        now, _ = ctx.mem_info()
        assert free - now < 82 << 20  # 77 MB, the cache, and whole 2 MiB pages of either
        cache.close()


def test_profile_and_lifetimes():
    """The launches show in the context's profile; a cache may outlive its context."""
    rng = np.random.default_rng(36)
    ctx = nx.Context(0)
    b = Batch(rng, [1, 100], [50, 100], 32)
    cache, _, _ = filled(ctx, rng, b, F16, 1, 64)
    ctx.profile(True)
    cache.attention(*b.args(), np.zeros((101, 41 * 64), np.float32), 41)
    names = ctx.profile_stats()
    assert {"attn_split", "attn_tile", "attn_join"} <= set(names)
    assert all(n == 1 and ms > 0 for n, ms in names.values())
    ctx.profile(False)
    other = nx.Context(0)
    ctx.close()
    q = rng.standard_normal((101, 1, 64)).astype(np.float32)
    cache.ctx = other
    assert np.all(np.isfinite(cache.attention(*b.args(), q, 1)))
    cache.close()
    other.close()
