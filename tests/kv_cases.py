"""Paged batches for the cache and attention tests, and both operators from
their formulas in 64 bits, one row at a time (numpy, no library code)."""
from __future__ import annotations

import numpy as np

F16, INT8 = 0, 1


class Batch:
    """Sequences of `lens` tokens whose last `ns` are the rows, on random pages.
    Table entries that no token needs name no page."""

    def __init__(self, rng, ns, lens, page_tokens, spare=3, max_pages=None, first_row=0, padding=0):
        self.ns, self.lens, self.page_tokens = list(ns), list(lens), page_tokens
        need = [-(-n // page_tokens) for n in lens]
        self.max_pages = max(max(need), 1) if max_pages is None else max_pages
        self.num_pages = sum(need) + spare
        order = rng.permutation(self.num_pages)
        self.pages = np.full((len(lens), self.max_pages), -1, np.int32)
        at = 0
        for s, k in enumerate(need):
            self.pages[s, :k] = order[at:at + k]
            at += k
        self.unused = order[at:]
        self.row_start = (first_row + np.concatenate([[0], np.cumsum(ns)])).astype(np.int32)
        self.kv_len = np.array(lens, np.int32)
        self.rows = int(self.row_start[-1]) + padding

    def whole(self):
        """The same sequences with every token as a row."""
        return np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32)

    def args(self):
        return self.row_start, self.kv_len, self.pages


def stored(fmt, x):
    """What a cache holds of the f32 rows x [..., D], as f32."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        if fmt == F16:
            return x.astype(np.float16).astype(np.float32)
        fine = np.isfinite(x).all(-1, keepdims=True)
        scale = (np.abs(x).max(-1, keepdims=True).astype(np.float64) / 127.0).astype(np.float32)
        s = np.where(fine & (scale > 0), scale, np.float32(1))
        # the quotient in 64 bits decides as the exact one: it is n + 1/2 only if
        # x = (n + 1/2) s exactly, else at least 2^-25 from it
        codes = np.rint(np.where(fine, x, 0).astype(np.float64) / s) + 0.0  # integers: no -0
        codes = np.clip(codes, -127, 127)  # a subnormal scale may be rounded far down
        y = (codes.astype(np.float32) * np.where(scale > 0, scale, np.float32(0))).astype(np.float32)
        return np.where(fine, y, np.float32(np.nan))


def seen_by(p, length, window, sinks):
    """The tokens that token p sees."""
    j = np.arange(min(p + 1, length))
    return j if not window else j[(j > p - window) | (j < sinks)]


def attention(batch, k, v, q, heads, scale, window=0, sinks=0):
    """out [rows x heads x D], and a bound of an f32 kernel's error per value.

    k, v: f32 values that the cache holds, [sum(lens) x G x D], sequence after
    sequence; q [rows x heads x D].

    The bound: a score's terms scale q k are each rounded some 2^-21 of their
    magnitude off (an operand split into two halves of 11 bits, a product's and
    the scales' roundings) and their sum over D at most D 2^-24 of the sum of
    magnitudes; exp adds 2^-21 of its own.  So a weight is off by
    e = 2 ((2^-21 + D 2^-24) sum |scale q k| + 2^-21) relative to itself, against the
    other weights, and the sums over N keys by at most (N + 64) 2^-24: in all
    (2 e + 2 (N + 64) 2^-24 + 2^-21) sum p |v| / sum p.  The largest weight
    p_j scale_j of a row is held at 2^8 or more, in halves whose places end at 2^-24:
    every weight may be off by 2^-25 for that, 2^-33 of the largest, and a value is up
    to max |v_j|: N 2^-33 max_j p_j max |v_j| / sum p besides.  (Non-finite keys and values are
    left out of the bound: where the result is finite their weight is 0, or they
    are other elements.)"""
    G, D = k.shape[1:]
    out = np.zeros((batch.rows, heads, D))
    bound = np.zeros_like(out)
    at = 0
    for s, (n, length) in enumerate(zip(batch.ns, batch.lens)):
        ks, vs = k[at:at + length].astype(np.float64), v[at:at + length].astype(np.float64)
        ka, va = (np.where(np.isfinite(x), np.abs(x), 0.0) for x in (ks, vs))
        for i in range(n):
            row = batch.row_start[s] + i
            j = seen_by(length - n + i, length, window, sinks)
            if not len(j):
                continue
            for g in range(G):
                hs = slice(g * heads // G, (g + 1) * heads // G)
                qr = q[row, hs].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = scale * (qr @ ks[j, g].T)
                    mag = abs(scale) * (np.abs(qr) @ ka[j, g].T).max(1, keepdims=True)
                    p = np.exp(x - x.max(1, keepdims=True))
                    total = p.sum(1, keepdims=True)
                    out[row, hs] = p @ vs[j, g] / total
                    e = 2 * ((2.0 ** -21 + D * 2.0 ** -24) * mag + 2.0 ** -21)
                    part = 2 * e + 2 * (len(j) + 64) * 2.0 ** -24 + 2.0 ** -21
                    bound[row, hs] = part * (p @ va[j, g]) / total
                    top = (p * va[j, g].max(1)).max(1, keepdims=True)
                    bound[row, hs] += len(j) * 2.0 ** -33 * top / total
        at += length
    return out, bound


def attention_dense(batch, k, v, q, heads, scale, window=0, sinks=0):
    """attention(), of finite keys and values, all rows of a sequence and head at once."""
    G, D = k.shape[1:]
    out = np.zeros((batch.rows, heads, D))
    bound = np.zeros_like(out)
    at = 0
    for s, (n, length) in enumerate(zip(batch.ns, batch.lens)):
        rows = slice(batch.row_start[s], batch.row_start[s] + n)
        p, j = np.arange(length - n, length)[:, None], np.arange(length)[None]
        seen = (j <= p) & ((p - j < window) | (j < sinks) if window else True)
        count = seen.sum(1)[:, None]
        for h in range(heads) if n else ():
            kg, vg = (x[at:at + length, h * G // heads].astype(np.float64) for x in (k, v))
            qh = q[rows, h].astype(np.float64)
            x = np.where(seen, scale * (qh @ kg.T), -np.inf)
            mag = np.where(seen, abs(scale) * (np.abs(qh) @ np.abs(kg).T), 0).max(1, keepdims=True)
            w = np.exp(x - x.max(1, keepdims=True))
            total = w.sum(1, keepdims=True)
            out[rows, h] = w @ vg / total
            part = 4 * ((2.0 ** -21 + D * 2.0 ** -24) * mag + 2.0 ** -21) + 2 * (count + 64) * 2.0 ** -24 + 2.0 ** -21
            top = (w * np.abs(vg).max(1)).max(1, keepdims=True)
            bound[rows, h] = (part * (w @ np.abs(vg)) + count * 2.0 ** -33 * top) / total
        at += length
    return out, bound


def assert_close(got, ref, bound, scores=8.0):
    """Within the bound per value, and as a whole as near as the roundings' root
    mean square.  For scores up to 8 that is some 2^-21 (two halves of q, eight
    sums of a score, exp's argument, the weights' halves, the sums): 2^-19 of the
    norm is allowed.  The first three grow with the scores."""
    got = np.asarray(got, np.float64)
    err = np.abs(got - ref)
    assert np.all(np.isfinite(got))
    assert np.all(err <= bound + 1e-38), f"{np.max(err / (bound + 1e-38)):.3g} times the bound"
    norm = np.linalg.norm(ref)
    limit = 2.0 ** -19 * max(1.0, scores / 8)
    assert np.linalg.norm(got - ref) <= limit * norm, np.linalg.norm(got - ref) / norm


def rel_l2(got, ref) -> float:
    return float(np.linalg.norm(np.asarray(got, np.float64) - ref) / np.linalg.norm(ref))


def random_kv(rng, tokens, G, D):
    """Keys with a few large channels, values: f32 [tokens x G x D]."""
    k = rng.standard_normal((tokens, G, D), dtype=np.float32)
    k[:, :, ::29] *= 3
    return k, rng.standard_normal((tokens, G, D), dtype=np.float32)
