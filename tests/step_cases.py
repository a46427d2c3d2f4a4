"""Heads normed and rotated, and log probabilities, from their formulas in 64 bits (numpy, no
library code), with bounds of what f32 kernels may be off."""
from __future__ import annotations

import numpy as np

HALVES, PAIRS = 0, 1
U = 2.0 ** -24  # half a step of f32, relative


def rope(positions, x, freq, style, weight=None, eps=1e-6):
    """Heads x [T x heads x D] rotated, and a bound of an f32 kernel's error per value.

    The bound, in units of 2^-24 of the head's largest normed value M: a normed value has its
    factor's rounding and two products' (3 units); cos and sin up to 3 units of their own, so a
    product p c is 6 off, the sum of two such 12, the first product's rounding and the sum's
    (up to 2 M) 3 more: 16 in all, and as many for the least normal value."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        if weight is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * weight.astype(np.float64)
        R = 2 * len(freq)
        # whole turns come off in long doubles, so the angle of a far position is right
        t = np.asarray(positions, np.longdouble)[:, None] * np.asarray(freq, np.float32).astype(np.longdouble)
        cos, sin = (f(t).astype(np.float64)[:, None] for f in (np.cos, np.sin))
        y = x.copy()
        i, j = ((slice(0, R // 2), slice(R // 2, R)) if style == HALVES else (slice(0, R, 2), slice(1, R, 2)))
        y[..., i] = x[..., i] * cos - x[..., j] * sin
        y[..., j] = x[..., i] * sin + x[..., j] * cos
    most = np.abs(x).max(-1, keepdims=True, initial=0)
    return y, np.broadcast_to(16 * U * most + 2.0 ** -126, y.shape)


def logprobs(x, tokens, top):
    """What nx_logprobs gives for rows x [T x V], and a bound of an f32 kernel's error per row (to which
    4 units of a log probability itself come).

    The bound: a term's exponent d log2 e is off by 2 units of 2^-24 of |d| and e^d by 2 more, and
    the sums of N terms, in chains of N / 256 + 16, by as many units of the sum of magnitudes:
    relative to S, e = (2 sum p |d| + N / 256 + 24) units, which is log S's error.  W's terms add
    |d| to that, so W / S is off by e times (1 + sum p |d|) and by 2 units of sum p d^2.  The log and the
    last differences round values up to |x_t - m| and log S: 4 units of those."""
    x = np.asarray(x, np.float64)
    T, V = x.shape
    lp, ent = np.zeros(np.shape(tokens)), np.zeros(T)
    ids, tlp = np.full((T, top), -1, np.int32), np.full((T, top), -np.inf)
    bound = np.zeros(T)
    for t in range(T):
        r = x[t]
        order = np.lexsort((np.arange(V), -np.where(np.isnan(r), -np.inf, r)))
        order = order[np.where(np.isnan(r), -np.inf, r)[order] > -np.inf][:top]
        ids[t, :len(order)] = order
        with np.errstate(all="ignore"):
            if np.isnan(r).any() or (r == np.inf).any():
                logp, ent[t] = np.full(V, np.nan), np.nan
            elif (r == -np.inf).all():
                logp, ent[t] = np.full(V, -np.inf), 0.0
            else:
                m = r.max()
                d = r - m
                p = np.exp(d)
                S = p.sum()
                logp = d - np.log(S)
                p /= S
                fine = p > 0
                ent[t] = -(p[fine] * logp[fine]).sum()
                a1, a2 = (p[fine] * -d[fine]).sum(), (p[fine] * d[fine] ** 2).sum()
                e = 2 * a1 + V / 256 + 24
                bound[t] = U * (e * (2 + a1) + 2 * a2 + 4 * np.log(S) + 8)
        for i, k in enumerate(tokens[t]):
            lp[t, i] = logp[k] if 0 <= k < V else 0.0
        tlp[t, :len(order)] = logp[order]
    return (lp, ent, ids, tlp), bound


def check_logprobs(got, x, tokens, top):
    ref, bound = logprobs(x, tokens, top)
    assert np.array_equal(got[2], ref[2]), "ids"
    for name, g, r in zip(("logprobs", "entropy", "ids", "top"), got, ref):
        if name == "ids":
            continue
        g = np.asarray(g, np.float64)
        b = bound.reshape((-1,) + (1,) * (r.ndim - 1))
        same = (np.isnan(g) & np.isnan(r)) | (g == r)
        with np.errstate(all="ignore"):
            off = np.where(same, 0, np.abs(g - r))
        b = b + np.where(same, 0, 4 * U * np.abs(r))
        assert (off <= b).all(), (name, float(np.nanmax(off / np.maximum(b, 1e-300))), off.max())


def evicted(mass, length, keep, sinks, recent):
    """The tokens of one head that stay, in their order: by a sort in Python of (weight, lower
    token), NaN below everything."""
    if length <= keep:
        return np.arange(length)
    middle = range(sinks, length - recent)
    weight = [(-np.inf, 0) if j >= len(mass) or np.isnan(mass[j]) else (float(mass[j]), 1) for j in range(length)]
    best = sorted(middle, key=lambda j: (-weight[j][1], -weight[j][0], j))[:keep - sinks - recent]
    return np.array(sorted(list(range(sinks)) + best + list(range(length - recent, length))), int)


def attention_mass(batch, k, q, heads, scale, before=None, width=None):
    """mass [seqs x G x width] of keys k [sum(lens) x G x D] that the cache holds, and a bound.

    The bound: a score's terms are each some 2^-21 off and their sum D 2^-24 of the sum of
    magnitudes, against the row's other scores too, and 2^x 2^-21: e of kv_cases.attention.  The row's
    log sum adds its N + 64 roundings, its own place and that of the difference to it, 2^-23 of
    the score's size and log2 N.  Then come as many sums as rows and heads, 2^-24 of the whole each."""
    G, D = k.shape[1:]
    width = width or max(max(batch.lens), 1)
    out = np.zeros((len(batch.ns), G, width)) if before is None else before.astype(np.float64)
    bound = np.zeros_like(out)
    at = 0
    for s, (n, length) in enumerate(zip(batch.ns, batch.lens)):
        if n:
            rows = slice(batch.row_start[s], batch.row_start[s] + n)
            hidden = np.arange(length)[None] > np.arange(length - n, length)[:, None]
            out[s, :, max(length - n, 0):length] = 0
            total, off = np.zeros((G, length)), np.zeros((G, length))
            for h in range(heads):
                g = h * G // heads
                ks = k[at:at + length, g].astype(np.float64)
                qh = q[rows, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = scale * (qh @ ks.T)
                    mag = np.where(hidden, 0, abs(scale) * (np.abs(qh) @ np.abs(ks).T)).max(1, keepdims=True)
                    x = np.where(hidden, -np.inf, x)
                    top = x.max(1, keepdims=True)
                    w = np.where(hidden, 0, np.exp(x - np.where(np.isfinite(top), top, 0)))
                    p = w / w.sum(1, keepdims=True)
                p = np.where(hidden.all(1)[:, None], 0, p)
                e = 2 * ((2.0 ** -21 + D * 2.0 ** -24) * mag + 2.0 ** -21)
                part = 2 * e + (length + 64) * U + 2 * U * (1.5 * mag + np.log2(length + 1))
                total[g] += p.sum(0)
                off[g] += (part * p).sum(0)
            m = min(length, width)
            out[s, :, :m] += total[:, :m]
            bound[s, :, :m] = off[:, :m] + (n * heads // G + 8) * U * out[s, :, :m] + 2.0 ** -120
        at += length
    return out, bound
