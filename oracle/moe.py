"""CPU oracle (TEST INFRASTRUCTURE, not product code): the mixture-of-experts layer and the log probabilities, from their
definitions in float64, with bounds on how far 32-bit arithmetic may take a result from them.
"""

from __future__ import annotations

import math

import numpy as np

from . import blocks, blocks_f1, product

U32 = 2.0 ** -24      # a rounding to fp32 is off by at most this share of the value


# ---------------------------------------------------------------- choice of the experts


def route(logits, top_k, scoring="softmax", renormalize=True, bias=None, scale=1.0):
    """(weights float64, ids) [tokens, top_k]."""
    z = np.asarray(logits, dtype=np.float64).copy()
    z[np.isnan(z)] = -np.inf
    z = np.minimum(z, np.finfo(np.float32).max)
    here = z > -np.inf
    with np.errstate(over="ignore", invalid="ignore"):
        if scoring == "softmax":
            top = np.where(here.any(1, keepdims=True), z.max(1, keepdims=True), 0.0)
            s = np.where(here, np.exp(z - top), 0.0)
            s = s / np.maximum(s.sum(1, keepdims=True), 1e-300)
        else:
            s = np.where(here, 1.0 / (1.0 + np.exp(-z)), 0.0)
    by = np.where(here, z if bias is None else s + np.asarray(bias, dtype=np.float64), -np.inf)
    m, n = z.shape
    w, ids = np.zeros((m, top_k)), np.full((m, top_k), -1, dtype=np.int64)
    for t in range(m):
        order = [e for e in sorted(range(n), key=lambda e: (-by[t, e], e)) if here[t, e]][:top_k]
        ids[t, :len(order)] = order
        w[t, :len(order)] = s[t, order]
    if renormalize:
        total = w.sum(1, keepdims=True)
        w = np.where(total > 0, w / np.where(total > 0, total, 1.0), 0.0)
    return w * scale, ids


# ---------------------------------------------------------------- experts


def q8(x):
    """(q [.., K], unit [.., K/32], t): round(127 x / amax) away from zero at ties, amax / 127, the unrounded quotient."""
    b = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    t = np.where(amax > 0, 127.0 * b / np.where(amax > 0, amax, 1.0), 0.0)
    q = np.trunc(t + np.copysign(0.5, t))
    return q.reshape(x.shape), (amax / 127.0)[..., 0], t.reshape(x.shape)


def _decode(raw, t):
    return blocks.decode(raw, t) if t in blocks.BLOCK_BYTES else blocks_f1.decode(raw, t)


def values(raw, t):
    return np.asarray((blocks if t in blocks.BLOCK_BYTES else blocks_f1).dequantize(raw, t), dtype=np.float64)


def _product(raw, t, q, unit):
    """[M, rows] of 8-bit activations: exact integer sums, scaled in float64 (the low-bit types with their truncating divisions)."""
    mod = product if t in blocks.BLOCK_BYTES else blocks_f1
    return mod.product_q81(_decode(raw, t), q.astype(np.int8), unit)


def _parts(raw, t):
    """Magnitude of the parts that a value's product is summed from: |value|, and where a block has minima the scaled quant and the
    scaled minimum, which may cancel in the value but are added up apart."""
    dec = _decode(raw, t)
    if getattr(dec, "imin", None) is None:
        return np.abs(values(raw, t))
    n, k = dec.w8.shape
    per = dec.imin.shape[1]
    low = np.repeat(np.repeat(dec.dmin.astype(np.float64), per // dec.dmin.shape[1], 1) * dec.imin, k // per, 1)
    return np.abs(values(raw, t) + low) + np.abs(low)


def _magnitudes(raw, t, q, unit):
    """Sum of the magnitudes of what is added in fp32."""
    return (np.abs(q) * np.repeat(unit, 32, -1)) @ _parts(raw, t).T


def _sum_error(k):
    """Relative to the sum of magnitudes: k / 32 slice terms (two where a superblock has minima) added one after another at worst, six
    roundings in each term, ten additions that join the parts."""
    return (2 * (k // 32) + 16) * U32


def _act(name, g):
    if name == "silu":
        with np.errstate(over="ignore"):
            return g / (1.0 + np.exp(-g))
    return 0.5 * g * np.array([math.erfc(-v / math.sqrt(2.0)) for v in g.ravel()]).reshape(g.shape)


def experts(x, raw13, raw2, t13, t2, weights, ids, act="silu", truncates=0.0):
    """(y, bound) float64 [tokens, hidden]: the layer's definition, and how far a sum in fp32 may be from it (before y is
    rounded to its type). The bound follows the errors through: the rounding of X to 8 bits, the gate and up products, the activation (four roundings and a
    function good to 2^-21), and the rounding of the activated product to 8 bits, where a value that is as near to a border as
    its own error may fall on either side. raw13 [experts][2 inter, bytes], raw2 [experts][hidden, bytes]."""
    m, hidden = x.shape
    y, bound = np.zeros((m, hidden)), np.zeros((m, hidden))
    xq, xu, xt = q8(x)
    # 127 x, rounded to fp32, against half * amax, in one fused step: a quotient moves by its own 2^-24 before it is compared, and not at
    # all where 127 x is an fp32 number (any 16-bit x)
    x127 = 127.0 * np.asarray(x, dtype=np.float64)
    xnear = (x127 != x127.astype(np.float32)) & (np.abs(np.abs(xt) - np.floor(np.abs(xt)) - 0.5) <= 1.01 * U32 * np.abs(xt))
    xstep = xnear * np.repeat(xu, 32, -1)
    for e in sorted({int(i) for i in np.asarray(ids).ravel() if 0 <= i < len(raw13)}):
        toks, slots = np.nonzero(np.asarray(ids) == e)
        inter = raw13[e].shape[0] // 2
        gu = _product(raw13[e], t13, xq[toks], xu[toks])
        err = _sum_error(hidden) * _magnitudes(raw13[e], t13, xq[toks], xu[toks])
        if xnear[toks].any():
            err = err + xstep[toks] @ np.abs(values(raw13[e], t13)).T
        g, u, dg, du = gu[:, :inter], gu[:, inter:], err[:, :inter], err[:, inter:]
        a = _act(act, g)
        h = a * u
        dh = 1.13 * dg * np.abs(u) + np.abs(a) * du + 1.13 * dg * du + (2.0 ** -20) * (np.abs(h) + np.abs(g * u) * 2.0 ** -3)
        hq, hu, t = q8(h)
        rel = np.repeat((dh.reshape(len(toks), -1, 32).max(-1) / np.maximum(hu * 127, 1e-300)) + 4 * U32, 32, -1)
        dt = dh / np.maximum(np.repeat(hu, 32, -1), 1e-300) + np.abs(t) * rel
        near = np.abs(np.abs(t) - np.floor(np.abs(t)) - 0.5) <= dt
        down = _product(raw2[e], t2, hq, hu)
        w2 = np.abs(values(raw2[e], t2))
        unit = np.repeat(hu, 32, -1)
        db = (near * unit + np.abs(hq) * unit * rel) @ w2.T + _sum_error(inter) * _magnitudes(raw2[e], t2, hq, hu)
        # a sum that is truncated after its scaling by an integer moves by one unit where it moves at all
        db += truncates * np.abs(w2).max() * unit.max() * (near.sum(-1, keepdims=True) + 1)
        wt = np.asarray(weights, dtype=np.float64)[toks, slots][:, None]
        np.add.at(y, toks, wt * down)
        np.add.at(bound, toks, np.abs(wt) * (db + 40 * U32 * np.abs(down)))
    return y, bound


# ---------------------------------------------------------------- log probabilities


def logprobs(x, ids, top_n):
    """Dict of float64 / int64 arrays (logprobs, ranks, entropy, top_logprobs, top_ids) and `tol`, `entropy_tol`: how far sums and
    exponentials in fp32 may take the log probabilities and the entropy."""
    x = np.asarray(x, dtype=np.float64) + 0.0
    m, v = x.shape
    out = {"logprobs": np.zeros(m), "ranks": np.zeros(m, np.int64), "entropy": np.zeros(m), "tol": np.zeros(m), "entropy_tol": np.zeros(m),
           "top_logprobs": np.full((m, top_n), -np.inf), "top_ids": np.full((m, top_n), -1, np.int64)}
    for r in range(m):
        row = x[r]
        order = np.lexsort((np.arange(v), -np.where(np.isnan(row), -np.inf, row), np.isnan(row)))
        place = np.empty(v, np.int64)
        place[order] = np.arange(v)
        bad = np.isnan(row).any() or (row == np.inf).any()
        top = row[order[0]]
        if bad:
            lp, out["entropy"][r] = np.full(v, np.nan), np.nan
        elif top == -np.inf:
            lp, out["entropy"][r] = np.full(v, -np.inf), 0.0
        else:
            y = row - top
            e = np.exp(y)
            s = e.sum()
            lp = y - math.log(s)
            z = np.where(e > 0, e * y, 0.0)
            out["entropy"][r] = math.log(s) - z.sum() / s
            # each exponential: its argument to (|y| + |x|) 2^-23, itself to 2^-21; the sums: v / 256 + 32 additions at worst
            fin = np.isfinite(row)
            arg = np.where(fin, np.abs(np.where(fin, y, 0)) + np.abs(np.where(fin, row, 0)), 0.0) * 2.0 ** -23 + 2.0 ** -21 + (v // 256 + 32) * U32
            ds = (e * arg).sum() / s
            out["tol"][r] = ds + 2.0 ** -21 * (1 + abs(math.log(s)))
            mean = abs(z.sum()) / s
            out["entropy_tol"][r] = out["tol"][r] + (np.abs(z) * arg).sum() / s + mean * ds + (mean + 1) * 2.0 ** -20
        n = min(top_n, v)
        out["top_ids"][r, :n] = order[:n]
        out["top_logprobs"][r, :n] = lp[order[:n]]
        i = int(ids[r])
        if 0 <= i < v:
            out["logprobs"][r], out["ranks"][r] = lp[i], place[i] + 1
        else:
            out["logprobs"][r] = 0.0 if i < 0 else np.nan
    return out
