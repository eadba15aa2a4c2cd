"""The paged cache of 4 bits a value, what reads caches back, and log probabilities, restated in numpy in 64 bits.

A cache is a dict: k, v [pages][kv][place][d / 2] bytes, k_scale, v_scale [pages][kv][d / 32][place] bytes (exponent + 127),
format "e2m1".  Element types as in serving_oracle.py.
"""

import numpy as np

import serving_oracle as so

GROUP, LEAST, MOST = 32, -23, 13
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LEVELS = np.concatenate([LEVELS, -LEVELS])
U = 2.0 ** -24


def codes(x):
    """Nearest e2m1 code, ties to the even one; magnitudes past 6 at it, NaN 0."""
    a = np.abs(np.where(np.isnan(x), 0.0, x))
    off = np.abs(np.minimum(a, 6.0)[..., None] - LEVELS[:8])
    near = off == off.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    return (code | np.where(np.signbit(x) & ~np.isnan(x), 8, 0)).astype(np.uint8)


def quantized(x):
    """(bytes, exponent bytes) of [..., d] values."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    most = np.abs(np.where(np.isfinite(g), g, 0.0)).max(-1)
    e = np.full(most.shape, LEAST)
    for up in range(LEAST, MOST):
        e = np.where(most > 6.0 * 2.0 ** up, up + 1, e)
    with np.errstate(invalid="ignore"):
        c = codes(g / 2.0 ** e[..., None].astype(np.float64)).reshape(x.shape)
    return c[..., 0::2] | c[..., 1::2] << 4, (e + 127).astype(np.uint8)


def append(cache, k, v, slots, page):
    out = {n: a.copy() if isinstance(a, np.ndarray) else a for n, a in cache.items()}
    for name, x in (("k", k), ("v", v)):
        c, e = quantized(x)
        for t, slot in enumerate(slots):
            if slot >= 0:
                out[name][slot // page, :, slot % page] = c[t]
                out[name + "_scale"][slot // page, :, :, slot % page] = e[t]
    return out


def values(cache, name):
    """[pages][kv][place][d] of a cache of any format."""
    c, s = cache[name], cache[name + "_scale"]
    if cache["format"] != "e2m1":
        x = so.values(np.ascontiguousarray(c if name == "k" else c.swapaxes(2, 3)), cache["format"])
        return x * s[:, :, None, None].astype(np.float64)
    x = np.stack([LEVELS[c & 15], LEVELS[c >> 4]], -1).reshape(*c.shape[:3], -1)
    return x * np.repeat(2.0 ** (s.astype(np.float64) - 127).swapaxes(2, 3), GROUP, -1)


def attention(cache, q, offsets, lengths, table, page, scale, causal=True, window=0, dtype="f32", drop=()):
    """(out, tolerance): 64-bit results and how far a binary32 evaluation in the documented operand widths may be off.
    drop: (request, column) pairs whose keys are left out.

    The tolerance counts, for z = scale * q.k with u = 2^-24:
      the first product: D roundings of the sum; the parts of q (two of 11 bits, 2^-22 of the row's largest value an
        element; one part is exact for f16 and bf16); the products with the scales and the maximum's subtraction, each
        a rounding of a number up to the row's largest |z| (in base 2, so 1.45 of it) and the headroom of 11: dz
      p = 2^z: dz, one step of exp (2^-23), and its parts: 2^-22 for two, half a step 2^-11 for one
      sums over n keys: n roundings each, in the numerator and the denominator; sixteen more for joins and the division
    each relative to the term, so against sum p |v| / sum p; the result's own rounding; and the smallest step of the
    binary16 parts: the largest p stands at 2^11 to 2^15, so p is off by up to 2^-25 / 2^11 = 2^-36 of the largest
    (twice that is allowed).
    """
    q = np.asarray(q, np.float64)
    t, heads, d = q.shape
    kv = cache["k"].shape[1]
    g = heads // kv
    kx, vx = values(cache, "k"), values(cache, "v")
    out, tol = np.zeros_like(q), np.zeros_like(q)
    for r in range(len(lengths)):
        n, o0, o1 = int(lengths[r]), int(offsets[r]), int(offsets[r + 1])
        if n == 0:
            continue
        pages = np.clip(table[r][: -(-n // page)], 0, None)
        gone = np.zeros(n, bool)
        for rr, col in drop:
            if rr == r:
                gone[col * page:(col + 1) * page] = True
        for h in range(kv):
            k, v = kx[pages, h].reshape(-1, d)[:n], vx[pages, h].reshape(-1, d)[:n]
            for i in range(o1 - o0):
                lo, hi = 0, n
                if causal:
                    at = n - (o1 - o0) + i
                    hi = max(0, at + 1)
                    lo = max(0, at + 1 - window) if window else 0
                keep = ~gone[lo:hi]
                if hi <= lo or not keep.any():
                    continue
                kk, vv = k[lo:hi][keep], v[lo:hi][keep]
                rows = q[o0 + i, h * g:(h + 1) * g]
                z = scale * (rows @ kk.T)
                p = np.exp(z - z.max(1, keepdims=True))
                l = p.sum(1, keepdims=True)
                got = (p @ vv) / l
                out[o0 + i, h * g:(h + 1) * g] = got
                part = 2.0 ** -22 * np.abs(rows).max(1, keepdims=True) * np.abs(kk).sum(1)[None] if dtype == "f32" else 0.0
                dz = abs(scale) * ((d + 4) * U * (np.abs(rows) @ np.abs(kk).T) + part) + U * (6 * np.abs(z).max(1, keepdims=True) + 32)
                rel = 2 * dz.max(1, keepdims=True) + 2.0 ** -22 + (2.0 ** -21 if dtype == "f32" else 2.0 ** -11) + (2 * len(kk) + 16) * U
                floor = 2.0 ** -35 * p.max(1, keepdims=True) * np.abs(vv).sum(0)[None]
                tol[o0 + i, h * g:(h + 1) * g] = (rel * (p @ np.abs(vv)) + floor) / l + so.HALF[dtype] * np.abs(got) + so.TINY[dtype]
    return out, tol * 1.01 + 1e-30


def logprobs(x, targets, top):
    """{name: (result, tolerance)} of rows x [tokens][vocab]; alternatives as whole numbers beside their log probabilities.

    The tolerance counts, with u = 2^-24, y = x - m and n = vocab / 256 + 64 (a lane's part of the row and the joins):
      e^y: y's rounding, its product with log2 e (rounded, as the constant is): 3 u |y| at most 88, past which the term
        is below 2^-126 of the largest; one step of exp: 2 u; n roundings of the sum; so s and t are off by the weighted
        mean of 3 u |y| plus (n + 6) u of themselves
      terms below binary32's least normal number, 2^-126 = e^-87.3, may come out as zero: what those with y < -87 add
        to s and to t, whole
      log1p(s) by what s / (1 + s) carries on, one step (2 u) of itself and of the subtractions from it.
    """
    tokens, vocab = x.shape
    n = vocab / 256 + 64
    got = {k: (np.zeros(tokens), np.zeros(tokens)) for k in ("logprobs", "entropy")}
    ids, lps, lps_tol = np.full((tokens, top), -1), np.full((tokens, top), -np.inf), np.zeros((tokens, top))
    for r in range(tokens):
        row = np.asarray(x[r], np.float64)
        m = row.max()
        if m == -np.inf:
            got["logprobs"][0][r] = 0.0 if targets[r] == -1 else -np.inf
            continue
        y = row - m
        e = np.exp(y)
        s = np.delete(e, int(np.argmax(row))).sum()
        log_s = np.log1p(s)
        fine = e > 0
        ey = (e[fine] * y[fine])
        mean = (e[fine] * np.minimum(np.abs(y[fine]), 88.0)).sum() / max(s, 1e-300)
        rel = 3 * U * mean + (n + 6) * U
        gone = y < -87.0
        lost = (e[gone] * (1 - np.maximum(y[gone], -1e4))).sum()
        tol_log = rel * s / (1 + s) + 4 * U * log_s + lost
        t = ey.sum() / (1 + s)
        second = (e[fine] * np.minimum(y[fine] ** 2, 88.0 ** 2)).sum() / (1 + s)
        got["entropy"][0][r] = log_s - t
        got["entropy"][1][r] = tol_log + abs(t) * ((2 * n + 16) * U + rel) + 3 * U * second + 2 * U * abs(log_s - t) + lost
        if targets[r] >= 0:
            lp = y[targets[r]] - log_s
            got["logprobs"][0][r] = lp
            got["logprobs"][1][r] = 0.0 if lp == -np.inf else tol_log + 2 * U * (abs(y[targets[r]]) + abs(lp))
        order = np.lexsort((np.arange(vocab), -(row + 0.0)))[:top]
        order = order[row[order] > -np.inf]
        ids[r, : len(order)] = order
        lps[r, : len(order)] = y[order] - log_s
        lps_tol[r, : len(order)] = tol_log + 2 * U * (np.abs(y[order]) + np.abs(y[order] - log_s))
    got.update(top_ids=(ids, None), top_logprobs=(lps, lps_tol))
    return got
