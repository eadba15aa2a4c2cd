"""The paged 8-bit cache and what reads and writes it, restated in numpy in 64 bits.

Element types are "f32", "f16", "bf16"; a bf16 array is its uint16 bits on the device side and
float32 here.  Caches are dicts: k [pages][kv][place][d], v [pages][kv][d][place] (uint8 bytes),
k_scale, v_scale [pages][kv], format "int8" or "e4m3".
"""

import numpy as np

QMAX = {"int8": 127.0, "e4m3": 448.0}
# Half a step, relative to the value.
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}  # half the smallest f16 step


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def to_device(x, dtype):
    """x rounded to the type, as the bytes a device holds."""
    x = np.asarray(x, np.float32)
    return {"f32": lambda: x, "f16": lambda: x.astype(np.float16), "bf16": lambda: bf16_bits(x)}[dtype]()


def from_device(a, dtype):
    if dtype == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def rounded(x, dtype):
    """Through binary32, then to the type."""
    return from_device(to_device(np.asarray(x, np.float64).astype(np.float32), dtype), dtype)


# ---- e4m3 ----------------------------------------------------------------------------------

_E4M3 = np.array([(m / 8.0 * 2.0 ** -6) if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)])
_E4M3[127] = np.nan
E4M3_VALUES = np.concatenate([_E4M3, -_E4M3])


def e4m3_codes(x):
    """Nearest code, ties to the even one; magnitudes up to 448."""
    a = np.abs(x)
    vals = _E4M3[:127]
    hi = np.clip(np.searchsorted(vals, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = vals[hi] - a, a - vals[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def codes(x, fmt):
    top = QMAX[fmt]
    x = np.where(np.isnan(x), 0.0, np.clip(x, -top, top))
    return np.rint(x).astype(np.int8).view(np.uint8) if fmt == "int8" else e4m3_codes(x)


def values(c, fmt):
    return c.view(np.int8).astype(np.float64) if fmt == "int8" else E4M3_VALUES[c]


# ---- the operators ---------------------------------------------------------------------------


def plan(lengths, added, table, free, count, page, max_tokens):
    """(new_lengths, offsets, positions, slots, owners, counts, table, free), or the refusal's."""
    r, cols = table.shape
    pages = lambda n: -(-n // page)  # noqa: E731
    table, free = table.copy(), free.copy()
    pos, slots, own = np.zeros(max_tokens, np.int32), np.full(max_tokens, -1, np.int32), np.full(max_tokens, -1, np.int32)
    total = sum(max(a, 0) for a in added)
    wrong = any(n < 0 or a < -1 or pages(n + max(a, 0)) > cols for n, a in zip(lengths, added)) or total > max_tokens
    back = [] if wrong else [table[i, j] for i in range(r) if added[i] == -1 for j in range(pages(lengths[i]))]
    wrong = wrong or not 0 <= count <= len(free) or count + len(back) > len(free)
    need = 0 if wrong else sum(pages(n + a) - pages(n) for n, a in zip(lengths, added) if a >= 0)
    short = max(0, need - count - len(back))
    if wrong or short:
        return np.array(lengths), np.zeros(r + 1, np.int64), pos, slots, own, [count, 0, 0, short], table, free
    free[count:count + len(back)] = back
    top = count + len(back)
    t, new, offsets = 0, [], [0]
    for i in range(r):
        if added[i] == -1:
            new.append(0)
            offsets.append(t)
            continue
        for j in range(pages(lengths[i]), pages(lengths[i] + added[i])):
            top -= 1
            table[i, j] = free[top]
        for p in range(lengths[i], lengths[i] + added[i]):
            pos[t], own[t], slots[t] = p, i, table[i, p // page] * page + p % page
            t += 1
        new.append(lengths[i] + added[i])
        offsets.append(t)
    return np.array(new), np.array(offsets), pos, slots, own, [top, t, need, 0], table, free


def rope(x, positions, freq, dims, interleaved, magnitude, norm=None, eps=0.0):
    y = np.asarray(x, np.float64)
    if norm is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps))) * np.asarray(norm, np.float64)
    out = y.copy()
    angle = np.asarray(positions, np.float64)[:, None] * freq
    c, s = (np.cos(angle) * magnitude)[:, None], (np.sin(angle) * magnitude)[:, None]
    ia, ib = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, dims // 2), slice(dims // 2, dims))
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    return out


def _append_one(code, scale, x, slots, page, fmt, swap):
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % page:
            n += 1
        pg, first = slots[t] // page, slots[t] % page
        for h in range(scale.shape[1]):
            run = x[t:t + n, h].astype(np.float64)
            most = np.abs(np.where(np.isfinite(run), run, 0)).max()
            e = -100
            if most > 0:
                e = max(-100, int(np.ceil(np.log2(most / QMAX[fmt]))) - 1)
                while most > QMAX[fmt] * 2.0 ** e:
                    e += 1
            old = float(scale[pg, h]) if first else 0.0
            new = max(old, 2.0 ** e)
            page_codes = code[pg, h].T if swap else code[pg, h]  # [place][d], a view
            if first and new != old:
                page_codes[:first] = codes(values(np.ascontiguousarray(page_codes[:first]), fmt) * (old / new), fmt)
            page_codes[first:first + n] = codes(run / new, fmt)
            scale[pg, h] = new
        t += n


def append(cache, k, v, slots, page):
    """A new cache with the tokens appended (slots well formed)."""
    c = {n: a.copy() if isinstance(a, np.ndarray) else a for n, a in cache.items()}
    _append_one(c["k"], c["k_scale"], k, slots, page, c["format"], False)
    _append_one(c["v"], c["v_scale"], v, slots, page, c["format"], True)
    return c


def gather(cache, row, n, h, page):
    """Keys and values [n][d] of one request and kv head."""
    fmt = cache["format"]
    pages = row[: -(-n // page)]
    d = cache["k"].shape[3]
    if n == 0:
        return np.zeros((0, d)), np.zeros((0, d))
    k = [values(cache["k"][p, h], fmt) * float(cache["k_scale"][p, h]) for p in pages]
    v = [values(np.ascontiguousarray(cache["v"][p, h].T), fmt) * float(cache["v_scale"][p, h]) for p in pages]
    return np.concatenate(k)[:n], np.concatenate(v)[:n]


def attention(cache, q, offsets, lengths, table, page, scale, causal=True, window=0, dtype="f32", drop=()):
    """(out, tolerance): 64-bit results and how far a binary32 evaluation in the documented operand
    widths may be off.  drop: (request, column) pairs whose keys are left out.

    The tolerance counts, for z = log2(e) * scale * q.k with u = 2^-24:
      the first product: D roundings of the sum and two of each product's scales; the parts of q (two of 11 bits,
        2^-22 of the row's largest value an element; one part is exact for f16 and bf16): dz
      p = 2^z: ln 2 * dz, one step of exp (2^-23), and its parts: 2^-22 for two, half a step 2^-11 for one
      sums over n keys: n roundings each, in the numerator and the denominator; six more for joins and the division
    each relative to the term, so against sum p |v| / sum p; and the result's own rounding.
      The probabilities times their page's value scale are held in binary16 with their largest at 2^11 to 2^15, where the
      smallest step is 2^-24: a term far below the largest is off by up to half of it, 2^-25 / 2^11 = 2^-36 of the largest
      p * v_scale for each unit of its code (twice that is allowed), however small the term itself is.
    """
    q = np.asarray(q, np.float64)
    t, heads, d = q.shape
    kv = cache["k"].shape[1]
    g = heads // kv
    out, tol = np.zeros_like(q), np.zeros_like(q)
    u = 2.0 ** -24
    for r in range(len(lengths)):
        n, o0, o1 = int(lengths[r]), int(offsets[r]), int(offsets[r + 1])
        for h in range(kv):
            k, v = gather(cache, table[r], n, h, page)
            gone = np.zeros(n, bool)
            for rr, col in drop:
                if rr == r:
                    gone[col * page:(col + 1) * page] = True
            v = np.where(gone[:, None], 0, v)
            for i in range(o1 - o0):
                lo, hi = 0, n
                if causal:
                    at = n - (o1 - o0) + i
                    hi = max(0, at + 1)
                    lo = max(0, at + 1 - window) if window else 0
                if hi <= lo:
                    continue
                keep = ~gone[lo:hi]
                if not keep.any():
                    continue
                kk, vv = k[lo:hi][keep], v[lo:hi][keep]
                rows = q[o0 + i, h * g:(h + 1) * g]
                z = scale * (rows @ kk.T)
                p = np.exp(z - z.max(1, keepdims=True))
                l = p.sum(1, keepdims=True)
                out[o0 + i, h * g:(h + 1) * g] = (p @ vv) / l
                part = 2.0 ** -22 * np.abs(rows).max(1, keepdims=True) * np.abs(kk).sum(1)[None] if dtype == "f32" else 0.0
                dz = abs(scale) * ((d + 4) * u * (np.abs(rows) @ np.abs(kk).T) + part) + 4 * u * np.abs(z - 0)
                # log2 of the value scale and the maximum enter the exponent: magnitudes up to 2^7.
                dz = dz + 128 * u
                rel = dz.max(1, keepdims=True) * 2 + 2.0 ** -22 + (2.0 ** -21 if dtype == "f32" else 2.0 ** -11) + (2 * len(kk) + 16) * u
                got = out[o0 + i, h * g:(h + 1) * g]
                vs = np.repeat(cache["v_scale"][np.clip(table[r], 0, None), h].astype(np.float64), page)[lo:hi][keep]
                code = np.abs(vv) / vs[:, None]
                floor = 2.0 ** -35 * (p * vs).max(1, keepdims=True) * code.sum(0)[None]
                tol[o0 + i, h * g:(h + 1) * g] = (rel * (p @ np.abs(vv)) + floor) / l + HALF[dtype] * np.abs(got) + TINY[dtype]
    return out, tol * 1.01 + 1e-30
