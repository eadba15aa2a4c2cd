"""The paged cache of 4 bits a value on the GPU, written, read back and attended over, against the 64-bit restatement of
cache4_oracle.py: codes and scales bit for bit, computed values within the roundings that their documentation counts.
"""

import ctypes

import numpy as np
import pytest

import cache4_oracle as co
import prism_hip as ph
import serving_oracle as so
import synth
from hiprt import DeviceBuffer, Graph, hip
from test_gpu_serving import BATCHES, DTYPE, EPS, NP, Rows, check, dev, i32, make_slots, make_table
from test_gpu_serving import Device as Device8
from test_gpu_serving import make_cache as make_cache8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ph.Context(0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def _announce(request):
    print(request.node.name, flush=True)


class At:
    def __init__(self, p):
        self.p = p

    def data_ptr(self):
        return self.p


def make_cache(rng, pages, kv, page, d, lo=-4, hi=1):
    c = {"format": "e2m1"}
    for n in ("k", "v"):
        c[n] = rng.integers(0, 256, (pages, kv, page, d // 2), dtype=np.uint8)
        c[n + "_scale"] = rng.integers(127 + lo, 127 + hi, (pages, kv, d // 32, page), dtype=np.uint8)
    return c


class Device:
    """A cache on the device."""

    def __init__(self, c, page):
        self.host, self.page = c, page
        self.buf = {n: dev(c[n]) for n in ("k", "v", "k_scale", "v_scale")}
        pages, kv, _, half = c["k"].shape
        self.desc = ph.KvCache(**self.buf, format=ph.CACHE_E2M1, pages=pages, page_size=page, kv_heads=kv, head_dim=2 * half)

    def check(self, want):
        for n in ("k", "v", "k_scale", "v_scale"):
            got = self.buf[n].to_numpy(np.uint8).reshape(want[n].shape)
            assert np.array_equal(got, want[n]), (n, np.argwhere(got != want[n])[:5])


def run_append(ctx, cache, k, v, slots, page):
    held = Device(cache, page)
    ctx.kv_append_device(held.desc, DTYPE[k.dtype], k, k.stride, v, v.stride, dev(np.asarray(slots, np.int32)), len(slots))
    return held, ctx.sync()


# ---- append -----------------------------------------------------------------------------------

RUNS = [[(0, 1)], [(5, 1), (0, 1), (15, 1)], [(3, 200), (0, 17)], [(1, 1)] * 40, [(7, 30), (0, 90), (15, 3), (9, 700)]]


@pytest.mark.parametrize("order", ["runs", "shuffled", "padded"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,kv,page", [(128, 4, 16), (64, 3, 32), (256, 1, 64), (128, 2, 128), (64, 5, 256)])
def test_gpu_append4(ctx, dtype, d, kv, page, order):
    rng = np.random.default_rng(d * kv + page)
    for runs in RUNS:
        slots = make_slots(rng, runs, page, sum(n for _, n in runs) // page + 2 * len(runs) + 3)
        if order == "shuffled":
            rng.shuffle(slots)
        elif order == "padded":
            slots = np.where(rng.random(len(slots)) < 0.3, -1, slots)
        tokens = len(slots)
        cache = make_cache(rng, tokens // page + 2 * len(runs) + 3, kv, page, d)
        spread = 2.0 ** rng.integers(-9, 9, (tokens, kv, d))
        k = Rows(rng.standard_normal((tokens, kv, d)) * spread, dtype, pad=9)
        v = Rows(rng.standard_normal((tokens, kv, d)) * spread, dtype, pad=4, shift=3)
        held, rc = run_append(ctx, cache, k, v, slots, page)
        assert rc == 0
        held.check(co.append(cache, k.x, v.x, slots, page))


@pytest.mark.parametrize("tokens", [1023, 4097, 20000])
def test_gpu_append4_of_many_tokens(ctx, tokens):
    rng = np.random.default_rng(tokens)
    kv, d, page = 2, 64, 16
    slots = make_slots(rng, [(3, tokens)], page, tokens // page + 5)
    cache = make_cache(rng, tokens // page + 5, kv, page, d)
    k, v = (Rows(rng.standard_normal((tokens, kv, d)), "bf16") for _ in range(2))
    held, rc = run_append(ctx, cache, k, v, slots, page)
    assert rc == 0
    held.check(co.append(cache, k.x, v.x, slots, page))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gpu_append4_borders(ctx, dtype):
    """Every code's borders on both sides at every exponent, magnitudes on both sides of 6 * 2^e, zeros of both signs, values
    below the smallest scale's steps."""
    rng = np.random.default_rng(2)
    d, page, kv = 64, 16, 1
    marks = np.array([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0])
    near = np.concatenate([marks, marks * (1 + 2.0 ** -7), marks * (1 - 2.0 ** -7)])
    rows = []
    for e in range(-30 if dtype != "f16" else -22, 14):
        x = rng.permutation(np.resize(np.concatenate([near, -near]), 2 * d)).reshape(2, d)
        x[1] *= 0.51  # no value at the top: the exponent below
        rows.append(np.minimum(np.abs(x * 2.0 ** e), 49152) * np.sign(x))
    x = np.concatenate(rows)
    x[0, :32], x[1, 32:] = 0.0, -0.0
    x = x[:, None]
    if dtype == "f32":
        x[3, 0, :32] = 1e-42  # a subnormal
        x[5, 0, 5] = 6.0 * 2.0 ** 3 * (1 + 2.0 ** -23)
    tokens = len(x)
    slots = rng.permutation(-(-tokens // page) * page)[:tokens]
    cache = make_cache(rng, -(-tokens // page), kv, page, d)
    k, v = Rows(x, dtype), Rows(x[::-1].copy(), dtype)
    held, rc = run_append(ctx, cache, k, v, slots, page)
    assert rc == 0
    held.check(co.append(cache, k.x, v.x, slots, page))


@pytest.mark.parametrize("dtype,past", [("f32", [np.nan, np.inf, -np.inf, 49153.0, -3e38]), ("f16", [np.nan, np.inf, -65504.0]),
                                        ("bf16", [np.nan, -np.inf, 49408.0])])
def test_gpu_append4_flags_what_it_cannot_hold(ctx, dtype, past):
    rng = np.random.default_rng(3)
    d, page, kv = 128, 16, 2
    cache = make_cache(rng, 2, kv, page, d)
    slots = np.array([4, 9, 20], np.int32)
    for which in ("k", "v"):
        for bad in past:
            x = {"k": rng.standard_normal((3, kv, d)), "v": rng.standard_normal((3, kv, d))}
            x[which][1, 1, 70] = bad
            k, v = Rows(x["k"], dtype), Rows(x["v"], dtype)
            held, rc = run_append(ctx, cache, k, v, slots, page)
            assert rc == ph.ERR_NONFINITE and ctx.sync() == 0
            held.check(co.append(cache, k.x, v.x, slots, page))


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gpu_append4_scales_follow_the_finite_values(ctx, dtype, rotated):
    """Infinities beside zeros, small values and nothing else, NaNs alone: each group by itself, its neighbours as ever."""
    rng = np.random.default_rng(22)
    d, page, kv, tokens = 64, 16, 2, 6
    x = rng.standard_normal((tokens, kv, d)) * 2.0 ** -5
    x[0, 0, :32], x[0, 0, 7] = 0.0, np.inf
    x[1, 1, 40] = -np.inf
    x[2, 0, 32:] = np.inf
    x[3, 1, :32] = np.nan
    x[4, 0, 5], x[4, 0, 6] = np.nan, np.inf
    x[5, :, 33:40] = -0.0
    k, v, q = Rows(x, dtype), Rows(x[::-1].copy(), dtype), Rows(np.zeros((tokens, 1, d)), dtype)
    slots, held = rng.permutation(2 * page)[:tokens], None
    cache = make_cache(rng, 2, kv, page, d)
    if rotated:  # by nothing: positions of zero
        held, rope = Device(cache, page), ph.Rope(ctx, 8, ph.rope_frequencies(8, 1e4))
        ctx.qkv_append_device(rope, held.desc, ph.QkvAppend(dtype=DTYPE[dtype], tokens=tokens, heads=1, q=q, k=k, v=v, q_stride=q.stride, k_stride=k.stride,
                                                            v_stride=v.stride, positions=i32(np.zeros(tokens)), slots=i32(slots), q_norm=None, k_norm=None,
                                                            eps=EPS, q_out=q, q_out_stride=q.stride))
        rc = ctx.sync()
        rope.close()
    else:
        held, rc = run_append(ctx, cache, k, v, slots, page)
    assert rc == ph.ERR_NONFINITE and ctx.sync() == 0
    kx = k.x.copy()
    if rotated:  # a pair's partner of an infinity, times a sine of 0, is NaN: of dimensions 0 to 3 and 4 to 7
        with np.errstate(invalid="ignore"):
            a, b = kx[..., :4].copy(), kx[..., 4:8].copy()
            kx[..., :4], kx[..., 4:8] = a * 1.0 - b * 0.0, b * 1.0 + a * 0.0
    held.check(co.append(cache, kx, v.x, slots, page))


def test_gpu_append4_flags_slots_outside(ctx):
    rng = np.random.default_rng(4)
    d, page, kv = 128, 16, 2
    cache = make_cache(rng, 2, kv, page, d)
    k, v = (Rows(rng.standard_normal((4, kv, d)), "f32") for _ in range(2))
    for bad in (32, -2, -(1 << 31), (1 << 31) - 1):
        slots = np.array([3, bad, -1, 17])
        held, rc = run_append(ctx, cache, k, v, slots, page)
        assert rc == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        held.check(co.append(cache, k.x, v.x, [3, -1, -1, 17], page))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,d,dims,heads,kv", [(1, 128, 64, 16, 4), (5, 64, 64, 3, 1), (37, 256, 64, 6, 2), (40, 64, 34, 2, 2), (700, 128, 128, 4, 2),
                                                    (9, 128, 8, 40, 8), (33, 256, 256, 4, 4), (6, 64, 16, 1, 1)])
def test_gpu_qkv_append4_is_its_parts(ctx, dtype, tokens, d, dims, heads, kv, normed, interleaved):
    """One call and its three parts, bit for bit; q in place."""
    rng = np.random.default_rng(tokens + d)
    page = 32
    x = rng.standard_normal((tokens, heads + 2 * kv, d))
    fused = Rows(x, dtype, pad=(8 if interleaved else 3))
    q, k, v = (fused.ptr + n * d * np.dtype(NP[dtype]).itemsize for n in (0, heads, heads + kv))
    positions = 1000 + np.arange(tokens)
    slots = make_slots(rng, [(11, tokens)], page, tokens // page + 4)
    slots[tokens // 2] = -1 if tokens > 4 else slots[tokens // 2]
    norms = [dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) if normed else None for _ in range(2)]
    cache = make_cache(rng, tokens // page + 4, kv, page, d)
    rope = ph.Rope(ctx, dims, ph.rope_frequencies(dims, 1e7), interleaved=interleaved, magnitude=1.25)
    one, parts = Device(cache, page), Device(cache, page)
    qr, kr = Rows(np.zeros((tokens, heads, d)), dtype), Rows(np.zeros((tokens, kv, d)), dtype)
    pb, sb = i32(positions), dev(slots)
    ctx.rope_device(rope, DTYPE[dtype], At(q), fused.stride, pb, tokens, heads, d, qr, qr.stride, norms[0], EPS)
    ctx.rope_device(rope, DTYPE[dtype], At(k), fused.stride, pb, tokens, kv, d, kr, kr.stride, norms[1], EPS)
    ctx.kv_append_device(parts.desc, DTYPE[dtype], kr, kr.stride, At(v), fused.stride, sb, tokens)
    ctx.qkv_append_device(rope, one.desc, ph.QkvAppend(dtype=DTYPE[dtype], tokens=tokens, heads=heads, q=q, k=k, v=v, q_stride=fused.stride,
                                                       k_stride=fused.stride, v_stride=fused.stride, positions=pb, slots=sb, q_norm=norms[0],
                                                       k_norm=norms[1], eps=EPS, q_out=q, q_out_stride=fused.stride))
    assert ctx.sync() == 0
    got = fused.read()
    assert np.array_equal(got[:, :heads], qr.read()) and np.array_equal(got[:, heads:], fused.x[:, heads:])
    want = co.append(cache, kr.read(), fused.x[:, heads + kv:], slots, page)
    parts.check(want)
    one.check(want)
    rope.close()


# ---- reading back -------------------------------------------------------------------------------


def held_cache(rng, fmt, pages, kv, page, d):
    if fmt == "e2m1":
        c = make_cache(rng, pages, kv, page, d, -10, 9)
        return c, Device(c, page)
    c = make_cache8(rng, pages, kv, page, d, fmt)
    if fmt == "e4m3":
        for n in ("k", "v"):
            c[n] = np.where(c[n] & 127 == 127, 126, c[n]).astype(np.uint8)
    c["k_scale"] *= np.float32(1.37)  # scales that are no powers of two round
    return c, Device8(c, page)


@pytest.mark.parametrize("fmt", ["e2m1", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,kv,page", [(128, 4, 16), (64, 3, 32), (256, 1, 64), (128, 2, 256)])
def test_gpu_read(ctx, fmt, dtype, d, kv, page):
    rng = np.random.default_rng(d + kv)
    cache, held = held_cache(rng, fmt, 9, kv, page, d)
    every = 9 * page
    kx, vx = (co.values(cache, n).swapaxes(1, 2).reshape(every, kv, d) for n in ("k", "v"))
    orders = {"one": [5], "run": np.arange(3, every - 2), "shuffled": rng.permutation(every), "twice": [7, 7, 3, 7], "padded": [-1, 4, -1, -1, 9],
              "runs": np.concatenate([np.arange(page - 1, page + 40), np.arange(5), np.arange(2 * page + 3, 2 * page + 4)])}
    for name, slots in orders.items():
        slots = np.asarray(slots)
        n = len(slots)
        k, v = (Rows(np.full((n, kv, d), 3.0), dtype, pad=(5 if name == "run" else 8), shift=sh) for sh in (1, 0))
        ctx.kv_read_device(held.desc, DTYPE[dtype], i32(slots), n, k, k.stride, v, v.stride)
        assert ctx.sync() == 0
        for out, x in ((k, kx), (v, vx)):
            want = np.where((slots >= 0)[:, None, None], so.rounded(x[slots], dtype), 3.0)
            assert np.array_equal(out.read(), want), name
        only = Rows(np.zeros((n, kv, d)), dtype)
        ctx.kv_read_device(held.desc, DTYPE[dtype], i32(slots), n, None, 0, only, only.stride)
        assert ctx.sync() == 0 and np.array_equal(only.read()[slots >= 0], v.read()[slots >= 0])
        ctx.kv_read_device(held.desc, DTYPE[dtype], i32(slots), n, only, only.stride, None, 0)
        assert ctx.sync() == 0 and np.array_equal(only.read()[slots >= 0], k.read()[slots >= 0])


@pytest.mark.parametrize("fmt", ["e2m1", "int8", "e4m3"])
def test_gpu_read_flags(ctx, fmt):
    """Slots outside leave their rows; values past the type, and scales that are no numbers."""
    rng = np.random.default_rng(5)
    d, kv, page = 64, 2, 16
    cache, held = held_cache(rng, fmt, 2, kv, page, d)
    for bad in (32, -2, -(1 << 31), (1 << 31) - 1):
        k, v = (Rows(np.full((3, kv, d), 3.0), "f32") for _ in range(2))
        ctx.kv_read_device(held.desc, ph.DTYPE_F32, i32([1, bad, 31]), 3, k, k.stride, v, v.stride)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        for out, n in ((k, "k"), (v, "v")):
            x = so.rounded(co.values(cache, n).swapaxes(1, 2).reshape(-1, kv, d), "f32")
            got = out.read()
            assert np.array_equal(got[[0, 2]], x[[1, 31]]) and (got[1] == 3.0).all()
    for n in ("k", "v"):
        for scale, dtype in ((147 if fmt == "e2m1" else 1e6, "f16"), (255 if fmt == "e2m1" else np.nan, "f32")):
            wrong = {m: a.copy() if isinstance(a, np.ndarray) else a for m, a in cache.items()}
            wrong[n][1, 0], wrong[n + "_scale"][1, 0] = 0x37 if fmt == "e2m1" else 0x70, scale
            there = Device(wrong, page) if fmt == "e2m1" else Device8(wrong, page)
            k, v = (Rows(np.zeros((2, kv, d)), dtype) for _ in range(2))
            ctx.kv_read_device(there.desc, DTYPE[dtype], i32([3, 20]), 2, k, k.stride, v, v.stride)
            assert ctx.sync() == ph.ERR_NONFINITE and ctx.sync() == 0
            ctx.kv_read_device(there.desc, DTYPE[dtype], i32([3, 4]), 2, k, k.stride, v, v.stride)
            assert ctx.sync() == 0


def test_gpu_read_after_append(ctx):
    """What the append wrote comes back within half a step of each group's scale."""
    rng = np.random.default_rng(6)
    d, kv, page, tokens = 128, 2, 16, 100
    k, v = (Rows(rng.standard_normal((tokens, kv, d)) * 2.0 ** rng.integers(-5, 5, (tokens, kv, 1)), "bf16") for _ in range(2))
    slots = rng.permutation(128)[:tokens]
    held, rc = run_append(ctx, make_cache(rng, 8, kv, page, d), k, v, slots, page)
    k2, v2 = (Rows(np.zeros((tokens, kv, d)), "f32") for _ in range(2))
    ctx.kv_read_device(held.desc, ph.DTYPE_F32, i32(slots), tokens, k2, k2.stride, v2, v2.stride)
    assert rc == 0 and ctx.sync() == 0
    for x, y in ((k.x, k2.read()), (v.x, v2.read())):
        g = x.reshape(tokens, kv, -1, 32)
        most = np.abs(g).max(-1, keepdims=True)
        # 6 * 2^e is less than twice the largest magnitude, and the widest step of codes, from 4 to 6, is 2 * 2^e.
        assert (np.abs(y.reshape(g.shape) - g) <= most / 3).all()
        again = co.quantized(y)
        assert np.array_equal(co.values({"k": again[0][None].swapaxes(1, 2), "k_scale": again[1][None].transpose(0, 2, 3, 1), "format": "e2m1"}, "k")[0],
                              y.swapaxes(0, 1))


# ---- attention --------------------------------------------------------------------------------


def attend(ctx, held, q, offsets, lengths, table, scale, causal=True, window=0, max_length=None, out=None):
    t, heads, d = q.shape
    out = out or Rows(np.full(q.shape, 3.0), q.dtype, pad=12)
    call = ph.Attention(dtype=DTYPE[q.dtype], requests=len(lengths), tokens=t, heads=heads, max_pages=table.shape[1],
                        max_length=max(max(lengths), 1) if max_length is None else max_length, q=q, q_stride=q.stride, out=out, out_stride=out.stride,
                        offsets=i32(offsets), lengths=i32(lengths), block_table=i32(table), scale=scale, causal=int(causal), window=window)
    ctx.attention_device(held.desc, call)
    return call, out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,heads,kv,page", [(128, 16, 4, 16), (64, 3, 1, 32), (256, 12, 2, 64), (128, 5, 5, 128), (64, 40, 5, 16), (256, 24, 4, 256)])
@pytest.mark.parametrize("batch", BATCHES)
def test_gpu_attention4(ctx, batch, d, heads, kv, page, dtype):
    rng = np.random.default_rng(len(batch) * d + page)
    added, lengths = (list(x) for x in zip(*BATCHES[batch]))
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)) * 2, dtype, pad=7, shift=1)
    for causal, window in ((True, 0), (True, 40), (False, 0)):
        call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, causal, window)
        assert ctx.sync() == 0
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, causal, window, dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch", [[(200, 200)], [(90, 150), (1, 1), (400, 433)], [(300, 1900)]])
def test_gpu_attention4_of_many_rows(ctx, batch, d, dtype):
    """Workgroups of 128 rows: taken for long keys, in binary32 for many tiles (heads of 64 and 128)."""
    rng = np.random.default_rng(len(batch) + d)
    page = 32
    heads, kv = (512, 256) if dtype == "f32" and d < 256 and len(batch) < 2 and batch[0][1] == 200 else (8, 2)
    added, lengths = (list(x) for x in zip(*batch))
    if heads == 512:
        added, lengths = [330], [330]
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)) * 2, dtype, pad=7, shift=1)
    for causal, window in ((True, 0), (True, 40), (False, 0)):
        call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, causal, window, max_length=2000)
        assert ctx.sync() == 0
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, causal, window, dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_length", [0, 3000, 1 << 20])
def test_gpu_attention4_splits_long_caches(ctx, dtype, max_length):
    """Keys split over workgroups and joined, whatever bound the caller gave for the lengths."""
    rng = np.random.default_rng(8)
    added, lengths, page, d, heads, kv = [1, 2, 1, 1], [2990, 1500, 1, 513], 16, 128, 8, 2
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((5, heads, d)), dtype)
    for window in (0, 1000):
        call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, True, window, max_length=max_length)
        assert ctx.sync() == 0
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, True, window, dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kind", ["single", "drafts", "many"])
def test_gpu_attention4_parts_of_many_blocks(ctx, kind, d, dtype):
    """Every kernel going through dozens of blocks a part (one part a tile, some, and as many as there may be, more than eight of
    them joined), with a page that is none and the start of a window far behind the first blocks."""
    rng = np.random.default_rng(d + len(kind))
    page, kv = 16, 2
    heads, added, lengths = {"single": (8, [1, 1, 1], [9000, 3000, 70]),       # 4 rows a request
                             "drafts": (16, [3, 4, 2], [9000, 3000, 70]),      # 24: two row tiles, but for heads of 256
                             "many": (2, [70, 90], [9000, 3000])}[kind]
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)), dtype, pad=4)
    wrong = table.copy()
    wrong[0, 8200 // page] = -1
    for window in (0, 1500):
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, True, window, dtype, drop=[(0, 8200 // page)])
        for max_length in (0, 9000, 100000):
            call, out = attend(ctx, held, q, offsets, lengths, wrong, d ** -0.5, True, window, max_length=max_length)
            assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
            check(out.read(), want, tol)


@pytest.mark.parametrize("added", [[1, 1, 1], [40, 3, 50]])
def test_gpu_attention4_rows_without_keys(ctx, added):
    """Requests without keys, tokens before the first key: zeros, and the rows behind the last request stay as they were."""
    rng = np.random.default_rng(9)
    page, d, heads, kv = 16, 64, 4, 2
    lengths = [0, 2, 37]  # fewer keys than tokens: the first tokens see none
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    t = offsets[-1] + 5
    q = Rows(rng.standard_normal((t, heads, d)), "f16")
    for causal in (True, False):
        call, out = attend(ctx, held, q, offsets, lengths, table, 0.125, causal)
        assert ctx.sync() == 0
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, 0.125, causal, 0, "f16")
        got = out.read()
        check(got, want, tol, slice(0, offsets[-1]))
        assert (got[offsets[-1]:] == 3.0).all() and (got[: added[0]] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("added", [1, 30, 100])
def test_gpu_attention4_masked_places_hold_anything(ctx, added, d):
    """Scales that are no numbers behind the keys, in pages no row sees, and missing pages before a window."""
    rng = np.random.default_rng(10)
    page, heads, kv, n = 16, 8, 2, 203
    lengths, offsets = [n], [0, added]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    dirty = {m: a.copy() if isinstance(a, np.ndarray) else a for m, a in cache.items()}
    used = table[0, : -(-n // page)]
    for m in ("k", "v"):
        dirty[m + "_scale"][used[-1], :, :, n % page:] = 255
        dirty[m][used[-1], :, n % page:] = 0x7F
        unused = np.setdiff1d(np.arange(pages), used)
        dirty[m + "_scale"][unused] = 255
    held = Device(dirty, page)
    q = Rows(rng.standard_normal((added, heads, d)), "f16")
    call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, max_length=2000)
    assert ctx.sync() == 0
    want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, True, 0, "f16")
    check(out.read(), want, tol)
    # The first column a window of 50 of the first token touches, and none before it.
    first = (n - added + 1 - 50) // page
    gone = table.copy()
    gone[0, :first] = -1
    for m in ("k", "v"):
        dirty[m + "_scale"][used[:first]] = 255
    held = Device(dirty, page)
    call, out = attend(ctx, held, q, offsets, lengths, gone, d ** -0.5, True, 50, max_length=2000)
    assert ctx.sync() == 0
    want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, True, 50, "f16")
    check(out.read(), want, tol)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (256, 256)])
@pytest.mark.parametrize("added", [1, 30, 100])
def test_gpu_attention4_places_before_a_window_hold_anything(ctx, added, d, page):
    """Scales that are no numbers in front of the first token's window, in the page where the window begins, at every place of
    16 neighbours it may begin at."""
    rng = np.random.default_rng(21)
    heads, kv = 8, 2
    n, windows = (203, [*range(37, 55), 1, 2, 100]) if added < 100 else (1830, range(1601, 1618))  # workgroups of 64 and 128 rows
    lengths, offsets = [n], [0, added]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    q = Rows(rng.standard_normal((added, heads, d)), "f16")
    at, place = np.divmod(np.arange(n), page)
    for window in windows:
        first = n - added + 1 - window
        dirty = {m: a.copy() if isinstance(a, np.ndarray) else a for m, a in cache.items()}
        for m in ("k", "v"):
            dirty[m + "_scale"][table[0, at[:first]], :, :, place[:first]] = 255
            dirty[m][table[0, at[:first]], :, place[:first]] = 0x7F
        call, out = attend(ctx, Device(dirty, page), q, offsets, lengths, table, d ** -0.5, True, window, max_length=2000)
        assert ctx.sync() == 0, window
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, True, window, "f16")
        check(out.read(), want, tol)


@pytest.mark.parametrize("added", [1, 40])
def test_gpu_attention4_leaves_out_pages_that_are_none(ctx, added):
    rng = np.random.default_rng(11)
    page, d, heads, kv = 32, 128, 4, 2
    lengths, offsets = [300, 250], [0, added, added + 1]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((added + 1, heads, d)), "bf16")
    for bad in (-1, pages, -(1 << 31), (1 << 31) - 1):
        wrong = table.copy()
        wrong[0, 3] = bad
        call, out = attend(ctx, held, q, offsets, lengths, wrong, 0.1)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, 0.1, True, 0, "bf16", drop=[(0, 3)])
        check(out.read(), want, tol)


def test_gpu_attention4_flags_lengths_and_offsets(ctx):
    rng = np.random.default_rng(12)
    page, d, heads, kv = 16, 64, 2, 1
    table, pages = make_table(rng, [40, 40, 40], page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((3, heads, d)), "f32")
    for offsets, lengths in (([0, 1, 2, 3], [40, -1, 40]), ([0, 1, 2, 3], [40, 1000, 40]), ([0, 2, 1, 3], [40, 40, 40]), ([0, 1, 2, 9], [40, 40, 40]),
                             ([-1, 1, 2, 3], [40, 40, 40])):
        call, out = attend(ctx, held, q, offsets, lengths, table, 0.1, max_length=48)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("added", [1, 9, 40])
def test_gpu_attention4_writes_the_valid_requests_alone(ctx, added, dtype):
    """Beside a request with a length that cannot be, the others are right; its rows, and whatever stands beside rows, stay as they were.
    Offsets out of order write no other memory than rows."""
    rng = np.random.default_rng(23)
    page, d, heads, kv = 16, 64, 8, 2
    good, offsets = [40, 33, 47], np.arange(4) * added
    table, pages = make_table(rng, good, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((3 * added + 2, heads, d)), dtype)
    want, tol = co.attention(cache, q.x, offsets, good, table, page, 0.1, True, 0, dtype)
    for wrong in range(3):
        for n in (-1, 1000, 65, -(1 << 31), (1 << 31) - 1):  # the table has four columns of 16
            lengths = [n if r == wrong else x for r, x in enumerate(good)]
            call, out = attend(ctx, held, q, offsets, lengths, table, 0.1, max_length=64)
            assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
            got, rows = out.read(), slice(added * wrong, added * wrong + added)
            assert (got[rows] == 3.0).all() and (got[3 * added:] == 3.0).all()
            others = np.r_[0:added * wrong, added * wrong + added:3 * added]
            check(got, want, tol, others)
    t = len(q.x)
    for bad in ([0, 2, 1, 3], [0, 1, 2, t + 1], [-1, 1, 2, 3], [0, t, 0, t], [0, -5, 2, 3], [0, (1 << 31) - 1, 2, 3]):
        call, out = attend(ctx, held, q, bad, good, table, 0.1, max_length=64)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        out.read()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("added", [1, 40])
def test_gpu_attention4_flags_nonfinite_rows(ctx, dtype, added):
    rng = np.random.default_rng(13)
    page, d, heads, kv = 16, 128, 4, 2
    lengths, offsets = [100, 90], [0, added, 2 * added]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    for bad in (np.nan, np.inf):
        x = rng.standard_normal((2 * added, heads, d))
        x[0, 1, 17] = bad
        q = Rows(x, dtype)
        call, out = attend(ctx, held, q, offsets, lengths, table, 0.1)
        assert ctx.sync() == ph.ERR_NONFINITE and ctx.sync() == 0
        x[0, 1] = 0
        want, tol = co.attention(cache, Rows(x, dtype).x, offsets, lengths, table, page, 0.1, True, 0, dtype)
        keep = np.ones((2 * added, heads), bool)
        keep[0, 1] = False
        check(out.read(), want, tol, keep)


@pytest.mark.parametrize("added", [1, 40])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gpu_attention4_ranges(ctx, dtype, added):
    """Scales over the format's whole range, large and small queries, scores that leave one key its weight, a negative scale."""
    rng = np.random.default_rng(14)
    page, d, heads, kv, n = 16, 128, 4, 2, 150
    lengths, offsets = [n], [0, added]
    table, pages = make_table(rng, lengths, page)
    for lo, hi, size, scale in ((13, 14, 1e-3, 0.1), (-23, -22, 100.0, 5.0), (-23, 14, 1e-4, 0.01), (-4, 1, 30.0, 0.5), (-4, 1, 1.0, -0.3),
                                (-4, 1, 0.0, 1.0), (-4, 1, 1.0, 0.0)):
        cache = make_cache(rng, pages, kv, page, d, lo, hi)
        held = Device(cache, page)
        q = Rows(rng.standard_normal((added, heads, d)) * size, dtype)
        call, out = attend(ctx, held, q, offsets, lengths, table, scale)
        assert ctx.sync() == 0
        want, tol = co.attention(cache, q.x, offsets, lengths, table, page, np.float32(scale), True, 0, dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("added", [1, 40])
def test_gpu_attention4_in_place(ctx, added):
    rng = np.random.default_rng(15)
    page, d, heads, kv = 16, 128, 8, 2
    lengths, offsets = [700, 60], [0, added, 2 * added]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((2 * added, heads, d)), "bf16", pad=8)
    want, tol = co.attention(cache, q.x, offsets, lengths, table, page, 0.1, True, 0, "bf16")
    call, out = attend(ctx, held, q, offsets, lengths, table, 0.1, out=q)
    assert ctx.sync() == 0
    check(q.read(), want, tol)


@pytest.mark.parametrize("requests", [1, 65, 3000])
def test_gpu_attention4_of_many_requests(ctx, requests):
    """Requests without tokens among thousands."""
    rng = np.random.default_rng(requests)
    page, d, heads, kv = 16, 64, 2, 1
    added = np.where(rng.random(requests) < 0.5, 0, 1)
    added[-1] = 1
    lengths = rng.integers(1, 40, requests).tolist()
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d)
    held = Device(cache, page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)), "f16")
    call, out = attend(ctx, held, q, offsets, lengths, table, 0.125)
    assert ctx.sync() == 0
    want, tol = co.attention(cache, q.x, offsets, lengths, table, page, 0.125, True, 0, "f16")
    check(out.read(), want, tol)


@pytest.mark.parametrize("added", [1, 6, 70, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_gpu_cache4_past_32_bits(ctx, added, d):
    """Pages whose codes stand past 4 GB: appended to, read back and attended over."""
    page, kv, heads = 256, 8, 8
    pages = (1 << 33) // (page * kv * d // 2) + 40  # 8 GB of codes each
    rng = np.random.default_rng(16)
    buf = {n: DeviceBuffer(pages * kv * page * d // 2) for n in ("k", "v")}
    buf.update({n: DeviceBuffer(pages * kv * page * d // 32) for n in ("k_scale", "v_scale")})
    desc = ph.KvCache(**buf, format=ph.CACHE_E2M1, pages=pages, page_size=page, kv_heads=kv, head_dim=d)
    use = [pages - 1, 3, pages // 2 + 5, pages - 9]
    n = 3 * page + 77
    x = {m: rng.standard_normal((n, kv, d)).astype(np.float32) for m in ("k", "v")}
    slots = np.array([use[i // page] * page + i % page for i in range(n)], np.int32)
    k, v = Rows(x["k"], "f32"), Rows(x["v"], "f32")
    sb = dev(slots)
    ctx.kv_append_device(desc, ph.DTYPE_F32, k, k.stride, v, v.stride, sb, n)
    k2, v2 = (Rows(np.zeros((n, kv, d)), "f32") for _ in range(2))
    ctx.kv_read_device(desc, ph.DTYPE_F32, sb, n, k2, k2.stride, v2, v2.stride)
    small = {"format": "e2m1"}
    for m in ("k", "v"):
        small[m], small[m + "_scale"] = np.zeros((4, kv, page, d // 2), np.uint8), np.zeros((4, kv, d // 32, page), np.uint8)
    small = co.append(small, x["k"], x["v"], np.arange(n), page)
    q = Rows(rng.standard_normal((added, heads, d)), "f16")
    held = type("Held", (), {"desc": desc})
    call, out = attend(ctx, held, q, [0, added], [n], np.array([use]), 0.1, max_length=2000)
    assert ctx.sync() == 0
    for got, m in ((k2, "k"), (v2, "v")):
        assert np.array_equal(got.read(), co.values(small, m).swapaxes(1, 2).reshape(-1, kv, d)[:n])
    want, tol = co.attention(small, q.x, [0, added], [n], np.arange(4)[None], page, 0.1, True, 0, "f16")
    check(out.read(), want, tol)


def far_cache4(d):
    """A cache of 8 GB of codes each, and the pages that are used."""
    page, kv = 256, 8
    pages = (1 << 33) // (page * kv * d // 2) + 40
    buf = {n: DeviceBuffer(pages * kv * page * d // 2) for n in ("k", "v")}
    buf.update({n: DeviceBuffer(pages * kv * page * d // 32) for n in ("k_scale", "v_scale")})
    return ph.KvCache(**buf, format=ph.CACHE_E2M1, pages=pages, page_size=page, kv_heads=kv, head_dim=d), buf, [pages - 1, 3, pages // 2 + 5, pages - 9]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("added", [1, 20, 70, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_gpu_attention4_past_32_bits_in_every_form(ctx, added, d, dtype):
    """Codes past 4 GB: one and two row tiles, 64 and 128 rows a workgroup, one part and several, binary32 and 16 bits."""
    page, kv, n = 256, 8, 3 * 256 + 77
    heads = 512 if added == 300 and dtype == "f32" and d < 256 else 8  # 128 rows a workgroup in binary32
    desc, buf, use = far_cache4(d)
    rng = np.random.default_rng(24)
    small = make_cache(rng, 4, kv, page, d)
    for m, b in buf.items():
        for i, at in enumerate(use):
            b.upload(small[m][i], at * small[m][i].nbytes)
    q = Rows(rng.standard_normal((added, heads, d)), dtype)
    held = type("Held", (), {"desc": desc})
    want, tol = co.attention(small, q.x, [0, added], [n], np.arange(4)[None], page, 0.1, True, 0, dtype)
    for max_length in (0, n, 2000):
        call, out = attend(ctx, held, q, [0, added], [n], np.array([use]), 0.1, max_length=max_length)
        assert ctx.sync() == 0
        check(out.read(), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("d", [64, 256])
def test_gpu_read8_past_32_bits(ctx, fmt, d):
    """Pages of an 8-bit cache whose codes stand past 4 GB, read back."""
    page, kv = 64, 8
    pages = (1 << 33) // (page * kv * d) + 40
    rng = np.random.default_rng(25)
    small = make_cache8(rng, 4, kv, page, d, fmt)
    if fmt == "e4m3":
        for n in ("k", "v"):
            small[n] = np.where(small[n] & 127 == 127, 126, small[n]).astype(np.uint8)
    buf = {n: DeviceBuffer(pages * kv * page * d) for n in ("k", "v")}
    buf.update({n: DeviceBuffer(4 * pages * kv) for n in ("k_scale", "v_scale")})
    desc = ph.KvCache(**buf, format={"int8": ph.CACHE_INT8, "e4m3": ph.CACHE_E4M3}[fmt], pages=pages, page_size=page, kv_heads=kv, head_dim=d)
    use = np.array([pages - 1, 3, pages // 2 + 5, pages - 9])
    for m, b in buf.items():
        for i, at in enumerate(use):
            b.upload(small[m][i], int(at) * small[m][i].nbytes)
    x = {m: so.rounded(co.values(small, m).swapaxes(1, 2).reshape(-1, kv, d), "f32") for m in ("k", "v")}
    for order in (np.arange(3, 4 * page - 5), rng.permutation(4 * page)):
        slots = use[order // page] * page + order % page
        k, v = (Rows(np.zeros((len(order), kv, d)), "f32") for _ in range(2))
        ctx.kv_read_device(desc, ph.DTYPE_F32, i32(slots), len(order), k, k.stride, v, v.stride)
        assert ctx.sync() == 0
        assert np.array_equal(k.read(), x["k"][order]) and np.array_equal(v.read(), x["v"][order])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_gpu_attention4_same_result_each_time_in_16_bits(ctx, d, dtype):
    """Single tokens over many parts and chunks, other calls between: every repeat gives the same bits."""
    rng = np.random.default_rng(26)
    page, heads, kv, lengths = 16, 16, 4, [5000, 900, 17]
    table, pages = make_table(rng, lengths, page)
    held = Device(make_cache(rng, pages, kv, page, d), page)
    other = Rows(rng.standard_normal((3, heads, d)), "f32")
    for added in ([1, 1, 1], [150, 90, 17]):
        offsets = np.concatenate([[0], np.cumsum(added)])
        q = Rows(rng.standard_normal((offsets[-1], heads, d)), dtype)
        first = None
        for _ in range(5):
            attend(ctx, held, other, [0, 1, 2, 3], lengths, table, 0.1)
            call, out = attend(ctx, held, q, offsets, lengths, table, 0.1)
            assert ctx.sync() == 0
            got = out.read()
            assert first is None or np.array_equal(first, got)
            first = got


def test_gpu_attention4_same_result_each_time(ctx):
    rng = np.random.default_rng(17)
    page, d, heads, kv = 16, 128, 32, 8
    lengths, offsets = [4000, 900, 17], [0, 1, 2, 3]
    table, pages = make_table(rng, lengths, page)
    held = Device(make_cache(rng, pages, kv, page, d), page)
    q = Rows(rng.standard_normal((3, heads, d)), "f32")
    first = None
    for _ in range(5):
        call, out = attend(ctx, held, q, offsets, lengths, table, 0.1)
        assert ctx.sync() == 0
        got = out.read()
        assert first is None or np.array_equal(first, got)
        first = got


def test_gpu_cache4_graphs_share_scratch(ctx):
    """Two captured steps of different sizes and eager calls between their replays: every one gives its own results."""
    rng = np.random.default_rng(18)
    page, d, heads, kv = 16, 128, 8, 2
    steps = []
    for lengths in ([3000, 5], [700, 900, 1100, 30]):
        n = len(lengths)
        table, pages = make_table(rng, lengths, page)
        cache = make_cache(rng, pages, kv, page, d)
        held = Device(cache, page)
        q = Rows(rng.standard_normal((n, heads, d)), "f32")
        call, out = attend(ctx, held, q, range(n + 1), lengths, table, 0.1)
        assert ctx.sync() == 0
        want, tol = co.attention(cache, q.x, range(n + 1), lengths, table, page, 0.1, True, 0, "f32")
        steps.append((held, q, call, out, want, tol))
    graphs = [Graph(ctx.stream(), lambda s=s: ctx.attention_device(s[0].desc, s[2])) for s in steps]
    long, big = make_table(rng, [9000], page)
    other = Device(make_cache(rng, big, kv, page, d), page)
    for i in (0, 1, 1, 0, 1):
        steps[i][3].buf.zero()
        graphs[i].launch()
        attend(ctx, other, Rows(np.ones((1, heads, d)), "f32"), [0, 1], [9000], long, 0.1)
        assert ctx.sync() == 0
        flat = steps[i][3].buf.to_numpy(np.float32)[steps[i][3].where].reshape(steps[i][4].shape)
        check(flat, steps[i][4], steps[i][5])


@pytest.mark.parametrize("fmt", ["e2m1", "int8", "e4m3"])
def test_gpu_append_and_read_replayed(ctx, fmt):
    """A captured append and read, replayed with other tokens, slots and eager calls between, gives what eager calls give."""
    rng = np.random.default_rng(20)
    page, d, kv, tokens = 16, 64, 3, 21
    (_, held), (_, eager) = (held_cache(np.random.default_rng(1), fmt, 8, kv, page, d) for _ in range(2))
    order = i32(np.arange(tokens))
    k, v = (Rows(np.zeros((tokens, kv, d)), "bf16") for _ in range(2))
    k2, v2 = (Rows(np.zeros((tokens, kv, d)), "f32") for _ in range(2))

    def run(cache):
        ctx.kv_append_device(cache.desc, ph.DTYPE_BF16, k, k.stride, v, v.stride, order, tokens)
        ctx.kv_read_device(cache.desc, ph.DTYPE_F32, order, tokens, k2, k2.stride, v2, v2.stride)

    run(held), run(eager)
    assert ctx.sync() == 0
    graph = Graph(ctx.stream(), lambda: run(held))
    for start in (0, 21, 42, 63):
        order.upload(np.arange(start, start + tokens, dtype=np.int32))
        for x in (k, v):
            x.buf.upload(so.to_device(rng.standard_normal(x.buf.nbytes // 2), "bf16"))
        run(eager)
        assert ctx.sync() == 0
        want = k2.read(), v2.read()
        assert np.abs(want[0]).max() > 0
        for x in (k2, v2):
            x.buf.upload(x.before)
        graph.launch()
        assert ctx.sync() == 0
        assert np.array_equal(k2.read(), want[0]) and np.array_equal(v2.read(), want[1])


def test_gpu_serving_step_with_the_4_bit_cache_and_log_probabilities(ctx):
    """Plan, projection, append, attention, projection, head and log probabilities, eager and as a graph that carries
    its own lengths: each operator's output against the restatement applied to what it was given."""
    rng = np.random.default_rng(19)
    hidden, heads, kv, d, page, r, vocab, top = 512, 4, 2, 128, 16, 3, 1000, 5
    rows = (heads + 2 * kv) * d
    wqkv = ctx.weight(ph.KIND_PTQ1, hidden, rows, synth.ptq1_weights(rows, hidden, seed=1))
    wo = ctx.weight(ph.KIND_PTQ1, heads * d, hidden, synth.ptq1_weights(hidden, heads * d, seed=2))
    head = ctx.weight(ph.KIND_PTQ1, hidden, vocab, synth.ptq1_weights(vocab, hidden, seed=3))
    cols, pages = 4, 12
    lengths = i32([30, 0, 17])
    cb, tb, fb = i32([pages - 4, 0, 0, 0]), i32([[0, 1, -1, -1], [-1] * 4, [2, 3, -1, -1]]), i32(np.arange(4, 16)[:pages])
    outs = {n: i32(np.zeros(k)) for n, k in (("offsets", r + 1), ("positions", r), ("slots", r), ("owners", r))}
    plan = ph.KvPlan(requests=r, max_pages=cols, max_tokens=r, page_size=page, free_capacity=pages, lengths=lengths, added=i32([1] * r), block_table=tb,
                     free_pages=fb, free_count=cb, new_lengths=lengths, counts=cb, **outs)
    cache = make_cache(rng, 16, kv, page, d)
    held = Device(cache, page)
    f = lambda *s: dev(np.zeros(s, np.float32))  # noqa: E731
    x, qkv, att, y, logits, lp, ent, tlp = dev(rng.standard_normal((r, hidden)).astype(np.float32)), f(r, rows), f(r, heads * d), f(r, hidden), \
        f(r, vocab), f(r), f(r), f(r, top)
    ids, targets = i32(np.zeros((r, top))), i32([5, -1, 999])
    rope = ph.Rope(ctx, 64, ph.rope_frequencies(64, 1e4))
    qp, kp, vp = (qkv.ptr + 4 * d * n for n in (0, heads, heads + kv))
    step = ph.QkvAppend(dtype=ph.DTYPE_F32, tokens=r, heads=heads, q=qp, k=kp, v=vp, q_stride=rows, k_stride=rows, v_stride=rows,
                        positions=outs["positions"], slots=outs["slots"], q_norm=None, k_norm=None, eps=EPS, q_out=qp, q_out_stride=rows)
    attn = ph.Attention(dtype=ph.DTYPE_F32, requests=r, tokens=r, heads=heads, max_pages=cols, max_length=64, q=qp, q_stride=rows, out=att,
                        out_stride=heads * d, offsets=outs["offsets"], lengths=lengths, block_table=tb, scale=d ** -0.5, causal=1, window=0)
    answer = ph.Logprobs(dtype=ph.DTYPE_F32, tokens=r, vocab=vocab, top=top, logits=logits, stride=vocab, targets=targets, logprobs=lp, entropy=ent,
                         top_ids=ids, top_logprobs=tlp)

    def run():
        ctx.kv_plan_device(plan)
        ctx.project_device(wqkv, ph.PATH_F32, x, r, False, qkv)
        ctx.qkv_append_device(rope, held.desc, step)
        ctx.attention_device(held.desc, attn)
        ctx.project_device(wo, ph.PATH_F32, att, r, False, y)
        ctx.project_device(head, ph.PATH_F32, y, r, False, logits)
        ctx.logprobs_device(answer)

    def verify():
        n = lengths.to_numpy(np.int32)
        table = tb.to_numpy(np.int32).reshape(r, cols)
        slots = outs["slots"].to_numpy(np.int32)
        now = {"format": "e2m1"}
        for m in ("k", "v", "k_scale", "v_scale"):
            now[m] = held.buf[m].to_numpy(np.uint8).reshape(cache[m].shape)
        got = qkv.to_numpy(np.float32).reshape(r, heads + 2 * kv, d)
        plain = got[:, heads:heads + kv].astype(np.float64)
        turned = so.rope(plain, outs["positions"].to_numpy(np.int32), ph.rope_frequencies(64, 1e4), 64, False, 1.0).astype(np.float32)
        want = co.append(verify.cache, turned, got[:, heads + kv:], slots, page)
        for m in ("k", "v", "k_scale", "v_scale"):
            assert np.array_equal(now[m], want[m]), m
        verify.cache = now
        o, tol = co.attention(now, got[:, :heads], range(r + 1), n, table, page, d ** -0.5)
        check(att.to_numpy(np.float32).reshape(r, heads, d), o, tol)
        w = co.logprobs(logits.to_numpy(np.float32).reshape(r, vocab), [5, -1, 999], top)
        assert np.array_equal(ids.to_numpy(np.int32).reshape(r, top), w["top_ids"][0])
        for b, name in ((lp, "logprobs"), (ent, "entropy"), (tlp, "top_logprobs")):
            check(b.to_numpy(np.float32).reshape(w[name][0].shape), *w[name])

    verify.cache = cache
    run()
    assert ctx.sync() == 0
    verify()
    graph = Graph(ctx.stream(), run)
    for _ in range(20):
        graph.launch()
        assert ctx.sync() == 0
        verify()
    assert lengths.to_numpy(np.int32).tolist() == [51, 21, 38]
    rope.close()
