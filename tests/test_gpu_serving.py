"""Block tables, rotary positions, the paged 8-bit cache and attention over it, on the GPU against
the 64-bit restatement of serving_oracle.py: codes, scales and whole numbers bit for bit,
computed values within the roundings that their documentation counts.
"""

import ctypes
import itertools

import numpy as np
import pytest

import prism_hip as ph
import serving_oracle as so
import synth
from hiprt import DeviceBuffer, Graph, hip, synchronize

pytestmark = pytest.mark.gpu

DTYPE = {"f32": ph.DTYPE_F32, "f16": ph.DTYPE_F16, "bf16": ph.DTYPE_BF16}
NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
FORMAT = {"int8": ph.CACHE_INT8, "e4m3": ph.CACHE_E4M3}
EPS = 1e-6


@pytest.fixture(scope="module")
def ctx():
    c = ph.Context(0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def _announce(request):
    print(request.node.name, flush=True)


def dev(a):
    return DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def i32(a):
    return dev(np.asarray(a, np.int32))


class Rows:
    """Rows [tokens][heads][d] inside wider, offset memory: pad elements before and behind each token's."""

    def __init__(self, x, dtype, pad=0, shift=0):
        self.dtype, self.shape = dtype, x.shape
        t, h, d = x.shape
        self.stride, self.shift = h * d + pad, shift
        flat = np.full(shift + t * self.stride + 8, 0x5A5A, np.uint16).view(NP[dtype]) if dtype != "f32" else \
            np.full(shift + t * self.stride + 8, 7.0, np.float32)
        self.where = shift + np.arange(t)[:, None] * self.stride + np.arange(h * d)[None]
        flat[self.where.reshape(-1)] = so.to_device(x, dtype).reshape(-1)
        self.before = flat.copy()
        self.buf = dev(flat)
        self.ptr = self.buf.data_ptr() + shift * flat.itemsize
        self.x = so.from_device(flat[self.where], dtype).reshape(x.shape)  # as rounded to the type

    def data_ptr(self):
        return self.ptr

    def read(self):
        flat = self.buf.to_numpy(NP[self.dtype])
        outside = np.ones(flat.size, bool)
        outside[self.where.reshape(-1)] = False
        assert np.array_equal(flat[outside].view(np.uint8), self.before[outside].view(np.uint8)), "wrote beside the rows"
        return so.from_device(flat[self.where], self.dtype).reshape(self.shape)


# ---- plan -----------------------------------------------------------------------------------


def run_plan(ctx, lengths, added, table, free, count, page, max_tokens, alias=False, times=1):
    r, cols = table.shape
    lb, cb = i32(lengths), i32([count, 99, 99, 99])
    new, counts = (lb, cb) if alias else (i32(np.full(r, 99)), i32(np.full(4, 99)))
    outs = {n: i32(np.full(k, 99)) for n, k in (("offsets", r + 1), ("positions", max_tokens), ("slots", max_tokens), ("owners", max_tokens))}
    tb, fb = i32(table), i32(free)
    plan = ph.KvPlan(requests=r, max_pages=cols, max_tokens=max_tokens, page_size=page, free_capacity=len(free), lengths=lb, added=i32(added),
                     block_table=tb, free_pages=fb, free_count=cb, new_lengths=new, counts=counts, **outs)
    for _ in range(times):
        ctx.kv_plan_device(plan)
    rc = ctx.sync()
    get = lambda b: b.to_numpy(np.int32)  # noqa: E731
    return rc, [get(new), get(outs["offsets"]), get(outs["positions"]), get(outs["slots"]), get(outs["owners"]), get(counts),
                get(tb).reshape(r, cols), get(fb)]


def make_plan(rng, r, page, longest, most, ended=0.2):
    lengths = rng.integers(0, longest + 1, r)
    added = np.where(rng.random(r) < ended, -1, rng.integers(0, most + 1, r))
    cols = max(1, max(-(-(n + max(a, 0)) // page) for n, a in zip(lengths, added)))
    order = rng.permutation(r * cols + 5).astype(np.int32)
    table, used = np.full((r, cols), -1, np.int32), 0
    for i, n in enumerate(lengths):
        k = -(-n // page)
        table[i, :k] = order[used:used + k]
        used += k
    free = np.concatenate([order[used:], np.full(used, -7, np.int32)])
    return lengths, added, table, free, len(order) - used


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("r,page,longest,most", [(1, 16, 0, 1), (1, 16, 40, 100), (3, 256, 5, 1), (64, 16, 200, 1), (65, 32, 100, 7),
                                                 (1025, 64, 90, 3), (2500, 16, 33, 9), (7, 128, 1000, 2000)])
def test_gpu_plan(ctx, r, page, longest, most, alias):
    rng = np.random.default_rng(r + page)
    case = make_plan(rng, r, page, longest, most)
    room = int(np.maximum(case[1], 0).sum()) + 3
    rc, got = run_plan(ctx, *case, page, room, alias)
    assert rc == 0
    for g, w in zip(got, so.plan(*case, page, room)):
        assert np.array_equal(g, np.asarray(w))


def test_gpu_plan_all_ended_or_idle(ctx):
    table = np.array([[4, 2], [1, -1], [0, 3]], np.int32)
    for added in ([-1, -1, -1], [0, 0, 0], [-1, 0, 5]):
        case = (np.array([20, 16, 32]), np.array(added), np.concatenate([table, np.full((3, 1), -1, np.int32)], 1), np.array([5, 6, -7, -7, -7, -7, -7], np.int32), 2)
        rc, got = run_plan(ctx, *case, 16, 9)
        assert rc == 0
        for g, w in zip(got, so.plan(*case, 16, 9)):
            assert np.array_equal(g, np.asarray(w)), added


@pytest.mark.parametrize("what", ["short", "tokens", "length", "added", "columns", "count", "room"])
def test_gpu_plan_refuses_a_step_as_a_whole(ctx, what):
    lengths, added = np.array([20, 3, 16]), np.array([13, 40, -1])
    table = np.array([[0, 1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1]], np.int32)
    free, count, room = np.array([4, 5, 6, 7, -7], np.int32), 4, 60
    if what == "short":
        count = 1  # one and the one given back, of three that are needed
    elif what == "tokens":
        room = 52
    elif what == "length":
        lengths[1] = -1
    elif what == "added":
        added[1] = -2
    elif what == "columns":
        added[0] = 45
    elif what == "count":
        count = 6
    else:
        free = free[:4]
    rc, got = run_plan(ctx, lengths, added, table, free, count, 16, room)
    assert rc == (ph.ERR_RESOURCE if what == "short" else ph.ERR_INVALID_INPUT)
    for g, w in zip(got, so.plan(lengths, added, table, free, count, 16, room)):
        assert np.array_equal(g, np.asarray(w))
    assert got[5][3] == (1 if what == "short" else 0)
    assert ctx.sync() == 0


@pytest.mark.parametrize("max_tokens", [40, 5000])
def test_gpu_plan_flags_negative_pages(ctx, max_tokens):
    """A held page and a free one below zero: their tokens have no slot, the others theirs."""
    table = np.array([[3, -1, -1], [-5, -1, -1], [1, -1, -1]], np.int32)
    free = np.array([7, -2, 8], np.int32)
    rc, got = run_plan(ctx, np.array([4, 10, 15]), np.array([20, 2, 2]), table, free, 3, 16, max_tokens)
    assert rc == ph.ERR_INVALID_INPUT and ctx.sync() == 0
    assert got[3][:12].tolist() == list(range(3 * 16 + 4, 4 * 16)) and got[3][12:20].tolist() == list(range(8 * 16, 8 * 16 + 8))
    assert got[3][20:22].tolist() == [-1, -1] and got[3][22:24].tolist() == [31, -1] and got[5].tolist() == [1, 24, 2, 0]


def test_gpu_plan_carries_its_state_through_a_graph(ctx):
    """Lengths and the free count in place: replays of one captured step are steps."""
    r, page = 5, 16
    lengths, added = np.array([0, 15, 16, 31, 7]), np.ones(5, np.int64)
    table, free = np.full((r, 6), -1, np.int32), np.arange(40, dtype=np.int32)
    want_free = 40
    for i, n in enumerate(lengths):
        for j in range(-(-n // page)):
            want_free -= 1
            table[i, j] = free[want_free]
    lb, cb, tb, fb = i32(lengths), i32([want_free, 0, 0, 0]), i32(table), i32(free)
    outs = {n: i32(np.zeros(k)) for n, k in (("offsets", r + 1), ("positions", 8), ("slots", 8), ("owners", 8))}
    plan = ph.KvPlan(requests=r, max_pages=6, max_tokens=8, page_size=page, free_capacity=40, lengths=lb, added=i32(added), block_table=tb,
                     free_pages=fb, free_count=cb, new_lengths=lb, counts=cb, **outs)
    ctx.kv_plan_device(plan)
    state = (lengths, table, want_free)
    w = so.plan(state[0], added, state[1], free, state[2], page, 8)
    graph = Graph(ctx.stream(), lambda: ctx.kv_plan_device(plan))
    for step in range(20):
        state = (w[0], w[6], w[5][0])
        assert np.array_equal(lb.to_numpy(np.int32), w[0]) and np.array_equal(tb.to_numpy(np.int32).reshape(r, 6), w[6])
        assert np.array_equal(outs["slots"].to_numpy(np.int32), w[3]), step
        graph.launch()
        assert ctx.sync() == 0
        w = so.plan(state[0], added, state[1], free, state[2], page, 8)


# ---- rotary positions -------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dims,tokens,heads", [(64, 64, 1, 1), (64, 2, 5, 3), (128, 64, 1, 16), (128, 66, 9, 5), (128, 128, 33, 40),
                                                 (256, 64, 6, 24), (256, 256, 3, 7), (64, 34, 130, 2)])
def test_gpu_rope(ctx, dtype, d, dims, tokens, heads):
    rng = np.random.default_rng(d + dims + tokens)
    freq = ph.rope_frequencies(dims, 1e7, 4.0, 2048.0)
    positions = rng.integers(0, 1 << 20, tokens)
    norm = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    for interleaved, normed, in_place in itertools.product((False, True), (False, True), (False, True)):
        x = Rows(rng.standard_normal((tokens, heads, d)), dtype, pad=(3 if tokens % 2 else 8), shift=1 if interleaved else 0)
        out = x if in_place else Rows(np.zeros((tokens, heads, d)), dtype, pad=5)
        rope = ph.Rope(ctx, dims, freq, interleaved=interleaved, magnitude=1.25)
        ctx.rope_device(rope, DTYPE[dtype], x, x.stride, i32(positions), tokens, heads, d, out, out.stride,
                        norm=dev(norm) if normed else None, eps=EPS)
        assert ctx.sync() == 0
        got = out.read()
        want = so.rope(x.x, positions, freq, dims, interleaved, 1.25, norm if normed else None, EPS)
        # Half a step of the type and of binary32; the binary64 work below that.
        tol = (so.HALF[dtype] + 2.0 ** -24) * np.abs(want) * 1.001 + so.TINY[dtype] + 1e-9 * np.abs(x.x).max()
        if dtype == "f32":
            tol = 2.0 ** -24 * np.abs(want) * 1.001 + 1e-12 * np.abs(x.x).max()
        assert (np.abs(got - want) <= tol).all(), (interleaved, normed, np.abs(got - want).max())
        rope.close()


def test_gpu_rope_flags_a_nonfinite_row_and_keeps_the_others(ctx):
    x = np.ones((4, 2, 64), np.float32)
    x[2, 1, 40] = np.nan
    rows, out = Rows(x, "f32"), Rows(np.zeros_like(x), "f32")
    freq = ph.rope_frequencies(64, 1e4)
    rope = ph.Rope(ctx, 64, freq)
    ctx.rope_device(rope, ph.DTYPE_F32, rows, rows.stride, i32(np.arange(4)), 4, 2, 64, out, out.stride)
    assert ctx.sync() == ph.ERR_NONFINITE and ctx.sync() == 0
    got, want = out.read(), so.rope(x, np.arange(4), freq, 64, False, 1.0)
    keep = np.ones((4, 2), bool)
    keep[2, 1] = False
    assert np.allclose(got[keep], want[keep], rtol=1e-6, atol=1e-6)
    rope.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dims", [(64, 8), (64, 34), (128, 64), (128, 66), (256, 64), (256, 192)])
def test_gpu_rope_leaves_what_stands_behind_the_rotated_dims(ctx, dtype, d, dims):
    """Without a norm the values behind the rotated ones come out bit for bit: zeros of both signs, subnormals, and what stands next to an
    infinity; with one, zeros keep their signs.  Several heads a wavefront and heads left over."""
    rng = np.random.default_rng(d + dims)
    tokens, heads = 5, 9
    x = rng.standard_normal((tokens, heads, d))
    x[:, :, dims::3] = -0.0
    x[:, ::2, dims + 1::5] = 0.0
    x[:, 1::3, dims + 5] = {"f32": 1e-42, "f16": 2.0 ** -24, "bf16": 2.0 ** -130}[dtype]
    freq = ph.rope_frequencies(dims, 1e4)
    bits = lambda v: np.ascontiguousarray(np.asarray(v, np.float64)).view(np.uint64)  # noqa: E731
    for interleaved in (False, True):
        rope = ph.Rope(ctx, dims, freq, interleaved=interleaved)
        for infinite, normed in ((False, False), (True, False), (False, True)):
            y = x.copy()
            if infinite:
                y[1, 2, dims + 6], y[3, 8, d - 1] = np.inf, -np.inf
            rows, out = Rows(y, dtype, pad=3), Rows(np.ones_like(y), dtype)
            norm = np.full(d, 1.5, np.float32)
            ctx.rope_device(rope, DTYPE[dtype], rows, rows.stride, i32(np.arange(tokens) * 7), tokens, heads, d, out, out.stride,
                            norm=dev(norm) if normed else None, eps=EPS)
            assert ctx.sync() == (ph.ERR_NONFINITE if infinite else 0)
            got = out.read()
            if normed:
                zero = rows.x[:, :, dims:] == 0
                assert np.array_equal(bits(got[:, :, dims:])[zero], bits(rows.x[:, :, dims:])[zero])
            else:
                assert np.array_equal(bits(got[:, :, dims:]), bits(rows.x[:, :, dims:]))
            want = so.rope(rows.x[:, :, :dims], np.arange(tokens) * 7, freq, dims, interleaved, 1.0)
            if not normed:
                assert (np.abs(got[:, :, :dims] - want) <= (so.HALF[dtype] + 2.0 ** -24) * np.abs(want) * 1.001 + so.TINY[dtype] + 1e-9).all()
        rope.close()


@pytest.mark.parametrize("dims", [64, 66])
@pytest.mark.parametrize("dtype,most", [("f32", 3e38), ("f16", 6e4), ("bf16", 3.3e38)])
def test_gpu_rope_flags_results_past_the_type(ctx, dtype, most, dims):
    x = np.full((2, 3, 128), 1.0)
    x[1, 2, :] = most  # turned by 45 degrees a pair is 1.4 times as long, or none
    freq = np.full(dims // 2, np.pi / 4)
    rope = ph.Rope(ctx, dims, freq)
    rows, out = Rows(x, dtype), Rows(np.zeros_like(x), dtype)
    for position, rc in ((1, ph.ERR_NONFINITE), (0, 0)):
        ctx.rope_device(rope, DTYPE[dtype], rows, rows.stride, i32([position] * 2), 2, 3, 128, out, out.stride)
        assert ctx.sync() == rc
    rope.close()


# ---- append -----------------------------------------------------------------------------------


def make_cache(rng, pages, kv, page, d, fmt):
    c = {"format": fmt}
    for n, shape in (("k", (pages, kv, page, d)), ("v", (pages, kv, d, page))):
        x = rng.standard_normal(shape) * (32 if fmt == "int8" else 100)
        c[n] = so.codes(x, fmt)
        c[n + "_scale"] = np.float32(2.0) ** rng.integers(-8, 2, (pages, kv)).astype(np.float32)
    return c


class Device:
    """A cache on the device."""

    def __init__(self, c, page):
        self.host, self.page = c, page
        self.buf = {n: dev(c[n]) for n in ("k", "v", "k_scale", "v_scale")}
        pages, kv, _, d = c["k"].shape
        self.desc = ph.KvCache(**self.buf, format=FORMAT[c["format"]], pages=pages, page_size=page, kv_heads=kv, head_dim=d)

    def check(self, want):
        for n in ("k", "v"):
            got = self.buf[n].to_numpy(np.uint8).reshape(want[n].shape)
            assert np.array_equal(got, want[n]), (n, np.argwhere(got != want[n])[:5])
            scale = self.buf[n + "_scale"].to_numpy(np.float32).reshape(want[n + "_scale"].shape)
            assert np.array_equal(scale, want[n + "_scale"], equal_nan=True), n


def make_slots(rng, runs, page, pages):
    """Slots of runs (first place, tokens) on pages in no order, split where a page ends."""
    order, slots = list(rng.permutation(pages)), []
    for first, n in runs:
        while n:
            m = min(n, page - first)
            slots += list(order.pop() * page + first + np.arange(m))
            n, first = n - m, 0
    return np.array(slots, np.int32)


RUNS = [[(0, 1)], [(5, 1), (0, 1), (15, 1)], [(3, 200), (0, 17)], [(1, 1)] * 40, [(7, 30), (0, 90), (15, 3), (9, 700)]]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,kv,page", [(128, 4, 16), (64, 3, 32), (256, 1, 64), (128, 2, 128), (64, 5, 256)])
def test_gpu_append(ctx, dtype, fmt, d, kv, page):
    rng = np.random.default_rng(d * kv + page)
    for runs in RUNS:
        tokens = sum(n for _, n in runs)
        cache = make_cache(rng, tokens // page + 2 * len(runs) + 3, kv, page, d, fmt)
        slots = make_slots(rng, runs, page, cache["k"].shape[0])
        spread = 2.0 ** rng.integers(-6, 6, (tokens, kv, 1))
        k = Rows(rng.standard_normal((tokens, kv, d)) * spread, dtype, pad=9)
        v = Rows(rng.standard_normal((tokens, kv, d)) * spread, dtype, pad=4, shift=3)
        held = Device(cache, page)
        ctx.kv_append_device(held.desc, DTYPE[dtype], k, k.stride, v, v.stride, dev(slots), tokens)
        assert ctx.sync() == 0
        held.check(so.append(cache, k.x, v.x, slots, page))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("runs", [[(3, 5000)], [(2, 1)] * 1500, [(0, 1), (15, 3)] * 1300, [(9, 40)] * 60], ids=["prompt", "single", "pairs", "chunks"])
def test_gpu_append_of_many_tokens(ctx, dtype, runs):
    """Each window of tokens a workgroup looks at, full of runs or of one."""
    rng = np.random.default_rng(len(runs))
    kv, d, page = 2, 64, 16
    tokens = sum(n for _, n in runs)
    cache = make_cache(rng, tokens // page + 2 * len(runs) + 3, kv, page, d, "int8")
    slots = make_slots(rng, runs, page, cache["k"].shape[0])
    k, v = (Rows(rng.standard_normal((tokens, kv, d)) * 2.0 ** rng.integers(-3, 3, (tokens, 1, 1)), dtype) for _ in range(2))
    held = Device(cache, page)
    ctx.kv_append_device(held.desc, DTYPE[dtype], k, k.stride, v, v.stride, dev(slots), tokens)
    assert ctx.sync() == 0
    held.check(so.append(cache, k.x, v.x, slots, page))


def test_gpu_append_edges_of_the_scale(ctx):
    """Magnitudes on both sides of qmax * 2^e, zeros, the smallest and the largest floats."""
    d, page = 64, 16
    for fmt, top in (("int8", 127.0), ("e4m3", 448.0)):
        most = [top, np.nextafter(np.float32(top), np.float32(1e9)), top * 2.0 ** -20, 0.0, 1e-45, 1e-38, 3.4e38, top * 2.0 ** -100,
                np.nextafter(np.float32(top * 2.0 ** 20), np.float32(1e30)), 1.0]
        k = np.zeros((len(most), 1, d), np.float32)
        k[:, 0] = np.float32(most)[:, None] * np.linspace(-1, 1, d, dtype=np.float32)
        k[:, 0, 5] = most
        v = -k[:, :, ::-1].copy()
        cache = make_cache(np.random.default_rng(1), len(most), 1, page, d, fmt)
        slots = np.arange(len(most), dtype=np.int32) * page + np.array([0, 3] * 5, np.int32)
        held = Device(cache, page)
        ctx.kv_append_device(held.desc, ph.DTYPE_F32, dev(k), d, dev(v), d, dev(slots), len(most))
        assert ctx.sync() == 0
        held.check(so.append(cache, k, v, slots, page))


def test_gpu_append_over_fresh_memory_token_by_token(ctx):
    """Pages whose memory holds anything, written one token a call: only what was written counts."""
    rng = np.random.default_rng(5)
    kv, d, page, n = 2, 64, 16, 35
    for fmt in ("int8", "e4m3"):
        cache = make_cache(rng, 4, kv, page, d, fmt)
        cache["k"][:], cache["v"][:] = 0xFF, 0x7F
        cache["k_scale"][:], cache["v_scale"][:] = np.nan, np.inf
        held = Device(cache, page)
        slots = np.concatenate([np.arange(16) + 32, np.arange(16), np.arange(3) + 48]).astype(np.int32)
        x = rng.standard_normal((n, 2, kv, d)).astype(np.float32) * 2.0 ** rng.integers(-4, 4, (n, 1, kv, 1)).astype(np.float32)
        want = cache
        for t in range(n):
            k, v = np.ascontiguousarray(x[t:t + 1, 0]), np.ascontiguousarray(x[t:t + 1, 1])
            ctx.kv_append_device(held.desc, ph.DTYPE_F32, dev(k), kv * d, dev(v), kv * d, dev(slots[t:t + 1]), 1)
            want = so.append(want, k, v, slots[t:t + 1], page)
        assert ctx.sync() == 0
        held.check(want)
        # Nothing is off by more than a step of its page's last scale, for all the rescaling.
        for t in range(n):
            p, o = slots[t] // page, slots[t] % page
            step = 1.0 if fmt == "int8" else np.maximum(2.0 ** -9, np.abs(x[t, 0]) / want["k_scale"][p][:, None] * 2.0 ** -4 + 2.0 ** -10)
            got = so.values(want["k"][p, :, o], fmt) * want["k_scale"][p][:, None]
            assert (np.abs(got - x[t, 0]) <= step * want["k_scale"][p][:, None]).all()


def test_gpu_append_skips_padding_and_refuses_bad_slots(ctx):
    rng = np.random.default_rng(6)
    kv, d, page = 2, 128, 16
    cache = make_cache(rng, 6, kv, page, d, "int8")
    # Padding among the tokens; a slot behind the cache, one below -1, and a second run in page 2.
    slots = np.array([-1, 5, 6, -1, 96, 32, 33, 40, -9, 95, -1], np.int32)
    good = np.array([-1, 5, 6, -1, -1, 32, 33, -1, -1, 95, -1], np.int32)
    k = rng.standard_normal((11, kv, d)).astype(np.float32)
    v = rng.standard_normal((11, kv, d)).astype(np.float32)
    for s, rc in ((good, 0), (slots, ph.ERR_INVALID_INPUT)):
        held = Device(cache, page)
        ctx.kv_append_device(held.desc, ph.DTYPE_F32, dev(k), kv * d, dev(v), kv * d, dev(s), 11)
        assert ctx.sync() == rc and ctx.sync() == 0
        held.check(so.append(cache, k, v, good, page))


def test_gpu_append_nonfinite(ctx):
    rng = np.random.default_rng(7)
    cache = make_cache(rng, 2, 1, 16, 64, "int8")
    k = rng.standard_normal((3, 1, 64)).astype(np.float32)
    v = k.copy()
    k[1, 0, 7], k[2, 0, 9], v[0, 0, 3] = np.nan, np.inf, -np.inf
    for fmt in ("int8", "e4m3"):
        cache["format"] = fmt
        held = Device(cache, 16)
        slots = np.array([4, 5, 6], np.int32)
        ctx.kv_append_device(held.desc, ph.DTYPE_F32, dev(k), 64, dev(v), 64, dev(slots), 3)
        assert ctx.sync() == ph.ERR_NONFINITE and ctx.sync() == 0
        held.check(so.append(cache, k, v, slots, 16))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 5, 40, 700])
def test_gpu_qkv_append_is_its_parts(ctx, dtype, tokens):
    """One call and its three parts, bit for bit; q in place."""
    rng = np.random.default_rng(tokens)
    heads, kv, d, page, dims = 6, 2, 128, 32, 64
    x = rng.standard_normal((tokens, heads + 2 * kv, d))
    fused = Rows(x, dtype)
    q, k, v = (fused.ptr + n * d * np.dtype(NP[dtype]).itemsize for n in (0, heads, heads + kv))
    P = ctypes.c_void_p

    class At:
        def __init__(self, p):
            self.p = p

        def data_ptr(self):
            return self.p

    positions = 1000 + np.arange(tokens)
    slots = make_slots(rng, [(11, tokens)], page, tokens // page + 4)
    norms = [dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2)]
    cache = make_cache(rng, tokens // page + 4, kv, page, d, "int8")
    freq = ph.rope_frequencies(dims, 1e7)
    rope = ph.Rope(ctx, dims, freq)
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
    want = so.append(cache, kr.read(), fused.x[:, heads + kv:], slots, page)
    parts.check(want)
    one.check(want)
    rope.close()


# ---- attention --------------------------------------------------------------------------------


def make_table(rng, lengths, page, spare=3):
    cols = max(1, max(-(-n // page) for n in lengths))
    order = rng.permutation(sum(-(-n // page) for n in lengths) + spare).astype(np.int32)
    table, used = np.full((len(lengths), cols + 1), -1, np.int32), 0
    for i, n in enumerate(lengths):
        k = -(-n // page)
        table[i, :k] = order[used:used + k]
        used += k
    return table, len(order)


def attend(ctx, held, q, offsets, lengths, table, scale, causal=True, window=0, max_length=None, out=None):
    t, heads, d = q.shape
    out = out or Rows(np.full(q.shape, 3.0), q.dtype, pad=12)
    call = ph.Attention(dtype=DTYPE[q.dtype], requests=len(lengths), tokens=t, heads=heads, max_pages=table.shape[1],
                        max_length=max(max(lengths), 1) if max_length is None else max_length, q=q, q_stride=q.stride, out=out, out_stride=out.stride,
                        offsets=i32(offsets), lengths=i32(lengths), block_table=i32(table), scale=scale, causal=int(causal), window=window)
    ctx.attention_device(held.desc, call)
    return call, out


def check(got, want, tol, rows=slice(None)):
    off = np.abs(got[rows] - want[rows])
    fine = bool((off <= tol[rows]).all())
    assert fine, (float(off.max()), float((off / tol[rows]).max()), np.argwhere(~(off <= tol[rows]))[:5].tolist())


# (new tokens, keys) of each request.
BATCHES = {
    "one": [(1, 1)],
    "step": [(1, n) for n in (1, 15, 16, 17, 63, 64, 65, 127, 500)],
    "draft": [(4, 4), (3, 300), (1, 2), (7, 64)],
    "chunk": [(70, 70), (33, 200), (1, 130)],
    "prompt": [(200, 200)],
    "mixed": [(90, 150), (1, 1), (1, 333), (2, 64), (130, 131)],
    "drafts": [(7, 64), (6, 200), (8, 8)],             # 17 to 32 rows a request
    "long-among-single": [(60, 60)] + [(1, 50)] * 20,  # many tiles of few rows for one request
}


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,heads,kv,page", [(128, 16, 4, 16), (64, 3, 1, 32), (256, 12, 2, 64), (128, 5, 5, 128)])
@pytest.mark.parametrize("batch", BATCHES)
def test_gpu_attention(ctx, batch, d, heads, kv, page, dtype, fmt):
    rng = np.random.default_rng(len(batch) * d + page)
    added, lengths = (list(x) for x in zip(*BATCHES[batch]))
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, fmt)
    cache["k_scale"] *= 0.25
    held = Device(cache, page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)) * 2, dtype, pad=7, shift=1)
    for causal, window in ((True, 0), (True, 40), (False, 0)):
        call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, causal, window)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, causal, window, dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_length", [0, 3000, 1 << 20])
def test_gpu_attention_splits_long_caches(ctx, dtype, max_length):
    """Keys split over workgroups and joined, whatever bound the caller gave for the lengths."""
    rng = np.random.default_rng(8)
    added, lengths, page, d, heads, kv = [1, 2, 1, 1], [2990, 1500, 1, 513], 16, 128, 8, 2
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["k_scale"] *= 0.25
    held = Device(cache, page)
    q = Rows(rng.standard_normal((5, heads, d)), dtype)
    for window in (0, 1000):
        call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, True, window, max_length=max_length)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5, True, window, dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("added", [[1, 1, 1], [40, 3, 50]])
def test_gpu_attention_rows_without_keys(ctx, fmt, added):
    """Requests without keys, tokens before the first key, other tokens of the batch: zeros, and the
    rows behind the last request stay as they were."""
    rng = np.random.default_rng(9)
    page, d, heads, kv = 16, 64, 4, 2
    lengths = [0, 2, 37]  # fewer keys than tokens: the first tokens see none
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, fmt)
    held = Device(cache, page)
    t = offsets[-1] + 5
    q = Rows(rng.standard_normal((t, heads, d)), "f16")
    for causal in (True, False):
        call, out = attend(ctx, held, q, offsets, lengths, table, 0.125, causal)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, offsets, lengths, table, page, 0.125, causal, 0, "f16")
        got = out.read()
        check(got, want, tol, slice(0, offsets[-1]))
        assert (got[offsets[-1]:] == 3.0).all()
        assert (got[: added[0]] == 0).all()


@pytest.mark.parametrize("added", [1, 30])
def test_gpu_attention_masked_places_hold_anything(ctx, added):
    """NaN codes and scales behind the keys, in pages no row sees, and missing pages before a window."""
    rng = np.random.default_rng(10)
    page, d, heads, kv, n = 16, 128, 8, 2, 203
    lengths, offsets = [n], [0, added]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, "e4m3")
    want_cache = {k: (a.copy() if isinstance(a, np.ndarray) else a) for k, a in cache.items()}
    last = table[0, n // page]
    cache["k"][last, :, n % page:] = 0x7F
    cache["v"][last, :, :, n % page:] = 0xFF
    used = set(table[0, : -(-n // page)].tolist())
    for p in set(range(pages)) - used:
        cache["k"][p], cache["v"][p], cache["k_scale"][p], cache["v_scale"][p] = 0x7F, 0x7F, np.nan, np.nan
    held = Device(cache, page)
    q = Rows(rng.standard_normal((added, heads, d)), "f32")
    for window in (0, 50):
        tb = table.copy()
        if window:
            tb[0, : (n - added + 1 - window) // page] = -1
        call, out = attend(ctx, held, q, offsets, lengths, tb, d ** -0.5, True, window)
        assert ctx.sync() == 0
        want, tol = so.attention(want_cache, q.x, offsets, lengths, table, page, d ** -0.5, True, window)
        check(out.read(), want, tol)


@pytest.mark.parametrize("added", [1, 70])
def test_gpu_attention_leaves_out_missing_pages(ctx, added):
    rng = np.random.default_rng(11)
    page, d, heads, kv, n = 32, 64, 4, 1, 150
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    held = Device(cache, page)
    q = Rows(rng.standard_normal((added, heads, d)), "f32")
    for entry in (-1, pages, 1 << 30):
        tb = table.copy()
        tb[0, 1] = entry
        call, out = attend(ctx, held, q, [0, added], [n], tb, 0.125)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        want, tol = so.attention(cache, q.x, [0, added], [n], table, page, 0.125, drop=[(0, 1)])
        check(out.read(), want, tol)


def test_gpu_attention_bad_lengths_and_offsets(ctx):
    rng = np.random.default_rng(12)
    page, d, heads, kv = 16, 64, 2, 1
    lengths, offsets = [20, 30, 40], [0, 1, 2, 3]
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    held = Device(cache, page)
    q = Rows(rng.standard_normal((3, heads, d)), "f32")
    want, tol = so.attention(cache, q.x, offsets, lengths, table, page, 0.125)
    for o, n, fine in (([0, 1, 2, 3], [20, -1, 40], [0, 2]), ([0, 1, 2, 3], [20, 16 * table.shape[1] + 1, 40], [0, 2]),
                       ([0, 1, 2, 9], lengths, [0, 1]), ([0, 2, 1, 3], lengths, [])):
        call, out = attend(ctx, held, q, o, n, table, 0.125, max_length=64)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        got = out.read()
        for t in fine:
            check(got, want, tol, t)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gpu_attention_ranges(ctx, dtype):
    """Queries and scales far from one: page scales 2^40 apart, tiny and large queries, sharp softmaxes."""
    rng = np.random.default_rng(13)
    page, d, heads, kv, n = 16, 128, 4, 1, 300
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["v_scale"] = np.float32(2.0) ** rng.integers(-30, 10, cache["v_scale"].shape).astype(np.float32)
    for q_mag, scale in ((2.0 ** -12, 1.0), (2.0 ** 12, 2.0 ** -14), (1.0, 1.0)):
        held = Device(cache, page)
        q = Rows(rng.standard_normal((2, heads, d)) * q_mag, dtype)
        call, out = attend(ctx, held, q, [0, 2], [n], table, scale)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, [0, 2], [n], table, page, scale, dtype=dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("batch", ["step", "mixed", "prompt", "drafts"])
def test_gpu_attention_in_place(ctx, batch):
    rng = np.random.default_rng(19)
    added, lengths = (list(x) for x in zip(*BATCHES[batch]))
    offsets, page, d, heads, kv = np.concatenate([[0], np.cumsum(added)]), 16, 128, 8, 2
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["k_scale"] *= 0.25
    held = Device(cache, page)
    for max_length in (max(lengths), 4000):
        q = Rows(rng.standard_normal((offsets[-1], heads, d)), "f32", pad=4)
        attend(ctx, held, q, offsets, lengths, table, d ** -0.5, max_length=max_length, out=q)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, offsets, lengths, table, page, d ** -0.5)
        check(q.read(), want, tol)


def test_gpu_attention_nonfinite_query(ctx):
    rng = np.random.default_rng(14)
    page, d, heads, kv, n = 16, 64, 4, 2, 40
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    held = Device(cache, page)
    x = rng.standard_normal((20, heads, d))
    q = Rows(x, "f32")
    want, tol = so.attention(cache, q.x, [0, 20], [n], table, page, 0.125)
    x[7, 2, 5] = np.nan
    q = Rows(x, "f32")
    call, out = attend(ctx, held, q, [0, 20], [n], table, 0.125)
    assert ctx.sync() == ph.ERR_NONFINITE and ctx.sync() == 0
    got = out.read()
    keep = np.ones((20, heads), bool)
    keep[7, 2] = False
    check(got[keep], want[keep], tol[keep])
    assert np.isnan(got[7, 2]).all()


def test_gpu_attention_of_thousands_of_requests(ctx):
    """More requests than one look-up step covers, some of them without tokens or keys."""
    rng = np.random.default_rng(16)
    r, page, d, heads, kv = 5000, 16, 64, 2, 1
    added, lengths = rng.choice([0, 1, 1, 1, 2], r), rng.integers(0, 41, r)
    offsets = np.concatenate([[0], np.cumsum(added)])
    table, pages = make_table(rng, lengths, page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    held = Device(cache, page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)), "f16")
    for max_length in (40, 4000):  # unsplit and split
        call, out = attend(ctx, held, q, offsets, lengths, table, 0.125, max_length=max_length)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, offsets, lengths, table, page, 0.125, dtype="f16")
        check(out.read(), want, tol)


@pytest.mark.parametrize("window", [1, 2, 65, 10000])
@pytest.mark.parametrize("added", [1, 40])
def test_gpu_attention_windows_and_a_negative_scale(ctx, window, added):
    rng = np.random.default_rng(window)
    page, d, heads, kv, n = 32, 128, 4, 2, 400
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["k_scale"] *= 0.25
    held = Device(cache, page)
    q = Rows(rng.standard_normal((added, heads, d)), "f32")
    for scale in (d ** -0.5, -d ** -0.5, 0.0):
        call, out = attend(ctx, held, q, [0, added], [n], table, scale, True, window)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, [0, added], [n], table, page, scale, True, window)
        check(out.read(), want, tol)


@pytest.mark.parametrize("added", [1, 9, 200])
def test_gpu_cache_past_32_bits(ctx, added):
    """Keys and values of 4.4 GB each: pages on both sides of the 4 GB line, appended and attended."""
    rng = np.random.default_rng(17)
    page, d, heads, kv, pages, n = 256, 128, 8, 8, 17000, 700
    unit = kv * page * d
    assert pages * unit > 1 << 32
    used = np.array([16999, 3, 16500, 16384], np.int32)  # the last and one beyond the line's page, and low ones
    small = make_cache(rng, len(used), kv, page, d, "int8")
    small["k_scale"] *= 0.25
    buf = {"k": DeviceBuffer(pages * unit), "v": DeviceBuffer(pages * unit), "k_scale": DeviceBuffer(pages * kv * 4), "v_scale": DeviceBuffer(pages * kv * 4)}

    def move(name, i, back=False):
        size = unit if name in "kv" else kv * 4
        host = np.ascontiguousarray(small[name][i])
        at = int(used[i]) * size
        if not back:
            buf[name].upload(host, at)
            return None
        got = np.empty_like(host)
        assert hip().hipMemcpy(got.ctypes.data, buf[name].data_ptr() + at, size, 2) == 0
        return got

    for i in range(len(used)):
        for name in buf:
            move(name, i)
    desc = ph.KvCache(**buf, format=ph.CACHE_INT8, pages=pages, page_size=page, kv_heads=kv, head_dim=d)
    k, v = (rng.standard_normal((added, kv, d)).astype(np.float32) for _ in range(2))
    first = n - added
    where = np.arange(first, n)
    slots = used[where // page] * page + where % page
    ctx.kv_append_device(desc, ph.DTYPE_F32, dev(k), kv * d, dev(v), kv * d, dev(slots.astype(np.int32)), added)
    q = Rows(rng.standard_normal((added, heads, d)), "bf16")
    table = used[None]

    class Held:
        pass

    Held.desc = desc
    call, out = attend(ctx, Held, q, [0, added], [n], table, d ** -0.5)
    assert ctx.sync() == 0
    want = so.append(small, k, v, (where // page * page + where % page).astype(np.int32), page)
    for i in range(len(used)):
        for name in buf:
            assert np.array_equal(move(name, i, True), want[name][i]), (name, i)
    exact, tol = so.attention(want, q.x, [0, added], [n], np.arange(len(used))[None], page, d ** -0.5, dtype="bf16")
    check(out.read(), exact, tol)


def test_gpu_attention_graphs_share_scratch(ctx):
    """Two captured calls whose partial results share the context's scratch, replayed in turn after a
    larger eager call, with eager work between; and a second context at the same time."""
    rng = np.random.default_rng(18)
    page, d, heads, kv = 16, 128, 8, 2
    cases, graphs = [], []
    with ph.Context(0) as other:
        for n, added in ((3000, 1), (1700, 2)):
            table, pages = make_table(rng, [n], page)
            cache = make_cache(rng, pages, kv, page, d, "int8")
            cache["k_scale"] *= 0.25
            held = Device(cache, page)
            q = Rows(rng.standard_normal((added, heads, d)), "f32")
            call, out = attend(ctx, held, q, [0, added], [n], table, d ** -0.5)
            assert ctx.sync() == 0
            cases.append((call, out, held, so.attention(cache, q.x, [0, added], [n], table, page, d ** -0.5)))
            graphs.append(Graph(ctx.stream(), lambda: ctx.attention_device(held.desc, call)))
        big, pages = make_table(rng, [20000], page)
        bigger = Device(make_cache(rng, pages, kv, page, d, "int8"), page)
        attend(ctx, bigger, Rows(rng.standard_normal((3, heads, d)), "f32"), [0, 3], [20000], big, d ** -0.5)
        for _ in range(3):
            for graph, (call, out, held, _) in zip(graphs, cases):
                other.attention_device(held.desc, call)  # the same rows from another stream
                assert other.sync() == 0
                out.buf.upload(out.before)
                graph.launch()
            assert ctx.sync() == 0
            for _, out, _, (want, tol) in cases:
                check(out.read(), want, tol)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("added,longest", [(1, 300), (1, 20000), (7, 300), (40, 300)], ids=["single", "split", "draft", "chunk"])
def test_gpu_attention_pages_before_a_window_hold_anything(ctx, added, longest, page, dtype, fmt):
    """Columns before a window name pages that may hold anything: NaN and infinite scales, NaN codes. The window begins
    inside a block of 64 keys, with pages between the block's first key and its own."""
    rng = np.random.default_rng(20)
    d, heads, kv, n = 128, 8, 2, 300
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, fmt)
    cache["k_scale"] *= 0.25
    q = Rows(rng.standard_normal((added, heads, d)), dtype)
    for lo in (128 + page, 128 + page + 5, 128 + 63):
        window = n - added + 1 - lo
        want, tol = so.attention(cache, q.x, [0, added], [n], table, page, d ** -0.5, True, window, dtype)
        for bad in (np.nan, np.inf):
            held = {k: (a.copy() if isinstance(a, np.ndarray) else a) for k, a in cache.items()}
            before = table[0, : lo // page]
            held["k"][before], held["v"][before], held["k_scale"][before], held["v_scale"][before] = 0x7F, 0xFF, bad, bad
            call, out = attend(ctx, Device(held, page), q, [0, added], [n], table, d ** -0.5, True, window, max_length=longest)
            assert ctx.sync() == 0, (lo, bad)
            check(out.read(), want, tol)


@pytest.mark.parametrize("dtype,scale", [("f16", 2.0 ** 10), ("bf16", 2.677e36)])
@pytest.mark.parametrize("added,n", [(1, 40), (1, 3000), (60, 90)], ids=["rows", "split", "tile"])
def test_gpu_attention_flags_results_past_the_type(ctx, added, n, dtype, scale):
    """Results that binary32 holds and the type does not: 127 * 2^10 in binary16, 3.3998e38 in bfloat16."""
    rng = np.random.default_rng(21)
    page, d, heads, kv = 16, 64, 4, 1
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["k"][:], cache["v"][:] = 0, 127
    q = Rows(rng.standard_normal((added, heads, d)), dtype)
    for factor, rc in ((1.0, ph.ERR_NONFINITE), (0.5, 0)):
        cache["v_scale"][:] = scale * factor
        call, out = attend(ctx, Device(cache, page), q, [0, added], [n], table, 0.125)
        assert ctx.sync() == rc and ctx.sync() == 0
        got, want = out.read(), 127.0 * float(np.float32(scale * factor))
        if rc:
            assert np.isposinf(got).all()
        else:  # equal probabilities: the division and the type's half step
            assert (np.abs(got - want) <= (so.HALF[dtype] + 2.0 ** -20) * want).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("added,longest", [(2, 300), (2, 20000), (40, 300), (40, 20000)], ids=["rows", "rows-split", "tile", "tile-split"])
@pytest.mark.parametrize("big", [2.0 ** 38, 2.0 ** 110])
@pytest.mark.parametrize("order", ["zeros first", "zeros last", "mixed", "random"])
def test_gpu_attention_value_scales_far_apart(ctx, order, big, added, longest, dtype):
    """Pages of zeros, whose scale is the smallest, beside pages of large values: their keys weigh as much as any."""
    rng = np.random.default_rng(22)
    page, d, heads, kv, n = 16, 64, 4, 1, 700
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["k_scale"][:] = 2.0 ** -7
    cols = np.arange(-(-n // page))
    zero = {"zeros first": cols < 22, "zeros last": cols >= 22, "mixed": cols % 3 == 0, "random": rng.random(len(cols)) < 0.1}[order]
    used = table[0, : len(cols)]
    cache["v_scale"][used, 0] = big
    if order == "random":
        cache["v_scale"][used, 0] = np.float32(1.3) * np.float32(2.0) ** rng.integers(-95, int(np.log2(big)), len(cols)).astype(np.float32)
    cache["v"][used[zero]], cache["v_scale"][used[zero]] = 0, 2.0 ** -100
    q = Rows(rng.standard_normal((added, heads, d)), dtype)
    held = Device(cache, page)
    for causal in (True, False):
        call, out = attend(ctx, held, q, [0, added], [n], table, d ** -0.5, causal, max_length=longest)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, [0, added], [n], table, page, d ** -0.5, causal, dtype=dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("added", [1, 20])
def test_gpu_attention_a_long_cache_of_zeros(ctx, added):
    """A million keys whose values are zero, then sixteen that are not: every key weighs the same."""
    page, d, heads, kv, columns = 16, 64, 4, 1, (1 << 16) + 1
    cache = make_cache(np.random.default_rng(23), 2, kv, page, d, "int8")
    cache["k"][:], cache["v"][0], cache["v"][1] = 0, 0, 64
    cache["v_scale"][:, 0] = 2.0 ** -100, 1.0
    table = np.zeros((1, columns), np.int32)
    table[0, -1] = 1
    q = Rows(np.ones((added, heads, d)), "f32")
    n = columns * page
    call, out = attend(ctx, Device(cache, page), q, [0, added], [n], table, 0.125, False, max_length=1)  # one part
    assert ctx.sync() == 0
    # Sums of equal powers of two: an ulp of exp2 and the division are all that rounds.
    assert (np.abs(out.read() * n / 1024 - 1) <= 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("added", [2, 40])
def test_gpu_attention_of_tiny_queries(ctx, added, dtype):
    """Queries below 2^-100 under a scale that brings their scores to one."""
    rng = np.random.default_rng(24)
    page, d, heads, kv, n = 16, 128, 4, 1, 200
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    cache["k_scale"] *= 0.25
    held = Device(cache, page)
    for power in (-98, -106, -112):
        q = Rows(rng.standard_normal((added, heads, d)) * 2.0 ** power, dtype)
        scale = float(np.float32(d ** -0.5)) * 2.0 ** -power
        call, out = attend(ctx, held, q, [0, added], [n], table, scale)
        assert ctx.sync() == 0
        want, tol = so.attention(cache, q.x, [0, added], [n], table, page, scale, dtype=dtype)
        check(out.read(), want, tol)


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("added", [1, 40])
def test_gpu_attention_at_the_longest_length(ctx, added, page):
    """The last positions below 2^31, through a window: the columns before it are not even there to be read."""
    rng = np.random.default_rng(25)
    d, heads, kv, window = 64, 4, 1, 150
    columns = (2 ** 31 - 1) // page
    n, near = columns * page, 640 + 64 - page  # the same place in a block of 64 keys
    table, pages = make_table(rng, [near], page)
    cache = make_cache(rng, pages, kv, page, d, "int8")
    held = Device(cache, page)
    q = Rows(rng.standard_normal((added, heads, d)), "f32")
    want, tol = so.attention(cache, q.x, [0, added], [near], table, page, 0.125, True, window)
    big = DeviceBuffer(columns * 4)
    tail = np.ascontiguousarray(table[0, : near // page])
    big.upload(tail, (columns - len(tail)) * 4)
    out = Rows(np.full(q.shape, 3.0), "f32")
    ctx.attention_device(held.desc, ph.Attention(dtype=ph.DTYPE_F32, requests=1, tokens=added, heads=heads, max_pages=columns, max_length=n, q=q,
                                                 q_stride=q.stride, out=out, out_stride=out.stride, offsets=i32([0, added]), lengths=i32([n]),
                                                 block_table=big, scale=0.125, causal=1, window=window))
    assert ctx.sync() == 0
    check(out.read(), want, tol)


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("tokens", ["few", "many"])
def test_gpu_plan_of_many_requests_without_tokens(ctx, tokens, alias):
    """More requests than one workgroup's LDS holds, hundreds in a row without a token."""
    r, page = 6000, 16
    rng = np.random.default_rng(26)
    lengths, added, table, free, count = make_plan(rng, r, page, 40, 3)
    added[:] = 0
    added[[0, 1, 70, 199, 200, 700, 5998]] = [3, 1, 2, 1, 40, 1, 5] if tokens == "few" else [3, 700, 2, 1, 4000, 1, 500]
    added[[5, 300, 5999]] = -1
    columns = -(-int((lengths + added).max()) // page)
    table = np.concatenate([table, np.full((r, columns), -1, np.int32)], 1)
    free = np.concatenate([free[:count], np.arange(len(free), len(free) + 400, dtype=np.int32), free[count:]])
    count += 400
    room = int(np.maximum(added, 0).sum()) + 130
    case = lengths, added, table, free, count
    rc, got = run_plan(ctx, *case, page, room, alias)
    assert rc == 0
    for g, w in zip(got, so.plan(*case, page, room)):
        assert np.array_equal(g, np.asarray(w))


@pytest.mark.parametrize("dtype,fmt,d,heads,kv,added", [("f32", "e4m3", 128, 24, 8, 8), ("bf16", "e4m3", 64, 48, 16, 7), ("f16", "int8", 128, 16, 8, 12),
                                                       ("bf16", "int8", 256, 8, 4, 1), ("f32", "e4m3", 256, 8, 4, 3), ("f16", "e4m3", 256, 8, 4, 40)])
def test_gpu_attention_past_32_bits_in_every_form(ctx, dtype, fmt, d, heads, kv, added):
    """One and two row tiles and whole tiles over codes of 4.4 GB."""
    rng = np.random.default_rng(27)
    page, n = 256, 900
    unit = kv * page * d
    pages = (1 << 32) // unit + 700
    used = np.array([pages - 1, 3, pages - 500, (1 << 32) // unit], np.int32)
    small = make_cache(rng, len(used), kv, page, d, fmt)
    small["k_scale"] *= 0.25 if fmt == "int8" else 0.0625
    buf = {"k": DeviceBuffer(pages * unit), "v": DeviceBuffer(pages * unit), "k_scale": DeviceBuffer(pages * kv * 4), "v_scale": DeviceBuffer(pages * kv * 4)}
    for name, b in buf.items():
        for i, p in enumerate(used):
            b.upload(np.ascontiguousarray(small[name][i]), int(p) * (unit if name in "kv" else kv * 4))

    class Held:
        desc = ph.KvCache(**buf, format=FORMAT[fmt], pages=pages, page_size=page, kv_heads=kv, head_dim=d)

    q = Rows(rng.standard_normal((added, heads, d)), dtype)
    call, out = attend(ctx, Held, q, [0, added], [n], used[None], d ** -0.5)
    assert ctx.sync() == 0
    want, tol = so.attention(small, q.x, [0, added], [n], np.arange(len(used))[None], page, d ** -0.5, dtype=dtype)
    check(out.read(), want, tol)


@pytest.mark.parametrize("batch,longest", [("step", 500), ("step", 20000), ("drafts", 4000), ("mixed", 333), ("prompt", 20000)])
def test_gpu_attention_repeats_itself(ctx, batch, longest):
    """The same call gives the same bits, split or not."""
    rng = np.random.default_rng(28)
    added, lengths = (list(x) for x in zip(*BATCHES[batch]))
    offsets, page, d, heads, kv = np.concatenate([[0], np.cumsum(added)]), 16, 128, 8, 2
    table, pages = make_table(rng, lengths, page)
    held = Device(make_cache(rng, pages, kv, page, d, "int8"), page)
    q = Rows(rng.standard_normal((offsets[-1], heads, d)), "f16")
    first = None
    for _ in range(5):
        call, out = attend(ctx, held, q, offsets, lengths, table, d ** -0.5, max_length=longest)
        assert ctx.sync() == 0
        got = out.read()
        first = got if first is None else first
        assert np.array_equal(got, first)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("added,longest", [(1, 80), (1, 4000), (40, 80)], ids=["rows", "split", "tile"])
def test_gpu_attention_of_the_largest_and_smallest_values(ctx, added, longest, fmt):
    """Appended pages of zeros, of the smallest floats and of the largest, attended together and each kind alone."""
    rng = np.random.default_rng(29)
    page, d, heads, kv, n = 16, 64, 4, 1, 80
    table, pages = make_table(rng, [n], page)
    cache = make_cache(rng, pages, kv, page, d, fmt)
    held = Device(cache, page)
    slots = (table[0, np.arange(n) // page] * page + np.arange(n) % page).astype(np.int32)
    k = rng.standard_normal((n, kv, d)).astype(np.float32)
    for kinds in ((0.0, 3.4e38, 1.0, 1e-38, 3.4e38), (0.0,) * 5, (1e-28,) * 5, (3.4e38,) * 5, (1e-20, 0.0, 1e-20, 0.0, 0.0)):
        v = (rng.choice([-1, 1], (n, kv, d)) * rng.uniform(0.5, 1, (n, kv, d)) * np.repeat(kinds, page)[:, None, None]).astype(np.float32)
        held = Device(cache, page)
        ctx.kv_append_device(held.desc, ph.DTYPE_F32, dev(k), kv * d, dev(v), kv * d, dev(slots), n)
        want_cache = so.append(cache, k, v, slots, page)
        q = Rows(rng.standard_normal((added, heads, d)), "f32")
        call, out = attend(ctx, held, q, [0, added], [n], table, d ** -0.5, max_length=longest)
        assert ctx.sync() == 0
        held.check(want_cache)
        want, tol = so.attention(want_cache, q.x, [0, added], [n], table, page, d ** -0.5)
        check(out.read(), want, tol)


# ---- together ---------------------------------------------------------------------------------


def test_gpu_serving_steps_in_a_graph(ctx):
    """A layer of three requests over steps, from the projection of q, k and v to that of the output:
    a prompt chunk each, then single tokens, every step of them a replay of one graph."""
    rng = np.random.default_rng(15)
    hidden, heads, kv, d, page, dims, r, cols = 512, 4, 2, 128, 16, 64, 3, 5
    width = (heads + 2 * kv) * d
    wq = ctx.weight(ph.KIND_PTQ1, hidden, width, synth.weights(ph.KIND_PTQ1, width, hidden, seed=1))
    wo = ctx.weight(ph.KIND_PTQ1, heads * d, hidden, synth.weights(ph.KIND_PTQ1, hidden, heads * d, seed=2))
    rope, freq = ph.Rope(ctx, dims, ph.rope_frequencies(dims, 1e7)), ph.rope_frequencies(dims, 1e7)
    cache = make_cache(rng, 12, kv, page, d, "int8")
    held = Device(cache, page)
    chunk = [20, 7, 33]
    most = sum(chunk)
    x, qkv, att, y = (DeviceBuffer(most * n * 4) for n in (hidden, width, heads * d, hidden))
    for b in (x, qkv, att, y):
        b.zero()
    lengths, counts, table, free = i32([0, 0, 0]), i32([12, 0, 0, 0]), i32(np.full((r, cols), -1)), i32(rng.permutation(12))
    added, offsets = i32(chunk), i32(np.zeros(r + 1))
    positions, slots, owners = (i32(np.zeros(most)) for _ in range(3))
    norm = dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32))

    def enqueue(tokens):
        ctx.kv_plan_device(ph.KvPlan(requests=r, max_pages=cols, max_tokens=tokens, page_size=page, free_capacity=12, lengths=lengths, added=added,
                                     block_table=table, free_pages=free, free_count=counts, new_lengths=lengths, offsets=offsets,
                                     positions=positions, slots=slots, owners=owners, counts=counts))
        ctx.project_device(wq, ph.PATH_F32, x, tokens, False, qkv)
        at = qkv.data_ptr()
        ctx.qkv_append_device(rope, held.desc, ph.QkvAppend(dtype=ph.DTYPE_F32, tokens=tokens, heads=heads, q=at, k=at + 4 * heads * d,
                                                            v=at + 4 * (heads + kv) * d, q_stride=width, k_stride=width, v_stride=width,
                                                            positions=positions, slots=slots, q_norm=norm, k_norm=norm, eps=EPS, q_out=at,
                                                            q_out_stride=width))
        ctx.attention_device(held.desc, ph.Attention(dtype=ph.DTYPE_F32, requests=r, tokens=tokens, heads=heads, max_pages=cols, max_length=cols * page,
                                                     q=at, q_stride=width, out=att, out_stride=heads * d, offsets=offsets, lengths=lengths,
                                                     block_table=table, scale=d ** -0.5, causal=1, window=0))
        ctx.project_device(wo, ph.PATH_F32, att, tokens, False, y)

    state = [np.zeros(r, np.int64), np.full((r, cols), -1, np.int32), free.to_numpy(np.int32), 12]
    want_cache = cache
    graph = None
    for step in range(12):
        n = np.array(chunk if step == 0 else [1, 1, 1] if step < 9 else [1, -1 if step == 9 else 0, 1])
        tokens = most if step == 0 else 3
        added.upload(n.astype(np.int32))
        xs = rng.standard_normal((tokens, hidden)).astype(np.float32)
        x.upload(xs)
        synchronize()
        if step < 2:
            enqueue(tokens)
        else:
            # The plan has run uncaptured with these sizes, so the step can be captured.
            graph = graph or Graph(ctx.stream(), lambda: enqueue(3))
            graph.launch()
        assert ctx.sync() == 0, ctx.last_error
        p = so.plan(state[0], n, state[1], state[2], state[3], page, tokens)
        state = [p[0], p[6], p[7], p[5][0]]
        assert np.array_equal(table.to_numpy(np.int32).reshape(r, cols), p[6]) and np.array_equal(lengths.to_numpy(np.int32), p[0])
        live = p[5][1]
        rows = ctx.project_f32(wq, width, xs, tokens=tokens).reshape(tokens, heads + 2 * kv, d)
        nh = norm.to_numpy(np.float32)
        q = so.rounded(so.rope(rows[:, :heads], p[2], freq, dims, False, 1.0, nh, EPS), "f32")
        k = so.rounded(so.rope(rows[:, heads:heads + kv], p[2], freq, dims, False, 1.0, nh, EPS), "f32")
        want_cache = so.append(want_cache, k, rows[:, heads + kv:], p[3], page)
        held.check(want_cache)
        want, tol = so.attention(want_cache, q, p[1], p[0], p[6], page, d ** -0.5)
        # q itself is off by half a step of binary32 from the device's.
        got = att.to_numpy(np.float32)[: tokens * heads * d].reshape(tokens, heads, d)
        check(got, want, tol + 1e-6 * np.abs(want).max(), slice(0, live))
        out = y.to_numpy(np.float32)[: tokens * hidden].reshape(tokens, hidden)
        assert np.array_equal(out[:live], ctx.project_f32(wo, hidden, got, tokens=tokens).reshape(tokens, hidden)[:live])
    rope.close()
    ctx.release(wq)
    ctx.release(wo)
