"""Log probabilities of given tokens, entropy and alternatives on the GPU against the 64-bit restatement of cache4_oracle.py:
the alternatives' ids exactly, values within the roundings that the restatement counts.
"""

import numpy as np
import pytest

import cache4_oracle as co
import prism_hip as ph
import serving_oracle as so
from hiprt import Graph
from test_gpu_serving import DTYPE, NP, check, dev, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ph.Context(0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def _announce(request):
    print(request.node.name, flush=True)


class Call:
    """Logits [tokens][vocab] in wider, offset memory, and guarded outputs."""

    def __init__(self, x, targets, top, dtype="f32", pad=0, shift=0, entropy=True):
        self.top, (t, n) = top, x.shape
        stride = n + pad
        flat = np.zeros(shift + t * stride, NP[dtype])
        flat.view(np.uint8)[:] = 0x7F  # NaN or a large value beside the rows
        where = shift + np.arange(t)[:, None] * stride + np.arange(n)[None]
        flat[where] = so.to_device(x, dtype)
        self.x = so.from_device(flat[where], dtype)
        self.buf = dev(flat)
        self.out = {m: dev(np.full(k + 3, 7.0, np.float32)) for m, k in (("logprobs", t), ("entropy", t), ("top_logprobs", t * top))}
        self.out["top_ids"] = i32(np.full(t * top + 3, 7))
        self.targets = None if targets is None else np.asarray(targets)
        self.tb = None if targets is None else i32(targets)
        self.shape, self.asked = {"logprobs": (t,), "entropy": (t,), "top_logprobs": (t, top), "top_ids": (t, top)}, \
            [m for m, on in (("logprobs", targets is not None), ("entropy", entropy), ("top_ids", top), ("top_logprobs", top)) if on]
        self.call = ph.Logprobs(dtype=DTYPE[dtype], tokens=t, vocab=n, top=top, logits=self.buf.ptr + shift * flat.itemsize, stride=stride, targets=self.tb,
                                **{m: b if m in self.asked else None for m, b in self.out.items()})

    def get(self, m):
        a = self.out[m].to_numpy(np.int32 if m == "top_ids" else np.float32)
        n = int(np.prod(self.shape[m])) if m in self.asked else 0
        assert (a[n:] == 7).all(), "wrote behind " + m
        return a[:n].reshape(self.shape[m]) if n else None

    def check(self, rows=slice(None)):
        want = co.logprobs(self.x, np.full(len(self.x), -1) if self.targets is None else self.targets, self.top)
        for m in self.out:
            got = self.get(m)
            if got is None:
                continue
            w, tol = want[m]
            if m == "top_ids":
                assert np.array_equal(got[rows], w[rows]), np.argwhere(got != w)[:5]
                continue
            none = np.isneginf(w)
            assert np.array_equal(np.isneginf(got[rows]), none[rows]), m
            check(np.where(none, 0, got), np.where(none, 0, w), tol, rows)


def logits(rng, tokens, vocab, masked=0.0):
    x = rng.standard_normal((tokens, vocab)) * 2.5
    x[np.arange(tokens), rng.integers(0, vocab, tokens)] += 12
    return np.where(rng.random((tokens, vocab)) < masked, -np.inf, x)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 63, 5), (5, 64, 64), (4, 65, 20), (7, 255, 1), (2, 1000, 64), (9, 4096, 20), (1, 4097, 5),
                                              (3, 32000, 20), (130, 5003, 5), (1, 151936, 20), (2, 151936, 64), (1, 262144, 5)])
def test_gpu_logprobs(ctx, dtype, tokens, vocab, top):
    rng = np.random.default_rng(vocab + top)
    for masked, pad, shift in ((0.0, 0, 0), (0.3, 5, 1), (0.98, 8, 3)):
        c = Call(logits(rng, tokens, vocab, masked), rng.integers(-1, vocab, tokens), top, dtype, pad, shift)
        ctx.logprobs_device(c.call)
        assert ctx.sync() == 0
        c.check()


@pytest.mark.parametrize("tokens,vocab", [(5000, 300), (600, 9001), (40, 151936)])
def test_gpu_logprobs_of_many_tokens(ctx, tokens, vocab):
    rng = np.random.default_rng(tokens)
    c = Call(logits(rng, tokens, vocab, 0.1), rng.integers(0, vocab, tokens), 7, "bf16", 3)
    ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [200, 5000, 70001])
def test_gpu_logprobs_orders_and_ties(ctx, dtype, vocab):
    """Rows that hold their largest words in the worst places: ascending, descending, all equal, few different values, zeros of
    both signs, one word, one word far above all others, the largest last."""
    rng = np.random.default_rng(vocab)
    i = np.arange(vocab)
    rows = [i / vocab * 20, -i / vocab * 20, np.zeros(vocab), rng.integers(0, 3, vocab), np.where(i % 2, -0.0, 0.0), np.where(i == vocab // 2, 1.0, -np.inf),
            np.where(i == 3, 100.0, rng.standard_normal(vocab)), np.where(i >= vocab - 30, 9.0, -9.0), np.where(i % 64 == 5, 3.0, 0.0),
            np.where(i % 256 < 4, i, -i) / vocab, np.full(vocab, -1e4), np.where(i < 10, -6e4, 6e4)]
    x = np.array(rows, np.float64)
    for top in (1, 20, 64):
        c = Call(x, rng.integers(0, vocab, len(x)), top, dtype)
        ctx.logprobs_device(c.call)
        assert ctx.sync() == 0
        c.check()


def test_gpu_logprobs_keeps_the_digits_of_sure_rows(ctx):
    """Entropies and losses far below one step of 1."""
    vocab = 1000
    x = np.zeros((6, vocab))
    for r, gap in enumerate((5.0, 20.0, 40.0, 60.0, 80.0, 500.0)):
        x[r, 17] = gap
    c = Call(x, [17] * 6, 1)
    ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    c.check()
    assert -1e-20 < c.get("logprobs")[3] < 0 and 0 < c.get("entropy")[4] < 1e-28


@pytest.mark.parametrize("vocab", [70, 40000])
def test_gpu_logprobs_rows_without_words(ctx, vocab):
    rng = np.random.default_rng(1)
    x = logits(rng, 4, vocab)
    x[1], x[3] = -np.inf, -np.inf
    c = Call(x, [0, 5, -1, -1], 3)
    ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    c.check()
    assert c.get("logprobs").tolist()[1::2] == [-np.inf, 0.0] and c.get("entropy")[1] == 0 and (c.get("top_ids")[1] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [70, 40000])
def test_gpu_logprobs_flags(ctx, dtype, vocab):
    """NaN, +infinity and targets out of range: flagged, their rows NaN, the others as ever."""
    rng = np.random.default_rng(2)
    for bad in (np.nan, np.inf):
        x = logits(rng, 3, vocab, 0.2)
        x[1, vocab - 3] = bad
        c = Call(x, [1, 2, 3], 4, dtype)
        ctx.logprobs_device(c.call)
        assert ctx.sync() == ph.ERR_NONFINITE and ctx.sync() == 0
        assert all(np.isnan(c.get(m)[1]).all() for m in ("logprobs", "entropy", "top_logprobs")) and (c.get("top_ids")[1] == -1).all()
        c.x[1, vocab - 3] = 0
        c.check([0, 2])
    for bad in (-2, vocab, -(1 << 31), (1 << 31) - 1):
        c = Call(logits(rng, 3, vocab), [1, bad, 3], 4, dtype)
        ctx.logprobs_device(c.call)
        assert ctx.sync() == ph.ERR_INVALID_INPUT and ctx.sync() == 0
        assert np.isnan(c.get("logprobs")[1])
        c.targets[1] = 0
        c.check([0, 2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [4, 260])
def test_gpu_logprobs_few_words_of_many(ctx, dtype, tokens):
    """Rows of a long vocabulary, whole and in parts, where fewer words than asked for are not masked by a large negative logit,
    and rows of one value."""
    rng = np.random.default_rng(6)
    vocab = 70001
    x = np.empty((tokens, vocab))
    for t in range(tokens):
        x[t] = (-1e9, 0.0, -3e38, -65504.0)[t % 4]
        some = rng.choice(vocab, 3 + t % 30, replace=False)
        x[t, some] = rng.standard_normal(len(some))
    for top in (5, 64):
        c = Call(x, rng.integers(0, vocab, tokens), top, dtype)
        ctx.logprobs_device(c.call)
        assert ctx.sync() == 0
        c.check()


@pytest.mark.parametrize("tokens,vocab", [(260, 70001), (300, 131072), (1, (1 << 20) + 5), (2, (1 << 24) - 3), (1, 1 << 24)])
def test_gpu_logprobs_of_long_rows(ctx, tokens, vocab):
    """Groups of several tiles."""
    rng = np.random.default_rng(vocab)
    c = Call(logits(rng, tokens, vocab, 0.1), rng.integers(0, vocab, tokens), 20, "f16", 1, 1)
    ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    c.check()


def test_gpu_logprobs_of_many_long_rows(ctx):
    """More than 256 rows past 2^20 words: parts of the largest groups.  Every row is the same."""
    from hiprt import DeviceBuffer
    rng = np.random.default_rng(7)
    tokens, vocab, top = 257, (1 << 20) + 70, 9
    row = so.to_device(logits(rng, 1, vocab, 0.1), "f16")
    big = DeviceBuffer(2 * tokens * vocab)
    for t in range(tokens):
        big.upload(row, 2 * t * vocab)
    c = Call(so.from_device(row, "f16"), [vocab - 5], top, "f16")
    out = {m: dev(np.zeros(tokens * k, np.float32)) for m, k in (("logprobs", 1), ("entropy", 1), ("top_logprobs", top))}
    ids = i32(np.zeros(tokens * top))
    ctx.logprobs_device(ph.Logprobs(dtype=DTYPE["f16"], tokens=tokens, vocab=vocab, top=top, logits=big, stride=vocab, targets=i32([vocab - 5] * tokens),
                                    top_ids=ids, **out))
    assert ctx.sync() == 0
    want = co.logprobs(c.x, [vocab - 5], top)
    assert (ids.to_numpy(np.int32).reshape(tokens, top) == want["top_ids"][0]).all()
    for m, b in out.items():
        w, tol = want[m]
        got = b.to_numpy(np.float32).reshape(tokens, -1)
        check(got, np.broadcast_to(w.reshape(1, -1), got.shape), np.broadcast_to(np.reshape(tol, (1, -1)), got.shape))


@pytest.mark.parametrize("vocab", [90, 40000])
def test_gpu_logprobs_of_the_whole_range(ctx, vocab):
    """Logits whose differences pass binary32's range."""
    i = np.arange(vocab)
    x = np.array([np.where(i % 7 == 0, 3e38, -3e38), np.where(i == vocab - 1, 3e38, -3e38), np.where(i == 0, 3.4e38, -3.4e38)])
    c = Call(x, [0, vocab - 1, 0], 5)
    ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    want = co.logprobs(c.x, [0, vocab - 1, 0], 1)
    for m in ("logprobs", "entropy"):
        check(c.get(m), *want[m])
    best = c.get("top_logprobs")
    check(best[:, :1], *want["top_logprobs"])
    assert np.isneginf(best[1:, 1:]).all() and c.get("top_ids").tolist()[1:] == [[vocab - 1, 0, 1, 2, 3], [0, 1, 2, 3, 4]]


def test_gpu_logprobs_of_what_is_asked(ctx):
    rng = np.random.default_rng(3)
    for vocab in (90, 50000):
        for targets, top, entropy in (([3, 4], 0, False), (None, 0, True), (None, 6, False), ([0, 1], 0, True), ([0, 1], 2, False)):
            c = Call(logits(rng, 2, vocab), targets, top, entropy=entropy)
            ctx.logprobs_device(c.call)
            assert ctx.sync() == 0
            c.check()


def test_gpu_logprobs_past_32_bits(ctx):
    """Rows that stand past 2^32 elements."""
    rng = np.random.default_rng(4)
    vocab, stride = 3001, (1 << 31) + 7
    from hiprt import DeviceBuffer
    x = so.to_device(logits(rng, 4, vocab), "f16")
    big = DeviceBuffer(2 * (3 * stride + vocab))
    for r in range(4):
        big.upload(x[r], 2 * r * stride)
    c = Call(so.from_device(x, "f16"), rng.integers(0, vocab, 4), 5, "f16")
    c.call.logits, c.call.stride = big.ptr, stride
    ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    c.check()


def test_gpu_logprobs_graphs_share_scratch(ctx):
    rng = np.random.default_rng(5)
    calls = [Call(logits(rng, t, n), rng.integers(0, n, t), top) for t, n, top in ((1, 151936, 20), (3, 60000, 64))]
    for c in calls:
        ctx.logprobs_device(c.call)
    assert ctx.sync() == 0
    graphs = [Graph(ctx.stream(), lambda c=c: ctx.logprobs_device(c.call)) for c in calls]
    other = Call(logits(rng, 2, 262144), [1, 2], 64)
    for i in (0, 1, 1, 0, 1):
        for b in calls[i].out.values():
            b.upload(np.full(b.nbytes // 4, 7, np.int32) if b is calls[i].out["top_ids"] else np.full(b.nbytes // 4, 7.0, np.float32))
        graphs[i].launch()
        ctx.logprobs_device(other.call)
        assert ctx.sync() == 0
        calls[i].check()
        other.check()
