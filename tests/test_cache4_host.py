"""The 4-bit cache's, the read's and the log probabilities' entry points on the CPU: what they refuse before any launch."""

import numpy as np

import cache4_oracle as co
from test_serving_host import stub  # noqa: F401

MORE = """
def cache4(**kw): return ph.KvCache(**{**CACHE, "format": ph.CACHE_E2M1, **kw})
def append4(**kw): ctx.kv_append_device(cache4(**kw), ph.DTYPE_F32, At(X), 256, At(Y), 256, At(Z), 3)
def attend4(**kw): ctx.attention_device(cache4(**kw), ph.Attention(**ATT))
def read(dtype=ph.DTYPE_F32, slots=Z, tokens=3, k=X, k_stride=256, v=Y, v_stride=256, **kw):
    ctx.kv_read_device(cache4(**kw), dtype, At(slots), tokens, At(k), k_stride, At(v), v_stride)
LP = dict(dtype=ph.DTYPE_F32, tokens=3, vocab=1000, top=5, logits=X, stride=1000, targets=Y, logprobs=Z, entropy=Z, top_ids=Z, top_logprobs=Z)
def score(**kw): ctx.logprobs_device(ph.Logprobs(**{**LP, **kw}))
"""


def dedent(code):
    import textwrap
    return MORE + textwrap.dedent(code)


def test_cache_refusals(stub):  # noqa: F811
    stub(dedent("""
        for call in (append4, attend4, read):
            assert runs(call) >= 1
            for bad in (dict(k=None) if call is not read else dict(k_scale=None), dict(k_scale=None), dict(v_scale=None), dict(format=3), dict(format=5),
                        dict(pages=0), dict(pages=1 << 27), dict(kv_heads=0), dict(k_scale=Z + 4), dict(v_scale=Z + 8)):
                refused(call, **bad)
            refused(call, ph.ERR_UNSUPPORTED, head_dim=96)
            refused(call, ph.ERR_UNSUPPORTED, page_size=8)
        """))


def test_read_refusals(stub):  # noqa: F811
    stub(dedent("""
        for fmt in (ph.CACHE_E2M1, ph.CACHE_INT8, ph.CACHE_E4M3):
            assert runs(read, format=fmt) >= 1 and runs(read, format=fmt, k=None) >= 1 and runs(read, format=fmt, v=None, v_stride=0) >= 1
            assert runs(read, format=fmt, tokens=0) == 0
        for bad in (dict(k=None, v=None), dict(slots=None), dict(dtype=3), dict(dtype=-1), dict(k=X + 2), dict(v=Y + 1), dict(k_stride=255), dict(v_stride=0),
                    dict(tokens=(1 << 23) + 1)):
            refused(read, **bad)
        assert runs(read, dtype=ph.DTYPE_F16, k=X + 2, k_stride=257) >= 1
        assert ph.lib().prism_hip_kv_read_device(ctx.handle, None, 0, None, 1, None, 0, None, 0, None) == ph.ERR_INVALID_INPUT
        """))


def test_logprobs_refusals(stub):  # noqa: F811
    stub(dedent("""
        assert runs(score) >= 1 and runs(score, tokens=0) == 0
        assert runs(score, targets=None, logprobs=None) >= 1 and runs(score, entropy=None) >= 1 and runs(score, top=0, top_ids=None, top_logprobs=None) >= 1
        for bad in (dict(dtype=3), dict(tokens=(1 << 23) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1, stride=1 << 25), dict(top=65), dict(targets=None),
                    dict(logprobs=None), dict(top=0), dict(top_ids=None), dict(top_logprobs=None), dict(logits=None), dict(logits=X + 2), dict(stride=999),
                    dict(targets=Y + 2), dict(entropy=Z + 1), dict(top_ids=Z + 2), dict(stride=1 << 41),
                    dict(targets=None, logprobs=None, entropy=None, top=0, top_ids=None, top_logprobs=None)):
            refused(score, **bad)
        assert runs(score, dtype=ph.DTYPE_BF16, logits=X + 2, stride=1001) >= 1
        assert ph.lib().prism_hip_logprobs_device(ctx.handle, None, None) == ph.ERR_INVALID_INPUT
        """))


def test_streams_faults_and_cancellation(stub):  # noqa: F811
    stub(dedent("""
        calls = [append4, attend4, read, score]
        flag = np.ones(1, np.int32)
        ctx.set_cancellation(flag)
        for call in calls:
            refused(call, ph.ERR_CANCELLED)
        ctx.set_cancellation(None)
        other = ctypes.c_void_p(0x5000)
        for f in (lambda: ctx.kv_read_device(cache4(), ph.DTYPE_F32, At(Z), 3, At(X), 256, At(Y), 256, other),
                  lambda: ctx.logprobs_device(ph.Logprobs(**LP), other)):
            refused(f)
        ctx.inject_fault()
        for call in calls:
            refused(call, ph.ERR_DEVICE_FAULT)
        """))


def test_a_call_made_once_uncaptured_can_be_captured(stub):  # noqa: F811
    stub(dedent("""
        long = lambda **k: ctx.attention_device(cache4(), ph.Attention(**{**ATT, "max_length": 60000, "max_pages": 4000, **k}))
        for call in (long, lambda **k: score(**{**dict(tokens=1, vocab=151936, stride=151936, top=64), **k})):
            call()
            S.stub_capture(1)
            call()
            S.stub_capture(0)
        S.stub_log()
        long(tokens=64, requests=2), score(tokens=2, vocab=1 << 20, stride=1 << 20, top=64)
        assert not [l for l in S.stub_log().decode().splitlines() if l.startswith("free")]
        """))


def test_log_probabilities_are_split_by_the_devices_size(stub):  # noqa: F811
    """Rows are split over workgroups up to a row a CU, until there are four workgroups a CU."""
    stub(dedent("""
        def grids(tokens, vocab=151936):
            S.stub_log()
            score(tokens=tokens, vocab=vocab, stride=vocab)
            return [int(l.split(" grid ")[1].split()[0]) for l in S.stub_log().decode().splitlines() if l.startswith("launch")]
        for cus in (256, 64, 32):
            S.stub_cus(cus)
            ctx = ph.Context(0)
            for tokens in (1, 5, cus // 4, cus // 2, cus - 1, cus, cus + 1, 3 * cus):
                got = grids(tokens)
                if tokens > cus:
                    assert got == [tokens], (cus, tokens, got)
                    continue
                # 38 tiles of four wavefronts, a part with a tile or more.
                parts = min(-(-4 * cus // tokens), 38)
                assert got == [tokens * -(-38 // -(-38 // parts)), tokens], (cus, tokens, got)
            assert grids(5, 4096) == [5]
        """))


def test_oracle_codes_are_the_nearest():
    """Each code's own value, the borders between neighbours and points on both sides of them."""
    levels = co.LEVELS[:8]
    assert np.array_equal(co.codes(levels), np.arange(8)) and np.array_equal(co.codes(-levels[1:]), np.arange(9, 16))
    for i in range(7):
        mid = (levels[i] + levels[i + 1]) / 2
        assert co.codes(np.array([mid]))[0] == (i if i % 2 == 0 else i + 1)
        assert co.codes(np.array([mid * (1 - 1e-9)]))[0] == i and co.codes(np.array([mid * (1 + 1e-9)]))[0] == i + 1
    x = np.concatenate([np.linspace(-9, 9, 4096), [np.nan, 0.0, -0.0]]).reshape(1, -1)
    c = co.codes(x)
    assert c[0, -3:].tolist() == [0, 0, 8]
    b, e = co.quantized(np.full((1, 64), 49153.0))
    assert (e == 140).all() and (b == 0x77).all()
    b, e = co.quantized(np.concatenate([np.full(32, 6.0), np.full(32, 6.0001)])[None])
    assert e.tolist() == [[127, 128]]


def test_oracle_scales_follow_the_finite_values():
    """An infinity takes the largest code at the exponent that the finite values ask for; a NaN is 0."""
    x = np.zeros((5, 32))
    x[0, 3], x[1, 3], x[2, 3], x[3, :] = np.inf, -np.inf, np.nan, np.inf
    x[4, 3], x[4, 9] = np.inf, 5.0
    b, e = co.quantized(x)
    values = co.values({"k": b[None, None], "k_scale": e.T[None, None], "format": "e2m1"}, "k")[0, 0]
    least = 6 * 2.0 ** -23
    assert e[:, 0].tolist() == [104, 104, 104, 104, 127]
    assert values[0, 3] == least and values[1, 3] == -least and values[2, 3] == 0 and (values[3] == least).all()
    assert values[4, 3] == 6 and values[4, 9] == 4  # 5 stands between 4 and 6, and 4 has the even code
