"""The serving entry points on the CPU: what they refuse before any launch, and the scratch of
captured calls, over the HIP runtime without a device; rotary frequencies against their formulas.
"""

import math
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import prism_hip as ph

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(os.path.dirname(HERE), "prism-inference_amd", "libprism_hip.so")

PRELUDE = """
import ctypes, sys
import numpy as np
S = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
S.stub_log.restype = ctypes.c_char_p
sys.path.insert(0, sys.argv[2])
import prism_hip as ph
X, Y, Z = 0x10000000, 0x20000000, 0x30000000  # device arrays of the caller; nothing reads them
ctx = ph.Context(0)
def log():
    return [l for l in S.stub_log().decode().splitlines() if l.startswith(("launch", "malloc"))]
CACHE = dict(k=X, v=Y, k_scale=Z, v_scale=Z + 4096, format=ph.CACHE_INT8, pages=100, page_size=16, kv_heads=2, head_dim=128)
PLAN = dict(requests=3, max_pages=4, max_tokens=9, page_size=16, free_capacity=12, lengths=X, added=X, block_table=X, free_pages=X,
            free_count=X, new_lengths=X, offsets=X, positions=X, slots=X, owners=X, counts=X)
QKV = dict(dtype=ph.DTYPE_F16, tokens=5, heads=6, q=X, k=X + 1536, v=X + 2048, q_stride=1280, k_stride=1280, v_stride=1280, positions=Z, slots=Z,
           q_norm=None, k_norm=None, eps=0.0, q_out=X, q_out_stride=1280)
ATT = dict(dtype=ph.DTYPE_F32, requests=3, tokens=5, heads=6, max_pages=4, max_length=64, q=X, q_stride=768, out=Y, out_stride=768, offsets=Z,
           lengths=Z, block_table=Z, scale=0.1, causal=1, window=0)
ROPE = ph.Rope(ctx, 64, ph.rope_frequencies(64, 1e4))
def plan(**kw): ctx.kv_plan_device(ph.KvPlan(**{**PLAN, **kw}))
def append(dtype=ph.DTYPE_F32, k=X, k_stride=256, v=Y, v_stride=256, slots=Z, tokens=3, **kw):
    ctx.kv_append_device(ph.KvCache(**{**CACHE, **kw}), dtype, At(k), k_stride, At(v), v_stride, At(slots), tokens)
def qkv(rope=ROPE, cache={}, **kw): ctx.qkv_append_device(rope, ph.KvCache(**{**CACHE, **cache}), ph.QkvAppend(**{**QKV, **kw}))
def attend(cache={}, **kw): ctx.attention_device(ph.KvCache(**{**CACHE, **cache}), ph.Attention(**{**ATT, **kw}))
def rope(rope=ROPE, dtype=ph.DTYPE_F32, x=X, x_stride=512, positions=Z, tokens=3, heads=4, head_dim=128, out=Y, out_stride=512, norm=None, eps=0.0):
    ctx.rope_device(rope, dtype, At(x), x_stride, At(positions), tokens, heads, head_dim, At(out), out_stride, norm, eps)
class At:
    def __init__(self, p): self.p = p
    def data_ptr(self): return self.p or 0
def refused(call, code=ph.ERR_INVALID_INPUT, **kw):
    log()
    try:
        call(**kw)
    except ph.PrismError as e:
        assert e.code == code and ctx.last_error, (call, kw, e)
    else:
        raise AssertionError((call, kw))
    assert not log(), kw
def runs(call, **kw):
    log()
    call(**kw)
    got = log()
    return sum(l.startswith("launch") for l in got)
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "hip_stub.cpp"), "-o", so], check=True)

    def run(code):
        p = subprocess.run([sys.executable, "-c", PRELUDE + textwrap.dedent(code), so, os.path.dirname(LIB)], capture_output=True, text=True,
                           timeout=300)
        assert p.returncode == 0, p.stdout + p.stderr
        return p.stdout

    return run


def test_plan_refusals(stub):
    stub("""
        assert runs(plan) == 1 and runs(plan, max_tokens=100000) == 2
        for name in ("lengths", "added", "block_table", "free_pages", "free_count", "new_lengths", "offsets", "positions", "slots", "owners", "counts"):
            refused(plan, **{name: None})
        for bad in (dict(requests=0), dict(requests=(1 << 23) + 1), dict(max_tokens=0), dict(max_tokens=(1 << 23) + 1), dict(max_pages=0),
                    dict(max_pages=1 << 28), dict(free_capacity=1 << 31)):
            refused(plan, **bad)
        for size in (0, 8, 24, 512):
            refused(plan, ph.ERR_UNSUPPORTED, page_size=size)
        """)


def test_cache_and_row_refusals(stub):
    stub("""
        for call in (lambda **k: append(**k), lambda **k: qkv(cache=k), lambda **k: attend(cache=k)):
            assert runs(call) >= 1
            for bad in (dict(k_scale=None), dict(v_scale=None), dict(format=2), dict(pages=0), dict(pages=1 << 27), dict(kv_heads=0)):
                refused(call, **bad)
            refused(call, ph.ERR_UNSUPPORTED, head_dim=96)
            refused(call, ph.ERR_UNSUPPORTED, page_size=8)
        for name in ("k", "v"):
            refused(qkv, cache={name: None}), refused(qkv, cache={name: X + 8}), refused(attend, cache={name: None})
            refused(append, **{name: None}), refused(append, **{name: X + 2}), refused(append, **{name + "_stride": 255})
        refused(append, dtype=3), refused(append, slots=None), refused(append, tokens=(1 << 23) + 1)
        assert runs(append, tokens=0) == 0
        assert runs(append, dtype=ph.DTYPE_BF16, k=X + 2, k_stride=257) == 1
        """)


def test_rotation_refusals(stub):
    stub("""
        assert runs(rope) == 1 and runs(rope, tokens=0) == 0
        other = ph.Context(0)
        foreign = ph.Rope(other, 64, ph.rope_frequencies(64, 1e4))
        wide = ph.Rope(ctx, 256, ph.rope_frequencies(256, 1e4))
        for bad in (dict(rope=foreign), dict(rope=wide), dict(dtype=-1), dict(x=None), dict(out=None), dict(positions=None), dict(x=X + 2),
                    dict(x_stride=511), dict(out_stride=511), dict(heads=0), dict(heads=5000), dict(eps=-1.0), dict(eps=float("nan")),
                    dict(out=X, out_stride=520), dict(tokens=1 << 23, heads=16)):
            refused(rope, **bad)
        refused(rope, ph.ERR_UNSUPPORTED, head_dim=32, x_stride=1 << 20)
        for bad in (dict(rope=foreign), dict(q=None), dict(q_out=None), dict(positions=None), dict(slots=None), dict(q_stride=767),
                    dict(k_stride=255), dict(q_out_stride=1290), dict(heads=0), dict(eps=float("inf")), dict(dtype=7)):
            refused(qkv, **bad)
        assert ph.lib().prism_hip_qkv_append_device(ctx.handle, ROPE.handle, None, None, None) == ph.ERR_INVALID_INPUT
        assert runs(qkv, tokens=0) == 0
        for bad in (dict(dims=0), dict(dims=3), dict(dims=258), dict(f=float("nan")), dict(f=1e7), dict(magnitude=float("inf"))):
            dims = bad.get("dims", 64)
            f = (ctypes.c_double * 200)(*[bad.get("f", 1.0)] * 200)
            assert not ph.lib().prism_hip_rope_create(ctx.handle, dims, 0, f, bad.get("magnitude", 1.0)) and ctx.last_error
        assert not ph.lib().prism_hip_rope_create(ctx.handle, 64, 0, None, 1.0)
        """)


def test_attention_refusals(stub):
    stub("""
        assert runs(attend) >= 1 and runs(attend, tokens=0) == 0 and runs(attend, requests=0) == 0
        for name in ("q", "out", "offsets", "lengths", "block_table"):
            refused(attend, **{name: None})
        for bad in (dict(dtype=9), dict(heads=0), dict(heads=5), dict(scale=float("nan")), dict(window=5, causal=0), dict(window=1 << 31),
                    dict(max_length=1 << 31), dict(max_pages=0), dict(max_pages=1 << 28), dict(requests=(1 << 22) + 1), dict(q=X + 2),
                    dict(q_stride=767), dict(out_stride=767), dict(out=X, out_stride=770), dict(tokens=1 << 24), dict(tokens=1 << 23, heads=16)):
            refused(attend, **bad)
        assert ph.lib().prism_hip_attention_device(ctx.handle, None, None, None) == ph.ERR_INVALID_INPUT
        """)


def test_streams_faults_and_cancellation(stub):
    stub("""
        calls = [plan, append, qkv, attend, rope]
        flag = np.ones(1, np.int32)
        ctx.set_cancellation(flag)
        for call in calls:
            refused(call, ph.ERR_CANCELLED)
        ctx.set_cancellation(None)
        other = ctypes.c_void_p(0x5000)
        for f in (lambda: ctx.kv_plan_device(ph.KvPlan(**PLAN), other), lambda: ctx.attention_device(ph.KvCache(**CACHE), ph.Attention(**ATT), other),
                  lambda: ctx.qkv_append_device(ROPE, ph.KvCache(**CACHE), ph.QkvAppend(**QKV), other)):
            refused(f)
        ctx.inject_fault()
        for call in calls:
            refused(call, ph.ERR_DEVICE_FAULT)
        assert not ph.lib().prism_hip_rope_create(ctx.handle, 64, 0, (ctypes.c_double * 32)(), 1.0)
        """)


def test_a_call_made_once_uncaptured_can_be_captured(stub):
    """Scratch never grows under capture, and what a captured call used outlives larger calls."""
    stub("""
        calls = [plan, qkv, lambda **k: attend(**{**dict(max_length=60000, max_pages=4000), **k})]
        for call in calls:
            S.stub_capture(1)
            refused(call, ph.ERR_UNSUPPORTED)
            S.stub_capture(0)
            call()
            S.stub_capture(1)
            call()
            S.stub_capture(0)
        S.stub_log()
        plan(requests=100000), qkv(tokens=4000), attend(max_length=60000, max_pages=4000, tokens=64, requests=2)
        assert not [l for l in S.stub_log().decode().splitlines() if l.startswith("free")]
        ctx.close()
        """)


def test_frequencies():
    f = ph.rope_frequencies(64, 1e7)
    assert np.allclose(f, 1e7 ** (-np.arange(0, 64, 2) / 64), rtol=1e-14)
    assert np.allclose(ph.rope_frequencies(64, 1e7, 8.0), f / 8, rtol=1e-14)
    got = ph.rope_frequencies(64, 1e7, 8.0, 4096.0, 1.0, 32.0)
    turns = 4096 * f / (2 * math.pi)
    assert np.allclose(got[turns >= 32], f[turns >= 32], rtol=1e-14) and np.allclose(got[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((got[mid] > f[mid] / 8) & (got[mid] < f[mid])).all()
    assert np.allclose(got[mid], f[mid] / 8 + (turns[mid] - 1) / 31 * (f[mid] - f[mid] / 8), rtol=1e-13)
    for bad in ((0, 1e4), (3, 1e4), (258, 1e4), (64, 0.0), (64, math.inf), (64, 1e4, 0.5), (64, 1e4, 2.0, -1.0), (64, 1e4, 2.0, 100.0, 5.0, 5.0)):
        with pytest.raises(ph.PrismError):
            ph.rope_frequencies(*bad)
