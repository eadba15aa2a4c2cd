"""Operators of the 4-bit paged cache and of the answers' log probabilities: what is measured, and their plain forms.

  append    q, k and v of a step: per-head RMSNorm, rotary positions, and k and v into 4-bit pages (prism_hip_qkv_append_device;
            without q and positions prism_hip_kv_append_device).
  read      keys and values of given slots back from a cache of any format (prism_hip_kv_read_device).
  attend    grouped-query attention over the 4-bit cache (prism_hip_attention_device).
  logprobs  log probabilities of given tokens, entropy and the most probable alternatives, from logits (prism_hip_logprobs_device).

The 4-bit format is e2m1: a code is a sign and a magnitude of 0, 0.5, 1, 1.5, 2, 3, 4 or 6, and each 32 consecutive dimensions of a token
and kv head share a scale 2^(byte - 127).  A page holds, for each kv head, k[page_size][head_dim / 2] and v[page_size][head_dim / 2] bytes (the
first of two dimensions in the low half) and the scales' bytes [head_dim / 32][page_size].  The cache is returned as it is held: equal codes
and scales are equal values.
"""

import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
GROUP = 32
LEAST, MOST = -23, 13  # exponents of a group's scale
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # A decode step of 32 requests: q and k normed and rotated, k and v into the pages in use.  Latency.
        {"name": "append-step", "op": "append", "dtype": "f32", "heads": 32, "kv_heads": 8, "head_dim": 128, "dims": 64,
         "interleaved": False, "page": 16, "requests": 32, "lo": 1, "hi": 2048, "new": 1, "norm": True, "scaled": False},
        # A long prompt at once.
        {"name": "append-prompt", "op": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "dims": 128,
         "interleaved": False, "page": 64, "requests": 1, "lo": 0, "hi": 0, "new": 8192, "norm": True, "scaled": True},
        # Chunks of 48 requests that begin and end inside pages; k and v alone, rotated elsewhere.
        {"name": "append-ragged", "op": "append", "dtype": "f16", "heads": 0, "kv_heads": 4, "head_dim": 256, "dims": 0,
         "interleaved": False, "page": 32, "requests": 48, "lo": 3, "hi": 900, "new": 201, "norm": False, "scaled": False},
        # A prefix of a long context handed to another cache or engine.
        {"name": "read-prefix", "op": "read", "dtype": "bf16", "kv_heads": 8, "head_dim": 128, "format": "e2m1", "page": 64,
         "requests": 1, "lo": 8192, "hi": 8192},
        # The last tokens of some requests out of an 8-bit cache, to be kept in another format.
        {"name": "read-ragged", "op": "read", "dtype": "f32", "kv_heads": 4, "head_dim": 128, "format": "int8", "page": 16,
         "requests": 40, "lo": 1, "hi": 333},
        # One request's decode step in the decoder's geometry at 1025 positions.  Latency.
        {"name": "attend-one", "op": "attend", "dtype": "f32", "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 16,
         "requests": 1, "lo": 1025, "hi": 1025, "new": 1, "prompts": 0, "causal": True, "window": 0},
        # A decode step of 64 requests of all lengths.
        {"name": "attend-batch", "op": "attend", "dtype": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "requests": 64, "lo": 1, "hi": 16384, "new": 1, "prompts": 0, "causal": True, "window": 0},
        # Long contexts, few requests, wide heads: the cache is all that counts.
        {"name": "attend-long", "op": "attend", "dtype": "bf16", "heads": 24, "kv_heads": 4, "head_dim": 256, "page": 64,
         "requests": 8, "lo": 20001, "hi": 131072, "new": 1, "prompts": 0, "causal": True, "window": 0},
        # A prompt of 8192 tokens at once.
        {"name": "attend-prompt", "op": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "requests": 1, "lo": 8192, "hi": 8192, "new": 8192, "prompts": 1, "causal": True, "window": 0},
        # Two chunks of 700 tokens among fourteen single tokens, in binary32 as the projections give them, windowed.
        {"name": "attend-chunk", "op": "attend", "dtype": "f32", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32,
         "requests": 16, "lo": 1000, "hi": 5000, "new": 700, "prompts": 2, "causal": True, "window": 2048},
        # The answer of one request's step: its token's log probability and five alternatives.  Latency.
        {"name": "logprobs-step", "op": "logprobs", "dtype": "f32", "tokens": 1, "vocab": 151936, "top": 5, "masked": False},
        # A prompt's tokens scored, twenty alternatives each, some words excluded.
        {"name": "logprobs-prompt", "op": "logprobs", "dtype": "f32", "tokens": 1024, "vocab": 151936, "top": 20, "masked": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(["append", "read", "attend", "logprobs"], [3, 2, 4, 3])[0]
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 262144)
        return {"op": op, "dtype": dtype, "tokens": _log(rng, 1, max(1, min(4096, 1024 * 151936 // vocab))), "vocab": vocab,
                "top": rng.choice([0, 1, 5, 20, 64]), "masked": rng.random() < 0.5}
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    if op == "read":
        requests = _log(rng, 1, 128)
        most = 8192 * 8 * 128 // (kv_heads * head_dim * requests)
        hi = _log(rng, 1, max(1, min(8192, most)))
        return {"op": op, "dtype": dtype, "kv_heads": kv_heads, "head_dim": head_dim, "format": rng.choice(["e2m1", "e2m1", "int8", "e4m3"]),
                "page": page, "requests": requests, "lo": rng.choice([1, (hi + 1) // 2]), "hi": hi}
    if op == "append":
        dims = rng.choice([head_dim, head_dim // 2, head_dim // 4, head_dim // 2 + 2])
        form = {"dtype": dtype, "heads": heads, "head_dim": head_dim, "dims": dims, "interleaved": rng.random() < 0.5,
                "scaled": rng.random() < 0.5, "norm": rng.random() < 0.5}
        requests = _log(rng, 1, 256)
        most = 8192 * 48 * 128 // ((heads + 2 * kv_heads) * head_dim * requests)
        if rng.random() < 0.25:
            form.update(heads=0, dims=0, norm=False, scaled=False, interleaved=False)
        return {"op": op, **form, "kv_heads": kv_heads, "page": page, "requests": requests, "lo": 0, "hi": _log(rng, 1, 4096),
                "new": _log(rng, 1, max(1, min(2048, most)))}
    while True:
        requests, hi, new = _log(rng, 1, 128), _log(rng, 1, 131072), 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        prompts = 0 if new == 1 else rng.randint(1, requests)
        causal = rng.random() < 0.9
        case = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "requests": requests,
                "lo": rng.choice([0, 1, (hi + 1) // 2]), "hi": hi, "new": new, "prompts": prompts, "causal": causal,
                "window": _log(rng, 1, 8192) if causal and rng.random() < 0.25 else 0}
        lengths, added = _lengths(case)
        w = work(case)
        # No more than the largest listed cases: operations, the cache's values, and the plain form's padded scores.
        if w["flops"] <= 1.5e11 and requests * max(lengths) * kv_heads * head_dim <= 6e8 and \
                requests * heads * max(added) * max(max(lengths), 1) <= 1e9 and max(lengths) > 0:
            return case


# ---- lengths: the case's own, spread evenly between its bounds ------------------------------


def _spread(r, lo, hi):
    return lo + int((hi - lo + 1) * ((r + 1) * 0.6180339887498949 % 1.0))


def _lengths(case):
    """Tokens in the cache and new ones of every request; attend's lengths count its new tokens (where causal)."""
    n = case["requests"]
    lengths = [_spread(r, case["lo"], case["hi"]) for r in range(n)]
    if case["op"] == "read":
        return lengths, [0] * n
    if case["op"] == "attend":
        added = [max(1, case["new"] - 37 * r) if r < case["prompts"] else 1 for r in range(n)]
        if case["causal"]:
            lengths = [max(a, b) for a, b in zip(lengths, added)]
        return lengths, added
    return lengths, [_spread(7 * r + 3, (case["new"] + 1) // 2, case["new"]) for r in range(n)]


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] == "logprobs":
        n = case["tokens"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + case["tokens"] * (12 + 8 * case["top"]), "flops": 5.0 * n}
    lengths, added = _lengths(case)
    d, kv, size = case["head_dim"], case["kv_heads"], SIZE[case["dtype"]]
    token = kv * (d + 2 * d // GROUP)  # bytes of one token's keys and values
    if case["op"] == "read":
        tokens = sum(lengths)
        if case["format"] != "e2m1":
            token = 2 * kv * d
        return {"bytes": tokens * (token + 2 * kv * d * size + 4), "flops": 2.0 * tokens * kv * d}
    tokens = sum(added)
    if case["op"] == "append":
        return {"bytes": tokens * ((2 * case["heads"] + 2 * kv) * d * size + token + 8), "flops": 8.0 * tokens * kv * d}
    pairs = seen = 0
    for total, a in zip(lengths, added):
        for_all = [min(total, total - a + i + 1) if case["causal"] else total for i in range(a)]
        pairs += sum(min(x, case["window"]) if case["window"] else x for x in for_all)
        seen += min(total, case["window"] + a - 1) if case["window"] else total
    return {"bytes": seen * token + 2 * tokens * case["heads"] * d * size, "flops": 4.0 * d * case["heads"] * pairs}


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1_000_003 + salt) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(shape, seed, salt, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV).to(dtype)


def _whole(lo, hi, shape, seed, salt, dtype):
    return torch.randint(lo, hi, shape, generator=_gen(seed, salt), device=DEV, dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _empty(shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device=DEV)


def _frequencies(dims, scaled):
    """Radians a position, in 64 bits: base 10^7; scaled: eight times the context, by turns over the original 32768."""
    f = 1e7 ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if not scaled:
        return f, 1.0
    keep = ((32768 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return (1 - keep) * f / 8.0 + keep * f, 0.1 * math.log(8.0) + 1.0


def _cache(case, seed, pages):
    """Pages as a run leaves them: codes that fill the scales' range."""
    kv, d, page, kind = case["kv_heads"], case["head_dim"], case["page"], case.get("format", "e2m1")
    s = {}
    for salt, name in ((11, "k"), (12, "v")):
        if kind == "e2m1":
            s[name] = _whole(0, 256, (pages, kv, page, d // 2), seed, salt, torch.uint8)
            s[name + "_scale"] = _whole(124, 127, (pages, kv, d // GROUP, page), seed, salt + 10, torch.uint8)
            continue
        x = _randn((pages, kv, page, d) if name == "k" else (pages, kv, d, page), seed, salt)
        s[name] = torch.round(x * 32).clamp(-127, 127).to(torch.int8) if kind == "int8" else \
            (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s[name + "_scale"] = torch.exp2(_whole(-6, -4, (pages, kv), seed, salt + 10, torch.int32).float())
    return s


def prepare(case, seed):
    s = {"case": case}
    op = case["op"]
    if op == "logprobs":
        n, vocab = case["tokens"], case["vocab"]
        # What a head gives: many words of little weight and a few of much.
        x = 2.5 * _randn((n, vocab), seed, 2)
        few = min(8, vocab)
        at = _whole(0, vocab, (n, few), seed, 3, torch.int64)
        x.scatter_add_(1, at, 4.0 * _randn((n, few), seed, 4).abs() + 4.0)
        if case["masked"]:
            x.masked_fill_(torch.rand((1, vocab), generator=_gen(seed, 5), device=DEV) < 0.3, -math.inf)
        targets = torch.where(_whole(0, 2, (n,), seed, 6, torch.int64) == 1, at[:, 0], _whole(0, vocab, (n,), seed, 7, torch.int64))
        s.update(logits=x.to(DTYPES[case["dtype"]]), targets=targets.to(torch.int32), logprobs=_empty(n, torch.float32),
                 entropy=_empty(n, torch.float32), top_ids=_empty((n, case["top"])), top_logprobs=_empty((n, case["top"]), torch.float32))
        if own:
            _handles(s)
        return s
    lengths, added = _lengths(case)
    tokens, page = sum(added), case["page"]
    dtype, d, kv = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    heads = case.get("heads", 0)
    if op == "attend":
        columns = max(1, max(_pages(n, page) for n in lengths))
        order = torch.randperm(case["requests"] * columns, generator=_gen(seed, 1), device=DEV).to(torch.int32)
        s.update(_cache(case, seed, order.numel()))
        s.update(table=order.view(case["requests"], columns), q=(1.5 * _randn((tokens, heads, d), seed, 2)).to(dtype),
                 out=_empty((tokens, heads, d), dtype), lengths=_i32(lengths),
                 offsets=_i32([sum(added[:r]) for r in range(case["requests"] + 1)]), longest=max(lengths), most=max(added))
    else:
        # Slots on pages in no order: of all the positions read, or of the new ones behind those the cache holds.
        new = lengths if op == "read" else added
        start = [0] * len(new) if op == "read" else lengths
        begun = [n // page for n in start]
        pages = [_pages(n + a, page) - b for n, a, b in zip(start, new, begun)]
        order = torch.randperm(sum(pages) + 7, generator=_gen(seed, 1), device=DEV)
        s.update(_cache(case, seed, order.numel()))
        total = sum(new)
        owner = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
        first = torch.tensor([sum(new[:r]) for r in range(len(new))], device=DEV)
        at = torch.tensor(start, device=DEV)[owner] + torch.arange(total, device=DEV) - first[owner]
        shift = torch.tensor([sum(pages[:r]) - begun[r] for r in range(len(new))], device=DEV)
        s.update(positions=at.to(torch.int32), slots=(order[at // page + shift[owner]] * page + at % page).to(torch.int32))
        if op == "read":
            s.update(k_out=_empty((total, kv, d), dtype), v_out=_empty((total, kv, d), dtype))
        else:
            # q, k and v as one projection leaves them, side by side in a token's row.
            x = _randn((tokens, (heads + 2 * kv) * d), seed, 2, dtype)
            s["q"], s["k_new"], s["v_new"] = (t.view(tokens, -1, d) for t in x.split([heads * d, kv * d, kv * d], 1))
            s["q_out"] = _empty((tokens, heads, d), dtype)
            for name, salt in (("q_norm", 3), ("k_norm", 4)):
                s[name] = 1 + 0.1 * _randn(d, seed, salt) if case["norm"] else None
    if case.get("dims"):
        s["frequencies"], s["magnitude"] = _frequencies(case["dims"], case["scaled"])
        s["frequencies"] = s["frequencies"].to(DEV)
    if own:
        _handles(s)
    return s


# ---- the framework's calls --------------------------------------------------------------------

_CTX = None


def _handles(s):
    """What a program keeps from step to step: the context, the rotation, and the calls' descriptions (structs of pointers and sizes)."""
    global _CTX
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "prism-inference_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import prism_hip as ph

    _CTX = _CTX or ph.Context(0)
    s["ctx"], case, op = _CTX, s["case"], s["case"]["op"]
    s["dtype"] = dtype = {"f32": ph.DTYPE_F32, "f16": ph.DTYPE_F16, "bf16": ph.DTYPE_BF16}[case["dtype"]]
    if op == "logprobs":
        top = case["top"] > 0
        s["call"] = ph.Logprobs(dtype=dtype, tokens=case["tokens"], vocab=case["vocab"], top=case["top"], logits=s["logits"],
                                stride=s["logits"].stride(0), targets=s["targets"], logprobs=s["logprobs"], entropy=s["entropy"],
                                top_ids=s["top_ids"] if top else None, top_logprobs=s["top_logprobs"] if top else None)
        return
    kind = {"e2m1": ph.CACHE_E2M1, "int8": ph.CACHE_INT8, "e4m3": ph.CACHE_E4M3}[case.get("format", "e2m1")]
    s["cache"] = ph.KvCache(k=s["k"], v=s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"], format=kind, pages=s["k"].shape[0],
                            page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["head_dim"])
    if case.get("dims"):
        s["rope"] = ph.Rope(_CTX, case["dims"], s["frequencies"].cpu().numpy(), interleaved=case["interleaved"], magnitude=s["magnitude"])
    if op == "append" and case["heads"]:
        s["call"] = ph.QkvAppend(dtype=dtype, tokens=s["slots"].numel(), heads=case["heads"], q=s["q"], q_stride=s["q"].stride(0),
                                 k=s["k_new"], k_stride=s["k_new"].stride(0), v=s["v_new"], v_stride=s["v_new"].stride(0),
                                 positions=s["positions"], slots=s["slots"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                                 q_out=s["q_out"], q_out_stride=s["q_out"].stride(0))
    elif op == "attend":
        s["call"] = ph.Attention(dtype=dtype, requests=case["requests"], tokens=s["q"].shape[0], heads=case["heads"],
                                 max_pages=s["table"].shape[1], max_length=s["longest"], q=s["q"], q_stride=s["q"].stride(0), out=s["out"],
                                 out_stride=s["out"].stride(0), offsets=s["offsets"], lengths=s["lengths"], block_table=s["table"],
                                 scale=case["head_dim"] ** -0.5, causal=int(case["causal"]), window=case["window"])


def _own(s):
    case, ctx, op = s["case"], s["ctx"], s["case"]["op"]
    if op == "append":
        if case["heads"]:
            ctx.qkv_append_device(s["rope"], s["cache"], s["call"])
        else:
            ctx.kv_append_device(s["cache"], s["dtype"], s["k_new"], s["k_new"].stride(0), s["v_new"], s["v_new"].stride(0), s["slots"],
                                 s["slots"].numel())
        return _appended(s)
    if op == "read":
        ctx.kv_read_device(s["cache"], s["dtype"], s["slots"], s["slots"].numel(), s["k_out"], s["k_out"].stride(0), s["v_out"],
                           s["v_out"].stride(0))
        return [s["k_out"], s["v_out"]]
    if op == "attend":
        ctx.attention_device(s["cache"], s["call"])
        return s["out"]
    ctx.logprobs_device(s["call"])
    return [s[n] for n in ("logprobs", "entropy", "top_ids", "top_logprobs")]


def _appended(s):
    got = [s[n] for n in ("k", "v", "k_scale", "v_scale")]
    return got + [s["q_out"]] if s["case"]["heads"] else got


def run(s):
    if own:
        return _own(s)
    return {"append": _append, "read": _read, "attend": _attend, "logprobs": _logprobs}[s["case"]["op"]](s)


# ---- the plain forms ---------------------------------------------------------------------------


def _rotated(x, s, norm):
    """[tokens][heads][head_dim] normed and rotated, in 64 bits (angles of far positions, values next to a code's border), rounded once."""
    case, y = s["case"], x.double()
    if norm is not None:
        y = y / torch.sqrt((y * y).mean(2, keepdim=True) + EPS) * norm.double()
    angle = (s["positions"].double()[:, None] * s["frequencies"])[:, None]
    c, n = torch.cos(angle) * s["magnitude"], torch.sin(angle) * s["magnitude"]
    d = case["dims"]
    pairs = y[:, :, :d].unflatten(2, (d // 2, 2) if case["interleaved"] else (2, d // 2))
    a, b = pairs.unbind(3 if case["interleaved"] else 2)
    turned = torch.stack([a * c - b * n, b * c + a * n], 3 if case["interleaved"] else 2).flatten(2)
    return torch.cat([turned, y[:, :, d:]], 2).float().to(x.dtype)


def _append_one(s, x, codes, scale):
    page = s["case"]["page"]
    at = s["slots"].long()
    x = x.float().unflatten(2, (-1, GROUP))
    m, e = torch.frexp(x.abs().amax(3))  # the least e with the largest magnitude at most 6 * 2^e
    e = torch.where(m <= 0.75, e, e + 1) - 3
    e = torch.where(m > 0, e, LEAST).clamp(LEAST, MOST)
    y = x * torch.exp2(-e.float())[..., None]
    a = y.abs()
    # Borders between the magnitudes, ties to the even code.
    c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0) + torch.signbit(y).to(torch.uint8) * 8).flatten(2)
    packed = c[..., 0::2] | c[..., 1::2] << 4
    h = torch.arange(codes.shape[1], device=DEV)[None]
    codes[(at // page)[:, None], h, (at % page)[:, None]] = packed
    g = torch.arange(scale.shape[2], device=DEV)
    scale[(at // page)[:, None, None], h[..., None], g, (at % page)[:, None, None]] = (e + 127).to(torch.uint8)


def _append(s):
    k = _rotated(s["k_new"], s, s["k_norm"]) if s["case"]["heads"] else s["k_new"]
    _append_one(s, k, s["k"], s["k_scale"])
    _append_one(s, s["v_new"], s["v"], s["v_scale"])
    got = [s[n] for n in ("k", "v", "k_scale", "v_scale")]
    return got + [_rotated(s["q"], s, s["q_norm"])] if s["case"]["heads"] else got


def _levels():
    """The two values of each byte."""
    half = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=DEV)
    return torch.stack([half.repeat(16), half.repeat_interleave(16)], 1)


def _values(codes, scale):
    """[..., kv_heads, places, head_dim / 2] bytes and [..., kv_heads, groups, places] scales as values."""
    x = _levels()[codes.int()].flatten(-2)
    return (x.unflatten(-1, (-1, GROUP)) * torch.exp2(scale.float() - 127.0).transpose(-1, -2)[..., None]).flatten(-2)


def _read(s):
    case, at = s["case"], s["slots"].long()
    page, place, h = (at // case["page"])[:, None], (at % case["page"])[:, None], torch.arange(case["kv_heads"], device=DEV)[None]
    got = []
    for name in ("k", "v"):
        codes, scale = s[name], s[name + "_scale"]
        if case["format"] == "e2m1":
            x = _levels()[codes[page, h, place].int()].flatten(2).unflatten(2, (-1, GROUP))
            x = (x * torch.exp2(scale.transpose(2, 3)[page, h, place].float() - 127.0)[..., None]).flatten(2)
        else:
            codes = codes if case["format"] == "int8" else codes.view(torch.float8_e4m3fn)
            x = codes[page, h, place] if name == "k" else codes.transpose(2, 3)[page, h, place]
            x = x.float() * scale[page, h][..., None]
        got.append(x.to(s["k_out"].dtype))
    return got


def _attend(s):
    case = s["case"]
    kv, d, r = case["kv_heads"], case["head_dim"], case["requests"]
    g, a, longest = case["heads"] // kv, s["most"], s["longest"]
    table = s["table"][:, : _pages(longest, case["page"])].long()
    # The keys and values of every request, [requests][kv_heads][keys][head_dim].
    k, v = (_values(s[n][table], s[n + "_scale"][table]).transpose(1, 2).reshape(r, kv, -1, d) for n in ("k", "v"))
    offsets, lengths = s["offsets"].long(), s["lengths"].long()
    added = offsets[1:] - offsets[:-1]
    i = torch.arange(a, device=DEV)
    rows = (offsets[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(r, a, kv, g, d).permute(0, 2, 1, 3, 4).reshape(r, kv, a * g, d)
    scores = torch.matmul(q * d ** -0.5, k.transpose(2, 3)).view(r, kv, a, g, -1)
    key = torch.arange(k.shape[2], device=DEV)[None, None]
    at = (lengths - added)[:, None, None] + i[None, :, None]
    allowed = key < lengths[:, None, None]
    if case["causal"]:
        allowed = allowed & (key <= at)
    if case["window"]:
        allowed = allowed & (key > at - case["window"])
    scores.masked_fill_(~allowed[:, None, :, None], float("-inf"))
    top = scores.amax(4, keepdim=True)
    p = scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(4, keepdim=True)
    out = torch.matmul(p.view(r, kv, a * g, -1), v).view(r, kv, a, g, d) / torch.where(total > 0, total, 1.0)
    t = torch.arange(s["q"].shape[0], device=DEV)
    owner = torch.searchsorted(offsets[1:], t, right=True)
    return out.permute(0, 2, 1, 3, 4)[owner, t - offsets[owner]].reshape(s["out"].shape).to(s["out"].dtype)


def _logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    y = x - x.amax(1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(1, keepdim=True, dtype=torch.float64)  # long sums
    z = torch.log(total).float()
    entropy = z[:, 0] - ((e * torch.where(e > 0, y, 0.0)).sum(1, dtype=torch.float64) / total[:, 0]).float()
    target = y.gather(1, s["targets"].long()[:, None]) - z
    # Largest first, the lowest index first among equals: keys of a value's order and, below it, its index.
    bits = (x + 0.0).view(torch.int32).long()
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)) * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=DEV))
    ids = (1 << 20) - 1 - (key.topk(top, 1).values & ((1 << 20) - 1))
    return [target[:, 0], entropy, ids.to(torch.int32), y.gather(1, ids) - z]


# ---- the same in 64 bits, from the definitions ---------------------------------------------------


def _turned64(x, s, norm):
    x = x.double()
    if norm is not None:
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
    d = s["case"]["dims"]
    turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEV), torch.outer(s["positions"].double(), s["frequencies"]))
    out = x.clone()
    at = slice(0, d, 2), slice(1, d, 2)
    if not s["case"]["interleaved"]:
        at = slice(0, d // 2), slice(d // 2, d)
    z = torch.complex(x[..., at[0]].contiguous(), x[..., at[1]].contiguous()) * turn[:, None]
    out[..., at[0]], out[..., at[1]] = z.real, z.imag
    return out


def _values64(codes, scale):
    """e2m1 by its fields: [places][head_dim / 2] bytes and [groups][places] scales of one kv head."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign, rest = 1.0 - 2.0 * torch.floor(c / 8), c % 8
    field, half = torch.floor(rest / 2), rest % 2
    x = sign * torch.where(field > 0, torch.exp2(field - 1) * (1 + half / 2), half / 2)
    return x * torch.exp2(scale.double() - 127).T.repeat_interleave(GROUP, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":  # codes and the scales' bytes are whole numbers
        return [None, None, None, None, _turned64(s["q"], s, s["q_norm"])] if case["heads"] else None
    if case["op"] == "logprobs":
        got = [[], [], [], []]
        for i in range(case["tokens"]):
            x = s["logits"][i].double()
            lp = x - torch.logsumexp(x, 0)
            p = lp.exp()
            got[0].append(lp[s["targets"][i].long()])
            got[1].append(-(p[p > 0] * lp[p > 0]).sum())
            got[3].append(lp.sort(descending=True, stable=True).values[: case["top"]])
        return [torch.stack(got[0]), torch.stack(got[1]), None, torch.stack(got[3])]
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "read":
        got, slots = [], s["slots"].long()
        for name in ("k", "v"):
            out = torch.zeros(s["k_out"].shape, dtype=torch.float64, device=DEV)
            for h in range(kv):
                codes, scale = s[name][:, h], s[name + "_scale"][:, h]
                if case["format"] == "e2m1":
                    x = _values64(codes.flatten(0, 1), scale.transpose(0, 1).flatten(1))
                else:
                    codes = codes.double() if case["format"] == "int8" else codes.view(torch.float8_e4m3fn).double()
                    x = ((codes if name == "k" else codes.transpose(1, 2)) * scale.double()[:, None, None]).flatten(0, 1)
                out[:, h] = x[slots]
            got.append(out)
        return got
    g = case["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lengths, added = _lengths(case)
    begin = 0
    for r, (n, a) in enumerate(zip(lengths, added)):
        mine = s["table"][r, : _pages(n, page)].long()
        for h in range(kv):
            # the pages' positions one after the other
            keys, vals = (_values64(s[m][mine, h].flatten(0, 1), s[m + "_scale"][mine, h].transpose(0, 1).flatten(1))[:n] for m in ("k", "v"))
            for i in range(0, a, 1024):
                m = min(1024, a - i)
                q = s["q"][begin + i: begin + i + m, h * g: (h + 1) * g].double()
                z = (q.reshape(-1, d) @ keys.T).view(m, g, n) / math.sqrt(d)
                if case["causal"]:
                    back = (n - a + i + torch.arange(m, device=DEV))[:, None] - torch.arange(n, device=DEV)[None]  # tokens behind the row
                    hidden = (back < 0) | (back >= case["window"]) if case["window"] else back < 0
                    z = z.masked_fill(hidden[:, None], -math.inf)
                if n:
                    w = torch.softmax(z, 2).nan_to_num(0.0)
                    out[begin + i: begin + i + m, h * g: (h + 1) * g] = (w.view(-1, n) @ vals).view(m, g, d)
        begin += a
    return out
