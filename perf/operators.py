"""Operators between the packed projections of many requests: what is measured, and their plain forms.

  plan    block tables, slots and positions of one step from the requests' lengths, pages given out and taken back
          on the GPU (prism_hip_kv_plan_device).
  rope    rotary positions of [tokens][heads][head_dim] rows (prism_hip_rope_device).
  append  per-head RMSNorm and rotary positions of q and k, and k and v into the paged 8-bit cache, one scale for each
          page and kv head (prism_hip_qkv_append_device; without q and positions prism_hip_kv_append_device).
  attend  grouped-query attention over that cache (prism_hip_attention_device).

A cache page holds, for each kv head, the codes k[page_size][head_dim] and v[head_dim][page_size]; a value is its code
(int8, or e4m3 in a byte) times the page's and head's binary32 scale, which the append makes a power of two.  The cache is
returned as it is held, its codes as whole numbers beside their scales: equal codes and scales are equal values.
"""

import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
QMAX = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6


def listed():
    return [
        # One decode step of 64 requests: a new token each, a page now and then.  Latency.
        {"name": "plan-step", "op": "plan", "requests": 64, "page": 16, "lo": 1, "hi": 4096, "new": 1, "ended": False},
        # A busy step: some thousand requests, prompts among them, finished ones giving their pages back.
        {"name": "plan-mixed", "op": "plan", "requests": 2048, "page": 64, "lo": 0, "hi": 8192, "new": 61, "ended": True},
        # The query heads of one token of the decoder's geometry, half of each head rotated.  Latency.
        {"name": "rope-step", "op": "rope", "dtype": "f32", "heads": 16, "head_dim": 128, "dims": 64, "interleaved": False,
         "tokens": 1, "first": 1024, "scaled": False, "norm": True},
        # A prompt's chunk far into a long context, interleaved pairs, frequencies scaled for it.
        {"name": "rope-prompt", "op": "rope", "dtype": "bf16", "heads": 24, "head_dim": 256, "dims": 64, "interleaved": True,
         "tokens": 4099, "first": 131072, "scaled": True, "norm": False},
        # A decode step of 32 requests: q and k normed and rotated, k and v into the pages in use.
        {"name": "append-step", "op": "append", "dtype": "f32", "heads": 32, "kv_heads": 8, "head_dim": 128, "dims": 64,
         "interleaved": False, "format": "int8", "page": 16, "requests": 32, "lo": 1, "hi": 2048, "new": 1, "norm": True,
         "scaled": False},
        # A long prompt at once, into e4m3 pages.
        {"name": "append-prompt", "op": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "dims": 128,
         "interleaved": False, "format": "e4m3", "page": 64, "requests": 1, "lo": 0, "hi": 0, "new": 8192, "norm": True,
         "scaled": True},
        # Chunks of 48 requests that begin and end inside pages; k and v alone, rotated elsewhere.
        {"name": "append-ragged", "op": "append", "dtype": "f16", "heads": 0, "kv_heads": 4, "head_dim": 256, "dims": 0,
         "interleaved": False, "format": "int8", "page": 32, "requests": 48, "lo": 3, "hi": 900, "new": 201, "norm": False,
         "scaled": False},
        # One request's decode step in the decoder's geometry at 1025 positions.  Latency.
        {"name": "attend-one", "op": "attend", "dtype": "f32", "heads": 16, "kv_heads": 4, "head_dim": 128, "format": "int8",
         "page": 16, "requests": 1, "lo": 1025, "hi": 1025, "new": 1, "prompts": 0, "causal": True, "window": 0},
        # A decode step of 64 requests of all lengths.
        {"name": "attend-batch", "op": "attend", "dtype": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128, "format": "int8",
         "page": 16, "requests": 64, "lo": 1, "hi": 8192, "new": 1, "prompts": 0, "causal": True, "window": 0},
        # Long contexts, few requests, wide heads: the cache is all that counts.
        {"name": "attend-long", "op": "attend", "dtype": "bf16", "heads": 24, "kv_heads": 4, "head_dim": 256, "format": "e4m3",
         "page": 64, "requests": 8, "lo": 20001, "hi": 65536, "new": 1, "prompts": 0, "causal": True, "window": 0},
        # A prompt of 8192 tokens at once.
        {"name": "attend-prompt", "op": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "format": "int8",
         "page": 64, "requests": 1, "lo": 8192, "hi": 8192, "new": 8192, "prompts": 1, "causal": True, "window": 0},
        # Two chunks of 700 tokens among fourteen single tokens, in binary32 as the projections give them, windowed.
        {"name": "attend-chunk", "op": "attend", "dtype": "f32", "heads": 32, "kv_heads": 8, "head_dim": 128, "format": "int8",
         "page": 32, "requests": 16, "lo": 1000, "hi": 5000, "new": 700, "prompts": 2, "causal": True, "window": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(["plan", "rope", "append", "attend"], [2, 2, 3, 5])[0]
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "plan":
        requests = _log(rng, 1, 2048)
        return {"op": op, "requests": requests, "page": page, "lo": 0, "hi": _log(rng, 16, 8192),
                "new": _log(rng, 1, max(2, 60000 // requests)), "ended": rng.random() < 0.5}
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    dims = rng.choice([head_dim, head_dim // 2, head_dim // 4, head_dim // 2 + 2])
    form = {"dtype": dtype, "heads": heads, "head_dim": head_dim, "dims": dims, "interleaved": rng.random() < 0.5,
            "scaled": rng.random() < 0.5, "norm": rng.random() < 0.5}
    if op == "rope":
        most = 4099 * 24 * 256 // (heads * head_dim)
        return {"op": op, **form, "tokens": _log(rng, 1, min(16384, most)), "first": _log(rng, 1, 1 << 20)}
    kind = rng.choice(["int8", "e4m3"])
    if op == "append":
        requests = _log(rng, 1, 256)
        most = 8192 * 48 * 128 // ((heads + 2 * kv_heads) * head_dim * requests)
        if rng.random() < 0.25:
            form.update(heads=0, dims=0, norm=False, scaled=False, interleaved=False)
        return {"op": op, **form, "kv_heads": kv_heads, "format": kind, "page": page, "requests": requests, "lo": 0,
                "hi": _log(rng, 1, 4096), "new": _log(rng, 1, max(1, min(2048, most)))}
    while True:
        requests, hi, new = _log(rng, 1, 128), _log(rng, 1, 65536), 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        prompts = 0 if new == 1 else rng.randint(1, requests)
        causal = rng.random() < 0.9
        case = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "format": kind, "page": page,
                "requests": requests, "lo": rng.choice([0, 1, (hi + 1) // 2]), "hi": hi, "new": new, "prompts": prompts,
                "causal": causal, "window": _log(rng, 1, 8192) if causal and rng.random() < 0.25 else 0}
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
    if case["op"] == "attend":
        added = [max(1, case["new"] - 37 * r) if r < case["prompts"] else 1 for r in range(n)]
        if case["causal"]:
            lengths = [max(a, b) for a, b in zip(lengths, added)]
        return lengths, added
    added = [_spread(7 * r + 3, (case["new"] + 1) // 2, case["new"]) for r in range(n)]
    if case.get("ended"):
        added = [-1 if r % 16 == 5 else a for r, a in enumerate(added)]
    return lengths, added


def _pages(tokens, page):
    return -(-tokens // page)


def _columns(case):
    lengths, added = _lengths(case)
    grow = [a if case["op"] != "attend" else 0 for a in added]
    return max(1, max(_pages(n + max(a, 0), case["page"]) for n, a in zip(lengths, grow)))


def work(case):
    if case["op"] == "rope":
        rows = case["tokens"] * case["heads"]
        return {"bytes": 2 * rows * case["head_dim"] * SIZE[case["dtype"]] + 4 * case["tokens"], "flops": 6.0 * rows * case["dims"]}
    lengths, added = _lengths(case)
    tokens, page, n = sum(max(a, 0) for a in added), case["page"], case["requests"]
    if case["op"] == "plan":
        new = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(lengths, added) if b >= 0)
        back = sum(_pages(a, page) for a, b in zip(lengths, added) if b < 0)
        # lengths, new tokens, lengths after, offsets; three words a token; pages read and written.
        return {"bytes": 4 * (4 * n + 1) + 12 * tokens + 8 * (new + back), "flops": 2.0 * (tokens + n)}
    d, kv, size = case["head_dim"], case["kv_heads"], SIZE[case["dtype"]]
    if case["op"] == "append":
        values = tokens * kv * d
        return {"bytes": tokens * (2 * case["heads"] + 2 * kv) * d * size + 2 * values + 8 * tokens, "flops": 8.0 * values}
    pairs = seen = 0
    for total, a in zip(lengths, added):
        for_all = [min(total, total - a + i + 1) if case["causal"] else total for i in range(a)]
        pairs += sum(min(x, case["window"]) if case["window"] else x for x in for_all)
        seen += min(total, case["window"] + a - 1) if case["window"] else total
    return {"bytes": 2 * seen * kv * d + 2 * tokens * case["heads"] * d * size, "flops": 4.0 * d * case["heads"] * pairs}


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1_000_003 + salt) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(shape, seed, salt, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV).to(dtype)


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


def _table(case, seed, spare=0):
    """A block table of distinct pages in no order, how many of them each request uses, and all pages there are."""
    lengths, _ = _lengths(case)
    columns = _columns(case)
    order = torch.randperm(case["requests"] * columns + spare, generator=_gen(seed, 1), device=DEV).to(torch.int32)
    table = order[spare:].view(case["requests"], columns)
    used = torch.tensor([_pages(n, case["page"]) for n in lengths], device=DEV)
    return table, used, order


def _cache(case, seed, pages):
    """Pages as a run leaves them: codes that fill the scales' range, scales a power of two each."""
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    s = {}
    for salt, name, shape in ((11, "k", (pages, kv, page, d)), (12, "v", (pages, kv, d, page))):
        x = torch.randn(shape, generator=_gen(seed, salt), device=DEV)
        s[name] = _codes(x * (32.0 if case["format"] == "int8" else 100.0), case["format"])
        e = torch.randint(0, 2, (pages, kv), generator=_gen(seed, salt + 10), device=DEV).float()
        s[name + "_scale"] = torch.exp2(e - (5.0 if case["format"] == "int8" else 7.0))
    return s


def prepare(case, seed):
    s = {"case": case}
    op = case["op"]
    if op == "plan":
        lengths, added = _lengths(case)
        table, used, order = _table(case, seed, 64)
        columns, n = table.shape[1], case["requests"]
        mine = torch.arange(columns, device=DEV)[None] < used[:, None]
        # The stack of free pages: those no request holds, with room for all.
        free = torch.zeros_like(order)
        rest = torch.cat([order[:64], table[~mine]])
        free[: rest.numel()] = rest
        s.update(lengths=_i32(lengths), added=_i32(added), table=torch.where(mine, table, -1), free=free,
                 free_count=_i32([rest.numel()]))
        tokens = sum(max(a, 0) for a in added) + 13  # room for a few more, as a program of fixed sizes keeps
        s.update(new_lengths=_empty(n), offsets=_empty(n + 1), positions=_empty(tokens), slots=_empty(tokens),
                 owner=_empty(tokens), counts=_empty(4))
    elif op == "rope":
        dtype, shape = DTYPES[case["dtype"]], (case["tokens"], case["heads"], case["head_dim"])
        s.update(x=_randn(shape, seed, 2, dtype), positions=case["first"] + torch.arange(case["tokens"], dtype=torch.int32, device=DEV),
                 out=_empty(shape, dtype), norm=1 + 0.1 * _randn(case["head_dim"], seed, 3) if case["norm"] else None)
    else:
        lengths, added = _lengths(case)
        tokens = sum(added)
        dtype, d, heads, kv = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
        owner = torch.repeat_interleave(torch.arange(case["requests"], device=DEV), torch.tensor(added, device=DEV))
        first = torch.tensor([sum(added[:r]) for r in range(case["requests"])], device=DEV)
        if op == "append":
            # A cache of the pages that the step writes, in no order, and seven more.
            begun = [n // case["page"] for n in lengths]
            pages = [_pages(n + a, case["page"]) - b for n, a, b in zip(lengths, added, begun)]
            order = torch.randperm(sum(pages) + 7, generator=_gen(seed, 1), device=DEV)
            s.update({n + "_codes" if n in "kv" else n: t for n, t in _cache(case, seed, order.numel()).items()})
            at = torch.tensor(lengths, device=DEV)[owner] + torch.arange(tokens, device=DEV) - first[owner]
            s["positions"] = at.to(torch.int32)
            shift = torch.tensor([sum(pages[:r]) - begun[r] for r in range(case["requests"])], device=DEV)
            s["slots"] = (order[at // case["page"] + shift[owner]] * case["page"] + at % case["page"]).to(torch.int32)
            # q, k and v as one projection leaves them, side by side in a token's row.
            x = _randn((tokens, (heads + 2 * kv) * d), seed, 2, dtype)
            s["q"], s["k"], s["v"] = (t.view(tokens, -1, d) for t in x.split([heads * d, kv * d, kv * d], 1))
            s["q_out"] = _empty((tokens, heads, d), dtype)
            for name, salt in (("q_norm", 3), ("k_norm", 4)):
                s[name] = 1 + 0.1 * _randn(d, seed, salt) if case["norm"] else None
        else:
            table, _, order = _table(case, seed)
            s.update(_cache(case, seed, order.numel()))
            s.update(table=table, q=(1.5 * _randn((tokens, heads, d), seed, 2)).to(dtype), out=_empty((tokens, heads, d), dtype),
                     lengths=_i32(lengths), offsets=_i32([sum(added[:r]) for r in range(case["requests"] + 1)]),
                     longest=max(lengths), most=max(added))
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
    dtype = {"f32": ph.DTYPE_F32, "f16": ph.DTYPE_F16, "bf16": ph.DTYPE_BF16}.get(case.get("dtype"))
    if case.get("dims"):
        s["rope"] = ph.Rope(_CTX, case["dims"], s["frequencies"].cpu().numpy(), interleaved=case["interleaved"], magnitude=s["magnitude"])
    if op == "plan":
        s["call"] = ph.KvPlan(requests=case["requests"], max_pages=s["table"].shape[1], max_tokens=s["slots"].numel(), page_size=case["page"],
                              free_capacity=s["free"].numel(), lengths=s["lengths"], added=s["added"], block_table=s["table"],
                              free_pages=s["free"], free_count=s["free_count"], new_lengths=s["new_lengths"], offsets=s["offsets"],
                              positions=s["positions"], slots=s["slots"], owners=s["owner"], counts=s["counts"])
    elif op == "rope":
        s["dtype"] = dtype
    else:
        s["cache"] = ph.KvCache(k=s["k_codes"] if op == "append" else s["k"], v=s["v_codes"] if op == "append" else s["v"],
                                k_scale=s["k_scale"], v_scale=s["v_scale"],
                                format=ph.CACHE_INT8 if case["format"] == "int8" else ph.CACHE_E4M3, pages=s["k_scale"].shape[0],
                                page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["head_dim"])
    if op == "append" and case["heads"]:
        s["call"] = ph.QkvAppend(dtype=dtype, tokens=s["slots"].numel(), heads=case["heads"], q=s["q"], q_stride=s["q"].stride(0),
                                 k=s["k"], k_stride=s["k"].stride(0), v=s["v"], v_stride=s["v"].stride(0), positions=s["positions"],
                                 slots=s["slots"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, q_out=s["q_out"],
                                 q_out_stride=s["q_out"].stride(0))
    elif op == "append":
        s["dtype"] = dtype
    elif op == "attend":
        s["call"] = ph.Attention(dtype=dtype, requests=case["requests"], tokens=s["q"].shape[0], heads=case["heads"],
                                 max_pages=s["table"].shape[1], max_length=s["longest"], q=s["q"], q_stride=s["q"].stride(0), out=s["out"],
                                 out_stride=s["out"].stride(0), offsets=s["offsets"], lengths=s["lengths"], block_table=s["table"],
                                 scale=case["head_dim"] ** -0.5, causal=int(case["causal"]), window=case["window"])


def _own(s):
    case, ctx, op = s["case"], s["ctx"], s["case"]["op"]
    if op == "plan":
        ctx.kv_plan_device(s["call"])
        return [s[n] for n in ("new_lengths", "offsets", "positions", "slots", "owner", "counts", "table", "free")]
    if op == "rope":
        ctx.rope_device(s["rope"], s["dtype"], s["x"], s["x"].stride(0), s["positions"], case["tokens"], case["heads"], case["head_dim"],
                        s["out"], s["out"].stride(0), s["norm"], EPS)
        return s["out"]
    if op == "append":
        if case["heads"]:
            ctx.qkv_append_device(s["rope"], s["cache"], s["call"])
        else:
            ctx.kv_append_device(s["cache"], s["dtype"], s["k"], s["k"].stride(0), s["v"], s["v"].stride(0), s["slots"], s["slots"].numel())
        return _appended(s)
    ctx.attention_device(s["cache"], s["call"])
    return s["out"]


def _appended(s):
    got = [s[n] for n in ("k_codes", "v_codes", "k_scale", "v_scale")]
    return got + [s["q_out"]] if s["case"]["heads"] else got


def run(s):
    if own:
        return _own(s)
    return {"plan": _plan, "rope": _rope, "append": _append, "attend": _attend}[s["case"]["op"]](s)


# ---- the plain forms ---------------------------------------------------------------------------


def _plan(s):
    page, added, table = s["case"]["page"], s["added"].long(), s["table"]
    lengths, count, room = s["lengths"].long(), s["free_count"].long()[0], s["free"].numel()
    ended, new = added < 0, added.clamp(min=0)
    after = torch.where(ended, 0, lengths + new)
    held, want = (lengths + page - 1) // page, (after + page - 1) // page
    back = torch.where(ended, held, 0)
    need = torch.where(ended, 0, want - held)
    total = count + back.sum()
    column = torch.arange(table.shape[1], device=DEV)[None]
    # Pages given back, on top of the stack; the place behind its end takes what is none.
    put = torch.where(ended[:, None] & (column < held[:, None]), (count + back.cumsum(0) - back)[:, None] + column, room)
    free = torch.cat([s["free"], s["free"].new_zeros(1)]).scatter(0, put.reshape(-1), table.reshape(-1))[:room]
    # Pages given out, from its top.
    take = total - 1 - ((need.cumsum(0) - need)[:, None] + column - held[:, None])
    fresh = ~ended[:, None] & (column >= held[:, None]) & (column < want[:, None])
    table = torch.where(fresh, free[take.clamp(0, room - 1)], table)
    ends = new.cumsum(0)
    t = torch.arange(s["slots"].numel(), device=DEV)
    owner = torch.searchsorted(ends, t, right=True)
    there, who = t < ends[-1], owner.clamp(max=added.numel() - 1)
    at = lengths[who] + t - (ends - new)[who]
    slot = table[who, (at // page).clamp(0, table.shape[1] - 1)].long() * page + at % page
    i32 = torch.int32
    counts = torch.stack([total - need.sum(), ends[-1], need.sum(), torch.zeros_like(total)])
    return [after.to(i32), torch.cat([ends.new_zeros(1), ends]).to(i32), torch.where(there, at, 0).to(i32),
            torch.where(there, slot, -1).to(i32), torch.where(there, owner, -1).to(i32), counts.to(i32), table, free]


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


def _rope(s):
    return _rotated(s["x"], s, s["norm"])


def _codes(x, kind):
    if kind == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, kind):
    return codes.float() if kind == "int8" else codes.view(torch.float8_e4m3fn).float()


def _append_one(s, x, codes, scale, swap):
    """Tokens x [tokens][kv_heads][head_dim] into the pages' codes; swap: the page's positions are its last axis."""
    case = s["case"]
    page, kind, qmax = case["page"], case["format"], QMAX[case["format"]]
    at = s["slots"].long()
    pages, place = at // page, at % page
    x = x.float()
    n, kv, d = scale.shape[0], case["kv_heads"], case["head_dim"]
    first = torch.full((n,), page, device=DEV).scatter_reduce(0, pages, place, "amin")
    most = torch.zeros((n, kv), device=DEV).scatter_reduce(0, pages[:, None].expand(-1, kv), x.abs().amax(2), "amax")
    m, e = torch.frexp(most)  # most <= qmax * 2^e, the least such e
    e = torch.where(m <= (qmax / 128 if kind == "int8" else qmax / 512), e, e + 1) - (7 if kind == "int8" else 9)
    least = torch.exp2(e.clamp(min=-100).float().where(most > 0, torch.full_like(most, -100.0)))
    old = torch.where((first == 0)[:, None], 0.0, scale)
    new = torch.where((first < page)[:, None], torch.maximum(old, least), scale)
    inv = 1.0 / new
    # What the page held before its first new token, at the new scale; then the new tokens.
    kept = (torch.arange(page, device=DEV)[None] < first[:, None]) & (first < page)[:, None]
    kept = kept[:, None, None, :] if swap else kept[:, None, :, None]
    again = _codes(_values(codes, kind) * (old * inv)[:, :, None, None], kind)
    codes = torch.where(kept, again, codes)
    got = _codes(x * inv[pages][:, :, None], kind)
    h = torch.arange(kv, device=DEV)
    if swap:
        codes[pages[:, None, None], h[None, :, None], torch.arange(d, device=DEV)[None, None], place[:, None, None]] = got
    else:
        codes[pages[:, None], h[None], place[:, None]] = got
    return codes, new


def _append(s):
    heads = s["case"]["heads"]
    k = _rotated(s["k"], s, s["k_norm"]) if heads else s["k"]
    k_codes, k_scale = _append_one(s, k, s["k_codes"], s["k_scale"], False)
    v_codes, v_scale = _append_one(s, s["v"], s["v_codes"], s["v_scale"], True)
    got = [k_codes, v_codes, k_scale, v_scale]
    return got + [_rotated(s["q"], s, s["q_norm"])] if heads else got


def _attend(s):
    case = s["case"]
    kv, d, page, r = case["kv_heads"], case["head_dim"], case["page"], case["requests"]
    g, a, longest = case["heads"] // kv, s["most"], s["longest"]
    table = s["table"][:, : _pages(longest, page)].long()
    # The keys and values of every request, [requests][kv_heads][keys][head_dim].
    k = (_values(s["k"][table], case["format"]) * s["k_scale"][table][:, :, :, None, None]).transpose(1, 2).reshape(r, kv, -1, d)
    v = (_values(s["v"][table], case["format"]) * s["v_scale"][table][:, :, :, None, None]).permute(0, 2, 1, 4, 3).reshape(r, kv, -1, d)
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


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned64(s["x"], s, s["norm"])
    if case["op"] == "append":
        # Codes are whole numbers; the scales are powers of two: the least that holds every new value, or the page's own.
        def scales(x, scale):
            got, qmax, page = scale.double().clone(), QMAX[case["format"]], case["page"]
            pages, places = (s["slots"] // page).tolist(), (s["slots"] % page).tolist()
            top = x.abs().amax(2).double().cpu()
            least = torch.exp2(torch.ceil(torch.log2(top / qmax)).clamp(min=-100.0))
            got, begun = got.cpu(), {}
            for t, p in enumerate(pages):
                if p not in begun:
                    begun[p] = True
                    if places[t] == 0:
                        got[p] = 0.0
                got[p] = torch.maximum(got[p], least[t])
            return got

        k = _turned64(s["k"], s, s["k_norm"]).float().to(s["k"].dtype) if case["heads"] else s["k"]
        got = [None, None, scales(k, s["k_scale"]), scales(s["v"], s["v_scale"])]
        return got + [_turned64(s["q"], s, s["q_norm"])] if case["heads"] else got
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    g = case["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lengths, added = _lengths(case)
    begin = 0
    for r, (n, a) in enumerate(zip(lengths, added)):
        mine = s["table"][r, : _pages(n, page)].long()
        for h in range(kv):
            # codes * scales, the page's positions one after the other
            keys = (_values(s["k"][mine, h], case["format"]).double() * s["k_scale"][mine, h].double()[:, None, None]).reshape(-1, d)[:n]
            vals = (_values(s["v"][mine, h], case["format"]).double() * s["v_scale"][mine, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:n]
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
