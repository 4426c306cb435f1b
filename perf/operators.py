"""A paged key/value cache and the attention that reads it, as timed cases.

Three operators: ``paged_cache_write`` (new tokens' K and V go into their pages, as they are or in
8 bits), ``paged_cache_read`` (a sequence's K and V come back out of them) and
``flash_attn_paged_func`` (a chunk of new tokens, or a single one, attends to everything cached).

A case has:
  op         "write", "read" or "attend"
  z n        batch entries, new tokens of each (the longest entry's where ``ragged``)
  ctx        tokens that an entry has cached before (write) or in all (read, attend); for z > 1 the
             entries' lengths are spread over [ctx/8, ctx], see ``_lengths``
  hq hkv d   query heads (attend), key/value heads, head dimension
  page       tokens per page
  dtype      "fp16" or "bf16": the model's type
  e4m3       the cache holds 8 bits with a power-of-two scale per token and head, else ``dtype``
  ragged     entries bring unequal numbers of new tokens, padded to ``n``
  causal     (attend) new token i of entry z sees the keys up to its own
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# exponents of the scale: what code * 2^e has to be in the model's type without rounding or overflow
_EXPONENTS = {torch.float16: (-15, 8), torch.bfloat16: (-120, 120)}


def _case(op, z, n, ctx, hkv, d, page, dtype, e4m3, hq=0, ragged=False, causal=True):
    return {"op": op, "z": z, "n": n, "ctx": ctx, "hq": hq, "hkv": hkv, "d": d, "page": page, "dtype": dtype,
            "e4m3": e4m3, "ragged": ragged, "causal": causal}


def listed():
    cases = {
        # one new token of each of 64 sequences into an 8-bit cache: a decode step's write, all latency
        "write_tokens_e4m3": _case("write", 64, 1, 128, 8, 128, 16, "bf16", True),
        # chunks of four long prompts into an 8-bit cache, from an odd position on
        "write_chunk_e4m3": _case("write", 4, 4096, 1001, 8, 128, 64, "bf16", True, ragged=True),
        # the same without a change of type, heads of 96
        "write_chunk_fp16_d96": _case("write", 3, 1000, 2016, 16, 96, 32, "fp16", False),
        # an 8-bit cache of eight conversations handed to a user of dense K and V
        "read_e4m3": _case("read", 8, 0, 8192, 8, 128, 64, "bf16", True),
        # a 16-bit cache read back, small pages, odd lengths
        "read_bf16_d64": _case("read", 5, 0, 2016, 16, 64, 16, "bf16", False),
        # one conversation, one new token: latency of a decode step
        "attend_token_alone": _case("attend", 1, 1, 4096, 8, 128, 64, "bf16", False, hq=32),
        # a served batch of unequal conversations, one new token each, 16-bit cache
        "attend_tokens_bf16": _case("attend", 32, 1, 16384, 8, 128, 64, "bf16", False, hq=32),
        # a larger one on an 8-bit cache
        "attend_tokens_e4m3": _case("attend", 64, 1, 16384, 8, 128, 64, "bf16", True, hq=32),
        # as many key/value heads as query heads, heads of 64, pages that end inside a tile
        "attend_tokens_mha_d64": _case("attend", 16, 1, 2048, 16, 64, 48, "fp16", False, hq=16),
        # five drafted tokens of each sequence against the cache, in one call
        "attend_drafts_e4m3": _case("attend", 8, 5, 8192, 4, 128, 16, "fp16", True, hq=32),
        # a chunk of a long prompt over what is cached of it
        "attend_chunk_bf16": _case("attend", 1, 2048, 16384, 8, 128, 64, "bf16", False, hq=32),
        # a step of a server that mixes prompts' chunks with single tokens, 8-bit cache
        "attend_mixed_e4m3": _case("attend", 6, 512, 8192, 8, 128, 32, "bf16", True, hq=32, ragged=True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _scores(c):
    return c["z"] * c["hq"] * c["n"] * c["ctx"]


def draw(rng):
    most = {c["op"]: c for c in listed()[::-1] if c["name"] in ("write_chunk_e4m3", "read_e4m3", "attend_chunk_bf16")}
    while True:
        op = rng.choice(("write", "read", "attend", "attend", "attend"))
        dtype, e4m3 = rng.choice(("fp16", "bf16")), rng.random() < 0.5
        d, page = rng.choice((64, 96, 128, 128)), rng.choice((16, 16, 32, 48, 64, 128, 256))
        hkv, group = rng.choice((1, 2, 4, 5, 8, 8, 16)), rng.choice((1, 2, 3, 4, 4, 7, 8, 16))
        z, ctx = _log(rng, 1, 64), _log(rng, 1, 32768)
        n = 1 if op == "attend" and rng.random() < 0.5 else _log(rng, 1, 4096)
        if op == "read":
            n = 0
        if op == "attend" and rng.random() < 0.9:  # (with fewer keys than new tokens the first ones see nothing)
            ctx = max(ctx, n)
        c = _case(op, z, n, ctx, hkv, d, page, dtype, e4m3, hq=hkv * group if op == "attend" else 0,
                  ragged=n > 1 and rng.random() < 0.4, causal=op != "attend" or rng.random() < 0.85)
        w = work(c)
        held = z * (ctx + (n if op == "write" else 0)) * hkv * d * 2
        if w["bytes"] + w["flops"] / 250 > 1.5e9 or held > 3e9:
            continue
        if op == "attend" and _scores(c) > _scores(most["attend"]):
            continue
        if op == "write" and z * n * hkv * d > 16 * 1024 * 1024 or op == "read" and held > 2 * 8 * 8192 * 8 * 128:
            continue
        return c


def _lengths(n, z):
    """Lengths of a batch's entries: even steps from n/8 to n, odd ones among them; the same set for
    every seed, in another order."""
    lo = max(1, n // 8)
    return [lo + (n - lo) * i // max(1, z - 1) for i in range(z)] if z > 1 else [n]


def _new_lengths(case):
    """New tokens of each entry: ``n``, or where ragged from one token (a decode step's) to ``n``."""
    z, n = case["z"], case["n"]
    return [1 + (n - 1) * i // max(1, z - 1) for i in range(z)] if case["ragged"] and z > 1 else [n] * z


def _plan(case, seed):
    """Lengths of the entries, in the seed's order: (cached before or in all, new)."""
    cpu = torch.Generator()
    cpu.manual_seed(int(seed))
    a, b = torch.randperm(case["z"], generator=cpu).tolist(), torch.randperm(case["z"], generator=cpu).tolist()
    ctx, new = _lengths(case["ctx"], case["z"]), _new_lengths(case)
    return [ctx[i] for i in a], [new[i] for i in b], cpu


def _encode(x):
    """Rows of (..., D) -> e4m3 codes and the exponent of each row's power-of-two scale: the smallest for
    which the row's largest finite value is at most 448, in the range the type allows.  Values that are
    not finite become NaN; what would round beyond the type's largest finite value is rounded towards zero."""
    low, high = _EXPONENTS[x.dtype]
    f = x.float()
    finite = torch.isfinite(f)
    top = torch.where(finite, f, 0.0).abs().amax(-1)
    m, ex = torch.frexp(top)
    e = torch.where(top > 0, torch.where(m > 0.875, ex - 8, ex - 9), low).clamp(low, high)
    most = torch.where(e == high, 240.0, 448.0).unsqueeze(-1)
    y = torch.ldexp(f, -e.unsqueeze(-1))
    y = torch.where(finite, torch.minimum(torch.maximum(y, -most), most), float("nan"))
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    z, n, hkv, d, page = case["z"], case["n"], case["hkv"], case["d"], case["page"]
    dtype = _DTYPES[case["dtype"]]
    ctx, new, cpu = _plan(case, seed)
    held = [c + (x if case["op"] == "write" else 0) for c, x in zip(ctx, new)]
    pages = [-(-c // page) for c in held]
    # the pool's pages in any order, as a server that has run for a while hands them out
    total = sum(held) // page + z + 3
    order = torch.randperm(total, generator=cpu).tolist()
    table, at = [], 0
    for p in pages:
        table.append(order[at:at + p] + [order[0]] * (max(pages) - p))
        at += p
    i32 = {"dtype": torch.int32, "device": "cuda"}
    state = {"case": case, "dtype": dtype, "table": torch.tensor(table, **i32),
             "lengths": torch.tensor(ctx, **i32), "most": max(ctx),
             "new": torch.tensor(new, **i32) if case["ragged"] else None}
    # (z, token) of every token that is real, for the plain form
    real = [(i, j) for i in range(z) for j in range(new[i])] if case["op"] == "write" else []
    state["real"] = torch.tensor(real, device="cuda").reshape(-1, 2).unbind(1)

    def values(*shape):
        # heads and tokens of unequal size, like projections' outputs
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        x *= torch.exp2(torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))
        return x.to(dtype)

    cache = []
    for _ in range(2):
        pool = values(total, page, hkv, d)
        cache.append(_encode(pool) if case["e4m3"] else (pool, None))
    (state["k_cache"], state["k_scale"]), (state["v_cache"], state["v_scale"]) = cache
    if case["op"] == "write":
        state["k"], state["v"] = values(z, n, hkv, d), values(z, n, hkv, d)
    if case["op"] == "attend":
        state["q"] = torch.randn((z, n, case["hq"], d), generator=g, device="cuda", dtype=torch.float32).to(dtype)
    return state


def _package():
    path = os.path.abspath("flash-attention-v100_b200")  # of the working folder
    if path not in sys.path:
        sys.path.insert(1, path)
    import flash_attn_v100

    return flash_attn_v100


def run(state):
    case = state["case"]
    if own:
        package = _package()
        cache = (state["k_cache"], state["v_cache"], state["table"])
        scales = {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        if case["op"] == "write":
            package.paged_cache_write(state["k"], state["v"], *cache, state["lengths"], state["new"], **scales)
            return {x: state[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")}
        if case["op"] == "read":
            return package.paged_cache_read(*cache, state["lengths"], state["most"], dtype=state["dtype"], **scales)
        return package.flash_attn_paged_func(state["q"], *cache, state["lengths"], state["new"],
                                             causal=case["causal"], return_lse=True, **scales)
    if case["op"] == "write":
        _plain_write(state)
        return {x: state[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if case["op"] == "read":
        return tuple(_plain_read(state, x).to(state["dtype"]) for x in "kv")
    return _plain_attend(state)


def _plain_write(state):
    z, i = state["real"]
    position = state["lengths"].long()[z] + i
    page, slot = state["table"].long()[z, position // state["case"]["page"]], position % state["case"]["page"]
    for x in "kv":
        rows = state[x][z, i]
        if state["k_scale"] is None:
            state[x + "_cache"][page, slot] = rows
        else:
            codes, scale = _encode(rows)
            state[x + "_cache"].view(torch.uint8)[page, slot] = codes.view(torch.uint8)
            state[x + "_scale"].view(torch.uint8)[page, slot] = scale.view(torch.uint8)


def _plain_read(state, x):
    """fp32 (z, most, hkv, d): what is cached, zeros behind each entry's last token."""
    table = state["table"].long()
    cache = state[x + "_cache"]
    if state["k_scale"] is None:
        pages = cache[table].float()
    else:
        pages = cache.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        e = state[x + "_scale"].view(torch.uint8)[table].int() - 127
        pages = torch.ldexp(pages, e.unsqueeze(-1))
    dense = pages.flatten(1, 2)[:, :state["most"]]
    at = torch.arange(state["most"], device="cuda")
    return torch.where((at < state["lengths"][:, None])[:, :, None, None], dense, 0.0)


def _plain_attend(state):
    case = state["case"]
    z, n, hq, hkv, d = (case[x] for x in ("z", "n", "hq", "hkv", "d"))
    group = hq // hkv
    k, v = _plain_read(state, "k").permute(0, 2, 3, 1), _plain_read(state, "v").permute(0, 2, 1, 3)
    q = state["q"].float().reshape(z, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(z, hkv, group * n, d)
    s = torch.matmul(q * d ** -0.5, k).reshape(z, hkv, group, n, -1)
    i, j = torch.arange(n, device="cuda"), torch.arange(state["most"], device="cuda")
    new = torch.full((z,), n, device="cuda") if state["new"] is None else state["new"]
    last = state["lengths"][:, None] - 1 + ((i - new[:, None] + 1) if case["causal"] else 0 * i)
    last = torch.where(i < new[:, None], last, -1)
    seen = j <= last[:, None, None, :, None]
    s = torch.where(seen, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(z, hkv, group * n, -1), v).reshape(z, hkv, group, n, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(z, n, hq, d)
    lse = (m + torch.log(total)).reshape(z, hq, n)
    return o.to(state["dtype"]), lse


def work(case):
    """Each input read once, each output written once.  A cached row is d values of 16 bits, or of 8 and a
    byte of scale.  Attention: two products over the pairs that the mask leaves; an entry's keys are read
    once, by whichever of its new tokens.  (Which lengths meet which numbers of new tokens is the seed's: they
    are taken in the order in which they are spread.)"""
    z, n, hq, hkv, d = (case[x] for x in ("z", "n", "hq", "hkv", "d"))
    row = d + 1 if case["e4m3"] else 2 * d
    ctx, new = _lengths(case["ctx"], z), _new_lengths(case)
    if case["op"] == "write":
        return {"bytes": 2.0 * hkv * sum(new) * (2 * d + row), "flops": 0}
    if case["op"] == "read":
        return {"bytes": 2.0 * hkv * (sum(ctx) * row + z * max(ctx) * 2 * d), "flops": 0}
    pairs = 0
    for c, x in zip(ctx, new):
        first = max(0, c - x)  # the first new token sees first + 1 keys
        rows = min(c, x)
        pairs += rows * first + rows * (rows + 1) // 2 if case["causal"] else c * x
    read = 2.0 * hkv * sum(ctx) * row + 2.0 * hq * d * sum(new)
    return {"bytes": read + hq * z * n * (2.0 * d + 4), "flops": 4.0 * hq * d * pairs}


def _value64(row, e4m3_scale):
    """A cached row in 64 bits."""
    x = row.to(torch.float64)
    return x if e4m3_scale is None else x * e4m3_scale.to(torch.float64).unsqueeze(-1)


def _nearest_e4m3(y):
    """The e4m3 number nearest to y (|y| <= 448), halves to even: steps of 2^(exponent - 3), at least 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)) + 1e-9) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    z, n, page = case["z"], case["n"], case["page"]
    ctx = state["lengths"].tolist()
    new = [n] * z if state["new"] is None else state["new"].tolist()
    low, high = _EXPONENTS[state["dtype"]]
    e4m3 = case["e4m3"]
    if case["op"] == "write":
        out = {}
        for x in "kv":
            cache = state[x + "_cache"].to(torch.float64)
            scale = state[x + "_scale"].to(torch.float64) if e4m3 else None
            for i in range(z):
                at = torch.arange(ctx[i], ctx[i] + new[i], device="cuda")
                where = (state["table"][i, at // page].long(), at % page)
                rows = state[x][i, :new[i]].to(torch.float64)
                if e4m3:
                    top = rows.abs().amax(-1, keepdim=True)
                    s = torch.exp2(torch.ceil(torch.log2(top / 448) - 1e-9).clamp(low, high))
                    scale[where] = s.squeeze(-1)
                    rows = _nearest_e4m3(rows / s)
                cache[where] = rows
            out[x + "_cache"], out[x + "_scale"] = cache, scale
        return out

    def entry(i, x, most):
        """(tokens, hkv, d) of entry i in 64 bits."""
        at = torch.arange(most, device="cuda")
        where = (state["table"][i, at // page].long(), at % page)
        scale = state[x + "_scale"].view(torch.uint8)[where].view(torch.float8_e8m0fnu) if e4m3 else None
        rows = state[x + "_cache"]
        rows = rows.view(torch.uint8)[where].view(rows.dtype) if e4m3 else rows[where]
        return _value64(rows, scale)

    if case["op"] == "read":
        out = [torch.zeros((z, state["most"], case["hkv"], case["d"]), dtype=torch.float64, device="cuda") for _ in "kv"]
        for t, x in zip(out, "kv"):
            for i in range(z):
                t[i, :ctx[i]] = entry(i, x, ctx[i])
        return tuple(out)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    o = torch.zeros((z, n, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((z, hq, n), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(z):
        k, v = entry(i, "k", ctx[i]), entry(i, "v", ctx[i])
        rows = torch.arange(new[i], device="cuda")[:, None]
        keys = torch.arange(ctx[i], device="cuda")[None, :]
        hidden = keys - ctx[i] > rows - new[i] if case["causal"] else torch.zeros_like(keys - rows, dtype=torch.bool)
        empty = hidden.all(-1)
        for h in range(hq):
            s = state["q"][i, :new[i], h].to(torch.float64) @ k[:, h // (hq // hkv)].T / math.sqrt(d)
            s.masked_fill_(hidden, -math.inf)
            lse[i, h, :new[i]] = torch.logsumexp(s, -1)
            o[i, :new[i], h] = torch.softmax(s, -1).masked_fill(empty[:, None], 0.0) @ v[:, h // (hq // hkv)]
    return o, lse
