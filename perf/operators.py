"""Workloads of the ragged paged-cache operators, in their plain form and through the package's own kernels.

Four operators over a paged KV cache ``[pages, page size, KV heads, head dim]``, whose ragged batch is packed along the
token axis (sequence b's tokens are rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]``, and they are the last ones of the
``cache_seqlens[b]`` tokens that the cache holds for it once the call's tokens are written):

* ``append``  -- writes the new tokens' K and V into their pages, as they are or quantised to e4m3 with a power-of-two
  scale for each token and KV head: ``s`` the smallest power of two (at least 2^-126) with ``max |x| <= 448 s``, the
  cache holds ``e4m3(x / s)``.
* ``gather``  -- reads tokens back from their pages into packed rows: ``e4m3 value * s``, rounded to 16 bits.
* ``chunk``   -- attention of the new tokens over the paged cache, 16-bit or quantised; query token i of n sees the first
  ``cache_seqlens[b] - n + i + 1`` tokens (causal).  ``out = softmax(q k / sqrt(d)) v``, with the row's log-sum-exp.
"""

import math
import random

import torch

own = False


# ------------------------------------------------------------------------------------------------------- the cases

def _case(name, op, **kw):
    base = dict(name=name, op=op, dtype="bf16", hq=32, hkv=8, d=128, page=16, batch=1, new=1, ctx=0, singles=0,
                ragged=False, lens=1, quant=False, fused=False)
    base.update(kw)
    return base


def listed():
    return [
        # one layer of a decode step writes one token of each of 128 sequences into a quantised cache: pure latency
        _case("append_step", "append", batch=128, singles=128, ctx=255, ragged=True, quant=True),
        # prompts of up to 15,000 tokens enter the quantised cache; k and v are slices of the fused qkv projection
        _case("append_prompt", "append", batch=4, new=15000, ragged=True, quant=True, fused=True, lens=5),
        # one sequence's quantised tokens read back, 64-wide heads, pages of 32
        _case("gather_one", "gather", dtype="fp16", hq=16, hkv=4, d=64, page=32, new=1000, quant=True),
        # eight long quantised sequences read back, for a handover to a 16-bit cache
        _case("gather_long", "gather", batch=8, new=16384, ragged=True, quant=True, lens=3),
        # a short prompt's last piece: 37 tokens after 475 that are in the cache
        _case("chunk_short", "chunk", new=37, ctx=475),
        # a 2,048-token piece of a 16,384-token prompt: the largest
        _case("chunk_long", "chunk", new=2048, ctx=14336),
        # a serving step that mixes one 512-token piece with 31 sequences that decode one token each
        _case("chunk_mixed", "chunk", batch=32, new=512, singles=31, ctx=4096, ragged=True, lens=7),
        # ragged pieces with 64-wide heads in fp16, pages of 32
        _case("chunk_ragged_d64", "chunk", dtype="fp16", hq=16, hkv=4, d=64, page=32, batch=8, new=600, ctx=2000,
              ragged=True, lens=2),
        # the decode step of 128 sequences over a quantised cache
        _case("q8_step", "chunk", batch=128, singles=128, ctx=1280, ragged=True, quant=True, lens=4),
        # one sequence decodes over 16,384 quantised tokens: few rows, a long axis
        _case("q8_single_long", "chunk", singles=1, ctx=16383, quant=True),
        # a 1,024-token piece over a quantised cache of 16,384
        _case("q8_chunk", "chunk", new=1024, ctx=15360, quant=True),
        # ragged pieces, eight query heads on one KV head, fp16
        _case("q8_ragged", "chunk", dtype="fp16", hq=8, hkv=1, batch=6, new=300, ctx=5000, ragged=True, quant=True,
              lens=6),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "chunk", "chunk", "chunk"])
    hkv = rng.choice([1, 2, 4, 8])
    case = _case("", op, dtype=rng.choice(["bf16", "fp16"]), hkv=hkv, hq=hkv * rng.choice([1, 2, 4, 8]),
                 d=rng.choice([64, 128, 128]), page=rng.choice([8, 16, 16, 24, 32, 64]), quant=rng.random() < 0.6,
                 ragged=rng.random() < 0.8, lens=rng.randrange(1 << 20))
    del case["name"]
    case["batch"] = _log_uniform(rng, 1, 128)
    if op == "chunk":
        case["new"] = _log_uniform(rng, 1, 2048)
        case["ctx"] = _log_uniform(rng, 1, 16384) - 1
        if rng.random() < 0.4:
            case["singles"] = rng.randrange(case["batch"] + 1)
        # the padded plain form's scores stay within those of the listed cases, and so does the arithmetic
        while case["batch"] * case["hq"] * case["new"] * (case["new"] + case["ctx"]) > 1.5e9 or work(case)["flops"] > 5e11:
            if case["batch"] > 1:
                case["batch"] = max(1, case["batch"] * 3 // 4)
            else:
                case["new"] = max(1, case["new"] * 3 // 4)
                case["ctx"] = case["ctx"] * 3 // 4
        case["singles"] = min(case["singles"], case["batch"])
    else:
        case["new"] = _log_uniform(rng, 1, 16384)
        case["ctx"] = _log_uniform(rng, 1, 1024) - 1
        case["fused"] = op == "append" and rng.random() < 0.5
        while case["batch"] * case["new"] * case["hkv"] * case["d"] > 4e7:
            if case["batch"] > 1:
                case["batch"] = max(1, case["batch"] // 2)
            else:
                case["new"] = case["new"] * 3 // 4
        while case["batch"] * (case["new"] + case["ctx"]) * case["hkv"] * case["d"] > 8e7:
            case["ctx"] = case["ctx"] // 2
    return case


def _lengths(case):
    """(new tokens, tokens in the cache before them) of each sequence: the first has the largest of both."""
    r = random.Random(case["lens"])
    new, ctx = [], []
    for b in range(case["batch"]):
        n = case["new"] if not case["ragged"] or b == 0 else 1 + r.randrange(case["new"])
        c = case["ctx"] if not case["ragged"] or b == 0 else r.randrange(case["ctx"] + 1)
        new.append(1 if b >= case["batch"] - case["singles"] else n)
        ctx.append(c)
    return new, ctx


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


# -------------------------------------------------------------------------------------------------------- the inputs

def _quantise(x):
    """e4m3 codes and the power-of-two scale's exponent byte of each row (last axis) of x, in 32 bits."""
    x = x.float()
    mant, expo = torch.frexp(x.abs().amax(dim=-1))
    expo = torch.where(mant > 0.875, expo - 8, expo - 9)  # 448 = 0.875 * 2^9
    expo = torch.where(mant == 0, torch.full_like(expo, -126), expo.clamp(min=-126))
    codes = (x * torch.ldexp(torch.ones_like(mant), -expo)[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (expo + 127).to(torch.uint8)


def _layout(case):
    """Host part of a paged batch: cu_seqlens, lengths, block table, page count (unused table entries are -1)."""
    new, ctx = _lengths(case)
    total = [n + c for n, c in zip(new, ctx)]
    page = case["page"]
    need = [-(-t // page) for t in total]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    order = list(range(sum(need)))
    random.Random(case["lens"] + 1).shuffle(order)
    width, at, rows = max(need), 0, []
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return cu, total, rows, max(1, sum(need)), max(new), max(total)


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = _dtype(case)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    cu, total, rows, pages, max_new, max_total = _layout(case)
    tokens = cu[-1]
    s = {"case": case, "tokens": tokens, "max_new": max_new, "max_total": max_total,
         "cu": torch.tensor(cu, dtype=torch.int32, device=dev),
         "lens": torch.tensor(total, dtype=torch.int32, device=dev),
         "table": torch.tensor(rows, dtype=torch.int32, device=dev),
         "k_scales": None, "v_scales": None, "plan": None}
    # keys have channels of unequal size, as projected and rotated keys do
    channel = torch.exp(0.5 * torch.randn((hkv, d), generator=gen, device=dev))
    if case["op"] == "append":
        if case["fused"]:
            qkv = torch.randn((tokens, hq + 2 * hkv, d), generator=gen, device=dev, dtype=dt)
            qkv[:, hq:hq + hkv] *= channel.to(dt)
            s["k"], s["v"] = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            s["k"] = torch.randn((tokens, hkv, d), generator=gen, device=dev, dtype=dt) * channel.to(dt)
            s["v"] = torch.randn((tokens, hkv, d), generator=gen, device=dev, dtype=dt)
        store = torch.float8_e4m3fn if case["quant"] else dt
        s["k_cache"] = torch.zeros((pages, page, hkv, d), device=dev, dtype=store)
        s["v_cache"] = torch.zeros((pages, page, hkv, d), device=dev, dtype=store)
        if case["quant"]:
            s["k_scales"] = torch.full((pages, hkv, page), 127, device=dev, dtype=torch.uint8).view(torch.float8_e8m0fnu)
            s["v_scales"] = torch.full((pages, hkv, page), 127, device=dev, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        return s
    kc = torch.randn((pages, page, hkv, d), generator=gen, device=dev, dtype=dt) * channel.to(dt)
    vc = torch.randn((pages, page, hkv, d), generator=gen, device=dev, dtype=dt)
    if case["quant"]:
        kc, ks = _quantise(kc)
        vc, vs = _quantise(vc)
        s["k_scales"] = ks.transpose(1, 2).contiguous().view(torch.float8_e8m0fnu)
        s["v_scales"] = vs.transpose(1, 2).contiguous().view(torch.float8_e8m0fnu)
    s["k_cache"], s["v_cache"] = kc, vc
    if case["op"] == "chunk":
        s["q"] = torch.randn((tokens, hq, d), generator=gen, device=dev, dtype=dt)
        if own:
            # a serving loop makes the step's plan once, after the lengths are final, and every layer uses it
            from mxflashattn_b200 import kvcache_chunk_plan

            s["plan"] = kvcache_chunk_plan(s["cu"], s["lens"], tokens, max_new, q_heads=hq, kv_heads=hkv, causal=True)
    return s


# ---------------------------------------------------------------------------------------------------- the operators

def _slots(s):
    """Row of the cache (page * page size + offset) of each packed token."""
    page = s["case"]["page"]
    tok = torch.arange(s["tokens"], device=s["cu"].device)
    seq = torch.searchsorted(s["cu"][1:].long(), tok, right=True)
    pos = s["lens"].long()[seq] - s["cu"].long()[seq + 1] + tok
    return s["table"].long()[seq, pos // page] * page + pos % page


def _append(s):
    case, slot = s["case"], _slots(s)
    page, hkv, d = case["page"], case["hkv"], case["d"]
    for x, cache, scales in ((s["k"], s["k_cache"], s["k_scales"]), (s["v"], s["v_cache"], s["v_scales"])):
        if scales is None:
            cache.view(-1, hkv, d)[slot] = x
        else:
            codes, expo = _quantise(x)
            cache.view(torch.uint8).view(-1, hkv, d)[slot] = codes.view(torch.uint8)
            scales.view(torch.uint8)[slot // page, :, slot % page] = expo
    return _appended(s)


def _appended(s):
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales") if s[n] is not None}


def _values(cache, scales):
    """The cache's values in 32 bits."""
    return cache.float() if scales is None else cache.float() * scales.float().transpose(1, 2)[..., None]


def _gather(s):
    case, slot = s["case"], _slots(s)
    flat = lambda cache, scales: _values(cache, scales).view(-1, case["hkv"], case["d"])[slot].to(_dtype(case))  # noqa: E731
    return {"k": flat(s["k_cache"], s["k_scales"]), "v": flat(s["v_cache"], s["v_scales"])}


def _chunk(s):
    """Attention over padded sequences: scores [batch, KV heads, heads of each, new tokens, cached tokens]."""
    case = s["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    dev = s["cu"].device
    cu, lens = s["cu"].long(), s["lens"].long()
    new = cu[1:] - cu[:-1]
    pos = torch.arange(s["max_total"], device=dev)
    slot = s["table"].long().clamp(min=0)[:, pos // page] * page + pos % page
    k = _values(s["k_cache"], s["k_scales"]).view(-1, hkv, d)[slot]
    v = _values(s["v_cache"], s["v_scales"]).view(-1, hkv, d)[slot]
    i = torch.arange(s["max_new"], device=dev)
    q = s["q"].float()[(cu[:-1, None] + i).clamp(max=s["tokens"] - 1)]
    q = q.view(-1, s["max_new"], hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    scores = (q.flatten(2, 3) @ k.permute(0, 2, 3, 1)).unflatten(2, (hq // hkv, s["max_new"])) / math.sqrt(d)
    seen = pos <= (lens - new)[:, None, None] + i[:, None]
    scores = scores.masked_fill(~(seen & (pos < lens[:, None, None]))[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = ((p / total).flatten(2, 3) @ v.permute(0, 2, 1, 3)).unflatten(2, (hq // hkv, s["max_new"]))
    lse = top + torch.log(total)
    tok = torch.arange(s["tokens"], device=dev)
    seq = torch.searchsorted(cu[1:], tok, right=True)
    at = tok - cu[seq]
    out = out.permute(0, 3, 1, 2, 4)[seq, at].reshape(s["tokens"], hq, d)
    lse = lse.permute(0, 3, 1, 2, 4)[seq, at].reshape(s["tokens"], hq)
    return {"out": out.to(_dtype(case)), "lse": lse}


def run(s):
    op = s["case"]["op"]
    if not own:
        return _append(s) if op == "append" else _gather(s) if op == "gather" else _chunk(s)
    import mxflashattn_b200 as fa

    if op == "append":
        fa.kvcache_append_varlen(s["k"], s["v"], s["k_cache"], s["v_cache"], s["cu"], s["lens"], s["table"],
                                 k_scales=s["k_scales"], v_scales=s["v_scales"])
        return _appended(s)
    if op == "gather":
        k, v = fa.kvcache_gather_varlen(s["k_cache"], s["v_cache"], s["cu"], s["lens"], s["table"], s["tokens"],
                                        k_scales=s["k_scales"], v_scales=s["v_scales"], dtype=_dtype(s["case"]))
        return {"k": k, "v": v}
    out, lse = fa.flash_attn_varlen_with_kvcache(
        s["q"], s["k_cache"], s["v_cache"], s["cu"], s["lens"], s["table"], s["max_new"], s["max_total"], causal=True,
        k_scales=s["k_scales"], v_scales=s["v_scales"], plan=s["plan"], return_softmax_lse=True)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------------------------ work and definition

def work(case):
    new, ctx = _lengths(case)
    tokens = sum(new)
    row = case["hkv"] * case["d"]
    # one cached token's K and V of all heads, with the scales' bytes
    cached = 2 * row + 2 * case["hkv"] if case["quant"] else 4 * row
    tables = 4 * (2 * case["batch"] + 1 + sum(-(-(n + c) // case["page"]) for n, c in zip(new, ctx)))
    if case["op"] != "chunk":
        # 16-bit rows on one side, the cache's on the other; a maximum and a product for each quantised value
        return {"bytes": tokens * (4 * row + cached) + tables, "flops": 4 * tokens * row if case["quant"] else 0}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    return {"bytes": sum(n + c for n, c in zip(new, ctx)) * cached + tokens * case["hq"] * (4 * case["d"] + 4) + tables,
            "flops": 4 * case["hq"] * case["d"] * pairs}


def _e4m3(y):
    """Values of y rounded to e4m3 (4 significant bits, exponents from -6, largest 448), nearest, ties to even."""
    mag = y.abs()
    expo = torch.floor(torch.log2(mag.clamp(min=2.0 ** -6)))
    step = torch.exp2(expo - 3)
    return torch.copysign(torch.clamp(torch.round(mag / step) * step, max=448.0), y)


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    cu, total, rows, pages, _, _ = _layout(case)
    places = []
    for b in range(case["batch"]):
        first = total[b] - (cu[b + 1] - cu[b]) if case["op"] != "chunk" else 0
        places.append([rows[b][t // page] * page + t % page for t in range(first, total[b])])
    if case["op"] == "append":
        flat = torch.tensor([x for p in places for x in p], device="cuda")
        got = {}
        for n in ("k", "v"):
            x = s[n].double()
            cache = torch.zeros((pages * page, hkv, d), dtype=torch.float64, device="cuda")
            if case["quant"]:
                top = x.abs().amax(dim=-1).clamp(min=2.0 ** -118)
                scale = torch.exp2(torch.round(torch.log2(top)) - 10.0)  # too small by 2 to 8 times
                for _ in range(4):
                    scale = torch.where(top > 448.0 * scale, 2.0 * scale, scale)
                scales = torch.ones((pages * page, hkv), dtype=torch.float64, device="cuda")
                scales[flat] = scale
                got[n + "_scales"] = scales.view(pages, page, hkv).transpose(1, 2).contiguous()
                x = _e4m3(x / scale[..., None])
            cache[flat] = x
            got[n + "_cache"] = cache.view(pages, page, hkv, d)
        return got
    values = []
    for n in ("k", "v"):
        x = s[n + "_cache"].double()
        if case["quant"]:
            x = x * s[n + "_scales"].double().transpose(1, 2)[..., None]
        values.append(x.view(pages * page, hkv, d))
    if case["op"] == "gather":
        flat = torch.tensor([x for p in places for x in p], device="cuda")
        return {"k": values[0][flat], "v": values[1][flat]}
    out = torch.zeros((cu[-1], hq, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((cu[-1], hq), dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, at = cu[b + 1] - cu[b], torch.tensor(places[b], device="cuda")
        seen = torch.arange(total[b], device="cuda") <= total[b] - n + torch.arange(n, device="cuda")[:, None]
        for h in range(hq):
            k, v = values[0][at, h * hkv // hq], values[1][at, h * hkv // hq]
            score = torch.where(seen, s["q"][cu[b]:cu[b + 1], h].double() @ k.T / d ** 0.5, -math.inf)
            lse[cu[b]:cu[b + 1], h] = torch.logsumexp(score, dim=1)
            out[cu[b]:cu[b + 1], h] = torch.softmax(score, dim=1) @ v
    return {"out": out, "lse": lse}
