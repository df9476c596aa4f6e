"""Cases, inputs and plain forms of the paged key-value cache operators.

Three operators share one cache, whose pages hold [kv_heads, page_size, head_dim] keys and values each:

  append   rotary positions on the new queries and keys, keys and values written into their pages
  decode   attention of one new token per sequence over its pages, optionally adding every cached
           token's share of the attention to a running weight
  evict    the tokens of least accumulated weight leave the cache, the survivors behind the budget
           move into their places

`listed` and `draw` give the cases, `prepare` their inputs, `run` one pass, `work` what a pass cannot
do without, `exact` the outputs in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0


def append_case(tokens, rows, heads, kv_heads, head_dim, rot, layout, scaling, page, dtype, cache, start):
    """`tokens` new tokens, shared out over `rows` sequences that hold about `start` tokens already."""
    return {"op": "append", "tokens": tokens, "rows": rows, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "rot": rot, "layout": layout, "scaling": scaling, "page": page, "dtype": dtype, "cache": cache, "start": start}


def decode_case(rows, low, high, heads, kv_heads, head_dim, page, dtype, cache, window=0, sinks=False, quiet=False,
                track=False):
    """`rows` sequences of `low` to `high` cached tokens."""
    return {"op": "decode", "rows": rows, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "cache": cache, "window": window, "sinks": sinks,
            "quiet": quiet, "track": track}


def evict_case(rows, low, high, budget, recent, kv_heads, head_dim, page, cache, aged):
    """`rows` sequences of `low` to `high` cached tokens, of which `budget` stay; `aged`: earlier evictions have
    left the cache out of order."""
    return {"op": "evict", "rows": rows, "low": low, "high": high, "budget": budget, "recent": recent, "sink": 4,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "cache": cache, "aged": aged}


def listed():
    return [
        # the next token of one conversation, with GPT-OSS heads and its YaRN-scaled positions: latency
        dict(append_case(1, 1, 64, 8, 64, 64, "half", "yarn", 16, "bf16", "bf16", 4000), name="append one token"),
        # four prompts enter the cache together
        dict(append_case(8192, 4, 64, 8, 64, 64, "half", "yarn", 16, "bf16", "bf16", 0), name="append prompts"),
        # chunks of prompts into an 8-bit cache, interleaved pairs on half of a wider head, 32-bit activations
        dict(append_case(1023, 5, 32, 8, 128, 64, "interleaved", "ntk", 32, "f32", "e4m3", 700),
             name="append partial 8-bit"),
        # one conversation in a sliding-window layer: latency
        dict(decode_case(1, 4000, 4000, 64, 8, 64, 16, "bf16", "bf16", window=128, sinks=True), name="decode window"),
        # a serving batch at mixed lengths, some of its places idle
        dict(decode_case(32, 0, 4096, 64, 8, 64, 16, "bf16", "bf16", sinks=True), name="decode ragged batch"),
        # a full batch at long lengths: the largest read
        dict(decode_case(64, 8192, 8192, 64, 8, 64, 64, "bf16", "bf16", sinks=True), name="decode full batch"),
        # long contexts in an 8-bit cache, wider heads, groups of four
        dict(decode_case(8, 2048, 16383, 32, 8, 128, 32, "bf16", "e4m3"), name="decode 8-bit"),
        # a batch whose cache will be thinned: the weights are kept beside the attention
        dict(decode_case(16, 1000, 4096, 64, 8, 64, 16, "bf16", "bf16", sinks=True, track=True), name="decode tracked"),
        # one very long sequence in 32 bits, odd page and length, quiet softmax
        dict(decode_case(1, 50001, 50001, 16, 2, 80, 24, "f32", "f32", quiet=True), name="decode long f32"),
        # every step of a conversation at its budget: one token in, one token out
        dict(evict_case(1, 2049, 2049, 2048, 256, 8, 64, 16, "bf16", True), name="evict one token"),
        # prompts thinned to the budget after they were read
        dict(evict_case(16, 1000, 8192, 2048, 256, 8, 64, 16, "bf16", False), name="evict after prompts"),
        # two very long prompts in an 8-bit cache
        dict(evict_case(2, 60001, 65536, 16384, 1024, 8, 128, 32, "e4m3", False), name="evict long 8-bit"),
    ]


def between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "evict"])
    cache = rng.choice(["bf16", "bf16", "e4m3", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    row_bytes = 2 * kv_heads * head_dim * BYTES[cache]
    most = 64 * 8192 * 2 * 8 * 64 * 2
    if op == "append":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        tokens = between(rng, 1, min(8192, 8192 * 80 * 64 // ((heads + 2 * kv_heads) * head_dim)))
        rows = tokens if rng.random() < 0.3 and tokens <= 256 else between(rng, 1, min(tokens, 16))
        rot = rng.choice([head_dim, head_dim, head_dim // 2, 32])
        return append_case(tokens, rows, heads, kv_heads, head_dim, rot, rng.choice(["half", "interleaved"]),
                           rng.choice(["none", "linear", "ntk", "yarn"]), page, rng.choice(["bf16", "f32"]), cache,
                           between(rng, 1, 30000) if rows == tokens else rng.choice([0, between(rng, 1, 3000)]))
    if op == "decode":
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8, 8, 16])
        rows = between(rng, 1, 64)
        high = between(rng, 1, max(1, min(131072, most // (rows * row_bytes) // 2)))
        track = rng.random() < 0.3
        return decode_case(rows, rng.choice([0, high // 4, high]), high, heads, kv_heads, head_dim, page,
                           rng.choice(["bf16", "bf16", "f32"]), cache,
                           window=0 if track else rng.choice([0, 0, between(rng, 1, 4096)]), sinks=rng.random() < 0.5,
                           quiet=rng.random() < 0.2, track=track)
    rows = between(rng, 1, 32)
    high = between(rng, 16, max(16, min(65536, most // (rows * row_bytes) // 4)))
    budget = max(8, rng.choice([high - 1, high // 2, high // 4]))
    return evict_case(rows, rng.choice([high, high // 2, 1]), high, budget, max(1, budget // rng.choice([2, 4, 8])) - 1
                      if budget > 16 else 1, kv_heads, head_dim, page, cache, rng.random() < 0.5)


def spread(low, high, n):
    """n whole numbers evenly over [low, high], its ends among them: the same ones for every seed."""
    return [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def frequencies(case):
    """The inverse frequencies of the rotated pairs in 64 bits, and the factor on cosine and sine: base 150000 and,
    where scaled, 32 times a first context of 4096 tokens."""
    half, base, factor, first = case["rot"] // 2, 150000.0, 32.0, 4096.0
    if case["scaling"] == "ntk" and half > 1:
        base *= factor ** (half / (half - 1))
    inv = base ** (-np.arange(half) / half)
    if case["scaling"] == "linear":
        inv = inv / factor
    if case["scaling"] == "yarn":
        low = half * math.log(first / (32.0 * 2 * math.pi)) / math.log(base)
        high = half * math.log(first / (1.0 * 2 * math.pi)) / math.log(base)
        keep = 1 - np.clip((np.arange(half) - low) / max(high - low, 1e-3), 0, 1)
        return inv / factor * (1 - keep) + inv * keep, 0.1 * math.log(factor) + 1
    return inv, 1.0


def pools(case, pages, gen):
    """Keys and values of the whole pool, and the 8-bit cache's scales by head."""
    shape, dt = (pages, case["kv_heads"], case["page"], case["head_dim"]), DTYPES[case["cache"]]

    def pool():
        x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16 if dt == torch.bfloat16 else torch.float32)
        return (x * 90).clamp_(-E4M3_MAX, E4M3_MAX).to(dt) if case["cache"] == "e4m3" else x.to(dt)

    k, v, scales = pool(), pool(), (None, None)
    if case["cache"] == "e4m3":
        scales = tuple((torch.rand(case["kv_heads"], device="cuda", generator=gen) + 0.5) / 90 for _ in range(2))
    return k, v, scales


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    s = {"case": dict(case)}
    H, hd, page, rows = case["kv_heads"], case["head_dim"], case["page"], case["rows"]
    if case["op"] == "append":
        new = np.diff([case["tokens"] * i // rows for i in range(rows + 1)])
        old = np.array([case["start"] * (8 + i % 3) // 10 for i in range(rows)])
        per_row = max(1, -(-int((old + new).max()) // page))
        old_pages = (old // page).astype(np.int64)
    else:
        lens = np.array(spread(case["low"], case["high"], rows))
        host.shuffle(lens)
        per_row = max(1, -(-case["high"] // page))
        old_pages = np.zeros(rows, np.int64)
    if case["op"] == "append":
        # only the pages that the new tokens touch are in the pool; those before them are other sequences' business
        used = [np.arange(old_pages[i], -(-(old[i] + new[i]) // page)) for i in range(rows)]
        n_pages = sum(len(u) for u in used) + 3
        order, tables, at = host.permutation(n_pages), np.zeros((rows, per_row), np.int32), 0
        for i, u in enumerate(used):
            tables[i, u] = order[at:at + len(u)]
            at += len(u)
    else:
        n_pages = rows * per_row + 3
        tables = host.permutation(n_pages)[:rows * per_row].reshape(rows, per_row).astype(np.int32)
    s["tables"] = torch.from_numpy(tables).cuda()
    s["k"], s["v"], (s["k_scale"], s["v_scale"]) = pools(case, n_pages, gen)
    if case["op"] == "append":
        # the tokens as they leave one projection of queries, keys and values together
        T, nH = case["tokens"], case["heads"]
        qkv = torch.randn(T, (nH + 2 * H) * hd, device="cuda", generator=gen).to(DTYPES[case["dtype"]])
        s["q"], s["k_new"], s["v_new"] = (t.unflatten(1, (-1, hd)) for t in qkv.split([nH * hd, H * hd, H * hd], 1))
        index = np.concatenate([old[i] + np.arange(new[i]) for i in range(rows)])
        s["index"] = torch.from_numpy(index.astype(np.int32)).cuda()
        s["rows"] = None if rows == T else torch.from_numpy(np.repeat(np.arange(rows), new).astype(np.int32)).cuda()
        inv, factor = frequencies(case)
        angle = torch.arange(int(index.max()) + 1, device="cuda", dtype=torch.float64)[:, None] * torch.from_numpy(inv).cuda()
        s["cos"], s["sin"] = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    else:
        s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    if case["op"] == "decode":
        q = torch.randn(rows, case["heads"], hd, device="cuda", generator=gen) * 2
        s["q"] = q.to(DTYPES[case["dtype"]])
        s["sinks"] = torch.randn(case["heads"], device="cuda", generator=gen) if case["sinks"] else None
    if case["op"] == "evict" or case.get("track"):
        # weights as attention leaves them: most tokens have little
        s["weight"] = torch.rand(n_pages, H, page, device="cuda", generator=gen).log().neg().square()
        s["position"] = torch.zeros(n_pages, H, page, device="cuda", dtype=torch.int32)
    if case["op"] == "evict":
        width = per_row * page
        at = torch.arange(width, device="cuda").expand(rows, H, width)
        if case["aged"]:
            # positions out of order, with gaps where earlier tokens were
            noise = torch.rand(rows, H, width, device="cuda", generator=gen)
            noise = torch.where(at < s["lens"][:, None, None], noise, 2.0)
            at = noise.argsort(-1).argsort(-1) * 3 + 2
        s["position"][s["tables"].long()] = at.reshape(rows, H, per_row, page).permute(0, 2, 1, 3).int()
        s["seen"] = s["lens"] * (3 if case["aged"] else 1)
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "burn-extended_b200"))
        from mxmoe.paged import PagedKvCache, RotaryTable
        s["paged"] = PagedKvCache.over(s["k"], s["v"], n_heads=case.get("heads", H), weight=s.get("weight"),
                                       position=s.get("position"), k_scale=s["k_scale"], v_scale=s["v_scale"])
        if case["op"] == "append":
            s["rotary"] = RotaryTable(s["cos"], s["sin"], interleaved=case["layout"] == "interleaved")
    return s


def run(s):
    return {"append": run_append, "decode": run_decode, "evict": run_evict}[s["case"]["op"]](s)


def run_append(s):
    if own:
        q = s["paged"].append(s["q"], s["k_new"], s["v_new"], s["tables"], s["index"], s["rotary"], rows=s["rows"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    c, index = s["case"], s["index"].long()
    cos, sin = s["cos"][index][:, None], s["sin"][index][:, None]
    rows = torch.arange(index.numel(), device="cuda") if s["rows"] is None else s["rows"].long()
    pages = s["tables"][rows, index // c["page"]].long()
    slots = index % c["page"]
    write(s["k"], pages, slots, rotated(s["k_new"].float(), cos, sin, c), s["k_scale"])
    write(s["v"], pages, slots, s["v_new"].float(), s["v_scale"])
    return {"q": rotated(s["q"].float(), cos, sin, c).to(s["q"].dtype), "k": s["k"], "v": s["v"]}


def rotated(x, cos, sin, c):
    r, h = c["rot"], c["rot"] // 2
    a, b = (x[..., :h], x[..., h:r]) if c["layout"] == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, w], -1) if c["layout"] == "half" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def write(pool, pages, slots, x, scale):
    if scale is not None:
        x = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(pool.dtype).view(torch.uint8)
        pool = pool.view(torch.uint8)
    pool[pages, :, slots] = x.to(pool.dtype)


def gathered(pool, tables, scale=None):
    """The pages of every row side by side, in 32 bits: [rows, kv_heads, length, head_dim]."""
    t = tables.long()
    x = pool.view(torch.uint8)[t].view(pool.dtype) if pool.dtype == torch.float8_e4m3fn else pool[t]
    x = x.float().permute(0, 2, 1, 3, 4).flatten(2, 3)
    return x if scale is None else x * scale[:, None, None]


def run_decode(s):
    c = s["case"]
    if own:
        out = s["paged"].decode(s["q"], s["tables"], s["lens"], window=c["window"], sinks=s["sinks"], quiet=c["quiet"],
                                track=c["track"])
        return {"out": out, "weight": s["weight"]} if c["track"] else {"out": out}
    B, H, hd, G = c["rows"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    k, v = gathered(s["k"], s["tables"], s["k_scale"]), gathered(s["v"], s["tables"], s["v_scale"])
    score = s["q"].float().view(B, H, G, hd) @ k.transpose(-1, -2) / math.sqrt(hd)
    at, lens = torch.arange(k.shape[2], device="cuda"), s["lens"][:, None].long()
    seen = (at < lens) & (at >= (lens - c["window"] if c["window"] else lens * 0))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    sink = None if s["sinks"] is None else s["sinks"].view(1, H, G, 1)
    top = top if sink is None else torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    total = total if sink is None else total + (sink - top).exp()
    total = total + (-top).exp() if c["quiet"] else total
    p = torch.where(total > 0, p / total, 0.0)
    out = (p @ v).view(B, c["heads"], hd).to(s["q"].dtype)
    if not c["track"]:
        return {"out": out}
    share = p.sum(2).unflatten(2, (-1, c["page"])).permute(0, 2, 1, 3)
    t = s["tables"].long()
    s["weight"][t] = s["weight"][t] + share
    return {"out": out, "weight": s["weight"]}


def run_evict(s):
    c = s["case"]
    if own:
        lens = s["paged"].evict(s["tables"], s["lens"], s["seen"], budget=c["budget"], sink=c["sink"], recent=c["recent"])
        return {"k": s["k"], "v": s["v"], "weight": s["weight"], "position": s["position"], "lens": lens}
    t, budget = s["tables"].long(), c["budget"]

    def flat(x):
        return x[t].transpose(1, 2).flatten(2)

    weight, position = flat(s["weight"]), flat(s["position"])
    at = torch.arange(weight.shape[-1], device="cuda")
    lens, seen = s["lens"][:, None, None].long(), s["seen"][:, None, None].long()
    safe = (position < c["sink"]) | (position >= seen - c["recent"])
    key = torch.where(weight.isnan(), math.inf, weight).double()
    key = torch.where(safe, torch.finfo(torch.float64).max, key)
    key = torch.where(at < lens, key, math.inf)
    rank = key.argsort(dim=-1, stable=True).argsort(-1)
    gone = rank < (lens - budget).clamp(min=0)
    over = lens > budget
    hole = gone & (at < budget)
    mover = ~gone & (at >= budget) & (at < lens) & over
    # hole i takes survivor i; there are as many of the one as of the other, and past them a token stays where it is
    last = at.numel()
    most = min(max(1, last - budget), budget)
    to = torch.where(hole, at, last).sort(-1).values[..., :most]
    by = torch.where(mover, at, last).sort(-1).values[..., :most]
    stay = (lens - 1).clamp(min=0).expand_as(to)
    to, by = torch.where(to == last, stay, to), torch.where(to == last, stay, by)
    head = torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    page_to, page_by = (t.gather(1, (x // c["page"]).flatten(1)).view_as(x) for x in (to, by))
    for x in (s["k"], s["v"], s["weight"], s["position"]):
        y = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
        y[page_to, head, to % c["page"]] = y[page_by, head, by % c["page"]]
    return {"k": s["k"], "v": s["v"], "weight": s["weight"], "position": s["position"],
            "lens": s["lens"].clamp(max=budget)}


def work(case):
    H, hd, es = case["kv_heads"], case["head_dim"], BYTES[case["cache"]]
    if case["op"] == "append":
        T, width = case["tokens"], BYTES[case["dtype"]]
        moved = T * hd * ((2 * case["heads"] + 2 * H) * width + 2 * H * es)
        return {"bytes": moved + T * (case["rot"] * 4 + 8), "flops": 3 * T * (case["heads"] + H) * case["rot"]}
    lens = spread(case["low"], case["high"], case["rows"])
    if case["op"] == "decode":
        read = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        b = 2 * read * H * hd * es + 2 * case["rows"] * case["heads"] * hd * BYTES[case["dtype"]]
        b += read // case["page"] * 4 + (8 * read * H if case["track"] else 0)
        return {"bytes": b, "flops": 4 * read * case["heads"] * hd}
    b = 0
    for n in lens:
        if n > case["budget"]:
            holes = (n - case["budget"]) * case["budget"] / n  # where weight does not go by place
            b += H * (8 * n + holes * 2 * (2 * hd * es + 8)) + n // case["page"] * 4
    return {"bytes": max(b, 8 * case["rows"]), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": exact_append, "decode": exact_decode, "evict": exact_evict}[case["op"]](s)


def exact_append(s):
    """Pairs as complex numbers, turned by e^(i position frequency)."""
    c, T = s["case"], s["index"].numel()
    inv, factor = frequencies(c)
    angle = s["index"].double()[:, None, None] * torch.from_numpy(inv).cuda()
    turn = torch.polar(torch.full_like(angle, factor), angle)

    def turned(x):
        x, r = x.double(), c["rot"]
        pairs = x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2) if c["layout"] == "half" else x[..., :r].unflatten(-1, (-1, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(-1, -2) if c["layout"] == "half" else z
        return torch.cat([z.flatten(-2), x[..., r:]], -1)

    out = {"q": turned(s["q"])}
    row = np.arange(T) if s["rows"] is None else s["rows"].cpu().numpy()
    index, tables = s["index"].cpu().numpy(), s["tables"].cpu().numpy()
    place = torch.from_numpy(tables[row, index // c["page"]].astype(np.int64) * c["page"] + index % c["page"]).cuda()
    for name, new, scale in (("k", turned(s["k_new"]), s["k_scale"]), ("v", s["v_new"].double(), s["v_scale"])):
        if scale is not None:
            new = (new / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        pool = s[name].double().transpose(1, 2).contiguous()
        pool.flatten(0, 1)[place] = new
        out[name] = pool.transpose(1, 2).contiguous()
    return out


def exact_decode(s):
    """Row by row, with the sink and the quiet one as columns of their own."""
    c = s["case"]
    H, hd, G = c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(c["rows"], H, G, hd, device="cuda", dtype=torch.float64)
    weight = s["weight"].double() if c["track"] else None
    for i, n in enumerate(s["lens"].tolist()):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        t = s["tables"][i, : -(-n // c["page"])].long()

        def cached(pool, scale):
            x = pool.view(torch.uint8)[t].view(pool.dtype) if scale is not None else pool[t]
            x = x.double().transpose(0, 1).flatten(1, 2)[:, first:n]
            return x if scale is None else x * scale.double()[:, None, None]

        k, v = cached(s["k"], s["k_scale"]), cached(s["v"], s["v_scale"])
        more = [] if s["sinks"] is None else [s["sinks"].double().view(H, G, 1)]
        more += [torch.zeros(H, G, 1, device="cuda", dtype=torch.float64)] if c["quiet"] else []
        score = torch.einsum("hgd,hnd->hgn", s["q"][i].double().view(H, G, hd), k) / math.sqrt(hd)
        p = torch.softmax(torch.cat([score] + more, -1), -1)[..., : n - first]
        out[i] = torch.einsum("hgn,hnd->hgd", p, v)
        if c["track"]:
            at = torch.arange(first, n, device="cuda")
            weight[t[at // c["page"]], :, at % c["page"]] += p.sum(1).T
    out = out.view(c["rows"], c["heads"], hd)
    return {"out": out, "weight": weight} if c["track"] else {"out": out}


def exact_evict(s):
    """Head by head on the host: the victims, then the survivors behind the budget into the victims' places."""
    c = s["case"]
    tables, lens, seen = (s[n].cpu().numpy().astype(np.int64) for n in ("tables", "lens", "seen"))
    weight, position = s["weight"].cpu().numpy(), s["position"].cpu().numpy()
    to, by = [], []
    for i, n in enumerate(lens.tolist()):
        if n <= c["budget"]:
            continue
        at = np.arange(n)
        page, slot = tables[i, at // c["page"]], at % c["page"]
        for h in range(c["kv_heads"]):
            w, p = weight[page, h, slot], position[page, h, slot]
            safe = (p < c["sink"]) | (p >= seen[i] - c["recent"])
            w = np.where(safe, 0, np.where(np.isnan(w), np.inf, w))
            victims = np.lexsort((at, w, safe))[: n - c["budget"]]
            gone = np.zeros(n, bool)
            gone[victims] = True
            holes, movers = at[gone & (at < c["budget"])], at[~gone & (at >= c["budget"])]
            to.append(np.stack([page[holes], np.full(len(holes), h), slot[holes]]))
            by.append(np.stack([page[movers], np.full(len(movers), h), slot[movers]]))
    out = {"lens": s["lens"].clamp(max=c["budget"]), "position": s["position"]}
    for name in ("k", "v", "weight"):
        out[name] = s[name].double() if name == "weight" or s[name].numel() <= 1 << 27 else s[name].float()
    if to:
        to, by = (torch.from_numpy(np.concatenate(x, 1)).cuda() for x in (to, by))
        for x in out.values():
            if x.dim() > 1:
                x[to[0], to[1], to[2]] = x[by[0], by[1], by[2]]
    return out
