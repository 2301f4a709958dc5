"""8-bit serving operators: what they are timed on, their plain forms and their values in 64 bits.

Four operators of a decoder layer served in 8 bits, one per "kind":

  linear   int8 linear layer: rows of activations quantised to int8 with one
           scale per token, times an int8 weight [N,K] with one scale per
           output channel
  attend   grouped-query attention over a paged cache held in e4m3 with one
           scale per page and head, from one query token per sequence to
           long chunks of prompts behind a cached prefix
  append   new keys and values quantised into such a cache
  copy     pages of such a cache copied (a forked sequence's last page, the
           moves of a compaction)

The cache: k [pages, n_kv, page, d] and v [pages, n_kv, d, page] in e4m3 (a
page of v is held transposed, so that a lane reads consecutive keys of one
channel), k_scale and v_scale [pages, n_kv] in fp32, powers of two.  Sequence
b's token t lies on page page_table[b, t // page]; kv_lens counts the tokens
with the new ones, which are its last.
"""
import functools
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@functools.lru_cache(None)
def _ops():
    import importlib

    return importlib.import_module("cuda-oxide-bench_amd").load_ops()


def listed():
    return [
        # one token of one user through a projection: the smallest call, all weight reads and latency
        {"name": "linear_1x7168x4096", "kind": "linear", "m": 1, "n": 7168, "k": 4096, "dtype": "bf16"},
        # a decode batch of 64
        {"name": "linear_64x4096x7168", "kind": "linear", "m": 64, "n": 4096, "k": 7168, "dtype": "bf16"},
        # a prompt whose length, width and depth are all off the tiles
        {"name": "linear_1003x2040x2064_f16", "kind": "linear", "m": 1003, "n": 2040, "k": 2064, "dtype": "f16"},
        # the largest product
        {"name": "linear_8192", "kind": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16"},
        # one user's next token behind a short context
        {"name": "attend_b1_t1001", "kind": "attend", "batch": 1, "ctx": 1001, "chunk": 1, "heads": 32, "kv_heads": 8,
         "d": 128, "page": 64, "dtype": "bf16"},
        # a decode batch with contexts of very different lengths up to 8192
        {"name": "attend_b64_t8192", "kind": "attend", "batch": 64, "ctx": 8192, "chunk": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # every query head its own keys, the small head dim, the smallest pages, an odd batch
        {"name": "attend_b33_t2000_d64_f16", "kind": "attend", "batch": 33, "ctx": 2000, "chunk": 1, "heads": 16,
         "kv_heads": 16, "d": 64, "page": 16, "dtype": "f16"},
        # three prompts' chunks behind cached prefixes
        {"name": "attend_b3_t4096_q2048", "kind": "attend", "batch": 3, "ctx": 4096, "chunk": 2048, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # the decode batch's new tokens into the cache
        {"name": "append_b64", "kind": "append", "batch": 64, "ctx": 512, "chunk": 1, "kv_heads": 8, "d": 128,
         "page": 64, "dtype": "bf16"},
        # chunks of prompts that begin and end inside pages
        {"name": "append_b4_q4096_f16", "kind": "append", "batch": 4, "ctx": 5000, "chunk": 4096, "kv_heads": 8,
         "d": 128, "page": 32, "dtype": "f16"},
        # the last pages of a few forked sequences
        {"name": "copy_12", "kind": "copy", "pool": 512, "moved": 12, "kv_heads": 8, "d": 128, "page": 64},
        # a compaction of a large pool
        {"name": "copy_2500", "kind": "copy", "pool": 6000, "moved": 2500, "kv_heads": 8, "d": 128, "page": 64},
    ]


def _log(rng, lo, hi, step=1):
    """A size between lo and hi, spread over its logarithm, a multiple of step."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(-(-lo // step) * step, x // step * step)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "attend", "attend", "attend", "append", "copy"])
    if kind == "linear":
        return {"kind": kind, "m": _log(rng, 1, 8192), "n": _log(rng, 256, 8192), "k": _log(rng, 256, 8192, 16),
                "dtype": rng.choice(["bf16", "f16"])}
    kv_heads, d, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if kind == "copy":
        pool = _log(rng, 64, max(64, 6000 * 8 * 64 * 128 // (kv_heads * d * page) // 4))
        return {"kind": kind, "pool": pool, "moved": _log(rng, 1, pool * 2 // 5), "kv_heads": kv_heads, "d": d,
                "page": page}
    dtype = rng.choice(["bf16", "f16"])
    if kind == "append":
        batch = _log(rng, 1, 64)
        ctx = _log(rng, 64, 20000 // batch)
        return {"kind": kind, "batch": batch, "ctx": ctx, "chunk": rng.choice([1, _log(rng, 1, ctx)]),
                "kv_heads": kv_heads, "d": d, "page": page, "dtype": dtype}
    group = rng.choice([1, 2, 4, 7, 8, 16])
    chunk = rng.choice(["one", "few", "long"])
    if chunk == "long":
        batch = _log(rng, 1, 4)
        heads = min(kv_heads * group, 32)
        kv_heads = heads // min(group, heads)
        heads = kv_heads * min(group, heads)
        ctx = _log(rng, 64, 4096)
        return {"kind": kind, "batch": batch, "ctx": ctx, "chunk": _log(rng, 16, min(2048, ctx)), "heads": heads,
                "kv_heads": kv_heads, "d": d, "page": page, "dtype": dtype}
    batch = _log(rng, 1, 64)
    most = 8192 * 64 * 8 * 128 // (batch * kv_heads * d)  # the largest listed cache
    ctx = _log(rng, 64, min(32768, most))
    return {"kind": kind, "batch": batch, "ctx": ctx, "chunk": 1 if chunk == "one" else rng.randint(2, 8),
            "heads": kv_heads * group, "kv_heads": kv_heads, "d": d, "page": page, "dtype": dtype}


def _lens(case):
    """(tokens in the cache with the new ones, new ones) of each sequence: the first is the longest."""
    rng = random.Random(case["batch"] * 1000003 + case["ctx"])
    lens = [case["ctx"]] + [rng.randint(max(1, case["ctx"] // 4), case["ctx"]) for _ in range(case["batch"] - 1)]
    chunk = case["chunk"]
    if chunk <= 8:
        return lens, [min(chunk, n) for n in lens]
    return lens, [min(n, chunk if b == 0 else rng.randint(max(1, chunk // 4), chunk)) for b, n in enumerate(lens)]


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    h, d, p = case["kv_heads"], case["d"], case["page"]
    if case["kind"] == "copy":
        return {"bytes": case["moved"] * (2 * (2 * h * p * d + 8 * h) + 8), "flops": 0}
    lens, news = _lens(case)
    if case["kind"] == "append":
        pages = sum((n - 1) // p - (n - new) // p + 1 for n, new in zip(lens, news))
        return {"bytes": 2 * sum(news) * h * d * 3 + pages * (8 * h + 4), "flops": 0}
    pages = sum(-(-n // p) for n in lens)
    pairs = sum(new * (n - new) + new * (new + 1) // 2 for n, new in zip(lens, news))
    return {"bytes": 2 * sum(lens) * h * d + pages * (8 * h + 4) + 4 * sum(news) * case["heads"] * d,
            "flops": 4 * pairs * case["heads"] * d}


def _two_to(x):
    """The smallest power of two s with x <= 448 s, at least 2^-32."""
    m, e = torch.frexp(x.double() / 448)
    return torch.ldexp(torch.ones_like(m), e - (m == 0.5).int()).clamp_min(2.0 ** -32).float()


def _pages_of(g, n, rows, cols, heads):
    """Codes and scales of n whole pages of a cache with N(0,1) values, each head and page of a magnitude of its own."""
    code = torch.empty((n, heads, rows, cols), dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty((n, heads), dtype=torch.float32, device="cuda")
    for i in range(0, n, 512):
        x = torch.randn((min(512, n - i), heads, rows, cols), generator=g, device="cuda")
        x *= torch.exp2(torch.rand((x.shape[0], heads, 1, 1), generator=g, device="cuda") * 3 - 2)
        s = _two_to(x.abs().amax((2, 3)))
        code[i:i + 512], scale[i:i + 512] = (x / s[..., None, None]).to(torch.float8_e4m3fn), s
    return code, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"kind": case["kind"]}
    if case["kind"] == "linear":
        x = torch.randn((case["m"], case["k"]), generator=g, device="cuda")
        x *= torch.exp(torch.randn(case["k"], generator=g, device="cuda") * 0.5)  # some channels are much larger
        w = torch.randn((case["n"], case["k"]), generator=g, device="cuda") / math.sqrt(case["k"])
        s["x"] = x.to(_DTYPES[case["dtype"]])
        s["sw"] = w.abs().amax(1) / 127
        s["w"] = torch.round(w / s["sw"][:, None]).to(torch.int8)
        return s
    heads, d, page = case["kv_heads"], case["d"], case["page"]
    if case["kind"] == "copy":
        pool = case["pool"]
        order = torch.randperm(pool, generator=g, device="cuda")[:2 * case["moved"]].int()
        s["src"], s["dst"] = order[:case["moved"]].contiguous(), order[case["moved"]:].contiguous()
    else:
        lens, news = _lens(case)
        most = -(-case["ctx"] // page)
        used = [-(-n // page) for n in lens]
        pool = sum(used) + 3
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        table, at = [], 0
        for n in used:
            table.append(order[at:at + n] + [-1] * (most - n))
            at += n
        total = sum(news)
        s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["cu"] = torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32, device="cuda")
        s["ragged"] = news != [1] * len(news)
        s["max_new"], s["max_kv"] = max(news), max(lens)
        # of each new token: its sequence and its place among that one's new tokens
        s["seq"] = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).cuda()
        s["row"] = torch.cat([torch.arange(n) for n in news]).cuda()
        if case["kind"] == "attend":
            s["q"] = torch.randn((total, case["heads"], d), generator=g, device="cuda").to(_DTYPES[case["dtype"]])
        else:
            for name in ("key", "value"):
                x = torch.randn((total, heads, d), generator=g, device="cuda")
                s[name] = x.to(_DTYPES[case["dtype"]])
    s["k"], s["k_scale"] = _pages_of(g, pool, page, d, heads)
    s["v"], s["v_scale"] = _pages_of(g, pool, d, page, heads)
    if own:
        s["cache"] = _ops().KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


def run(s):
    if own:
        return _run_own(s, _ops())
    return {"linear": _linear, "attend": _attend, "append": _append, "copy": _copy}[s["kind"]](s)


def _run_own(s, ops):
    if s["kind"] == "linear":
        return ops.linear_int8(s["x"], s["w"], s["sw"])
    if s["kind"] == "copy":
        ops.kv8_copy_pages(s["cache"], s["src"], s["dst"])
        return s["k"], s["v"], s["k_scale"], s["v_scale"]
    more = {"cu_q": s["cu"], "max_q": s["max_new"]} if s["ragged"] else {}
    if s["kind"] == "attend":
        return ops.gqa_kv8(s["q"], s["cache"], s["table"], s["lens"], max_kv=s["max_kv"], **more)
    ops.kv8_append(s["key"], s["value"], s["cache"], s["table"], s["lens"], **more)
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _linear(s):
    """q = round(x / sx), sx = max |x| / 127 of each row; y = (q . w^T) sx sw.  The quotient next to a half in 64 bits."""
    x = s["x"].float()
    most = x.abs().amax(1)
    sx = torch.where(most > 0, most / 127, 1.0)
    q = torch.round(x.double() / sx.double()[:, None]).float()
    return ((q @ s["w"].float().t()) * sx[:, None] * s["sw"]).to(s["x"].dtype)


def _at(code, pages):
    return code.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()


def _attend(s):
    q, table, lens = s["q"], s["table"].clamp_min(0).long(), s["lens"].long()
    batch, most = table.shape
    pool, heads, page, d = s["k"].shape
    t = most * page
    group = q.shape[1] // heads
    key = _at(s["k"], table) * s["k_scale"][table][..., None, None]    # [batch, most, heads, page, d]
    key = key.permute(0, 2, 1, 3, 4).reshape(batch, heads, t, d)
    value = _at(s["v"], table) * s["v_scale"][table][..., None, None]  # [batch, most, heads, d, page]
    value = value.permute(0, 2, 1, 4, 3).reshape(batch, heads, t, d)
    n = s["max_new"]
    padded = torch.zeros((batch, n, heads, group, d), device=q.device)
    padded[s["seq"], s["row"]] = q.float().view(-1, heads, group, d)
    rows = padded.permute(0, 2, 3, 1, 4).reshape(batch, heads, group * n, d)
    p = (rows @ key.transpose(2, 3)).view(batch, heads, group, n, t) / math.sqrt(d)
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    last = (lens - new)[:, None] + torch.arange(n, device=q.device)  # the last key that each row sees
    p.masked_fill_(torch.arange(t, device=q.device) > last[:, None, None, :, None], -math.inf)
    p -= p.amax(-1, keepdim=True)
    p.exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(batch, heads, group * n, t) @ value).view(batch, heads, group, n, d) / total
    return out.permute(0, 3, 1, 2, 4)[s["seq"], s["row"]].reshape(q.shape).to(q.dtype)


def _append(s):
    """Of every page that new tokens reach: its scale grows to the smallest power of two that holds them too (one
    that a page's first token is among starts anew), the codes that were there move to the new scale, the new follow."""
    lens, new = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    page = s["k"].shape[2]
    batch = lens.shape[0]
    start = lens - new
    most = (s["max_new"] + page - 2) // page + 1  # pages that a sequence's new tokens can reach
    at = start[:, None] // page + torch.arange(most, device=lens.device)  # [batch, most] of the sequence's pages
    reached = at * page < lens[:, None]
    pages = s["table"].long().gather(1, at.clamp_max(s["table"].shape[1] - 1)).clamp_min(0).view(-1)
    # where a sequence reaches fewer pages, its last one is written more than once, with the same values
    lasts = (lens - 1) // page - start // page
    same = torch.arange(batch, device=lens.device)[:, None] * most + torch.arange(most, device=lens.device).clamp(
        max=lasts[:, None])
    same = same.view(-1)
    place = start[s["seq"]] + s["row"]
    slot = (s["seq"] * most + place // page - start[s["seq"]] // page, place % page)
    held = (start[:, None] - at * page).clamp(0, page).view(-1)  # tokens that were on it
    whole = torch.arange(page, device=lens.device)
    is_old = whole < held[:, None]
    is_new = ~is_old & (whole < (lens[:, None] - at * page).view(-1)[:, None])
    for code, scale, x, turned in ((s["k"], s["k_scale"], s["key"], False), (s["v"], s["v_scale"], s["value"], True)):
        fresh = torch.zeros((batch * most, page, x.shape[1], x.shape[2]), device=x.device)
        fresh[slot] = x.float()
        fresh = fresh.permute(0, 2, 1, 3)  # [pages, heads, page, d]
        was = _at(code, pages)
        was = was.transpose(2, 3) if turned else was
        grown = _two_to(fresh.abs().amax((2, 3)))
        old = scale[pages]
        grown = torch.where(held[:, None] > 0, torch.maximum(grown, old), grown)[..., None, None]
        kept = (was * (old[..., None, None] / grown)).to(torch.float8_e4m3fn)
        came = (fresh / grown).to(torch.float8_e4m3fn)
        now = torch.where(is_old[:, None, :, None], kept.view(torch.uint8), torch.where(
            is_new[:, None, :, None], came.view(torch.uint8), was.to(torch.float8_e4m3fn).view(torch.uint8)))
        now = now.transpose(2, 3) if turned else now
        code.view(torch.uint8)[pages[same]] = now[same]
        scale[pages[same]] = grown[..., 0, 0][same]
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for x in (s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["k_scale"], s["v_scale"]):
        x[dst] = x[src]
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "linear":
        x = s["x"].double()
        sx = (s["x"].float().abs().max(1, keepdim=True).values / 127).double()  # the scale as it is stored
        sx[sx == 0] = 1
        return (torch.round(x / sx) * sx) @ (s["w"].double() * s["sw"].double()[:, None]).t()
    if s["kind"] == "attend":
        return _exact_attend(case, s)
    k, v = s["k"].double(), s["v"].double()
    ks, vs = s["k_scale"].double(), s["v_scale"].double()
    if s["kind"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[b], v[b], ks[b], vs[b] = k[a], v[a], ks[a], vs[a]
        return k, v, ks, vs
    return _exact_append(case, s, k, v, ks, vs)


def _exact_attend(case, s):
    q, out = s["q"].double(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    first = 0
    for b, (n, new) in enumerate(zip(*_lens(case))):
        pages = s["table"][b, :-(-n // case["page"])].long()
        for h in range(case["kv_heads"]):
            key = (s["k"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, case["d"])[:n]
            value = s["v"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]
            value = value.transpose(1, 2).reshape(-1, case["d"])[:n]
            for j in range(h * group, (h + 1) * group):
                score = q[first:first + new, j] @ key.t() * case["d"] ** -0.5
                hidden = torch.ones((new, n), dtype=torch.bool, device="cuda").triu(n - new + 1)
                out[first:first + new, j] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ value
        first += new
    return out


def _nearest(x):
    """The e4m3 values nearest to x (ties to the even code), |x| at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(case, s, k, v, ks, vs):
    page, first = case["page"], 0
    for b, (n, new) in enumerate(zip(*_lens(case))):
        for j in range((n - new) // page, (n - 1) // page + 1):
            lo, hi = max(n - new, j * page), min(n, (j + 1) * page)
            at, held = int(s["table"][b, j]), lo - j * page
            for code, scale, x in ((k, ks, s["key"]), (v.transpose(2, 3), vs, s["value"])):
                fresh = x[first + lo - (n - new):first + hi - (n - new)].double().transpose(0, 1)  # [heads, tokens, d]
                most = fresh.abs().amax((1, 2)).clamp_min(448 * 2.0 ** -32) / 448
                grown = torch.exp2(torch.ceil(torch.log2(most)))
                grown = torch.maximum(grown, scale[at]) if held else grown
                code[at, :, :held] = _nearest(code[at, :, :held] * (scale[at] / grown)[:, None, None])
                code[at, :, held:hi - j * page] = _nearest(fresh / grown[:, None, None])
                scale[at] = grown
        first += new
    return k, v, ks, vs
