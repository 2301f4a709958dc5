"""A step over the 8-bit cache, from projection to answer: what its operators are timed on, their plain forms and
their values in 64 bits.

Four operators, one per "kind":

  rope     RMS norm of every query and key head and the position rotation, in one pass
  window   grouped-query attention over the paged e4m3 cache where a row sees the last `window` tokens up to itself
           and the sequence's first `sinks`, for single tokens and prompts
  tree     grouped-query attention over that cache for drafted tokens that form a tree: a row sees what came before
           them and those of them whose bits are set in its mask
  logprob  log probabilities of given tokens, the entropy and the top alternatives of rows of logits

The cache: k [pages, n_kv, page, d] and v [pages, n_kv, d, page] in e4m3 (a
page of v is held transposed), k_scale and v_scale [pages, n_kv] in fp32,
powers of two.  Sequence b's token t lies on page page_table[b, t // page];
kv_lens counts the tokens with the new ones, which are its last.
"""
import functools
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@functools.lru_cache(None)
def _ops():
    import importlib

    return importlib.import_module("cuda-oxide-bench_amd").load_ops()


def listed():
    return [
        # one user's next token: the smallest call, all latency
        {"name": "rope_t1", "kind": "rope", "tokens": 1, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128,
         "pairs": "halves", "dtype": "bf16"},
        # the ragged tokens of a mixed step, a rotation of a part of each head, neighbouring channels as pairs
        {"name": "rope_t777_d64_part_f16", "kind": "rope", "tokens": 777, "heads": 14, "kv_heads": 2, "d": 64,
         "rot": 32, "pairs": "neighbours", "dtype": "f16"},
        # prompts of together 16384 tokens
        {"name": "rope_t16384", "kind": "rope", "tokens": 16384, "heads": 32, "kv_heads": 8, "d": 128, "rot": 128,
         "pairs": "halves", "dtype": "bf16"},
        # one user's next token far into a text, the small head dim, the smallest pages, a window off the pages
        {"name": "window_b1_t8000_w1000_d64_f16", "kind": "window", "batch": 1, "ctx": 8000, "chunk": 1,
         "window": 1000, "sinks": 4, "heads": 16, "kv_heads": 4, "d": 64, "page": 16, "dtype": "f16"},
        # a decode batch with contexts of very different lengths up to 8192
        {"name": "window_b64_t8192_w2048", "kind": "window", "batch": 64, "ctx": 8192, "chunk": 1, "window": 2048,
         "sinks": 16, "heads": 32, "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # two prompts' chunks behind cached prefixes
        {"name": "window_b2_t8192_q4096_w1024", "kind": "window", "batch": 2, "ctx": 8192, "chunk": 4096,
         "window": 1024, "sinks": 4, "heads": 32, "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # one user's small draft behind a short context
        {"name": "tree_b1_t1001_n13", "kind": "tree", "batch": 1, "ctx": 1001, "drafts": 13, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # a batch of drafts of up to 32 tokens
        {"name": "tree_b16_t4096_n32", "kind": "tree", "batch": 16, "ctx": 4096, "drafts": 32, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "dtype": "bf16"},
        # wide trees of up to 100 tokens, every query head its own keys, the small head dim, the smallest pages
        {"name": "tree_b33_t2000_n100_d64_f16", "kind": "tree", "batch": 33, "ctx": 2000, "drafts": 100, "heads": 16,
         "kv_heads": 16, "d": 64, "page": 16, "dtype": "f16"},
        # one user's next token over a small vocabulary
        {"name": "logprob_t1_v32000", "kind": "logprob", "rows": 1, "vocab": 32000, "given": 1, "top": 5, "pad": 0,
         "masked": False, "dtype": "bf16"},
        # a decode batch whose logits are 32 bits wide, some rows held to a grammar, a few given tokens each
        {"name": "logprob_t64_v128000_f32", "kind": "logprob", "rows": 64, "vocab": 128000, "given": 4, "top": 20,
         "pad": 0, "masked": True, "dtype": "f32"},
        # a prompt's tokens scored, an odd vocabulary inside padded rows
        {"name": "logprob_t2048_v100003", "kind": "logprob", "rows": 2048, "vocab": 100003, "given": 1, "top": 8,
         "pad": 29, "masked": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi, step=1):
    """A size between lo and hi, spread over its logarithm, a multiple of step."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(-(-lo // step) * step, x // step * step)


def draw(rng):
    kind = rng.choice(["rope", "window", "window", "tree", "tree", "logprob"])
    if kind == "logprob":
        vocab, dtype = _log(rng, 1000, 200000), rng.choice(["bf16", "f16", "f32"])
        most = 2048 * 100003 // (vocab * (2 if dtype == "f32" else 1))
        return {"kind": kind, "rows": _log(rng, 1, min(most, 4096)), "vocab": vocab, "given": rng.randint(1, 6),
                "top": rng.choice([0, rng.randint(1, 20)]), "pad": rng.choice([0, rng.randint(1, 64)]),
                "masked": rng.random() < 0.3, "dtype": dtype}
    kv_heads, dtype = rng.choice([1, 2, 4, 8, 16]), rng.choice(["bf16", "f16"])
    group = rng.choice([1, 2, 4, 7, 8, 16])
    if kind == "rope":
        d = rng.choice([64, 80, 128, 256])
        heads = kv_heads * group
        most = min(16384 * 40 * 128 // ((heads + kv_heads) * d), 32768)
        return {"kind": kind, "tokens": _log(rng, 1, most), "heads": heads, "kv_heads": kv_heads, "d": d,
                "rot": rng.choice([d, d // 32 * 16]), "pairs": rng.choice(["halves", "neighbours"]), "dtype": dtype}
    d, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if kind == "tree":
        heads = min(kv_heads * group, 64)
        group = heads // kv_heads
        batch = _log(rng, 1, 64)
        ctx = _log(rng, 128, min(16384, 16 * 4096 * 5 * 128 // (batch * kv_heads * d)))
        most = min(128, ctx // 2, 16 * 4096 * 32 * 20 * 128 // (batch * ctx * kv_heads * group * d))
        return {"kind": kind, "batch": batch, "ctx": ctx, "drafts": _log(rng, 2, max(2, most)),
                "heads": kv_heads * group, "kv_heads": kv_heads, "d": d, "page": page, "dtype": dtype}
    chunk = rng.choice(["one", "one", "few", "long"])
    if chunk == "long":
        batch = _log(rng, 1, 4)
        heads = min(kv_heads * group, 32)
        kv_heads = heads // min(group, heads)
        heads = kv_heads * min(group, heads)
        ctx = _log(rng, 64, 4096)
        new = _log(rng, 16, min(2048, ctx))
    else:
        batch = _log(rng, 1, 64)
        heads = kv_heads * group
        ctx = _log(rng, 64, min(32768, 8192 * 64 * 5 * 128 // (batch * kv_heads * d)))
        new = 1 if chunk == "one" else rng.randint(2, 8)
    return {"kind": kind, "batch": batch, "ctx": ctx, "chunk": new, "window": _log(rng, 16, 4096),
            "sinks": rng.choice([0, 1, 4, rng.randint(5, 128)]), "heads": heads, "kv_heads": kv_heads, "d": d,
            "page": page, "dtype": dtype}


def _lens(case):
    """(tokens in the cache with the new ones, new ones) of each sequence: the first has the most of both."""
    rng = random.Random(case["batch"] * 1000003 + case["ctx"])
    lens = [case["ctx"]] + [rng.randint(max(1, case["ctx"] // 4), case["ctx"]) for _ in range(case["batch"] - 1)]
    if case["kind"] == "window" and case["chunk"] <= 8:
        return lens, [min(case["chunk"], n) for n in lens]
    most = case["chunk"] if case["kind"] == "window" else case["drafts"]
    return lens, [min(n, most if b == 0 else rng.randint(max(1, most // 4), most)) for b, n in enumerate(lens)]


def _in_view(case, n, new):
    """(tokens of a sequence that any new row sees, pairs of rows and tokens that they see; trees: the most)"""
    if case["kind"] == "tree":
        return n, new * (n - new) + new * (new + 1) // 2
    w, s = case["window"], case["sinks"]
    pairs = sum(min(p + 1, w) + min(s, max(p + 1 - w, 0)) for p in range(n - new, n))
    behind = max(n - new + 1 - w, 0)  # tokens that have left the first row's window
    return n - behind + min(s, behind), pairs


def work(case):
    if case["kind"] == "logprob":
        t, v = case["rows"], case["vocab"]
        out = t * (8 * case["given"] + 4 + 8 * case["top"])
        return {"bytes": t * v * (4 if case["dtype"] == "f32" else 2) + out, "flops": 6 * t * v}
    if case["kind"] == "rope":
        t, values = case["tokens"], case["tokens"] * (case["heads"] + case["kv_heads"]) * case["d"]
        return {"bytes": 4 * values + t * (4 * case["rot"] + 4) + 4 * case["d"], "flops": 7 * values}
    h, d, p = case["kv_heads"], case["d"], case["page"]
    lens, news = _lens(case)
    seen = [_in_view(case, n, new) for n, new in zip(lens, news)]
    pages = sum(-(-n // p) for n, _ in seen)
    masks = 8 * -(-max(news) // 64) * sum(news) if case["kind"] == "tree" else 0
    return {"bytes": 2 * sum(n for n, _ in seen) * h * d + pages * (8 * h + 4) + 4 * sum(news) * case["heads"] * d + masks,
            "flops": 4 * sum(pairs for _, pairs in seen) * case["heads"] * d}


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


def _tree(rng, n, words):
    """Masks of a random tree of n drafted tokens, in whole numbers of 64 bits each: a row sees its ancestors and itself."""
    rows = []
    for i in range(n):
        parent = rng.randint(max(0, i - 12), i - 1) if i else -1
        rows.append((rows[parent] if parent >= 0 else 0) | 1 << i)
    whole = [[r >> 64 * w & 0xFFFFFFFFFFFFFFFF for w in range(words)] for r in rows]
    return [[x - (1 << 64) if x >> 63 else x for x in r] for r in whole]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    s = {"kind": case["kind"]}
    dtype = _DTYPES[case["dtype"]]
    if case["kind"] == "logprob":
        t, v = case["rows"], case["vocab"]
        x = torch.randn((t, v + case["pad"]), generator=g, device="cuda").mul_(2.5)
        # a few favourites a row, some far ahead of the rest
        best = torch.randint(0, v, (t, 6), generator=g, device="cuda")
        x.scatter_add_(1, best, torch.rand((t, 6), generator=g, device="cuda") * 16)
        if case["masked"]:  # every third row may take one token in fifty
            x[::3].masked_fill_(torch.rand(x[::3].shape, generator=g, device="cuda") > 0.02, -math.inf)
            x[::3, 7] = 0.5
        s["logits"] = x.to(dtype)[:, :v]
        given = torch.randint(0, v, (t, case["given"]), generator=g, device="cuda")
        given[:, 0] = best[:, 0]
        s["given"], s["top"] = given.int(), case["top"]
        return s
    if case["kind"] == "rope":
        t, n, m, d, rot = case["tokens"], case["heads"], case["kv_heads"], case["d"], case["rot"]
        qkv = (torch.randn((t, (n + 2 * m) * d), generator=g, device="cuda") * 3).to(dtype)
        s["q"] = qkv[:, :n * d].unflatten(1, (n, d))  # views of a fused projection
        s["k"] = qkv[:, n * d:(n + m) * d].unflatten(1, (m, d))
        for name in ("wq", "wk"):
            s[name] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)
        angle = torch.arange(32768, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        place, positions = 0, []
        while len(positions) < t:  # sequences' tokens, one behind the other
            place = rng.randint(0, 16000)
            positions += range(place, place + rng.randint(1, max(1, min(t // 3, 16000))))
        s["positions"] = torch.tensor(positions[:t], dtype=torch.int32, device="cuda")
        s["eps"], s["neighbours"] = 1e-6, case["pairs"] == "neighbours"
        return s
    heads, d, page = case["kv_heads"], case["d"], case["page"]
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
    s["page_table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["cu"] = torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32, device="cuda")
    s["ragged"] = news != [1] * len(news)
    s["max_new"], s["max_kv"] = max(news), max(lens)
    # of each new token: its sequence and its place among that one's new tokens
    s["seq"] = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).cuda()
    s["row"] = torch.cat([torch.arange(n) for n in news]).cuda()
    s["q"] = torch.randn((total, case["heads"], d), generator=g, device="cuda").to(dtype)
    if case["kind"] == "tree":
        words = -(-max(news) // 64)
        s["tree"] = torch.tensor([r for n in news for r in _tree(rng, n, words)], dtype=torch.int64, device="cuda")
    else:
        s["window"], s["sinks"] = case["window"], case["sinks"]
    s["k"], s["k_scale"] = _pages_of(g, pool, page, d, heads)
    s["v"], s["v_scale"] = _pages_of(g, pool, d, page, heads)
    if own:
        s["cache"] = _ops().KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


def run(s):
    if own:
        return _run_own(s, _ops())
    return {"rope": _rope, "window": _attend, "tree": _attend, "logprob": _logprob}[s["kind"]](s)


def _run_own(s, ops):
    if s["kind"] == "rope":
        return ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["table"], s["positions"], eps=s["eps"],
                                neighbours=s["neighbours"])
    if s["kind"] == "logprob":
        return ops.token_logprobs(s["logits"], s["given"], top=s["top"])
    more = {"cu_q": s["cu"], "max_q": s["max_new"]} if s["ragged"] else {}
    if s["kind"] == "window":
        return ops.gqa_kv8_window(s["q"], s["cache"], s["page_table"], s["lens"], s["window"], s["sinks"],
                                  max_kv=s["max_kv"], **more)
    return ops.gqa_kv8_tree(s["q"], s["cache"], s["page_table"], s["lens"], s["tree"], max_kv=s["max_kv"], **more)


def _rope(s):
    """y = x / sqrt(mean(x^2) + eps) * w; its pairs (a, b) become (a cos - b sin, b cos + a sin)."""
    at = s["table"][s["positions"].long()]
    rot = at.shape[1]
    cos, sin = at[:, None, :rot // 2], at[:, None, rot // 2:]
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w.float()
        if s["neighbours"]:
            a, b = y[..., :rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([turned, y[..., rot:]], -1).to(x.dtype))
    return tuple(out)


def _bits(masks, i):
    """Bit i (a tensor of numbers below 64 times the masks' words) of each row of masks."""
    return (masks[:, i // 64] >> (i % 64) & 1).bool()


def _hidden(s, t, n):
    """[batch, n, t]: the tokens that a sequence's new rows do not see."""
    device = s["lens"].device
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    first = s["lens"].long() - new  # of the new tokens
    token = torch.arange(t, device=device)
    if s["kind"] == "window":
        last = (first[:, None] + torch.arange(n, device=device))[..., None]
        return (token > last) | ((token <= last - s["window"]) & (token >= s["sinks"]))
    bits = torch.zeros((len(first), n, n), dtype=torch.bool, device=device)
    bits[s["seq"], s["row"]] = _bits(s["tree"], torch.arange(n, device=device))
    among = (token - first[:, None])[:, None].expand(-1, n, -1)  # a token's number among the drafted ones
    return ~((among < 0) | (bits.gather(2, among.clamp(0, n - 1)) & (among < n)))


def _attend(s):
    q, table, lens = s["q"], s["page_table"].clamp_min(0).long(), s["lens"].long()
    batch, most = table.shape
    pool, heads, page, d = s["k"].shape
    t = most * page
    group = q.shape[1] // heads

    def at(code):
        return code.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()

    key = at(s["k"]) * s["k_scale"][table][..., None, None]    # [batch, most, heads, page, d]
    key = key.permute(0, 2, 1, 3, 4).reshape(batch, heads, t, d)
    value = at(s["v"]) * s["v_scale"][table][..., None, None]  # [batch, most, heads, d, page]
    value = value.permute(0, 2, 1, 4, 3).reshape(batch, heads, t, d)
    n = s["max_new"]
    padded = torch.zeros((batch, n, heads, group, d), device=q.device)
    padded[s["seq"], s["row"]] = q.float().view(-1, heads, group, d)
    rows = padded.permute(0, 2, 3, 1, 4).reshape(batch, heads, group * n, d)
    p = (rows @ key.transpose(2, 3)).view(batch, heads, group, n, t) / math.sqrt(d)
    hidden = _hidden(s, t, n) | (torch.arange(t, device=q.device) >= lens[:, None, None])
    p.masked_fill_(hidden[:, None, None], -math.inf)
    p -= p.amax(-1, keepdim=True).clamp_min(-3e38)  # (a padded row may see nothing)
    p.exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(batch, heads, group * n, t) @ value).view(batch, heads, group, n, d) / total
    return out.permute(0, 3, 1, 2, 4)[s["seq"], s["row"]].reshape(q.shape).to(q.dtype)


def _logprob(s):
    """log p = x - m - log S, S = sum exp(x - m); the entropy is log S - sum p (x - m).  The order of the alternatives is
    that of one whole number each: the value's bits, made to rise with it, above the place counted from the end."""
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total[:, 0] - torch.where(e > 0, e * y, 0.0).sum(1) / total[:, 0]
    given = y.gather(1, s["given"].long()) - log_total
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32
    order += torch.arange(x.shape[1] - 1, -1, -1, device=x.device)
    best = x.shape[1] - 1 - (order.topk(s["top"], 1).values & 0xFFFFFFFF)
    return given, entropy, best.int(), y.gather(1, best) - log_total


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "rope":
        return _exact_rope(s)
    if s["kind"] == "logprob":
        return _exact_logprob(s)
    return _exact_attend(case, s)


def _exact_rope(s):
    """Pairs as complex numbers, multiplied by cos + i sin."""
    at = s["table"].double()[s["positions"].long()]
    half = at.shape[1] // 2
    turn = torch.complex(at[:, :half], at[:, half:])[:, None]
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        y = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
        first = slice(0, 2 * half, 2) if s["neighbours"] else slice(0, half)
        second = slice(1, 2 * half, 2) if s["neighbours"] else slice(half, 2 * half)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_logprob(s):
    rows = []
    for x, given in zip(s["logits"], s["given"]):
        x = x.double()
        log_p = x - torch.logsumexp(x, 0)
        p = torch.exp(log_p)
        order = torch.sort(x, descending=True, stable=True).indices[:s["top"]]
        rows.append((log_p[given.long()], -torch.special.xlogy(p, p).sum(), order.int(), log_p[order]))
    return tuple(torch.stack(x) for x in zip(*rows))


def _exact_attend(case, s):
    q, out = s["q"].double(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    first = 0
    for b, (n, new) in enumerate(zip(*_lens(case))):
        pages = s["page_table"][b, :-(-n // case["page"])].long()
        seen = torch.ones((new, n), dtype=torch.bool, device="cuda")
        if case["kind"] == "window":
            near = seen.tril(n - new) & ~seen.tril(n - new - case["window"])
            near[:, :case["sinks"]] = True
            seen = near & seen.tril(n - new)
        else:
            masks = s["tree"][first:first + new].tolist()
            seen[:, n - new:] = torch.tensor([[bool(row[j // 64] >> j % 64 & 1) for j in range(new)] for row in masks])
        for h in range(case["kv_heads"]):
            key = (s["k"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, case["d"])[:n]
            value = s["v"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]
            value = value.transpose(1, 2).reshape(-1, case["d"])[:n]
            for j in range(h * group, (h + 1) * group):
                score = q[first:first + new, j] @ key.t() * case["d"] ** -0.5
                out[first:first + new, j] = torch.softmax(score.masked_fill(~seen, -math.inf), 1) @ value
        first += new
    return out
