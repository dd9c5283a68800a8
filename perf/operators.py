"""The packed-batch operators of the language model, as they are measured.

Four operators that serve many requests of the VLM in one step: `layout` (block tables and slot maps
from request lengths), `rope` (per-head norms of queries and keys with the multi-axis rotation, K / V
written into their cache pages), `attention` (packed causal grouped-query attention over prompts,
chunks and single tokens) and `prefix` (the same for a batch whose requests share a long prefix).

With `own` false, `run` computes an operator in its plain form (elementary torch operations in 32
bits, rounded once at the end); with `own` true it makes the framework's calls. `exact` is the
definition in 64 bits, written apart.
"""
import math
import random

import torch

own = False

PAGE = 128  # rows per K/V cache page
DEV = "cuda"


def listed():
    return [
        # the answer of one request grows by a token: everything is latency
        dict(name="layout one answer", op="layout", batch=1, longest=1, decoding=100, past=1424, mix=1),
        # a full house: new prompts among answers in progress
        dict(name="layout 2048 requests", op="layout", batch=2048, longest=1500, decoding=50, past=6000, mix=2),
        # one decoding step of 61 answers, three position axes, normalised heads
        dict(name="rope 61 answers", op="rope", tokens=61, heads=28, kv_heads=4, dim=128, axes=3, norm=True),
        # one image of 1296 merged tokens and 128 text tokens, rotation alone
        dict(name="rope image prompt", op="rope", tokens=1424, heads=28, kv_heads=4, dim=128, axes=3, norm=False),
        # a batch of images in a vision tower: two axes, as many key heads as query heads
        dict(name="rope 20011 patches", op="rope", tokens=20011, heads=16, kv_heads=16, dim=64, axes=2, norm=True),
        # three short text prompts of a small model, keys beside the queries (no cache)
        dict(name="attention short texts", op="attention", batch=3, q_lo=1, q_hi=37, past_lo=0, past_hi=0, heads=4,
             kv_heads=2, dim=64, paged=False, mix=3),
        # the prompt of one image and its text, over its cache pages
        dict(name="attention image prompt", op="attention", batch=1, q_lo=1424, q_hi=1424, past_lo=0, past_hi=0,
             heads=28, kv_heads=4, dim=128, paged=True, mix=4),
        # four long prompts of different lengths, one of them a chunk after cached tokens
        dict(name="attention long prompts", op="attention", batch=4, q_lo=700, q_hi=5001, past_lo=0, past_hi=600,
             heads=28, kv_heads=4, dim=128, paged=True, mix=5),
        # one decoding step of 96 answers of any age
        dict(name="attention 96 answers", op="attention", batch=96, q_lo=1, q_hi=1, past_lo=60, past_hi=6000,
             heads=28, kv_heads=4, dim=128, paged=True, mix=6),
        # five questions about one image, all decoding
        dict(name="prefix five questions", op="prefix", batch=5, q=1, prefix=1312, own_lo=1, own_hi=60, heads=28,
             kv_heads=4, dim=128, mix=7),
        # the same with four drafted tokens each, on narrow heads
        dict(name="prefix drafted tokens", op="prefix", batch=24, q=4, prefix=2777, own_lo=4, own_hi=300, heads=16,
             kv_heads=2, dim=64, mix=8),
        # many answers after one long document
        dict(name="prefix 128 answers", op="prefix", batch=128, q=1, prefix=6000, own_lo=16, own_hi=1500, heads=28,
             kv_heads=4, dim=128, mix=9),
    ]


# ------------------------------------------------------------------------------------ cases
def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 0.6)), math.log(max(hi, 0.6) + 0.4)))))))


def _lengths(case):
    """(new tokens, tokens before them) of every request: a function of the case alone."""
    rng = random.Random(case["mix"])
    if case["op"] == "layout":
        q = [1 if rng.randrange(100) < case["decoding"] else _spread(rng, 1, case["longest"]) for _ in range(case["batch"])]
        past = [_spread(rng, 0, case["past"]) for _ in q]
        past[0] = case["past"]
    elif case["op"] == "attention":
        q = [_spread(rng, case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
        q[rng.randrange(len(q))] = case["q_hi"]
        past = [_spread(rng, case["past_lo"], case["past_hi"]) if case["past_hi"] else 0 for _ in q]
    else:
        q = [case["q"]] * case["batch"]
        past = [_spread(rng, case["own_lo"], case["own_hi"]) - case["q"] for _ in q]
        past = [max(p, 0) for p in past]
    return q, past


def _pages(n):
    return -(-n // PAGE)


def work(case):
    if case["op"] == "layout":
        q, past = _lengths(case)
        new = sum(_pages(a + b) - _pages(b) for a, b in zip(q, past))
        # lengths in; starts and lengths out; row, request and position of every token; new pages in and out
        return {"bytes": 4 * (2 * len(q) + 2 * len(q) + 1 + 3 * sum(q) + 2 * new), "flops": 0}
    if case["op"] == "rope":
        n, width = case["tokens"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        turned = (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * n * width + 4 * n * (case["axes"] + 1), "flops": n * turned * (3 + 4 * case["norm"])}
    q, past = _lengths(case)
    shared = case.get("prefix", 0)
    pairs = sum(a * (b + shared) + a * (a + 1) // 2 for a, b in zip(q, past))
    rows = shared + sum(q) + sum(past)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 4 * dim * (sum(q) * heads + rows * kv_heads), "flops": 4 * pairs * heads * dim}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _room(case):
    """Bytes of the plain form's scores."""
    if case["op"] not in ("attention", "prefix"):
        return 0
    q, past = _lengths(case)
    return 4 * len(q) * max(q) * (max(a + b for a, b in zip(q, past)) + case.get("prefix", 0)) * case["heads"]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        mix = rng.randrange(1, 1 << 30)
        op = rng.choice(("layout", "rope", "attention", "attention", "prefix", "prefix"))
        kv_heads = rng.choice((1, 2, 4, 8, 16))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
        dim = rng.choice((64, 128))
        if op == "layout":
            case = dict(op=op, batch=_spread(rng, 1, 4000), longest=_spread(rng, 1, 2500), decoding=rng.choice((0, 50, 90, 100)),
                        past=_spread(rng, 1, 16000), mix=mix)
        elif op == "rope":
            case = dict(op=op, tokens=_spread(rng, 1, 24000), heads=heads, kv_heads=kv_heads, dim=dim,
                        axes=rng.choice((1, 2, 3)), norm=rng.random() < 0.5)
        elif op == "attention" and rng.random() < 0.5:  # prompts, or chunks after what is cached
            q_hi = _spread(rng, 1, 6000)
            past_hi = rng.choice((0, _spread(rng, 1, 3000)))
            case = dict(op=op, batch=_spread(rng, 1, 16), q_lo=_spread(rng, 1, q_hi), q_hi=q_hi, past_lo=0, past_hi=past_hi,
                        heads=heads, kv_heads=kv_heads, dim=dim, paged=bool(past_hi) or rng.random() < 0.5, mix=mix)
        elif op == "attention":  # answers in progress
            past_hi = _spread(rng, 1, 12000)
            case = dict(op=op, batch=_spread(rng, 1, 300), q_lo=1, q_hi=rng.choice((1, 1, 1, 2, 5)), past_lo=_spread(rng, 0, past_hi),
                        past_hi=past_hi, heads=heads, kv_heads=kv_heads, dim=dim, paged=True, mix=mix)
        else:
            own_hi = _spread(rng, 1, 2000)
            case = dict(op=op, batch=_spread(rng, 1, 300), q=rng.choice((1, 1, 1, 3, 4, 17)), prefix=_spread(rng, 1, 16000),
                        own_lo=_spread(rng, 1, own_hi), own_hi=own_hi, heads=heads, kv_heads=kv_heads, dim=dim, mix=mix)
            case["own_lo"], case["own_hi"] = max(case["own_lo"], case["q"]), max(case["own_hi"], case["q"])
        if _cost(case) <= most and _room(case) <= 13e9 and work(case)["bytes"] <= 1.5e9:
            return case


# ------------------------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32).mul_(std).to(torch.bfloat16)


def _heads_like(gen, rows, heads, dim, std):
    """Rows of heads whose channels have offsets of their own, as projected queries and keys have."""
    at = torch.randn(heads * dim, generator=gen, device=DEV) * 0.3
    return torch.randn(rows, heads * dim, generator=gen, device=DEV).mul_(std).add_(at).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return dict(layout=_prepare_layout, rope=_prepare_rope, attention=_prepare_attention, prefix=_prepare_attention)[case["op"]](case, gen)


def _prepare_layout(case, gen):
    q, past = _lengths(case)
    have, need = [_pages(p) for p in past], sum(_pages(a + b) - _pages(b) for a, b in zip(q, past))
    width = max(_pages(a + b) for a, b in zip(q, past)) + 1
    held = sum(have)
    order = torch.randperm(held + need + 9, generator=gen, device=DEV).to(torch.int32)
    at = torch.arange(width, device=DEV)
    own_pages = at[None] < _ints(have)[:, None]
    table = torch.full((len(q), width), -1, dtype=torch.int32, device=DEV)
    table[own_pages] = order[:held]
    empty = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
    n = sum(q)
    return dict(op="layout", q_len=_ints(q), past=_ints(past), table=table, free_pages=order[held:].clone(), free_start=_ints([3]),
                q_start=empty(len(q) + 1), kv_len=empty(len(q)), rows=empty(n), req=empty(n), pos=empty(n), free_next=empty(2))


def _prepare_rope(case, gen):
    n, heads, kv_heads, dim, axes = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "axes"))
    half = dim // 2
    if axes == 2:  # a ladder of frequencies for each of row and column
        inv = (10000.0 ** -(torch.arange(half // 2, dtype=torch.float64) / (half // 2))).repeat(2)
        axis = torch.arange(half) // (half // 2)
        side = max(1, int(math.sqrt(n)))
        at = torch.arange(n)
        pos = torch.stack([at // side, at % side])
    else:
        inv = 1e6 ** -(torch.arange(half, dtype=torch.float64) / half)
        first, second = half // 4, half * 5 // 8
        axis = ((torch.arange(half) >= first).long() + (torch.arange(half) >= second).long()) if axes == 3 else torch.zeros(half)
        before = n // 16  # text, an image, text
        side = max(1, int(math.sqrt(n * 7 // 8)))
        at = torch.arange(n)
        in_image = (at >= before) & (at < before + side * side)
        k = (at - before).clamp(min=0)
        after = before + side + (at - before - side * side)
        line = torch.where(at < before, at, after)
        grid = torch.stack([torch.full((n,), before), before + k // side, before + k % side])
        pos = torch.where(in_image[None], grid, line[None])[:axes] + int(torch.randint(0, 3000, (1,), generator=gen, device=DEV))
    pages = _pages(n) + 2
    place = torch.randperm(pages, generator=gen, device=DEV)
    at = torch.arange(n, device=DEV)
    weight = lambda: (1 + 0.2 * torch.randn(dim, generator=gen, device=DEV)).to(torch.bfloat16) if case["norm"] else None  # noqa: E731
    return dict(op="rope", heads=heads, kv_heads=kv_heads, dim=dim, qkv=_heads_like(gen, n, heads + 2 * kv_heads, dim, 2.0),
                pos=pos.to(device=DEV, dtype=torch.int32).contiguous(), inv_freq=inv.float().to(DEV), axis=axis.to(device=DEV, dtype=torch.int32),
                rows=(place[at // PAGE] * PAGE + at % PAGE).to(torch.int32), q_weight=weight(), k_weight=weight(), eps=1e-6,
                q_out=torch.empty(n, heads * dim, device=DEV, dtype=torch.bfloat16),
                k_cache=_normal(gen, pages * PAGE, kv_heads * dim), v_cache=_normal(gen, pages * PAGE, kv_heads * dim))


def _prepare_attention(case, gen):
    q, past = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    kv = [a + b for a, b in zip(q, past)]
    n = sum(q)
    start = [0]
    for a in q:
        start.append(start[-1] + a)
    s = dict(op=case["op"], heads=heads, kv_heads=kv_heads, dim=dim, scale=dim ** -0.5, q_most=max(q), kv_most=max(kv),
             q=_heads_like(gen, n, heads, dim, 1.5), o=torch.empty(n, heads * dim, device=DEV, dtype=torch.bfloat16), q_start=_ints(start),
             kv_len=_ints(kv), prefix=case.get("prefix", 0), table=None, k_start=None, prefix_table=None)
    if case["op"] == "attention" and not case["paged"]:
        s["k_start"] = _ints(start[:-1])
        rows = n
    else:
        blocks = [_pages(x) for x in kv]
        shared = _pages(s["prefix"])
        pages = sum(blocks) + shared + 3
        place = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        width = max(blocks) + 1
        table = torch.zeros(len(q), width, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV)[None] < _ints(blocks)[:, None]] = place[:sum(blocks)]
        s["table"] = table
        s["prefix_table"] = place[sum(blocks):sum(blocks) + shared].clone()
        rows = pages * PAGE
    s["k"], s["v"] = _heads_like(gen, rows, kv_heads, dim, 1.0), _normal(gen, rows, kv_heads * dim)
    return s


# ------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        return _run_own(s)
    return dict(layout=_plain_layout, rope=_plain_rope, attention=_plain_attention, prefix=_plain_attention)[s["op"]](s)


def _run_own(s):
    from appcorr_b200.ops import packed

    if s["op"] == "layout":
        packed.packed_layout(s["q_len"], s["past"], s["table"], s["free_pages"], s["free_start"], q_start=s["q_start"],
                             kv_len=s["kv_len"], rows=s["rows"], req=s["req"], pos=s["pos"], free_next=s["free_next"])
        return {k: s[k] for k in ("q_start", "kv_len", "rows", "req", "pos", "table", "free_next")}
    if s["op"] == "rope":
        packed.qk_norm_rope(s["qkv"], s["pos"], s["inv_freq"], s["axis"], s["q_out"], s["k_cache"], s["v_cache"], heads=s["heads"],
                            kv_heads=s["kv_heads"], head_dim=s["dim"], rows=s["rows"], q_weight=s["q_weight"],
                            k_weight=s["k_weight"], eps=s["eps"])
        return {k: s[k] for k in ("q_out", "k_cache", "v_cache")}
    if s["op"] == "attention":
        return packed.packed_attention(s["q"], s["k"], s["v"], s["o"], q_start=s["q_start"], kv_len=s["kv_len"], heads=s["heads"],
                                       kv_heads=s["kv_heads"], head_dim=s["dim"], table=s["table"], k_start=s["k_start"], scale=s["scale"])
    return packed.shared_prefix_attention(s["q"], s["k"], s["v"], s["o"], q_start=s["q_start"], kv_len=s["kv_len"], table=s["table"],
                                          prefix_table=s["prefix_table"], prefix_len=s["prefix"], heads=s["heads"],
                                          kv_heads=s["kv_heads"], head_dim=s["dim"], scale=s["scale"])


def _plain_layout(s):
    q, past, table, free = s["q_len"].long(), s["past"].long(), s["table"], s["free_pages"]
    batch, width = table.shape
    end = q.cumsum(0)
    kv = past + q
    have = (past + PAGE - 1) // PAGE
    total = (kv + PAGE - 1) // PAGE
    need = (total.clamp(max=width) - have).clamp(min=0)
    first = need.cumsum(0) - need
    begin = s["free_start"].long()
    at = torch.arange(width, device=DEV)[None] - have[:, None]
    source = begin + first[:, None] + at
    new = (at >= 0) & (at < need[:, None])
    given = new & (source < free.numel())
    table.copy_(torch.where(given, free[source.clamp(0, free.numel() - 1)], torch.where(new, -1, table)))
    n = torch.arange(s["rows"].numel(), device=DEV)
    b = torch.searchsorted(end, n, right=True).clamp(max=batch - 1)
    pos = past[b] + n - (end - q)[b]
    page = torch.where(pos // PAGE < width, table[b, (pos // PAGE).clamp(max=width - 1)], -1)
    inside = n < end[-1]
    rows = torch.where(inside & (page >= 0), page * PAGE + pos % PAGE, -1)
    asked = need.sum()
    following = torch.minimum(begin[0] + asked, torch.full_like(asked, free.numel()))
    missing = begin[0] + asked - following + (total - width).clamp(min=0).sum()
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(q_start=whole(torch.cat([end.new_zeros(1), end])), kv_len=whole(kv), rows=whole(rows), req=whole(torch.where(inside, b, -1)),
                pos=whole(torch.where(inside, pos, -1)), table=table, free_next=whole(torch.stack([following, missing])))


def _plain_rope(s):
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    n = s["qkv"].shape[0]
    x = s["qkv"].float().view(n, heads + 2 * kv_heads, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    angle = s["pos"].float()[s["axis"].long()].T * s["inv_freq"]
    sin, cos = angle.sin()[:, None], angle.cos()[:, None]

    def turned(t, weight):
        if weight is not None:
            t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + s["eps"]) * weight.float()
        a, b = t[..., :dim // 2], t[..., dim // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).reshape(n, -1).to(torch.bfloat16)

    rows = s["rows"].long()
    s["q_out"].copy_(turned(q, s["q_weight"]))
    s["k_cache"][rows] = turned(k, s["k_weight"])
    s["v_cache"][rows] = v.reshape(n, -1).to(torch.bfloat16)
    return {k: s[k] for k in ("q_out", "k_cache", "v_cache")}


def _plain_attention(s):
    """Queries and keys padded to the longest request's, the scores in one product."""
    heads, kv_heads, dim, shared = s["heads"], s["kv_heads"], s["dim"], s["prefix"]
    group = heads // kv_heads
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    q_len = start[1:] - start[:-1]
    batch, t, length = kv_len.numel(), s["q_most"], s["kv_most"]
    at = torch.arange(length, device=DEV)
    if s["table"] is None:
        rows = s["k_start"].long()[:, None] + at
    else:
        rows = s["table"].long()[:, at // PAGE] * PAGE + at % PAGE
    rows = torch.where(at < kv_len[:, None], rows, 0)
    if shared:
        before = torch.arange(shared, device=DEV)
        rows = torch.cat([(s["prefix_table"].long()[before // PAGE] * PAGE + before % PAGE).expand(batch, -1), rows], 1)
    k = s["k"][rows].float().view(batch, -1, kv_heads, dim).permute(0, 2, 3, 1)
    v = s["v"][rows].float().view(batch, -1, kv_heads, dim).permute(0, 2, 1, 3)
    step = torch.arange(t, device=DEV)
    token = start[:-1, None] + step
    live = step < q_len[:, None]
    q = s["q"][token.clamp(max=s["q"].shape[0] - 1)].float().view(batch, t, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    last = (kv_len - q_len)[:, None] + step
    seen = torch.arange(shared + length, device=DEV) <= shared + last[..., None]
    scores = (q.reshape(batch, kv_heads, group * t, dim) @ k).view(batch, kv_heads, group, t, -1).mul_(s["scale"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(batch, kv_heads, group * t, -1) @ v).view(batch, kv_heads, group, t, dim) / total.clamp(min=1e-30)
    s["o"][token[live]] = out.permute(0, 3, 1, 2, 4).reshape(batch, t, -1)[live].to(torch.bfloat16)
    return s["o"]


# ------------------------------------------------------------------------------------ the definition
def exact(case, seed):
    if case["op"] == "layout":
        return None  # whole numbers
    s = prepare(case, seed)
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    half, group = dim // 2, heads // kv_heads
    if case["op"] == "rope":
        n = case["tokens"]
        angle = torch.stack([s["pos"][int(a)].double() * f for a, f in zip(s["axis"].tolist(), s["inv_freq"].double())], 1)
        unit = torch.polar(torch.ones_like(angle), angle)
        out = []
        for lo, count, weight in ((0, heads, s["q_weight"]), (heads, kv_heads, s["k_weight"])):
            x = s["qkv"][:, lo * dim:(lo + count) * dim].double().view(n, count, dim)
            if weight is not None:
                x = x / ((x ** 2).sum(-1, keepdim=True) / dim + s["eps"]).sqrt() * weight.double()
            z = torch.complex(x[..., :half], x[..., half:]) * unit[:, None]
            out.append(torch.cat([z.real, z.imag], -1).reshape(n, -1))
        k, v = s["k_cache"].double(), s["v_cache"].double()
        k[s["rows"].long()] = out[1]
        v[s["rows"].long()] = s["qkv"][:, (heads + kv_heads) * dim:].double()
        return dict(q_out=out[0], k_cache=k, v_cache=v)
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    start, kv = s["q_start"].tolist(), s["kv_len"].tolist()
    shared = s["prefix"]
    pages = lambda t, length: (t.long()[:, None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(-1)[:length]  # noqa: E731
    front = pages(s["prefix_table"], shared) if shared else torch.zeros(0, dtype=torch.long, device=DEV)
    for b, length in enumerate(kv):
        lo, hi = start[b], start[b + 1]
        if s["table"] is None:
            rows = int(s["k_start"][b]) + torch.arange(length, device=DEV)
        else:
            rows = torch.cat([front, pages(s["table"][b], length)])
        k, v = s["k"][rows].double(), s["v"][rows].double()
        last = torch.arange(shared + length - (hi - lo), shared + length, device=DEV).repeat_interleave(group)
        for h in range(kv_heads):
            mine = slice(h * dim, (h + 1) * dim)
            q = s["q"][lo:hi, h * group * dim:(h + 1) * group * dim].double().reshape(-1, dim)
            x = q @ k[:, mine].T * s["scale"]
            x[torch.arange(shared + length, device=DEV)[None] > last[:, None]] = -math.inf
            o[lo:hi, h * group * dim:(h + 1) * group * dim] = (torch.softmax(x, 1) @ v[:, mine]).reshape(hi - lo, -1)
            del x
    return o
