"""Attention over chosen pages of a paged cache, as a program calls it through this package: what is measured and what is right.

Four calls, one after the other in an attention layer whose tokens read a few pages of a long context each:

    append   head norms, rotation, keys and values into their pages, and the mean key of each page that becomes full
    scores   per token, key/value head and full page: the largest product of the group's queries with the page's mean key
    choose   per token and key/value head: first pages, last pages and the best-scored of the rest, ascending, -1 behind them
    attend   softmax attention of every token over the keys of its chosen pages up to its own position

A case names the call (``call``), the heads and sizes, and the batch (``requests``: ``history+new`` per request; one that brings one
token is a decoded token, one that brings more is a portion of a prompt).  Where ``own`` is false the calls are written out in
elementary torch operations in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------- the cases
def _case(name, call, requests, heads=32, kv_heads=8, dim=128, page=64, top=16, first=1, recent=2, rot=128, style="neox",
          norm=True, dtype="bfloat16"):
    return dict(name=name, call=call, requests=requests, heads=heads, kv_heads=kv_heads, dim=dim, page=page, top=top, first=first,
                recent=recent, rot=rot, style=style, norm=norm, dtype=dtype)


def _decodes(count, lowest, step):
    return ",".join("%d+1" % (lowest + step * i) for i in range(count))


def listed():
    return [
        # one chat on the smallest model of the benchmark: launches count; the token fills its page
        _case("append_chat", "append", "1023+1", heads=16),
        # a step's portions of three prompts: a long one going on inside a page, a new one, the end of another
        _case("append_portions", "append", "7001+2800,0+1203,12222+93"),
        # the 32-bit engine, half of each head turned in neighbouring pairs, no head norm
        _case("append_float32", "append", "100+333,17+1", heads=16, rot=64, style="interleaved", norm=False, dtype="float32"),
        # a loaded server's decode step at contexts all over the range
        _case("scores_decode_b32", "scores", _decodes(32, 700, 1000)),
        # a prompt's portion behind a long history
        _case("scores_portion", "scores", "28672+4096"),
        # a few users' decode step
        _case("choose_decode_b8", "choose", _decodes(8, 3000, 4001)),
        # portions of two long prompts
        _case("choose_portions", "choose", "24000+2500,9000+1596"),
        # one user's long chat
        _case("attend_chat", "attend", "16000+1"),
        # a loaded server's decode step
        _case("attend_decode_b64", "attend", _decodes(64, 300, 499)),
        # a prompt's portion behind a long history: the largest
        _case("attend_portion", "attend", "28672+4096"),
        # a mixed step on other sizes: portions beside decoded tokens, small heads, larger groups, small pages
        _case("attend_mixed", "attend", "9000+1500,0+333,20001+77," + _decodes(9, 1111, 1777), kv_heads=4, dim=64, page=32, top=24, rot=64),
        # the 32-bit engine on a short portion
        _case("attend_float32", "attend", "4000+300", heads=16, dtype="float32"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        call = rng.choice(["append", "scores", "choose", "attend", "attend"])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8])
        dim = rng.choice([64, 128])
        page = rng.choice([16, 32, 64, 64, 128])
        dtype = "float32" if rng.random() < 0.15 else "bfloat16"
        recent, first = rng.randint(1, 4), rng.randint(0, 2)
        top = max(first + recent, _spread(rng, 4, 40))
        form = rng.choice(["decode", "portion", "mixed"])
        requests = []
        if form != "portion":
            requests += ["%d+1" % _spread(rng, 1, 30000) for _ in range(_spread(rng, 1, 64))]
        if form != "decode":
            longest = 400 if dtype == "float32" else 4000
            requests += ["%d+%d" % (_spread(rng, 1, 28000) - 1, _spread(rng, 2, longest)) for _ in range(rng.randint(1, 3))]
        rng.shuffle(requests)
        case = _case("", call, ",".join(requests), heads, kv_heads, dim, page, top, first, recent, rng.choice([dim, dim // 2]),
                     rng.choice(["neox", "interleaved"]), rng.random() < 0.7, dtype)
        del case["name"]
        if _cost(case) <= 1.0:
            return case


def _cost(case):
    """The work of a case's plain form and its state against the largest listed one's."""
    reqs = _requests(case)
    tokens = sum(n for _, n in reqs)
    pages = sum(_pages(h + n, case["page"]) for h, n in reqs)
    most = max(_pages(h + n, case["page"]) for h, n in reqs)
    k = min(case["top"], most)
    state = pages * case["page"] * case["kv_heads"] * case["dim"] / 1.1e9
    read = {"append": 0, "scores": tokens * case["kv_heads"] * most / (4096.0 * 8 * 512),
            "choose": tokens * case["kv_heads"] * most / (4096.0 * 8 * 512),
            "attend": tokens * case["heads"] * k * case["page"] * case["dim"] / (4096.0 * 32 * 1024 * 128)}[case["call"]]
    wide = tokens * case["kv_heads"] * case["dim"] * (most if case["call"] == "scores" else case["page"] * (k if case["call"] == "attend" else 1))
    return max(state, read, tokens / 4096.0, wide / (4096.0 * 8 * 1024 * 128))


def _requests(case):
    return [tuple(int(x) for x in r.split("+")) for r in case["requests"].split(",")]


def _pages(tokens, page):
    return -(-tokens // page)


# ---------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, dev = DTYPES[case["dtype"]], torch.device("cuda")
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rand = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device=dev, dtype=dtype)  # noqa: E731
    reqs = _requests(case)
    T = sum(n for _, n in reqs)
    held = [_pages(h + n, P) for h, n in reqs]
    width = max(held)
    total = sum(held)
    # pages lie in the pool in no order; requests hold what their tokens need
    order = torch.randperm(total + 3, generator=g, device=dev)[:total].to(torch.int32)
    table = torch.full((len(reqs), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    cu = [0]
    for _, n in reqs:
        cu.append(cu[-1] + n)
    positions = torch.cat([torch.arange(h, h + n, dtype=torch.int32) for h, n in reqs]).to(dev)
    request = torch.repeat_interleave(torch.arange(len(reqs)), torch.tensor([n for _, n in reqs])).to(dev)
    s = dict(case=case, T=T, width=width, table=table, cu=torch.tensor(cu, dtype=torch.int32, device=dev), positions=positions,
             request=request, scale=1.0 / math.sqrt(D))
    if case["call"] == "append":
        s["cache"] = rand(total + 3, 2, G, P, D, dtype=dt)
        s["means"] = s["cache"][:, 0].float().mean(2).to(dt)
        s["qkv"] = (2.0 * rand(T, (H + 2 * G) * D)).to(dt)
        s["slots"] = (table[request, (positions // P).long()] * P + positions % P).to(torch.int32)
        s["q_weight"], s["k_weight"] = ((1.0 + 0.1 * rand(D)).to(dt) for _ in range(2)) if case["norm"] else (None, None)
        rot = case["rot"]
        angle = torch.arange(width * P, dtype=torch.float64, device=dev)[:, None] * 1e6 ** (
            -2.0 * torch.arange(rot // 2, dtype=torch.float64, device=dev) / rot)
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        s["q"] = torch.empty(T, H * D, dtype=dt, device=dev)
        return s
    if case["call"] == "scores":
        s["q"] = rand(T, H * D).to(dt)
        s["means"] = (rand(total + 3, G, D) / math.sqrt(P)).to(dt)
        return s
    # scores: part of them the page's own, part shared by a run of tokens, part the token's own, so that neighbours
    # choose much the same pages; an eighth of the pages repeats the page before (repeated text: equal scores)
    own_page, run = rand(len(reqs), G, width), rand(T // 64 + 1, G, width)
    at = torch.arange(T, device=dev)
    scores = rand(T, G, width).mul_(0.7).add_(own_page[request]).add_(run[at // 64])
    scores[:, :, 1:] = torch.where(torch.arange(1, width, device=dev) % 8 == 3, scores[:, :, :-1], scores[:, :, 1:])
    full = (positions // P).long()
    scores.masked_fill_(torch.arange(width, device=dev) >= full[:, None, None], -math.inf)
    if case["call"] == "choose":
        s["scores"] = scores
        return s
    s["chosen"] = _choice(scores, full, case)
    s["q"] = rand(T, H * D).to(dt)
    s["cache"] = rand(total + 3, 2, G, P, D, dtype=dt)
    return s


# ---------------------------------------------------------------- the plain forms
def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)


def _turned(x, cos, sin, style):
    """x [T, heads, D], cos and sin [T, 1, rot / 2]."""
    half = cos.shape[-1]
    y = x.clone()
    if style == "neox":
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
    return y


def _append(s):
    c = s["case"]
    H, G, D, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].float().reshape(s["T"], H + 2 * G, D)
    at = s["cos_sin"][s["positions"].long()][:, None]
    cos, sin = at.chunk(2, -1)
    q = _turned(_normed(x[:, :H], s["q_weight"]), cos, sin, c["style"])
    k = _turned(_normed(x[:, H:H + G], s["k_weight"]), cos, sin, c["style"])
    cache, slots = s["cache"], s["slots"].long()
    cache[slots // P, 0, :, slots % P] = k.to(cache.dtype)
    cache[slots // P, 1, :, slots % P] = x[:, H + G:].to(cache.dtype)
    full = (slots // P)[slots % P == P - 1]
    s["means"][full] = cache[full, 0].float().mean(2).to(cache.dtype)
    return q.reshape(s["T"], H * D).to(cache.dtype), cache, s["means"]


def _scores(s):
    c = s["case"]
    T, G, D, P = s["T"], c["kv_heads"], c["dim"], c["page"]
    pages = s["table"].clamp(min=0).long()[s["request"]]
    q = s["q"].float().reshape(T, G, -1, D)
    got = torch.einsum("tghd,tjgd->tghj", q, s["means"].float()[pages]).amax(2)
    return got.masked_fill_(torch.arange(s["width"], device=q.device) >= (s["positions"] // P)[:, None, None], -math.inf)


def _choice(scores, full, c):
    """int32 [T, G, top] from scores [T, G, N]; a token's own page is ``full``."""
    T, G, N = scores.shape
    j = torch.arange(N, device=scores.device)
    at = full[:, None, None]
    forced = ((j < c["first"]) | (j > at - c["recent"])) & (j <= at)
    rank = torch.where(forced, math.inf, torch.where(j <= at, scores, -math.inf).nan_to_num(nan=-math.inf, posinf=3e38, neginf=-3e38))
    rank = torch.where(j <= at, rank, -math.inf)
    k = min(c["top"], N)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :k]
    best = torch.where(torch.arange(k, device=scores.device) <= at, best, N).sort(-1).values
    out = torch.full((T, G, c["top"]), -1, dtype=torch.int32, device=scores.device)
    out[..., :k] = torch.where(best < N, best, -1).to(torch.int32)
    return out


def _attend(s):
    c = s["case"]
    T, H, G, D, P = s["T"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    chosen = s["chosen"].long()
    pages = s["table"][s["request"][:, None, None], chosen.clamp(min=0)].long().clamp(min=0)
    head = torch.arange(G, device=pages.device)[None, :, None]
    at = chosen[..., None] * P + torch.arange(P, device=pages.device)
    seen = ((at <= s["positions"][:, None, None, None]) & (chosen >= 0)[..., None]).reshape(T, G, 1, -1)
    q = s["q"].float().reshape(T, G, H // G, D)
    score = torch.matmul(q, s["cache"][pages, 0, head].float().reshape(T, G, -1, D).transpose(2, 3)) * s["scale"]
    score = score.masked_fill_(~seen, -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(p, s["cache"][pages, 1, head].float().reshape(T, G, -1, D)) / p.sum(-1, keepdim=True)
    return out.reshape(T, H * D).to(s["q"].dtype)


# ---------------------------------------------------------------- one pass
def run(state):
    s = state
    c = s["case"]
    H, G, D, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if c["call"] == "append":
        if not own:
            return _append(s)
        from dinfer_b200.kernels import page_ops
        page_ops.append(s["qkv"], s["positions"], H, G, D, EPS, s["q_weight"], s["k_weight"], s["cos_sin"], s["q"], s["cache"],
                        s["slots"], s["means"], interleaved=c["style"] == "interleaved")
        return s["q"], s["cache"], s["means"]
    if c["call"] == "scores":
        if not own:
            return _scores(s)
        from dinfer_b200.kernels import page_ops
        return page_ops.page_scores(s["q"], s["means"], s["table"], s["cu"], s["positions"], H, P)
    if c["call"] == "choose":
        if not own:
            return _choice(s["scores"], (s["positions"] // P).long(), c)
        from dinfer_b200.kernels import page_ops
        return page_ops.choose_pages(s["scores"], s["positions"], P, c["top"], first=c["first"], recent=c["recent"])
    if not own:
        return _attend(s)
    from dinfer_b200.kernels import page_ops
    out = torch.empty_like(s["q"])
    return page_ops.attention_pages(s["q"], out, s["cache"], s["table"], s["cu"], s["positions"], s["chosen"], H, s["scale"])


def work(case):
    reqs = _requests(case)
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    e = 4 if case["dtype"] == "float32" else 2
    T = sum(n for _, n in reqs)
    full = [p // P for h, n in reqs for p in range(h, h + n)]        # per token: the full pages before its own
    if case["call"] == "append":
        begun = sum(h % P for h, n in reqs if h % P + n >= P)        # keys of earlier steps in pages that become full
        done = sum((h + n) // P - h // P for h, n in reqs)
        moved = 2 * T * (H + 2 * G) * D + begun * G * D + done * G * D
        return {"bytes": moved * e + T * (case["rot"] + 2) * 4, "flops": T * (H + G) * (3 * D + 3 * case["rot"])}
    width = max(_pages(h + n, P) for h, n in reqs)
    if case["call"] == "scores":
        means = sum((h + n - 1) // P for h, n in reqs) * G * D
        return {"bytes": (T * H * D + means) * e + T * G * width * 4, "flops": 2 * H * D * sum(full)}
    if case["call"] == "choose":
        return {"bytes": 4 * G * (sum(full) + T * case["top"]), "flops": G * sum(full)}
    keys = sum(min(case["top"], f + 1) * P - (P - 1 - p % P) for f, p in zip(full, (p for h, n in reqs for p in range(h, h + n))))
    held = 0
    for h, n in reqs:                                                # pages that some token of the request chose, at most
        held += min(_pages(h + n, P), sum(min(case["top"], p // P + 1) for p in range(h, h + n)))
    return {"bytes": (2 * T * H * D + 2 * held * P * G * D) * e + T * G * case["top"] * 4, "flops": 4 * H * D * keys}


# ---------------------------------------------------------------- the definitions in 64 bits, token by token or head by head
def exact(case, seed):
    s = prepare(case, seed)
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    T, f8 = s["T"], torch.float64
    if case["call"] == "append":
        rot, pos = case["rot"], s["positions"].double()
        i = torch.arange(rot // 2, device=pos.device, dtype=f8)
        angle = torch.outer(pos, torch.exp(-2.0 * i / rot * math.log(1e6)))
        turn = torch.polar(torch.ones_like(angle), angle)            # e^(i angle)

        def finished(x, weight):
            if weight is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * weight.double()
            first, rest = x[..., :rot], x[..., rot:]
            pairs = first.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["style"] == "neox" else first.unflatten(-1, (rot // 2, 2))
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
            z = z.transpose(-1, -2) if case["style"] == "neox" else z
            return torch.cat([z.flatten(-2), rest], -1)

        q, k, v = s["qkv"].double().split([H * D, G * D, G * D], 1)
        q, k = finished(q.unflatten(1, (H, D)), s["q_weight"]), finished(k.unflatten(1, (G, D)), s["k_weight"])
        cache, means = s["cache"].double(), s["means"].double()
        rows = cache.permute(0, 3, 1, 2, 4).reshape(-1, 2, G, D)     # by slot
        rows[s["slots"].long()] = torch.stack([k, v.unflatten(1, (G, D))], 1)
        cache = rows.reshape(-1, P, 2, G, D).permute(0, 2, 3, 1, 4).contiguous()
        ends = {int(x) // P for x in s["slots"].tolist() if int(x) % P == P - 1}
        for page in ends:
            means[page] = cache[page, 0].sum(1) / P
        return q.reshape(T, H * D), cache, means
    cu, table = s["cu"].tolist(), s["table"].tolist()
    if case["call"] == "scores":
        out = torch.full((T, G, s["width"]), -math.inf, dtype=f8, device="cuda")
        for r, (h, n) in enumerate(_requests(case)):
            full = (h + n - 1) // P
            if not full:
                continue
            m = s["means"].double()[table[r][:full]]
            q = s["q"][cu[r]:cu[r + 1]].double().unflatten(1, (G, H // G, D))
            own_page = s["positions"][cu[r]:cu[r + 1]] // P
            for g in range(G):
                best = (q[:, g] @ m[:, g].T).max(1).values
                best[torch.arange(full, device="cuda")[None] >= own_page[:, None]] = -math.inf
                out[cu[r]:cu[r + 1], g, :full] = best
        return out
    if case["call"] == "choose":
        return None
    out = torch.empty(T, G, H // G, D, dtype=f8, device="cuda")
    slab = max(1, (1 << 28) // (case["top"] * P * D))
    for g in range(G):
        for a in range(0, T, slab):
            z = min(T, a + slab)
            chosen = s["chosen"][a:z, g].long()
            pages = s["table"].long()[s["request"][a:z, None], chosen.clamp(min=0)].clamp(min=0)
            k, v = (s["cache"][:, plane, g][pages].double().flatten(1, 2) for plane in (0, 1))
            x = torch.einsum("thd,tkd->thk", s["q"][a:z].double().unflatten(1, (G, H // G, D))[:, g], k) / math.sqrt(D)
            at = (chosen[:, :, None] * P + torch.arange(P, device="cuda")).flatten(1)
            x[((at > s["positions"][a:z, None]) | (at < 0))[:, None].expand_as(x)] = -math.inf
            out[a:z, g] = torch.einsum("thk,tkd->thd", torch.softmax(x, -1), v)
    return out.reshape(T, H * D)
