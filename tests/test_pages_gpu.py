"""Attention over chosen pages, call by call against plain forms in 64 bits, and the calls as a layer makes them."""
import math

import pytest
import torch

from page_cases import (BF16, F32, HALF_STEP, Batch, angles, attention_bound, finished, gen, plain_attention, plain_choice,
                        plain_scores)

pytestmark = pytest.mark.gpu


def c(t):
    return None if t is None else t.cuda()


# requests, page, heads, kv heads, head size
SIZES = [
    ([(0, 1)], 16, 4, 1, 16),
    ([(0, 1), (15, 1), (16, 1), (63, 1), (200, 1)], 16, 8, 2, 64),
    ([(30, 40), (0, 0), (0, 33), (129, 1)], 32, 6, 2, 80),
    ([(63, 66), (0, 64), (500, 7)], 64, 8, 2, 128),
    ([(1000, 130)], 128, 16, 2, 128),
    ([(100, 50), (7, 1)], 24, 5, 5, 48),
    ([(70, 20)], 64, 20, 4, 64),
    ([(90, 9)], 16, 32, 2, 128),
    ([(40, 60)], 32, 3, 1, 256),
]


def qkv_of(b, H, G, D, dtype, g, stride=0):
    x = torch.randn(b.T, (H + 2 * G) * D + stride, generator=g).to(dtype)
    return x, c(x)[:, :(H + 2 * G) * D], x[:, :(H + 2 * G) * D]


@pytest.mark.parametrize("form", ["norm neox", "norm interleaved part", "plain", "neox part wide"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_append(size, dtype, form):
    from dinfer_b200.kernels import page_ops
    requests, P, H, G, D = size
    g = gen(len(form) + D)
    b = Batch(requests, P, seed=1, pad=2)
    _, dev, x = qkv_of(b, H, G, D, dtype, g, stride=0 if form == "plain" else 8)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(F32 if "wide" in form else dtype) for _ in range(2))
    if "norm" not in form:
        wq = wk = None
    rot = 0 if form == "plain" else (D // 4 * 2 if "part" in form else D)
    table = angles(int(b.positions.max()) + 1, rot) if rot else None
    cache0 = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    means0 = torch.randn(b.num_pages, G, D, generator=g).to(dtype)
    cache, means = c(cache0), c(means0)
    q = torch.full((b.T, H * D + 16), 7.0, dtype=dtype, device="cuda")
    for _ in range(2):                                       # a second time gives the same
        page_ops.append(dev, c(b.positions), H, G, D, 1e-6, c(wq), c(wk), c(table), q[:, :H * D], cache, c(b.slots), means,
                        interleaved="interleaved" in form)
    q, cache, means = q.cpu(), cache.cpu(), means.cpu()
    assert (q[:, H * D:] == 7.0).all()
    # a handful of 32-bit operations on elements up to `size`, then one rounding (none where nothing is done)
    noise = 16 * 2.0 ** -24

    def close(got, want, size):
        got = got.double()
        assert bool(((got - want).abs() <= HALF_STEP[dtype] * want.abs() * 1.001 + noise * size + 1e-30).all()), (got - want).abs().max()

    heads = x.double().reshape(b.T, H + 2 * G, D)
    interleaved = "interleaved" in form
    want_cache = cache0.double().clone()
    kept = torch.zeros(b.num_pages, P, dtype=torch.bool)
    for t in range(b.T):
        p, slot = int(b.positions[t]), int(b.slots[t])
        row = table[p] if rot else None
        for h in range(H):
            w = finished(heads[t, h], wq, 1e-6, row, interleaved)
            close(q[t, h * D:(h + 1) * D], w, w.abs().max())
        if slot < 0:
            continue
        page, o = divmod(slot, P)
        kept[page, o] = True
        for k in range(G):
            w = finished(heads[t, H + k], wk, 1e-6, row, interleaved)
            close(cache[page, 0, k, o], w, w.abs().max())
            assert torch.equal(cache[page, 1, k, o], x.reshape(b.T, H + 2 * G, D)[t, H + G + k])
    untouched = ~kept[:, None, None, :, None].expand_as(cache0)
    assert torch.equal(cache[untouched], cache0[untouched])
    full = {int(s) // P for s in b.slots.tolist() if s >= 0 and s % P == P - 1}
    for page in range(b.num_pages):
        if page in full:
            want = cache[page, 0].double().mean(1)
            assert bool(((means[page].double() - want).abs() <= HALF_STEP[dtype] * want.abs() * 1.001
                         + P * 2.0 ** -24 * cache[page, 0].abs().max()).all())
        else:
            assert torch.equal(means[page], means0[page])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 48])
def test_means_do_not_depend_on_the_portions(D, dtype):
    """One prompt whole, token by token and in odd portions: the same cache and the same means, bit by bit."""
    from dinfer_b200.kernels import page_ops
    P, H, G, n = 32, 4, 2, 650
    g = gen(3)
    whole = Batch([(0, n)], P, seed=2)
    x = torch.randn(n, (H + 2 * G) * D, generator=g).to(dtype).cuda()
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda()
    table, slots, positions = angles(n, D).cuda(), c(whole.slots), c(whole.positions)
    got = []
    for cuts in ([n], [1] * n, [31, 2, 30, 1, 40, 46, 500]):
        cache = torch.zeros(whole.num_pages, 2, G, P, D, dtype=dtype, device="cuda")
        means = torch.zeros(whole.num_pages, G, D, dtype=dtype, device="cuda")
        q = torch.empty(n, H * D, dtype=dtype, device="cuda")
        at = 0
        for m in cuts:
            s = slice(at, at + m)
            page_ops.append(x[s], positions[s], H, G, D, 1e-6, w, w, table, q[s], cache, slots[s], means)
            at += m
        got.append((q.cpu(), cache.cpu(), means.cpu()))
    for other in got[1:]:
        for a, z in zip(got[0], other):
            assert torch.equal(a, z)
    assert float(got[0][2].float().abs().sum()) > 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("n", [45, 500, 650])
def test_tokens_of_a_page_in_any_order(n, D, dtype):
    """The rows of a step lie in the batch in any order: the same cache and the same means, bit by bit."""
    from dinfer_b200.kernels import page_ops
    P, H, G, old = 32, 4, 2, 20
    g = gen(n)
    b = Batch([(0, old + n)], P, seed=2)
    x = torch.randn(old + n, (H + 2 * G) * D, generator=g).to(dtype).cuda()
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda()
    table, slots, positions = angles(old + n, D).cuda(), c(b.slots), c(b.positions)
    got = []
    for order in (torch.arange(n), torch.arange(n).flip(0), torch.randperm(n, generator=g)):
        cache = torch.zeros(b.num_pages, 2, G, P, D, dtype=dtype, device="cuda")
        means = torch.zeros(b.num_pages, G, D, dtype=dtype, device="cuda")
        for rows in (torch.arange(old), old + order):
            rows = rows.cuda()
            q = torch.empty(len(rows), H * D, dtype=dtype, device="cuda")
            page_ops.append(x[rows], positions[rows], H, G, D, 1e-6, w, w, table, q, cache, slots[rows], means)
        got.append((cache.cpu(), means.cpu()))
    for other in got[1:]:
        for a, z in zip(got[0], other):
            assert torch.equal(a, z)
    assert int((got[0][1].float().abs().sum((1, 2)) > 0).sum()) == (old + n) // P


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES + [([(1700, 40), (33, 1), (0, 90), (640, 3)], 16, 8, 2, 128), ([(900, 1)] * 9, 16, 4, 2, 64),
                                          ([(2500, 150), (0, 40), (4100, 300)], 16, 8, 2, 128), ([(300, 90)], 16, 5, 5, 64), ([(700, 200)], 32, 10, 2, 64),
                                          ([(600, 70)], 16, 12, 4, 128), ([(520, 66)], 16, 32, 2, 64), ([(0, 64), (64, 64)], 64, 16, 2, 64)], ids=str)
def test_scores(size, dtype):
    from dinfer_b200.kernels import page_ops
    requests, P, H, G, D = size
    g = gen(D)
    b = Batch(requests, P, seed=3, extra_width=5, pad=3)
    if b.width > 7:
        b.table[0, 1] = -1                                   # a page given back
    q = torch.randn(b.T, H * D + 8, generator=g).to(dtype)
    means = (0.2 * torch.randn(b.num_pages, G, D, generator=g)).to(dtype)
    for pages in (b.width, b.width - 5):
        out = torch.full((b.T, G, pages + 3), 5.0, dtype=F32, device="cuda")
        page_ops.page_scores(c(q)[:, :H * D], c(means), c(b.table), c(b.cu), c(b.positions), H, P, out=out[..., :pages], pages=pages)
        got = out.cpu().double()
        assert (got[b.live:] == 5.0).all() and (got[..., pages:] == 5.0).all()
        got = got[:b.live, :, :pages]
        want, size_ = (x[:b.live] for x in plain_scores(q[:, :H * D], means, b, H, pages))
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        fine = torch.isfinite(want)
        # D products summed in 32 bits, each step off by 2^-22 of what has been summed at most
        assert bool(((got - want).abs()[fine] <= (D * 2.0 ** -22 * size_[fine] + 1e-30)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new", [1, 40, 100])
def test_scores_of_what_is_no_number(new, dtype):
    """A NaN or infinity in one query or one mean stays with its own scores; in a page not scored it changes nothing."""
    from dinfer_b200.kernels import page_ops
    P, H, G, D = 16, 8, 2, 64
    b = Batch([(40 * P, new)], P, seed=4)
    g = gen(5)
    q, means = torch.randn(b.T, H * D, generator=g).to(dtype), torch.randn(b.num_pages, G, D, generator=g).to(dtype)
    clean = page_ops.page_scores(c(q), c(means), c(b.table), c(b.cu), c(b.positions), H, P).cpu()
    q[b.T - 1, 3] = math.nan                                 # a head of key head 0
    means[int(b.table[0, 7]), 1, 9] = math.inf
    means[int(b.table[0, (40 * P + new - 1) // P]), 0, 0] = math.nan
    got = page_ops.page_scores(c(q), c(means), c(b.table), c(b.cu), c(b.positions), H, P).cpu()
    want = plain_scores(q, means, b, H, b.width)[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)], want[torch.isinf(want)].float())
    same = torch.isfinite(want)
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("top,first,recent", [(1, 0, 1), (4, 1, 1), (8, 2, 3), (16, 1, 2), (31, 0, 1), (33, 1, 1), (64, 4, 4), (100, 1, 2), (300, 0, 1)])
@pytest.mark.parametrize("pages", [1, 7, 31, 33, 100, 257, 700, 1500, 2100, 5000, 8300, 16500])
def test_choice(pages, top, first, recent):
    from dinfer_b200.kernels import page_ops
    P, T, G = 16, 24, 3
    g = gen(pages + top)
    scores = torch.randn(T, G, pages + 2, generator=g)
    scores[3:6] = scores[3:6].round()                        # many equal scores
    scores[6] = 1.5
    scores[7] = -math.inf
    scores[8, :, ::3] = math.inf
    scores[9, :, ::2] = math.nan
    scores[10] = math.nan
    scores[11] = torch.where(torch.rand(G, pages + 2, generator=g) < 0.5, 0.0, -0.0)
    scores[12, :, 1:] = scores[12, :, :-1] * 1e-42           # numbers below the normal ones
    scores[13] = torch.arange(pages + 2.0)
    scores[14] = -torch.arange(pages + 2.0)
    positions = torch.randint(0, pages * P, (T,), generator=g).to(torch.int32)
    positions[6:15] = pages * P - 1
    positions[0], positions[1], positions[2] = 0, P - 1, -1
    positions[15] = pages * P + 5                            # beyond the scores' last page
    got = page_ops.choose_pages(c(scores)[..., :pages], c(positions), P, top, first=first, recent=recent).cpu()
    assert torch.equal(got, plain_choice(scores[..., :pages], positions, P, top, first, recent))


def choices(b, G, top, g, kind):
    """Hand-made choices: ascending ones in the main, and what else the call allows."""
    out = torch.full((b.T, G, top), -1, dtype=torch.int32)
    for t, (r, p) in enumerate(b.where):
        own = p // b.page
        for k in range(G):
            n = min(top, own + 1)
            picks = sorted(set(torch.randperm(own + 1, generator=g)[:n].tolist()) | ({own} if kind != "far" else set()))[-top:]
            out[t, k, :len(picks)] = torch.tensor(picks, dtype=torch.int32)
    if kind == "odd" and b.live > 1:
        out[0] = -1                                          # nothing
        out[1, :, 0] = out[1, :, -1] = 0                     # the same page twice, in no order
        out[b.live - 1, 0, :] = 10 ** 9                      # no such page
        out[b.live - 1, -1, 0] = b.width - 1                 # behind the token, or not held
    return out


ATTENTION = SIZES + [([(2000, 200), (0, 300)], 16, 8, 2, 128), ([(777, 300)], 64, 16, 1, 64), ([(640, 150)], 32, 12, 4, 128),
                     ([(256, 130), (31, 1), (100, 1), (2, 2)], 64, 8, 8, 128), ([(400, 90)], 128, 4, 2, 64), ([(50, 40)] * 5, 16, 10, 2, 128),
                     ([(3000, 500), (20, 90), (500, 1)], 64, 8, 2, 128), ([(70, 300)], 32, 6, 2, 64), ([(0, 129), (4000, 64)], 16, 32, 2, 64),
                     ([(1, 200)], 16, 3, 3, 128), ([(900, 700)], 64, 8, 1, 64), ([(300, 20), (5, 3)], 64, 48, 3, 128)]


@pytest.fixture(params=["by rule", "together"])
def form(request, monkeypatch):
    """Which kernel runs: the one that the sizes choose, or, wherever it takes the call, the one in which neighbouring tokens walk the
    pages that they chose together (at these sizes the rule seldom takes it)."""
    from dinfer_b200.kernels import page_ops
    calls, real = [], page_ops._call

    def counted(lib, *args):
        calls.append(lib)
        return real(lib, *args)
    monkeypatch.setattr(page_ops, "_call", counted)
    if request.param == "together":
        rule = page_ops._portions
        monkeypatch.setattr(page_ops, "_portions", lambda head: rule(head, True))
        monkeypatch.setattr(page_ops, "PORTION_TOKENS", 1)
    return request.param, calls


@pytest.mark.parametrize("kind", ["usual", "far", "odd"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", ATTENTION, ids=str)
def test_attention(size, dtype, kind, form):
    from dinfer_b200.kernels import page_ops
    requests, P, H, G, D = size
    if dtype == F32 and sum(n for _, n in requests) > 120:
        requests = [(h, min(n, 60)) for h, n in requests]
    g = gen(D + H)
    b = Batch(requests, P, seed=6, extra_width=1, pad=2)
    q = torch.randn(b.T, H * D + 8, generator=g).to(dtype)
    cache = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    seen = torch.zeros(b.num_pages, P, dtype=torch.bool)
    for r, (h, n) in enumerate(requests):
        for p in range(h + n):
            seen[int(b.table[r, p // P]), p % P] = True
    cache.transpose(2, 3).transpose(1, 2)[~seen] = math.nan  # what nobody has written may hold anything
    if kind == "odd" and b.width > 4:
        b.table[0, 1] = -1                                   # a page given back
    chosen = choices(b, G, 5, g, kind)
    out = torch.full((b.T, H * D + 8), 3.0, dtype=dtype, device="cuda")
    scale = D ** -0.5
    page_ops.attention_pages(c(q)[:, :H * D], out[:, :H * D], c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, scale)
    got = out.cpu()
    assert (got[b.live:] == 3.0).all() and (got[:, H * D:] == 3.0).all()
    want, size_, qk = plain_attention(q[:, :H * D], cache, b, chosen, H, scale)
    off = (got[:b.live, :H * D].double() - want).abs()
    bound = attention_bound(dtype, D, want, size_, qk)
    assert bool((off <= bound).all()), float((off / bound).max())
    if form[0] == "together" and dtype == BF16 and D in (64, 128) and P in (16, 32, 64, 128) and b.T > len(requests):
        assert form[1] == ["attention_pages_umma"]


@pytest.mark.parametrize("requests", [[(700, 1)], [(300, 1)] * 40 + [(0, 1), (23, 1)], [(500, 3), (0, 0), (90, 30), (7, 1)]], ids=["one", "many", "mixed"])
@pytest.mark.parametrize("P,H,G,D", [(8, 2, 2, 128), (24, 6, 3, 64), (40, 6, 2, 128), (64, 5, 1, 64), (16, 16, 2, 128), (200, 8, 1, 128),
                                     (64, 18, 2, 128), (12, 4, 2, 64), (64, 6, 2, 96), (33, 3, 1, 512)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_single_tokens(requests, P, H, G, D, dtype):
    """Groups of one to nine heads, pages of any length, a token alone (a cluster shares its keys) and many."""
    from dinfer_b200.kernels import page_ops
    g = gen(P + H)
    b = Batch(requests, P, seed=P, extra_width=1, pad=1)
    q, cache = torch.randn(b.T, H * D, generator=g).to(dtype), torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    seen = torch.zeros(b.num_pages, P, dtype=torch.bool)
    for r, (h, n) in enumerate(requests):
        for p in range(h + n):
            seen[int(b.table[r, p // P]), p % P] = True
    cache.transpose(2, 3).transpose(1, 2)[~seen] = math.inf
    chosen = choices(b, G, 7, g, "odd")
    out = torch.full((b.T, H * D), 3.0, dtype=dtype, device="cuda")
    page_ops.attention_pages(c(q), out, c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, D ** -0.5)
    got = out.cpu()
    assert (got[b.live:] == 3.0).all()
    want, size_, qk = plain_attention(q, cache, b, chosen, H, D ** -0.5)
    bound = attention_bound(dtype, D, want, size_, qk)
    off = (got[:b.live].double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("new", [1, 5, 100, 400])
@pytest.mark.parametrize("what", ["value", "key"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_token_sees_a_later_one(dtype, what, new, form):
    """A NaN in a token's own key or value reaches the tokens from it on that read its page, and nothing before or beside: those are
    what they are without it, up to the bound that every result keeps (the kernel for portions makes the rows beside such a value
    again, one by one, with sums in another order)."""
    from dinfer_b200.kernels import page_ops
    if dtype == F32 and new > 100:
        new = 100
    P, H, G, D = 64, 8, 2, 128
    g = gen(new)
    b = Batch([(100, new), (40, 3)], P, seed=8)
    q = torch.randn(b.T, H * D, generator=g).to(dtype)
    cache = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    chosen = choices(b, G, 3, g, "usual")
    args = (c(b.table), c(b.cu), c(b.positions), c(chosen), H, 0.1)
    clean, size, qk = plain_attention(q, cache, b, chosen, H, 0.1)
    at = 100 + new // 2
    cache[int(b.table[0, at // P]), 0 if what == "key" else 1, 1, at % P, 7] = math.nan
    got = page_ops.attention_pages(c(q), torch.empty_like(c(q)), c(cache), *args).cpu()
    reaches = torch.tensor([r == 0 and p >= at and at // P in chosen[t, 1].tolist() for t, (r, p) in enumerate(b.where)])
    heads = torch.arange(H * D) // D >= H // G
    hit = reaches[:, None] & heads[None] & (torch.ones(H * D, dtype=torch.bool) if what == "key" else torch.arange(H * D) % D == 7)
    assert torch.equal(torch.isnan(got), hit)
    assert bool(((got.double() - clean).abs() <= attention_bound(dtype, D, clean, size, qk))[~hit].all())


@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores(dtype, new, form):
    """Scores far apart (a softmax that keeps one key) and far from zero, and keys of the type's lowest value."""
    from dinfer_b200.kernels import page_ops
    P, H, G, D = 32, 8, 2, 64
    if dtype == F32:
        new = min(new, 50)
    g = gen(9)
    b = Batch([(300, new)], P, seed=9)
    q = (40 * torch.randn(b.T, H * D, generator=g)).to(dtype)
    cache = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    cache[:, 0] *= 30
    chosen = choices(b, G, 6, g, "usual")
    got = page_ops.attention_pages(c(q), torch.empty_like(c(q)), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, 1.0).cpu()
    want, size, qk = plain_attention(q, cache, b, chosen, H, 1.0)
    bound = attention_bound(dtype, D, want, size, qk)
    assert bool(((got.double() - want).abs() <= bound).all())
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_layer_prompt_whole_and_token_by_token(dtype, form):
    """The four calls as a layer makes them: a prompt in portions and then single tokens, beside another request, against the plain
    form of every token on the cache and means that were built."""
    from dinfer_b200.kernels import page_ops
    P, H, G, D, top = 16, 8, 2, 64, 4
    g = gen(11)
    lens = [200, 90]
    end = Batch([(n, 0) for n in lens], P, seed=10)
    rows = [torch.randn(n, (H + 2 * G) * D, generator=g).to(dtype) for n in lens]
    w = torch.ones(D, dtype=dtype)
    table = angles(max(lens), D)
    cache = torch.zeros(end.num_pages, 2, G, P, D, dtype=dtype, device="cuda")
    means = torch.zeros(end.num_pages, G, D, dtype=dtype, device="cuda")
    at = [0, 0]
    for step in ([150, 0], [1, 60], [0, 7], [40, 1], [1, 1], [1, 1], [7, 20]):
        b = Batch([(a, n) for a, n in zip(at, step)], P, seed=10)
        b.table, b.width, b.num_pages = end.table, end.width, end.num_pages
        b.slots = torch.tensor([int(b.table[r, p // P]) * P + p % P for r, p in b.where], dtype=torch.int32)
        x = torch.cat([rows[r][a:a + n] for r, (a, n) in enumerate(zip(at, step))])
        q = torch.empty(b.T, H * D, dtype=dtype, device="cuda")
        dev = (c(b.table), c(b.cu), c(b.positions))
        page_ops.append(c(x), dev[2], H, G, D, 1e-6, c(w), c(w), c(table), q, cache, c(b.slots), means)
        scores = page_ops.page_scores(q, means, *dev, H, P)
        chosen = page_ops.choose_pages(scores, dev[2], P, top, first=1, recent=2)
        out = page_ops.attention_pages(q, torch.empty_like(q), cache, *dev, chosen, H, D ** -0.5)
        want, size = plain_scores(q.cpu(), means.cpu(), b, H, b.width)
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(scores.cpu()), fine)
        assert bool(((scores.cpu().double() - want).abs()[fine] <= D * 2.0 ** -22 * size[fine]).all())
        assert torch.equal(chosen.cpu(), plain_choice(scores.cpu(), b.positions, P, top, 1, 2))
        want, size, qk = plain_attention(q.cpu(), cache.cpu(), b, chosen.cpu(), H, D ** -0.5)
        assert bool(((out.cpu().double() - want).abs() <= attention_bound(dtype, D, want, size, qk)).all())
        at = [a + n for a, n in zip(at, step)]


@pytest.mark.parametrize("new", [[(700, 1), (90, 1), (300, 1)], [(700, 200), (90, 1), (0, 90)]])
def test_replayed_from_a_graph_on_another_stream(new, form):
    """The four calls captured once and replayed on other inputs, and eager calls on a stream of their own: the same as eager."""
    from dinfer_b200.kernels import page_ops
    P, H, G, D, top = 32, 8, 2, 128, 6
    b = Batch(new, P, seed=12)
    T = b.T
    dev = (c(b.table), c(b.cu), c(b.positions))
    slots, table, w = c(b.slots), angles(1000, D).cuda(), torch.ones(D, dtype=BF16, device="cuda")
    x = torch.empty(T, (H + 2 * G) * D, dtype=BF16, device="cuda")
    cache0 = torch.randn(b.num_pages, 2, G, P, D, generator=gen(1)).to(BF16).cuda()
    means0 = cache0[:, 0].float().mean(2).to(BF16)
    cache, means = cache0.clone(), means0.clone()

    def layer():
        q = torch.empty(T, H * D, dtype=BF16, device="cuda")
        page_ops.append(x, dev[2], H, G, D, 1e-6, w, w, table, q, cache, slots, means)
        scores = page_ops.page_scores(q, means, *dev, H, P)
        chosen = page_ops.choose_pages(scores, dev[2], P, top, first=1, recent=2)
        return page_ops.attention_pages(q, torch.empty_like(q), cache, *dev, chosen, H, D ** -0.5)

    inputs = [torch.randn(T, (H + 2 * G) * D, generator=gen(s)).to(BF16).cuda() for s in (1, 2, 3)]
    want = []
    for i in inputs:
        x.copy_(i)
        cache.copy_(cache0), means.copy_(means0)
        want.append(layer().clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.copy_(inputs[1])
        cache.copy_(cache0), means.copy_(means0)
        assert torch.equal(layer(), want[1])
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                       # two graphs of the same call share one pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = layer()
        graphs.append((graph, out))
    for i, wanted in list(zip(inputs, want)) * 2:
        for graph, out in graphs:
            x.copy_(i)
            cache.copy_(cache0), means.copy_(means0)
            graph.replay()
            assert torch.equal(out, wanted)


def test_another_device_is_refused(monkeypatch):
    """Tensors off the current device are refused by name, not read."""
    from dinfer_b200.kernels import page_ops
    from dinfer_b200.kernels.lib import KernelError
    x = torch.zeros(1, 1, 4, device="cuda")
    monkeypatch.setattr(page_ops, "_device", lambda: 1)
    with pytest.raises(KernelError, match="current device is 1"):
        page_ops.choose_pages(x, torch.zeros(1, dtype=torch.int32, device="cuda"), 16, 4)


def test_no_tokens():
    from dinfer_b200.kernels import page_ops
    H, G, D, P = 4, 2, 64, 16
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")          # noqa: E731
    i = lambda *s: z(*s, dtype=torch.int32)                                          # noqa: E731
    q, cache, means = z(0, H * D), z(3, 2, G, P, D), z(3, G, D)
    page_ops.append(z(0, (H + 2 * G) * D), i(0), H, G, D, 1e-6, None, None, None, q, cache, i(0), means)
    s = page_ops.page_scores(q, means, i(1, 3), i(2), i(0), H, P)
    chosen = page_ops.choose_pages(s, i(0), P, 4)
    assert page_ops.attention_pages(q, z(0, H * D), cache, i(1, 3), i(2), i(0), chosen, H, 0.1).shape == (0, H * D)
    torch.cuda.synchronize()
