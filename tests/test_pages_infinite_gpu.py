"""Attention over chosen pages where scores are infinite or large: what the softmax makes of them."""
import math

import pytest
import torch

from page_cases import BF16, F32, Batch, attention_bound, gen, plain_attention
from test_pages_gpu import c, choices, form  # noqa: F401  (form: a fixture)

pytestmark = pytest.mark.gpu

# requests, page, heads, kv heads, head size: together, blocks of a cluster share a list where the context is long
SIZES = [([(700, 1)], 64, 8, 2, 128), ([(300, 40), (0, 30)], 64, 8, 2, 128), ([(3000, 40), (90, 1)], 64, 8, 2, 128), ([(2000, 70)], 16, 16, 2, 64),
         ([(500, 30)], 32, 4, 4, 64), ([(200, 1)] * 30, 32, 6, 2, 64), ([(90, 9), (0, 20)], 24, 6, 2, 80), ([(900, 1)], 16, 2, 1, 256)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_scores_of_minus_infinity(size, dtype, form):  # noqa: F811
    """Every key of a page scores -inf with every query of a key head: beside other pages it has no weight; a token that sees such
    keys alone gets what is not a number, a token that sees none gets zeros, and nothing else changes."""
    from dinfer_b200.kernels import page_ops
    requests, P, H, G, D = size
    g = gen(D + P)
    b = Batch(requests, P, seed=31, pad=1)
    q = torch.randn(b.T, H, D, generator=g)
    q[..., 3] = q[..., 3].abs() + 0.25
    q = q.reshape(b.T, H * D).to(dtype)
    cache = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    chosen = choices(b, G, 5, g, "usual")
    for t in range(0, b.live, 3):                            # the first page alone; every ninth token nothing
        chosen[t] = -1
        if t % 9:
            chosen[t, :, 1] = 0
        elif t % 2:
            chosen[t, :, 0] = b.width                        # (no such page)
    if b.live == 1:
        chosen[0, 0] = torch.tensor([0, -1, -1, -1, -1])
    finite = plain_attention(q, cache, b, chosen, H, 0.2)[2]
    for r in range(len(requests)):
        cache[int(b.table[r, 0]), 0, 0, :, 3] = -math.inf    # key head 0 only
    want, size_, _ = plain_attention(q, cache, b, chosen, H, 0.2)
    assert bool(torch.isnan(want).any()) and not bool(torch.isnan(want[:, (H // G) * D:]).any())
    got = page_ops.attention_pages(c(q), torch.full_like(c(q), 3.0), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, 0.2).cpu()
    assert (got[b.live:] == 3.0).all()
    got, nan = got[:b.live].double(), torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert bool(((got - want).abs() <= attention_bound(dtype, D, want, size_, finite))[~nan].all())


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -9])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_scores_of_whole_numbers(size, dtype, scale, form):  # noqa: F811
    """Queries and keys of whole numbers, so that every partial sum of a score is one below 2^24 and exact in 32 bits in any order, cut off or
    rounded, and the scale a power of two.  What is off then is the score's way through the exponential (log2 e times the scale, the
    product, the maximum taken off: less than 8 x 2^-24 of the largest score), not the sum of its D products: a bound of a few percent
    where scores lie thousands apart, of a rounding where many keys have weight."""
    from dinfer_b200.kernels import page_ops
    requests, P, H, G, D = size
    g = gen(D + P + 1)
    b = Batch(requests, P, seed=32, pad=1)
    q = torch.randint(-40, 41, (b.T, H * D), generator=g).to(dtype)
    cache = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    cache[:, 0] = torch.randint(-30, 31, (b.num_pages, G, P, D), generator=g).to(dtype)
    chosen = choices(b, G, 5, g, "usual")
    got = page_ops.attention_pages(c(q), torch.full_like(c(q), 3.0), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, scale).cpu()
    assert (got[b.live:] == 3.0).all()
    want, size_, qk = plain_attention(q, cache, b, chosen, H, scale)
    assert float(qk.max()) / scale < 2 ** 24
    bound = attention_bound(dtype, 1, want, size_, 1.4427 * qk)          # 2 x 2^-22 of the largest score instead of 2 D x 2^-22
    assert bool((bound <= (0.08 if dtype == F32 else 0.09) * size_ + 1e-30).all())
    off = (got[:b.live].double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_a_score_of_infinity(size, dtype, form):  # noqa: F811
    """One key scores +inf with every query of a key head: infinity over infinity for the tokens that see it, nothing for the others."""
    from dinfer_b200.kernels import page_ops
    requests, P, H, G, D = size
    g = gen(D + P + 2)
    b = Batch(requests, P, seed=33, pad=1)
    q = torch.randn(b.T, H, D, generator=g)
    q[..., 3] = q[..., 3].abs() + 0.25
    q = q.reshape(b.T, H * D).to(dtype)
    cache = torch.randn(b.num_pages, 2, G, P, D, generator=g).to(dtype)
    chosen = choices(b, G, 5, g, "usual")
    finite = plain_attention(q, cache, b, chosen, H, 0.2)[2]
    for r, (h, n) in enumerate(requests):
        at = h + n // 2
        cache[int(b.table[r, at // P]), 0, G - 1, at % P, 3] = math.inf
    want, size_, _ = plain_attention(q, cache, b, chosen, H, 0.2)
    got = page_ops.attention_pages(c(q), torch.full_like(c(q), 3.0), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, 0.2).cpu()
    assert (got[b.live:] == 3.0).all()
    got, nan = got[:b.live].double(), torch.isnan(want)
    assert bool(nan.any()) and torch.equal(torch.isnan(got), nan)
    assert bool(((got - want).abs() <= attention_bound(dtype, D, want, size_, finite))[~nan].all())
