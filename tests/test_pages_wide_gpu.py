"""Attention over chosen pages on groups of many heads and lists of many pages: the kernel in which neighbouring tokens walk their pages
together, as the rule gives calls to it, with lists beyond what its shared memory holds."""
import math

import pytest
import torch

from page_cases import BF16, Batch, attention_bound, gen, plain_attention
from test_pages_gpu import c, choices

pytestmark = pytest.mark.gpu


@pytest.fixture
def libraries(monkeypatch):
    """The kernel libraries that calls run on."""
    from dinfer_b200.kernels import page_ops
    got, real = [], page_ops._call

    def counted(lib, *args):
        got.append(lib)
        return real(lib, *args)
    monkeypatch.setattr(page_ops, "_call", counted)
    return got


def compare(b, q, cache, chosen, H):
    from dinfer_b200.kernels import page_ops
    D = cache.shape[-1]
    got = page_ops.attention_pages(c(q), torch.full_like(c(q), 3.0), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, D ** -0.5).cpu()
    assert (got[b.live:] == 3.0).all()
    want, size, qk = plain_attention(q, cache, b, chosen, H, D ** -0.5)
    off, bound = (got[:b.live].double() - want).abs(), attention_bound(BF16, D, want, size, qk)
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("requests,page,H,G,D,top", [
    ([(700, 1)], 64, 64, 1, 128, 16), ([(700, 1)] * 5 + [(0, 1), (63, 1)], 64, 80, 2, 128, 16), ([(3000, 9)], 64, 64, 1, 128, 40),
    ([(900, 30), (1500, 1), (20, 1)], 32, 48, 2, 64, 24), ([(2000, 60), (0, 0), (0, 5)], 16, 17, 1, 128, 100), ([(300, 20)], 128, 128, 1, 64, 3),
    ([(20000, 2)], 16, 4, 2, 64, 1100), ([(17000, 1)] * 2, 16, 2, 2, 128, 1030)], ids=str)
@pytest.mark.parametrize("kind", ["usual", "odd"])
def test_what_the_kernel_for_tokens_does_not_take(requests, page, H, G, D, top, kind, libraries):
    """Groups above 16 heads, more than 1024 pages: single tokens and portions, by rule."""
    g = gen(H + page)
    b = Batch(requests, page, seed=41, extra_width=1, pad=1)
    q, cache = torch.randn(b.T, H * D, generator=g).to(BF16), torch.randn(b.num_pages, 2, G, page, D, generator=g).to(BF16)
    if kind == "odd":
        b.table[0, 1] = -1
    compare(b, q, cache, choices(b, G, top, g, kind), H)
    assert libraries == ["attention_pages_umma"]


@pytest.mark.parametrize("new", [1, 300])
def test_a_cache_without_pages(new):
    """Nothing is held, so nothing is seen: zeros, however many tokens."""
    from dinfer_b200.kernels import page_ops
    H, G, D, P = 8, 2, 128, 64
    b = Batch([(900, new)], P, seed=42, pad=1)
    q, cache = torch.randn(b.T, H * D, generator=gen(1)).to(BF16), torch.empty(0, 2, G, P, D, dtype=BF16)
    chosen = choices(b, G, 16, gen(2), "usual")
    got = page_ops.attention_pages(c(q), torch.full_like(c(q), 3.0), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, 0.1).cpu()
    assert (got[:b.live] == 0).all() and (got[b.live:] == 3.0).all()


@pytest.mark.parametrize("scale", [1e-46, 1e-41, 0.0, -0.1])
@pytest.mark.parametrize("new", [1, 300])
def test_scales_that_are_not_positive_in_32_bits(new, scale):
    from dinfer_b200.kernels import page_ops
    H, G, D, P = 8, 2, 128, 64
    b = Batch([(900, new)], P, seed=43)
    g = gen(3)
    q, cache = torch.randn(b.T, H * D, generator=g).to(BF16), torch.randn(b.num_pages, 2, G, P, D, generator=g).to(BF16)
    chosen = choices(b, G, 16, g, "usual")
    got = page_ops.attention_pages(c(q), torch.empty_like(c(q)), c(cache), c(b.table), c(b.cu), c(b.positions), c(chosen), H, scale).cpu()
    want, size, qk = plain_attention(q, cache, b, chosen, H, scale)
    assert bool(((got.double() - want).abs() <= attention_bound(BF16, D, want, size, qk.abs())).all())


@pytest.mark.parametrize("new", [3, 16])
def test_scores_of_more_pages_than_a_grid_counts_by_the_128(new):
    """8388481 pages of one token: the kernel with 128 pages a block would need more blocks than a launch may have."""
    from dinfer_b200.kernels import page_ops
    D, pages = 64, 128 * 65535 + 1
    table = torch.full((1, pages), -1, dtype=torch.int32)
    places = [0, 127, 128, 5000, pages // 2, pages - 2, pages - 1]
    table[0, places] = torch.arange(len(places), dtype=torch.int32)
    g = gen(5)
    q, means = torch.randn(new, D, generator=g).to(BF16), torch.randn(len(places), 1, D, generator=g).to(BF16)
    positions = torch.full((new,), pages - 1, dtype=torch.int32)
    positions[0] = 5000
    got = page_ops.page_scores(c(q), c(means), c(table), c(torch.tensor([0, new], dtype=torch.int32)), c(positions), 1, 1)[:, 0]
    want = (q.double() @ means[:, 0].double().T).masked_fill(torch.tensor(places)[None] >= positions[:, None], -math.inf)
    size = q.double().abs() @ means[:, 0].double().abs().T
    found = got[:, c(torch.tensor(places))].cpu().double()
    assert torch.equal(torch.isinf(found), torch.isinf(want))
    fine = torch.isfinite(want)
    assert bool(((found - want).abs()[fine] <= D * 2.0 ** -22 * size[fine]).all())
    assert int(torch.isfinite(got).sum()) == int(fine.sum())


# heads, kv heads, page, history, new tokens: lists of more entries than shared memory holds (256 for a group of one head, 1024 for four
# and more) of contexts of more pages than one window of the lists' kernel (1024 and 4096)
LONG = [(2, 2, 16, 40000, 300, 64), (16, 4, 16, 70000, 1300, 64), (2, 2, 32, 40000, 270, 128)]


@pytest.mark.parametrize("H,G,page,history,new,D", LONG)
@pytest.mark.parametrize("kind", ["usual", "odd"])
def test_long_lists_over_several_windows(H, G, page, history, new, D, kind, libraries, monkeypatch):
    """Prompt portions far along, 40 chosen pages of a token all over the context; odd: pages of the second window that are not held, and
    one that a token names twice."""
    from dinfer_b200.kernels import page_ops
    rule = page_ops._portions
    monkeypatch.setattr(page_ops, "_portions", lambda head: rule(head, True))
    g = gen(H + new)
    b = Batch([(history, new), (0, 3)], page, seed=44, extra_width=1)
    window = 1024 if H == G else 4096
    assert b.width > window + 100 or page != 16
    q, cache = torch.randn(b.T, H * D, generator=g).to(BF16), torch.randn(b.num_pages, 2, G, page, D, generator=g).to(BF16)
    chosen = choices(b, G, 40, g, "far")
    far = history // page
    if kind == "odd":
        b.table[0, far - 50:far - 20] = -1
        chosen[new // 2, :, 3] = chosen[new // 2, :, 30] = far - 5
        chosen[new - 1, :, 7] = far - 30
    compare(b, q, cache, chosen, H)
    assert libraries == ["attention_pages_umma"]
