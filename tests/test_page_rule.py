"""Which kernel attention over chosen pages runs on (no GPU needed: the calls end where the library would be called)."""
import pytest
import torch

from dinfer_b200.kernels import page_ops

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def kernel_of(monkeypatch):
    """The kernel library that a call names, for tensors that lie nowhere in particular."""
    got = []
    monkeypatch.setattr(page_ops, "_here", lambda what, *tensors: None)
    monkeypatch.setattr(page_ops, "_device", lambda: 0)
    monkeypatch.setattr(page_ops, "_multiprocessors", lambda: 148)
    monkeypatch.setattr(page_ops, "_call", lambda lib, *args: got.append(lib))
    monkeypatch.setattr(page_ops.gemm_ops, "_state", lambda device: {"status": torch.zeros(1, dtype=torch.int32)})

    def kernel(new, history, H, G, D, top, page, dtype=BF16, scale=0.1, pages=None):
        T, B, width = sum(new), len(new), -(-(history + max(new)) // page)
        i = lambda *s: torch.zeros(*s, dtype=torch.int32)                            # noqa: E731
        cache = torch.empty(2 if pages is None else pages, 2, G, page, D, dtype=dtype)
        q = torch.empty(T, H * D, dtype=dtype)
        page_ops.attention_pages(q, torch.empty_like(q), cache, i(B, width), i(B + 1), i(T), i(T, G, top), H, scale)
        assert len(got) == 1
        return got.pop()
    return kernel


# new tokens of the requests, history, heads, kv heads, head size, pages a token reads, tokens of a page
@pytest.mark.parametrize("call,wanted", [
    # the tensor-core kernel for tokens against neighbours together
    (([1], 16000, 32, 8, 128, 16, 64), "attention_pages"), (([1] * 64, 8000, 32, 8, 128, 16, 64), "attention_pages"),
    (([4096], 28672, 32, 8, 128, 16, 64), "attention_pages_umma"), (([256], 8000, 32, 8, 128, 16, 64), "attention_pages_umma"),
    (([16], 8000, 32, 8, 128, 16, 64), "attention_pages"), (([64] + [1] * 16, 8000, 32, 8, 128, 16, 64), "attention_pages"),
    # groups above 16 heads or more than 1024 pages: there is only the kernel for any sizes token by token, which is longer from few
    # tokens on
    (([100], 8000, 64, 1, 128, 16, 64), "attention_pages_umma"), (([300], 8000, 64, 1, 128, 16, 64), "attention_pages_umma"),
    (([2], 8000, 64, 1, 128, 16, 64), "attention_pages_umma"), (([1] * 24, 8000, 64, 1, 128, 16, 64), "attention_pages_umma"),
    (([100], 8000, 40, 2, 128, 16, 64), "attention_pages_umma"), (([300], 8000, 128, 1, 128, 8, 64), "attention_pages_umma"),
    (([300], 8000, 48, 2, 64, 4, 64), "attention_pages_umma"), (([2], 20000, 8, 2, 128, 1100, 16), "attention_pages_umma"),
    (([100], 20000, 8, 2, 128, 1100, 16), "attention_pages_umma"),
    (([2], 8000, 24, 1, 64, 8, 16), "attention_pages"), (([24], 8000, 24, 1, 64, 8, 16), "attention_pages"), (([100], 8000, 24, 1, 64, 8, 16), "attention_pages_umma"),
    # what the kernel of neighbours does not take
    (([300], 8000, 129, 1, 128, 16, 64), "attention_pages"), (([300], 8000, 64, 1, 80, 16, 64), "attention_pages"),
    (([300], 8000, 64, 1, 128, 16, 24), "attention_pages"), (([300], 8000, 64, 1, 128, 16, 64, F32), "attention_pages")], ids=str)
def test_which_kernel_runs(kernel_of, call, wanted):
    assert kernel_of(*call) == wanted


@pytest.mark.parametrize("more", [dict(pages=0), dict(scale=1e-46), dict(scale=0.0), dict(scale=-1.0)], ids=str)
def test_a_cache_without_pages_and_a_scale_that_is_no_positive_number(kernel_of, more):
    """The kernel of neighbouring tokens refuses them: the others give zeros, and weights that are right."""
    assert kernel_of([256], 8000, 32, 8, 128, 16, 64, **more) == "attention_pages"


@pytest.mark.parametrize("top,takes", [(1 << 20, True), ((1 << 23) - 1, True), (1 << 23, False), (1 << 30, False)])
def test_tokens_times_pages_beyond_31_bits(top, takes):
    """The lists of a block's 256 tokens count their tokens' entries in 32 bits: a call with more goes to the other kernels."""
    from dinfer_b200.kernels.lib import library
    f = library("attention_pages_umma").dinfer_attention_pages_umma_workspace
    f.argtypes, f.restype = [page_ops.c_int] * 9, page_ops.c_int64
    assert (f(1, 5000, top, 300, 1, 1, 64, 16, 0) > 0) is takes      # 256 tokens of one head


@pytest.mark.parametrize("call,refused", [
    ("the same", True), ("a row further", True), ("half a row further", True), ("half a row before", True), ("columns that meet", True),
    ("columns side by side", False), ("columns the other way", False), ("behind", False), ("rows of another width", True), ("one token", True),
    ("one token beside", False)])
def test_outputs_over_queries(monkeypatch, call, refused):
    """A row may be made twice, and blocks read queries while others write: no part of ``out`` may lie on ``q``."""
    from dinfer_b200.kernels.lib import KernelError
    H, G, D, page, T = 4, 2, 64, 16, 5
    w, launched = H * D, []
    monkeypatch.setattr(page_ops, "_here", lambda what, *tensors: None)
    monkeypatch.setattr(page_ops, "_device", lambda: 0)
    monkeypatch.setattr(page_ops, "_call", lambda lib, *args: launched.append(lib))
    x = torch.zeros(T * 4 * w, dtype=BF16)
    rows = lambda at, ld, n=T: x[at:].as_strided((n, w), (ld, 1), at)                # noqa: E731
    q, out = {"the same": (rows(0, w), rows(0, w)), "a row further": (rows(0, w), rows(w, w)), "half a row further": (rows(0, w), rows(w // 2, w)),
              "half a row before": (rows(w // 2, w), rows(0, w)), "columns that meet": (rows(0, 3 * w), rows(w - 8, 3 * w)),
              "columns side by side": (rows(0, 2 * w), rows(w, 2 * w)), "columns the other way": (rows(2 * w, 3 * w), rows(w, 3 * w)),
              "behind": (rows(0, w), rows(T * w, w)), "rows of another width": (rows(0, 2 * w), rows(w, 3 * w)),
              "one token": (rows(0, 7, 1), rows(8, 9, 1)), "one token beside": (rows(0, w, 1), rows(w, w, 1))}[call]
    n = q.shape[0]
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)                                # noqa: E731
    args = (q, out, torch.zeros(2, 2, G, page, D, dtype=BF16), i(1, 3), i(2), i(n), i(n, G, 4), H, 0.1)
    if refused:
        with pytest.raises(KernelError, match="out must not be q's memory"):
            page_ops.attention_pages(*args)
    else:
        page_ops.attention_pages(*args)
    assert len(launched) == (not refused)
