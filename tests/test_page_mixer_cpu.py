"""What the page-attention mixer hands to its calls (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from dinfer_b200.kernels import page_ops
from dinfer_b200.parts import page_attention  # noqa: F401  (registers the mixer)
from dinfer_b200.parts.base import MIXERS, BuildEnv, CacheBinding

HEADS, KV_HEADS, DIM, PAGE, TOKENS = 4, 2, 16, 16, 5


@pytest.fixture
def calls(monkeypatch):
    """The four calls' names and arguments in order; nothing is computed."""
    got = []
    for name in ("append", "page_scores", "choose_pages", "attention_pages"):
        monkeypatch.setattr(page_ops, name, lambda *a, _name=name, **k: got.append((_name, a, k)))
    return got


def mixer_and_step(page=PAGE):
    m = MIXERS.get("page_attention")(dict(num_heads=HEADS, num_kv_heads=KV_HEADS, head_dim=DIM, top=4, page=page),
                                     BuildEnv(torch.device("cpu"), torch.float32, 64, 128))
    m.qkv = lambda x: torch.zeros(x.shape[0], (HEADS + 2 * KV_HEADS) * DIM)
    m.o = lambda x: x
    group = SimpleNamespace(slot_mapping=torch.arange(TOKENS, dtype=torch.int32), block_table=torch.zeros(1, 8, dtype=torch.int32))
    ctx = SimpleNamespace(groups=[group], derived={}, positions=torch.arange(TOKENS, dtype=torch.int32),
                          cu_seqlens=torch.tensor([0, TOKENS], dtype=torch.int32), decode_splits=0, max_seq_len=TOKENS)
    return m, ctx


def binding(write=True, page=PAGE, means=True):
    kv = torch.zeros(3, 2, KV_HEADS, page, DIM)
    return CacheBinding(kv=kv, group=0, write=write, means=torch.zeros(3, KV_HEADS, DIM) if means else None)


def tensors_of(value):
    if isinstance(value, torch.Tensor):
        return [value]
    if isinstance(value, dict):
        value = value.values()
    return [t for v in value for t in tensors_of(v)] if not isinstance(value, (int, float, str, bool, type(None))) else []


def test_a_layer_that_reads_anothers_cache_keeps_no_tensor_beyond_its_run(calls):
    """A step's context may run several times, a graph's warm-up before its capture among them.  What one run makes is not there for the
    next: a graph that recorded the address of a warm-up's tensor would read memory that has gone back."""
    m, ctx = mixer_and_step()
    cache = binding(write=False)
    slots = []
    for _ in range(3):
        m.forward(torch.zeros(TOKENS, 64), ctx, cache)
        name, args, _ = calls[-4]
        assert name == "append"
        slots.append(args[11])
        assert torch.equal(slots[-1], torch.full((TOKENS,), -1, dtype=torch.int32))
        assert tensors_of(ctx.derived) == []
    assert len({t.data_ptr() for t in slots}) == len(slots)
    m.forward(torch.zeros(TOKENS, 64), ctx, binding())
    assert calls[-4][1][11] is ctx.groups[0].slot_mapping


@pytest.mark.parametrize("page,means", [(PAGE, False), (2 * PAGE, True), (PAGE // 2, True)])
def test_another_entrys_cache_without_means_or_of_other_pages_is_refused(calls, page, means):
    """Scores and choice count in the layer's own pages, attention in the cache's: unlike ones would read other keys than were chosen."""
    m, ctx = mixer_and_step()
    with pytest.raises(ValueError, match="another entry's cache"):
        m.forward(torch.zeros(TOKENS, 64), ctx, binding(write=False, page=page, means=means))
    assert calls == []
