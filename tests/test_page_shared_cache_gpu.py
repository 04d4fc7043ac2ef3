"""Attention over chosen pages in schedule entries that read an earlier entry's pages and means instead of keeping their own: step by step
and through captured decode and mixed steps, against the plain implementation."""
import dataclasses
import random

import pytest
import torch

import helpers as H
import plain_model
from test_page_attention_gpu import sparse

pytestmark = pytest.mark.gpu

NAME = "SharedPagesForTest"


@pytest.fixture
def shared_pages():
    """A registered architecture: the layers of Qwen3 twice over, the second time on the first one's pages."""
    from dinfer_b200.config.model_config import Qwen3Config
    from dinfer_b200.config.registry import register_architecture, unregister_architecture
    from dinfer_b200.models.qwen3 import qwen3_spec
    from dinfer_b200.parts.spec import ScheduleEntry

    def spec(cfg):
        s = qwen3_spec(cfg)
        n = len(s.layers)
        return dataclasses.replace(s, schedule=tuple(ScheduleEntry(i) for i in range(n)) + tuple(ScheduleEntry(i, cache_from=i) for i in range(n)))
    register_architecture(NAME, lambda d: Qwen3Config.from_dict({**d, "architectures": ["Qwen3ForCausalLM"]}), spec, replace=True)
    yield NAME
    unregister_architecture(NAME)


def plain_logits(W, cfg, ids, monkeypatch):
    """The plain implementation over the same schedule: the runs of the second half attend to the first half's keys and values."""
    n = cfg["num_hidden_layers"]
    attention, kept, at = sparse(cfg), {}, [0]

    def shared(q, k, v, scale, window=None):
        i = at[0]
        at[0] += 1
        if i < n:
            kept[i] = (k, v)
        else:
            k, v = kept[i - n]
        return attention(q, k, v, scale, window)
    with monkeypatch.context() as m:
        m.setattr(plain_model, "causal_gqa_attention", shared)
        return plain_model.qwen3_logits(W, cfg, ids, schedule=list(range(n)) * 2).numpy()


def model(tmp_path, name, top, dtype):
    cfg = {**H.CONFIGS[name], "architectures": [NAME], "page_attention": {"top": top, "page": 16, "recent": 2}}
    seed, std, jit = H.INIT[name]
    return cfg, H.make_model_dir(str(tmp_path / "model"), cfg, seed, std, jit, getattr(torch, dtype))


# few pages a token in 32 bits; in bfloat16, where a near-tie between pages may fall either way, room for all of them
FORMS = [("D", "float32", 4), ("E", "float32", 5), ("D", "bfloat16", 40), ("E", "bfloat16", 40)]


@pytest.mark.parametrize("name,dtype,top", FORMS)
def test_step_by_step(tmp_path, monkeypatch, shared_pages, name, dtype, top):
    cfg, d = model(tmp_path, name, top, dtype)
    W = H.load_plain_weights(d)
    rng = random.Random(21)
    lengths = {"a": 170, "b": 60, "c": 9}
    tokens = {r: H.random_tokens(rng, n, cfg["vocab_size"]) for r, n in lengths.items()}
    want = {r: plain_logits(W, cfg, t, monkeypatch) for r, t in tokens.items()}
    rp = H.LocalReplay(d, dtype, 512, block_size=16)
    for tag, steps in (("whole/", H.schedule_whole(lengths)), ("mixed/", H.schedule_mixed(lengths, rng))):
        got = H.run_schedule(rp, steps, tokens, tag=tag)
        worst = max(H.rel_err(got[r], want[r]) for r in tokens)
        assert worst <= H.TOLERANCE[dtype], (tag, worst)
    assert rp.close() == 0


def churn(slots):
    """Small tensors full of slots that requests hold, on every stream of the pool that side streams come from: what a graph reads without
    owning it holds such numbers by now."""
    for _ in range(32):
        with torch.cuda.stream(torch.cuda.Stream()):
            _kept = [torch.randint(0, slots, (n,), dtype=torch.int32, device="cuda") for n in (8, 64, 128, 200, 300, 400, 512) for _ in range(3)]
    torch.cuda.synchronize()


@pytest.mark.parametrize("name,dtype,top", FORMS)
def test_through_captured_steps(tmp_path, monkeypatch, shared_pages, name, dtype, top):
    """Requests that join and finish in steps that replay graphs: the logits of every entry's last token, so that pages of a request that
    another one's step has written over would show."""
    from dinfer_b200.config.engine_config import EngineConfig
    from dinfer_b200.engine.batch import StepEntry
    from dinfer_b200.engine.runner import ModelRunner
    cfg, d = model(tmp_path, name, top, dtype)
    W = H.load_plain_weights(d)
    rng = random.Random(22)
    steps, lengths = H.schedule_rolling([f"r{i}" for i in range(8)], [50, 40], 6)
    tokens = {r: H.random_tokens(rng, n, cfg["vocab_size"]) for r, n in lengths.items()}
    want = {r: plain_logits(W, cfg, t, monkeypatch) for r, t in tokens.items()}
    pages = H.max_live_tokens(steps) // 16
    r = ModelRunner.from_dir(d, EngineConfig(max_model_len=512, max_num_seqs=8, max_num_batched_tokens=256, num_blocks=pages, block_size=16,
                                             dtype=dtype, enable_cuda_graph=True, mixed_cuda_graph=True))
    worst = 0.0
    for entries, end in steps:
        out = r.step([StepEntry(q, tokens[q][lo:hi], [hi - lo - 1]) for q, lo, hi in entries]).cpu().numpy()
        worst = max([worst] + [H.rel_err(out[i], want[q][hi - 1]) for i, (q, lo, hi) in enumerate(entries)])
        for q in end:
            r.finish(q)
        churn(pages * 16)
    r.check_device_status()
    r.manager.check_invariants()
    assert any(isinstance(k, int) for k in r._graphs) and any(isinstance(k, tuple) for k in r._graphs), list(r._graphs)
    assert worst <= H.TOLERANCE[dtype], worst
