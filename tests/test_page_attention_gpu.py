"""Attention over chosen pages inside the engine: a Qwen3 model whose configuration asks for it, against the plain implementation."""
import math
import random

import pytest
import torch

import helpers as H
import plain_model

pytestmark = pytest.mark.gpu


def config(name, top, page, **more):
    return {**H.CONFIGS[name], "page_attention": {"top": top, "page": page, **more}}


def folder(tmp_path, name, cfg, dtype):
    seed, std, jit = H.INIT[name]
    return H.make_model_dir(str(tmp_path / "model"), cfg, seed, std, jit, dtype)


def sparse(cfg):
    """The plain attention of ``plain_model``, of the chosen pages only."""
    a = cfg["page_attention"]
    page, top, first, recent = a["page"], a["top"], a.get("first", 1), a.get("recent", 1)

    def attention(q, k, v, scale, window=None):
        T, Hh, D = q.shape
        G = k.shape[1]
        out = torch.empty_like(q)
        means = torch.stack([k[j * page:(j + 1) * page].mean(0) for j in range(T // page)]) if T >= page else None
        for t in range(T):
            own = t // page
            for g in range(G):
                x = q[t, g * (Hh // G):(g + 1) * (Hh // G)]
                forced = [j for j in range(own + 1) if j < first or j > own - recent]
                rest = [j for j in range(own + 1) if j not in forced]
                if rest:
                    s = (x @ means[:own, g].T).amax(0)
                    rest = sorted(rest, key=lambda j: (-float(s[j]), j))[:max(0, top - len(forced))]
                keys = torch.cat([torch.arange(j * page, min((j + 1) * page, t + 1)) for j in sorted(forced + rest)])
                w = torch.softmax(x @ k[keys, g].T * scale, -1)
                out[t, g * (Hh // G):(g + 1) * (Hh // G)] = w @ v[keys, g]
        return out
    return attention


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,page", [("B", 16), ("D", 16), ("E", 64), ("C", 24)])
def test_with_room_for_every_page_it_is_the_whole_attention(tmp_path, name, page, dtype):
    """Whole, token by token, in portions and mixed, pages used again: the logits of the plain implementation."""
    cfg = config(name, 40, page)
    d = folder(tmp_path, name, cfg, getattr(torch, dtype))
    rng = random.Random(7)
    lengths = {"a": 3, "b": 64, "c": 90, "d": min(230, cfg["max_position_embeddings"])}
    tokens = {r: H.random_tokens(rng, n, cfg["vocab_size"]) for r, n in lengths.items()}
    oracle = H.PlainOracle(d)
    want = {r: oracle.logits(t) for r, t in tokens.items()}
    rp = H.LocalReplay(d, dtype, 1024, block_size=8)
    for tag, steps in (("whole/", H.schedule_whole(lengths)), ("tail/", H.schedule_tail(lengths, 20)),
                       ("mixed/", H.schedule_mixed(lengths, rng))):
        got = H.run_schedule(rp, steps, tokens, tag=tag)
        worst = max(H.rel_err(got[r], want[r]) for r in tokens)
        assert worst <= H.TOLERANCE[dtype], (tag, worst)
    rp.runner.check_device_status()
    assert rp.close() == 0


@pytest.mark.parametrize("name,page,top", [("D", 16, 5), ("E", 16, 4)])
def test_chosen_pages_in_32_bit(tmp_path, monkeypatch, name, page, top):
    """Few pages a token, 32-bit: the plain implementation's own choice of pages and its logits, however the prompt is cut."""
    cfg = config(name, top, page, first=1, recent=2)
    d = folder(tmp_path, name, cfg, torch.float32)
    monkeypatch.setattr(plain_model, "causal_gqa_attention", sparse(cfg))
    rng = random.Random(8)
    lengths = {"a": 300, "b": 150, "c": 20}
    tokens = {r: H.random_tokens(rng, n, cfg["vocab_size"]) for r, n in lengths.items()}
    oracle = H.PlainOracle(d)
    want = {r: oracle.logits(t) for r, t in tokens.items()}
    monkeypatch.undo()
    dense = H.PlainOracle(d).logits(tokens["a"])
    assert H.rel_err(want["a"].astype("float32"), dense) > 100 * H.TOLERANCE["float32"]        # another attention indeed
    rp = H.LocalReplay(d, "float32", 1024, block_size=16)
    for tag, steps in (("whole/", H.schedule_whole(lengths)), ("tail/", H.schedule_tail(lengths, 30)),
                       ("mixed/", H.schedule_mixed_large(lengths, rng, portions=(40, 70, 100)))):
        got = H.run_schedule(rp, steps, tokens, tag=tag)
        worst = max(H.rel_err(got[r], want[r]) for r in tokens)
        assert worst <= H.TOLERANCE["float32"], (tag, worst)
    assert rp.close() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_through_graphs_is_generation_without(tmp_path, dtype):
    """The engine's entry point with captured decode and mixed steps, a prefix cache and few pages: the same tokens as step by step."""
    from dinfer_b200 import LLM, SamplingParams
    cfg = config("D", 4, 16, recent=2)
    d = folder(tmp_path, "D", cfg, getattr(torch, dtype))
    rng = random.Random(9)
    prompts = [H.random_tokens(rng, n, cfg["vocab_size"]) for n in (200, 33, 90, 7)]
    got = []
    for graphs in (False, True):
        llm = LLM(d, dtype=dtype, max_model_len=512, max_num_seqs=3, max_num_batched_tokens=64, num_blocks=80, enable_cuda_graph=graphs,
                  mixed_cuda_graph=graphs)
        outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True))
        llm.runner.check_device_status()
        got.append([o.output_ids for o in outs])
        del llm
    if dtype == "float32":
        assert got[0] == got[1]
    else:                                                    # (steps cut otherwise round otherwise: a near-tie may fall the other way)
        assert sum(a == b for x, y in zip(*got) for a, b in zip(x, y)) >= 40


def test_pages_shared_between_requests_keep_their_means(tmp_path):
    """With the prefix cache a later request with the same beginning reads pages (and means) that an earlier one filled."""
    from dinfer_b200 import LLM, SamplingParams
    cfg = config("E", 4, 16, recent=1)
    d = folder(tmp_path, "E", cfg, torch.float32)
    rng = random.Random(10)
    beginning = H.random_tokens(rng, 160, cfg["vocab_size"])
    prompts = [beginning + H.random_tokens(rng, n, cfg["vocab_size"]) for n in (5, 40)]
    got = []
    for prefix in (False, True):
        llm = LLM(d, dtype="float32", max_model_len=512, max_num_seqs=2, max_num_batched_tokens=512, num_blocks=80,
                  enable_prefix_caching=prefix)
        got.append([llm.generate([p], SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True))[0].output_ids for p in prompts * 2])
        del llm
    assert got[0] == got[1]
