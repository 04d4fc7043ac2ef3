"""Attention over chosen pages inside the engine on prompts long enough for the kernel in which neighbouring tokens walk their pages
together, and in bfloat16 with few pages a token: the plain implementation over the pages that the engine chose."""
import random

import numpy as np
import pytest
import torch

import helpers as H
import plain_model
from test_page_attention_gpu import config, folder

pytestmark = pytest.mark.gpu


@pytest.fixture
def recorded(monkeypatch):
    """The kernel libraries that calls run on and the pages that ``choose_pages`` chose, call by call."""
    from dinfer_b200.kernels import page_ops
    libraries, choices = [], []
    real_call, real_choice = page_ops._call, page_ops.choose_pages

    def call(lib, *args):
        libraries.append(lib)
        return real_call(lib, *args)

    def choose(*args, **kw):
        choices.append(real_choice(*args, **kw))
        return choices[-1]
    monkeypatch.setattr(page_ops, "_call", call)
    monkeypatch.setattr(page_ops, "choose_pages", choose)
    return libraries, choices


@pytest.mark.parametrize("name,page", [("D", 16), ("E", 64), ("D", 128), ("E", 32)])
def test_long_prompts_with_room_for_every_page(tmp_path, recorded, name, page):
    """Whole, and mixed with another's decoded tokens: the logits of the plain implementation, and the kernel that was meant."""
    cfg = config(name, 64, page)
    d = folder(tmp_path, name, cfg, torch.bfloat16)
    rng = random.Random(31)
    lengths = {"a": 900, "b": 500}
    tokens = {r: H.random_tokens(rng, n, cfg["vocab_size"]) for r, n in lengths.items()}
    oracle = H.PlainOracle(d)
    want = {r: oracle.logits(t) for r, t in tokens.items()}
    rp = H.LocalReplay(d, "bfloat16", 2048, block_size=16)
    for tag, steps in (("whole/", H.schedule_whole(lengths)), ("mixed/", H.schedule_mixed_large(lengths, rng, portions=(130, 300, 400)))):
        recorded[0].clear()
        got = H.run_schedule(rp, steps, tokens, tag=tag)
        worst = max(H.rel_err(got[r], want[r]) for r in tokens)
        assert worst <= H.TOLERANCE["bfloat16"], (tag, worst)
        assert "attention_pages_umma" in recorded[0], tag
    rp.runner.check_device_status()
    assert rp.close() == 0


@pytest.mark.parametrize("name,page,top", [("D", 16, 20), ("E", 32, 12), ("D", 16, 4)])
def test_few_pages_in_bfloat16(tmp_path, monkeypatch, recorded, name, page, top):
    """The plain implementation reads the pages that the engine chose (a near-tie may fall either way); and no page that was left out
    scores higher by the plain implementation than one that was taken, beyond what activations off by the tolerance explain."""
    cfg = config(name, top, page, recent=2)
    d = folder(tmp_path, name, cfg, torch.bfloat16)
    rng = random.Random(32)
    n, layers = 800, cfg["num_hidden_layers"]
    tokens = {"a": H.random_tokens(rng, n, cfg["vocab_size"])}
    rp = H.LocalReplay(d, "bfloat16", 1024, block_size=16)
    got = H.run_schedule(rp, H.schedule_tail({"a": n}, 15), tokens)["a"]
    rp.runner.check_device_status()
    assert rp.close() == 0
    assert ("attention_pages_umma" in recorded[0]) is (top > 4) and "attention_pages" in recorded[0]
    chosen = [torch.cat([c.cpu() for c in recorded[1][l::layers]]) for l in range(layers)]       # [tokens, key heads, top] a layer
    assert all(c.shape[0] == n for c in chosen)
    at, tolerance = [0], H.TOLERANCE["bfloat16"]

    def attention(q, k, v, scale, window=None):
        mine = chosen[at[0]]
        at[0] += 1
        heads, G = q.shape[1], k.shape[1]
        out = torch.empty_like(q)
        means = k[:n // page * page].reshape(n // page, page, G, -1).mean(1)
        for t in range(n):
            own = t // page
            for g in range(G):
                x = q[t, g * (heads // G):(g + 1) * (heads // G)]
                pages = [j for j in mine[t, g].tolist() if j >= 0]
                assert pages == sorted(set(pages)) and {0, own, max(own - 1, 0)} <= set(pages) and len(pages) == min(top, own + 1)
                rest = [j for j in range(own + 1) if j not in pages]
                if rest:
                    s = (x @ means[:own, g].T).amax(0)
                    taken = [j for j in pages if 0 < j < own - 1]
                    size = float(x.norm(dim=1).max() * means[:own, g].norm(dim=1).max())
                    assert float(s[rest].max()) - float(s[taken].min()) <= 2 * (2 * tolerance + tolerance ** 2) * size
                keys = torch.cat([torch.arange(j * page, min((j + 1) * page, t + 1)) for j in pages])
                out[t, g * (heads // G):(g + 1) * (heads // G)] = torch.softmax(x @ k[keys, g].T * scale, -1) @ v[keys, g]
        return out
    with monkeypatch.context() as m:
        m.setattr(plain_model, "causal_gqa_attention", attention)
        want = plain_model.qwen3_logits(H.load_plain_weights(d), cfg, tokens["a"]).numpy()
    assert H.rel_err(got, want) <= tolerance
    if top <= 4:                                             # another attention indeed
        assert H.rel_err(want.astype(np.float32), H.PlainOracle(d).logits(tokens["a"])) > tolerance
