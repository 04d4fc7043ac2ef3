"""What the calls of attention over chosen pages refuse: by name, before anything is launched."""
import pytest
import torch

from dinfer_b200.kernels import page_ops
from dinfer_b200.kernels.lib import KernelError

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
H, G, D, P, T, B = 4, 2, 64, 16, 5, 2


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    """The checks run on CPU tensors; a call that passes them all ends in ``Launched`` instead of the library."""
    monkeypatch.setattr(page_ops, "_here", lambda what, *tensors: None)

    def library(*args):
        raise Launched
    monkeypatch.setattr(page_ops, "_call", library)
    monkeypatch.setattr(page_ops, "_device", lambda: 0)
    monkeypatch.setattr(page_ops.gemm_ops, "_state", lambda device: {"status": torch.zeros(1, dtype=I32)})


class Launched(Exception):
    pass


def args(call):
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)
    i = lambda *s: z(*s, dtype=I32)
    cache, means, batch = z(3, 2, G, P, D), z(3, G, D), dict(block_table=i(B, 3), cu_seqlens=i(B + 1), positions=i(T))
    return {"append": dict(qkv=z(T, (H + 2 * G) * D), positions=i(T), num_heads=H, num_kv_heads=G, head_dim=D, eps=1e-6,
                           q_weight=z(D), k_weight=z(D), cos_sin=z(9, D, dtype=F32), q_out=z(T, H * D), cache=cache, slots=i(T), means=means),
            "page_scores": dict(q=z(T, H * D), means=means, num_heads=H, page_size=P, **batch),
            "choose_pages": dict(scores=z(T, G, 3, dtype=F32), positions=i(T), page_size=P, top=4),
            "attention_pages": dict(q=z(T, H * D), out=z(T, H * D), cache=cache, chosen=i(T, G, 4), num_heads=H, scale=0.1, **batch)}[call]


@pytest.mark.parametrize("call", ["append", "page_scores", "choose_pages", "attention_pages"])
def test_what_is_right_is_launched(call):
    with pytest.raises(Launched):
        getattr(page_ops, call)(**args(call))


def other(*s, dtype=BF16):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("call,change", [
    ("append", dict(qkv=other(T, (H + 2 * G) * D + 1))),
    ("append", dict(qkv=other(T, 2 * (H + 2 * G) * D)[:, ::2])),
    ("append", dict(q_out=other(T + 1, H * D))),
    ("append", dict(q_out=other(T, H * D, dtype=F32))),
    ("append", dict(cache=other(3, 2, G, P, D, dtype=F32))),
    ("append", dict(cache=other(3, 1, G, P, D))),
    ("append", dict(cache=other(3, 2, G, D, P).transpose(3, 4))),
    ("append", dict(cache=other(3, 2, G + 1, P, D))),
    ("append", dict(means=other(2, G, D))),
    ("append", dict(means=other(3, G, D, dtype=F32))),
    ("append", dict(slots=other(T, dtype=torch.int64))),
    ("append", dict(slots=other(T - 1, dtype=I32))),
    ("append", dict(positions=other(2 * T, dtype=I32)[::2])),
    ("append", dict(q_weight=None)),
    ("append", dict(k_weight=other(D, dtype=F32))),
    ("append", dict(q_weight=other(2 * D)[::2], k_weight=other(D))),
    ("append", dict(cos_sin=other(9, D))),
    ("append", dict(num_heads=3)),
    ("page_scores", dict(q=other(T, H * D, dtype=F32))),
    ("page_scores", dict(q=other(T, H * D + 2))),
    ("page_scores", dict(means=other(3, G, D).transpose(0, 1))),
    ("page_scores", dict(block_table=other(B + 1, 3, dtype=I32))),
    ("page_scores", dict(cu_seqlens=other(B + 1, dtype=torch.int64))),
    ("page_scores", dict(positions=other(T + 1, dtype=I32))),
    ("page_scores", dict(num_heads=3)),
    ("page_scores", dict(pages=4)),
    ("page_scores", dict(pages=-1)),
    ("page_scores", dict(page_size=0)),
    ("page_scores", dict(out=other(T, G, 4, dtype=F32))),
    ("page_scores", dict(out=other(T, G, 3))),
    ("page_scores", dict(out=other(T, 3, G, dtype=F32).transpose(1, 2))),
    ("choose_pages", dict(scores=other(T, G, 3))),
    ("choose_pages", dict(scores=other(T, 3, dtype=F32))),
    ("choose_pages", dict(scores=other(T, G, 0, dtype=F32))),
    ("choose_pages", dict(scores=other(T, 3, G, dtype=F32).transpose(1, 2))),
    ("choose_pages", dict(positions=other(T, dtype=F32))),
    ("choose_pages", dict(positions=other(T + 1, dtype=I32))),
    ("choose_pages", dict(recent=0)),
    ("choose_pages", dict(first=-1)),
    ("choose_pages", dict(first=3, recent=2)),
    ("choose_pages", dict(page_size=0)),
    ("choose_pages", dict(out=other(T, G, 3, dtype=I32))),
    ("choose_pages", dict(out=other(T, G, 4))),
    ("attention_pages", dict(q=other(T, H * D, dtype=torch.float16))),
    ("attention_pages", dict(out=other(T, H * D, dtype=F32))),
    ("attention_pages", dict(out=other(T + 1, H * D))),
    ("attention_pages", dict(out=other(T, H * D * 2)[:, ::2])),
    ("attention_pages", dict(cache=other(3, 2, G, P, D + 1))),
    ("attention_pages", dict(cache=other(3, 2, G, D, P).transpose(3, 4))),
    ("attention_pages", dict(chosen=other(T, G, 4, dtype=torch.int64))),
    ("attention_pages", dict(chosen=other(T, G + 1, 4, dtype=I32))),
    ("attention_pages", dict(chosen=other(T, G, 0, dtype=I32))),
    ("attention_pages", dict(chosen=other(G, T, 4, dtype=I32).transpose(0, 1))),
    ("attention_pages", dict(num_heads=5)),
    ("attention_pages", dict(block_table=other(0, 3, dtype=I32), cu_seqlens=other(1, dtype=I32))),
])
def test_refusals(call, change):
    with pytest.raises(KernelError):
        getattr(page_ops, call)(**{**args(call), **change})


def test_tensors_off_the_device_are_refused(monkeypatch):
    monkeypatch.undo()
    for call in ("append", "page_scores", "choose_pages", "attention_pages"):
        with pytest.raises(KernelError, match="CUDA tensors only"):
            getattr(page_ops, call)(**{k: v for k, v in args(call).items()})


# ---------------------------------------------------------------- the model's configuration and the part

def test_configuration_and_spec():
    import helpers as H
    from dinfer_b200.config.model_config import Qwen3Config
    from dinfer_b200.models.qwen3 import qwen3_spec
    plain = Qwen3Config.from_dict(H.TINY_D)
    assert plain.page_attention is None and "page_attention" not in plain.to_dict()
    assert all(l.mixer.kind == "gqa_attention" for l in qwen3_spec(plain).layers)
    c = Qwen3Config.from_dict({**H.TINY_D, "page_attention": {"top": 8}})
    assert c.page_attention == {"page": 64, "top": 8, "first": 1, "recent": 1} and Qwen3Config.from_dict(c.to_dict()) == c
    mixers = [l.mixer for l in qwen3_spec(c).layers]
    assert all(m.kind == "page_attention" and m.params["top"] == 8 and m.params["num_heads"] == 8 for m in mixers)


@pytest.mark.parametrize("value", [{}, {"page": 16}, {"top": 4, "size": 16}, {"top": 1, "first": 1, "recent": 1}, {"top": 4, "recent": 0},
                                   {"top": 4, "first": -1}, {"top": 4, "page": 0}, {"top": "4"}, [4], {"top": 4.0}])
def test_configuration_refusals(value):
    import helpers as H
    from dinfer_b200.config.model_config import ConfigError, Qwen3Config
    with pytest.raises(ConfigError):
        Qwen3Config.from_dict({**H.TINY_D, "page_attention": value})


@pytest.mark.parametrize("change", [dict(top=1), dict(recent=0), dict(first=-1), dict(page=0), dict(num_kv_heads=3), dict(head_dim=513)])
def test_part_refusals(change):
    from dinfer_b200.parts.base import BuildEnv, MIXERS
    from dinfer_b200.parts import page_attention  # noqa: F401
    env = BuildEnv(torch.device("cpu"), BF16, 64, 128)
    params = dict(num_heads=4, num_kv_heads=2, head_dim=16, top=6, page=16)
    mixer = MIXERS.get("page_attention")(params, env)
    need = mixer.cache_need()
    assert need.key_means and need.block_size == 16 and [d.shape for d in mixer.declare()] == [(64, 64), (32, 64), (32, 64), (64, 64)]
    with pytest.raises(ValueError):
        MIXERS.get("page_attention")({**params, **change}, env)


def test_attention_does_not_write_over_its_queries():
    a = args("attention_pages")
    with pytest.raises(KernelError, match="out must not be q's memory"):
        page_ops.attention_pages(**{**a, "out": a["q"]})
