"""Grouped-query attention over chosen pages of a long context: a token reads, per key/value head, the first pages of its
request, the last ones up to its own, and of the full pages between the few that score best for it; a page's score is the largest
product of the group's queries with the mean of the page's keys.  Up to as many pages as a token may choose it is the attention over
everything before it.

Data flow of one step:
  qkv = x Wqkv^T                                     one fused product, rows laid out q heads | k heads | v heads
  q <- rope(headnorm(q)); k, v, page means -> cache   one kernel (the projection's rows are only read)
  s = page_scores(q, means)                          per token, key/value head and full page
  c = choose_pages(s)                                the pages, ascending
  o = attention_pages(q, cache, c)                   keys of the chosen pages up to the token's position
  y = o Wo^T
"""
from __future__ import annotations

import math
from typing import Dict, List, Optional

import torch

from ..kernels import page_ops
from .base import MIXERS, POSITION_ENCODINGS, BuildEnv, CacheBinding, KvCacheNeed, Mixer, StepContext, build_part
from . import rope  # noqa: F401  (the position encodings)
from .linear import Linear
from .spec import PartSpec, TensorDecl


@MIXERS.register("page_attention")
class PageAttention(Mixer):
    """params: ``num_heads``, ``num_kv_heads``, ``head_dim``, ``top`` (pages a token reads at most, per key/value head), optional ``page``
    (tokens of a page, 64), ``first`` (pages from the request's beginning that are always read, 1), ``recent`` (pages up to the token's
    own that are always read, itself included, 1), ``qk_norm`` (bool), ``eps``, ``position`` (a PartSpec), ``scale``, and the tensor
    names ``q_proj``, ``k_proj``, ``v_proj``, ``o_proj``, ``q_norm``, ``k_norm`` (after the prefix).  Heads of 64 and 128 in groups of up to
    16 on pages of 16, 32, 64 or 128 tokens run on the tensor cores in bfloat16; other sizes, and the scores of the 32-bit engine, on
    kernels for any sizes, many times slower.  An entry that reads another's cache has to have pages of the same size."""

    def __init__(self, params, env: BuildEnv, prefix=""):
        super().__init__(params, env, prefix)
        p = self.params
        self.H, self.Hkv, self.D = int(p["num_heads"]), int(p["num_kv_heads"]), int(p["head_dim"])
        self.page, self.top = int(p.get("page", 64)), int(p["top"])
        self.first, self.recent = int(p.get("first", 1)), int(p.get("recent", 1))
        if min(self.H, self.Hkv, self.D, self.page) <= 0 or self.H % self.Hkv or self.D > 512:
            raise ValueError(f"page attention: heads {self.H} / kv heads {self.Hkv} of {self.D}, pages of {self.page}")
        if self.first < 0 or self.recent < 1 or self.top < self.first + self.recent:
            raise ValueError(f"page attention: {self.first} first and {self.recent} recent pages of {self.top} (a token's own is always read)")
        self.qk_norm = bool(p.get("qk_norm", False))
        self.eps = float(p.get("eps", 1e-6))
        self.scale = float(p.get("scale", 1.0 / math.sqrt(self.D)))
        self.position = build_part(POSITION_ENCODINGS, p.get("position") or PartSpec("none"), env, prefix)
        if not self.position.fused:
            raise NotImplementedError("page attention needs a position encoding that is a table rotation")
        n = lambda key, default: prefix + p.get(key, default)
        self.names = {"q": n("q_proj", "q_proj.weight"), "k": n("k_proj", "k_proj.weight"), "v": n("v_proj", "v_proj.weight"),
                      "o": n("o_proj", "o_proj.weight"), "qn": n("q_norm", "q_norm.weight"), "kn": n("k_norm", "k_norm.weight")}
        self.qkv: Optional[Linear] = None
        self.o: Optional[Linear] = None
        self.q_norm_w = self.k_norm_w = None

    def declare(self) -> List[TensorDecl]:
        H, Hkv, D, h, N = self.H, self.Hkv, self.D, self.env.hidden_size, self.names
        d = [TensorDecl(N["q"], (H * D, h)), TensorDecl(N["k"], (Hkv * D, h)), TensorDecl(N["v"], (Hkv * D, h)), TensorDecl(N["o"], (h, H * D))]
        if self.qk_norm:
            d += [TensorDecl(N["qn"], (D,), init="ones"), TensorDecl(N["kn"], (D,), init="ones")]
        return d

    def bind(self, tensors: Dict[str, torch.Tensor]) -> None:
        rows = [tensors[self.names[x]] for x in ("q", "k", "v")]
        dt = torch.float32 if any(t.dtype == torch.float32 for t in rows) else rows[0].dtype
        self.qkv = Linear(torch.cat([t.to(dt) for t in rows], dim=0))
        self.o = Linear(tensors[self.names["o"]])
        if self.qk_norm:
            self.q_norm_w = tensors[self.names["qn"]].contiguous()
            self.k_norm_w = tensors[self.names["kn"]].to(self.q_norm_w.dtype).contiguous()

    def cache_need(self):
        return KvCacheNeed(self.Hkv, self.D, None, self.page, key_means=True)

    def kernel_libraries(self):
        return ["page_append", "page_choice", "attention_pages", "attention_pages_umma"] + self.qkv.kernel_libraries() + self.o.kernel_libraries()

    def takes_half_normed(self, rows: int) -> bool:
        return self.qkv.fuses_norm(rows, self.env.act_dtype)

    def makes_norm(self, rows: int) -> bool:
        return self.qkv.makes_norm(rows, self.env.act_dtype)

    def adds_into_residual(self, rows: int) -> bool:
        return self.o.fuses_norm(rows, self.env.act_dtype)

    def forward(self, x, ctx: StepContext, cache: CacheBinding, sink=None):
        g = ctx.groups[cache.group]
        qkv = self.qkv(x)
        slots = g.slot_mapping
        if not cache.write:                                  # another layer's keys and values: only q is made
            if cache.means is None or cache.kv.shape[3] != self.page:
                raise ValueError(f"page attention in pages of {self.page} reads another entry's cache, which has to keep key means in "
                                 f"pages as large (pages of {cache.kv.shape[3]}, {'no ' if cache.means is None else ''}means)")
            # made by every run: a graph has to own and fill what it reads (a tensor kept in the context would be its warm-up's)
            slots = torch.full_like(slots, -1)
        q = torch.empty((qkv.shape[0], self.H * self.D), dtype=qkv.dtype, device=qkv.device)
        page_ops.append(qkv, ctx.positions, self.H, self.Hkv, self.D, self.eps, self.q_norm_w, self.k_norm_w,
                        self.position.fused_table(), q, cache.kv, slots, cache.means,
                        interleaved=getattr(self.position, "interleaved", False))
        # the pages there may be: of the longest request (inside a captured graph the longest that the engine admits)
        longest = int(self.env.max_positions) if ctx.decode_splits else ctx.max_seq_len
        pages = max(1, min(g.block_table.shape[1], -(-longest // self.page)))
        scores = page_ops.page_scores(q, cache.means, g.block_table, ctx.cu_seqlens, ctx.positions, self.H, self.page, pages=pages)
        chosen = page_ops.choose_pages(scores, ctx.positions, self.page, self.top, first=self.first, recent=self.recent)
        out = torch.empty_like(q)
        page_ops.attention_pages(q, out, cache.kv, g.block_table, ctx.cu_seqlens, ctx.positions, chosen, self.H, self.scale)
        if sink is not None:                                 # (residual, the norm behind this mixer)
            return self.o.into_residual(out, sink[0], sink[1])
        return self.o(out)
