"""Wrappers of attention over chosen pages of the paged cache: a token reads a few pages of its request's context, the ones a
cheap score picks for it (per key/value head, shared by the heads of its group).  In an attention layer, in this order:

    append           head norms, rotation, keys and values into their pages, the mean key of each page that becomes full
    page_scores      per token, key/value head and full page: the largest product of the group's queries with the mean key
    choose_pages     first pages, last pages and the best-scored of the rest
    attention_pages  softmax attention over the keys of the chosen pages up to the token's position

All four take the step's tokens as one batch (portions of prompts beside decoded tokens), float32 or bfloat16, any head size
up to 512, any number of heads per key/value head, any page size.  Bfloat16 with head sizes 64 and 128 and pages of 16, 32, 64 or
128 tokens runs on kernels of its own.  Tensors lie on the current device; the calls run on its current stream.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_int64, c_void_p
from typing import Optional

import torch

from . import gemm_ops
from .lib import DTYPE_CODE, KernelError, check, dtype_code, library, num_sms, ptr, require_cuda, stream_handle
from .ops import _fn


# Steps of at least so many tokens, and so many a request, walk the pages that neighbouring tokens chose together
PORTION_TOKENS = 64
PORTION_TOKENS_A_REQUEST = 4


def _portions(q, out, cache, block_table, top: int, scale: float) -> int:
    """Bytes of workspace of the kernel for portions where it takes this call, else 0: bfloat16 rows that TMA can address, a positive
    scale, enough tokens."""
    T, B = q.shape[0], block_table.shape[0]
    if T < PORTION_TOKENS or T < PORTION_TOKENS_A_REQUEST * B or q.dtype != torch.bfloat16 or not scale > 0:
        return 0
    if q.stride(0) % 8 or out.stride(0) % 8 or (q.data_ptr() | out.data_ptr() | cache.data_ptr()) % 16 or cache.numel() // cache.shape[-1] > 0x7fffffff:
        return 0
    f = library("attention_pages_umma").dinfer_attention_pages_umma_workspace
    f.argtypes, f.restype = [c_int] * 8, c_int64
    return f(B, block_table.shape[1], top, T, q.shape[1] // cache.shape[4], cache.shape[2], cache.shape[4], cache.shape[3])


def _here(what: str, *tensors) -> None:
    """On CUDA, all on the current device (the kernels run there, whatever the tensors say)."""
    require_cuda(*tensors)
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise KernelError(f"{what}: a tensor on device {t.get_device()}, the current device is {here}")


def _ints(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise KernelError(f"{what}: {name} must be contiguous int32")


def _batch(what: str, T: int, block_table, cu_seqlens, positions) -> None:
    _ints(what, block_table=block_table, cu_seqlens=cu_seqlens, positions=positions)
    if block_table.dim() != 2 or cu_seqlens.dim() != 1 or cu_seqlens.numel() != block_table.shape[0] + 1 or positions.numel() != T \
            or block_table.shape[0] == 0:
        raise KernelError(f"{what}: block_table [B, width] with B > 0, cu_seqlens [B + 1], positions [T]")


def _heads(what: str, q, num_heads: int, num_kv_heads: int, head_dim: int) -> None:
    if q.dim() != 2 or q.stride(1) != 1 or q.shape[1] != num_heads * head_dim:
        raise KernelError(f"{what}: rows [T, {num_heads} * {head_dim}] with a contiguous last axis, not {tuple(q.shape)}")
    if num_heads <= 0 or num_kv_heads <= 0 or num_heads % num_kv_heads or head_dim > 512:
        raise KernelError(f"{what}: {num_heads} heads of {head_dim} over {num_kv_heads} key/value heads")


def append(qkv: torch.Tensor, positions: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, eps: float,
           q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
           q_out: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, means: torch.Tensor,
           interleaved: bool = False) -> torch.Tensor:
    """From the projection's rows ``qkv`` [T, (H + 2 Hkv) D] (q heads | k heads | v heads; only read): q, normed and turned, into
    ``q_out`` [T, H * D]; k, normed and turned, and v into ``cache`` [pages, 2, Hkv, page, D] at ``slots`` (int32 [T], page *
    page_size + offset; -1: a row that is not kept); and the mean of the keys, as cached, of every page whose last offset this
    step writes into ``means`` [pages, Hkv, D].  Other pages' means are left as they are.  ``q_weight`` / ``k_weight`` [D]: head norm
    ``x / sqrt(mean(x^2) + eps) * w``, or None for both; ``cos_sin`` f32 [positions, rot]: the angle table (``cos | sin``) of the
    first ``rot`` elements, pairs (i, i + rot/2) or with ``interleaved`` (2i, 2i + 1), which reaches every position; None: no
    rotation.  A slot is written by one token of the step at most.  Returns ``q_out``."""
    what = "page append"
    _here(what, qkv, positions, q_weight, k_weight, cos_sin, q_out, cache, slots, means)
    dt = qkv.dtype
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (num_heads + 2 * num_kv_heads) * head_dim:
        raise KernelError(f"{what}: qkv rows [T, ({num_heads} + 2 * {num_kv_heads}) * {head_dim}] with a contiguous last axis")
    T = qkv.shape[0]
    _heads(what, q_out, num_heads, num_kv_heads, head_dim)
    if q_out.shape[0] != T or q_out.dtype != dt or cache.dtype != dt or means.dtype != dt:
        raise KernelError(f"{what}: q_out, cache and means of the rows' dtype, q_out [T, H * D]")
    if cache.dim() != 5 or tuple(cache.shape[1:3]) != (2, num_kv_heads) or cache.shape[4] != head_dim or cache.shape[3] == 0 \
            or not cache.is_contiguous():
        raise KernelError(f"{what}: cache shape {tuple(cache.shape)} is not [pages, 2, {num_kv_heads}, page, {head_dim}], contiguous")
    if tuple(means.shape) != (cache.shape[0], num_kv_heads, head_dim) or not means.is_contiguous():
        raise KernelError(f"{what}: means [pages, Hkv, D], contiguous, not {tuple(means.shape)}")
    _ints(what, positions=positions, slots=slots)
    if positions.numel() != T or slots.numel() != T:
        raise KernelError(f"{what}: positions and slots int32 [T]")
    if (q_weight is None) != (k_weight is None):
        raise KernelError(f"{what}: q and k norm weights come together")
    w_dt = dt
    if q_weight is not None:
        w_dt = q_weight.dtype
        if q_weight.numel() != head_dim or k_weight.numel() != head_dim or k_weight.dtype != w_dt \
                or not q_weight.is_contiguous() or not k_weight.is_contiguous():
            raise KernelError(f"{what}: norm weights [head_dim], contiguous, of one dtype")
    rot = rows = 0
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
            raise KernelError(f"{what}: angle table must be contiguous float32 [positions, rot]")
        rows, rot = cos_sin.shape
    lib, f = _fn("page_append", "dinfer_page_append",
                 [c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_int, c_int, c_int, c_void_p, c_int64,
                  c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p])
    check(lib, f(ptr(qkv), qkv.stride(0), ptr(positions), ptr(q_weight), ptr(k_weight), eps, ptr(cos_sin), rows, rot,
                 int(bool(interleaved)), ptr(q_out), q_out.stride(0), ptr(cache), ptr(means), ptr(slots), cache.shape[0],
                 cache.shape[3], T, num_heads, num_kv_heads, head_dim, dtype_code(dt), dtype_code(w_dt), stream_handle()), what)
    return q_out


def page_scores(q: torch.Tensor, means: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                positions: torch.Tensor, num_heads: int, page_size: int, out: Optional[torch.Tensor] = None,
                pages: Optional[int] = None) -> torch.Tensor:
    """``out[t, g, j] = max over the heads h of group g of q[t, h] . means[page, g]`` for the full pages j before token t's own
    (``j < positions[t] // page_size``), -inf for the others and for pages the table does not hold (-1): float32 [T, Hkv, pages].
    ``q`` [T, H * D] may be strided rows; ``pages`` (default: the table's width) bounds the pages looked at.  A product that
    is not a number makes the page's score one that is not.  Rows behind the last request's tokens are left as they are."""
    what = "page_scores"
    _here(what, q, means, block_table, cu_seqlens, positions, out)
    if means.dim() != 3 or not means.is_contiguous() or means.dtype != q.dtype:
        raise KernelError(f"{what}: means [pages, Hkv, D], contiguous, of q's dtype")
    num_pages, Hkv, D = means.shape
    _heads(what, q, num_heads, Hkv, D)
    T = q.shape[0]
    _batch(what, T, block_table, cu_seqlens, positions)
    width = block_table.shape[1]
    pages = width if pages is None else pages
    if not 0 <= pages <= width or page_size <= 0:
        raise KernelError(f"{what}: {pages} pages of {page_size} tokens, the table holds {width}")
    if out is None:
        out = torch.empty((T, Hkv, pages), dtype=torch.float32, device=q.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != (T, Hkv, pages) or (pages > 1 and out.stride(2) != 1):
        raise KernelError(f"{what}: out float32 [T, Hkv, pages] with a contiguous last axis")
    lib, f = _fn("page_choice", "dinfer_page_scores",
                 [c_void_p, c_int64, c_void_p, c_int, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p, c_int64, c_int64,
                  c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p])
    check(lib, f(ptr(q), q.stride(0), ptr(means), num_pages, ptr(block_table), width, ptr(cu_seqlens), block_table.shape[0],
                 ptr(positions), ptr(out), out.stride(0), out.stride(1), T, num_heads, Hkv, D, page_size, pages,
                 dtype_code(q.dtype), stream_handle()), what)
    return out


def choose_pages(scores: torch.Tensor, positions: torch.Tensor, page_size: int, top: int, first: int = 1, recent: int = 1,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 [T, Hkv, top]: per token and key/value head the pages its attention reads, ascending, -1 behind the last.  Of the
    pages up to the token's own (``positions[t] // page_size``, the last column of ``scores`` at most): the first ``first``, the
    last ``recent`` (the own one included, hence at least 1), and of those between the ones with the largest ``scores`` (float32 [T,
    Hkv, pages], the last axis contiguous) up to ``top`` in all; of equal scores the lower page, and what is not a number behind
    every number.  A negative position chooses no page."""
    what = "choose_pages"
    _here(what, scores, positions, out)
    if scores.dim() != 3 or scores.dtype != torch.float32 or (scores.shape[2] > 1 and scores.stride(2) != 1) or scores.shape[2] == 0:
        raise KernelError(f"{what}: scores float32 [T, Hkv, pages] with a contiguous last axis and at least one page")
    T, Hkv, pages = scores.shape
    _ints(what, positions=positions)
    if positions.numel() != T:
        raise KernelError(f"{what}: positions int32 [T]")
    if page_size <= 0 or first < 0 or recent < 1 or top < first + recent:
        raise KernelError(f"{what}: {first} first and {recent} recent pages of {top}, pages of {page_size} tokens")
    if out is None:
        out = torch.empty((T, Hkv, top), dtype=torch.int32, device=scores.device)
    elif out.dtype != torch.int32 or tuple(out.shape) != (T, Hkv, top) or not out.is_contiguous():
        raise KernelError(f"{what}: out int32 [T, Hkv, top], contiguous")
    lib, f = _fn("page_choice", "dinfer_choose_pages",
                 [c_void_p, c_int64, c_int64, c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p])
    check(lib, f(ptr(scores), scores.stride(0), scores.stride(1), ptr(positions), page_size, first, recent, top, pages, ptr(out),
                 T, Hkv, stream_handle()), what)
    return out


def attention_pages(q: torch.Tensor, out: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, positions: torch.Tensor, chosen: torch.Tensor, num_heads: int,
                    scale: float) -> torch.Tensor:
    """``out[t, h] = softmax over the seen keys (scale * q[t, h] . k) v``: token t sees the keys of its request's pages
    ``chosen[t, g]`` (int32 [T, Hkv, top]; g the head's key/value head) at positions up to ``positions[t]``.  Numbers outside the
    table's columns and pages the table does not hold are no pages, a page named twice counts twice, and a token that sees
    nothing gets zeros.  ``q`` and ``out`` [T, H * D] may be strided rows; ``cache`` [pages, 2, Hkv, page, D].  Rows behind
    the last request's tokens are left as they are.  Returns ``out``."""
    what = "attention_pages"
    _here(what, q, out, cache, block_table, cu_seqlens, positions, chosen)
    if q.dtype not in DTYPE_CODE or out.dtype != q.dtype or cache.dtype != q.dtype:
        raise KernelError(f"{what}: q, out and cache of one dtype, float32 or bfloat16")
    if cache.dim() != 5 or cache.shape[1] != 2 or cache.shape[3] == 0 or not cache.is_contiguous():
        raise KernelError(f"{what}: cache shape {tuple(cache.shape)} is not [pages, 2, Hkv, page, D], contiguous")
    num_pages, _, Hkv, page_size, D = cache.shape
    _heads(what, q, num_heads, Hkv, D)
    _heads(what, out, num_heads, Hkv, D)
    T = q.shape[0]
    if out.shape[0] != T:
        raise KernelError(f"{what}: out [T, H * D] of q's shape")
    _batch(what, T, block_table, cu_seqlens, positions)
    _ints(what, chosen=chosen)
    if chosen.dim() != 3 or tuple(chosen.shape[:2]) != (T, Hkv) or chosen.shape[2] == 0:
        raise KernelError(f"{what}: chosen int32 [T, Hkv, top] with top > 0")
    top = chosen.shape[2]
    head = (ptr(q), q.stride(0), ptr(out), out.stride(0), ptr(cache), num_pages, ptr(block_table), block_table.shape[1],
            ptr(cu_seqlens), block_table.shape[0], ptr(positions), ptr(chosen), top, T, num_heads, Hkv, D, page_size, scale)
    types = [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p,
             c_int, c_int, c_int, c_int, c_int, c_int, c_float]
    size = _portions(q, out, cache, block_table, top, scale)
    if size:
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
        lib, f = _fn("attention_pages_umma", "dinfer_attention_pages_umma", types + [c_void_p, c_int64, c_void_p, c_void_p])
        check(lib, f(*head, ptr(work), size, ptr(gemm_ops._state(q.device)["status"]), stream_handle()), "attention_pages_umma")
        return out
    lib, f = _fn("attention_pages", "dinfer_attention_pages", types + [c_int, c_int, c_void_p])
    check(lib, f(*head, num_sms(), DTYPE_CODE[q.dtype], stream_handle()), what)
    return out
