"""Wrappers of attention over chosen pages of the paged cache: a token reads a few pages of its request's context, the ones a
cheap score picks for it (per key/value head, shared by the heads of its group).  In an attention layer, in this order:

    append           head norms, rotation, keys and values into their pages, the mean key of each page that becomes full
    page_scores      per token, key/value head and full page: the largest product of the group's queries with the mean key
    choose_pages     first pages, last pages and the best-scored of the rest
    attention_pages  softmax attention over the keys of the chosen pages up to the token's position

All four take the step's tokens as one batch (portions of prompts beside decoded tokens), float32 or bfloat16, any head size
up to 512, any number of heads per key/value head, any page size.  Head sizes 64 and 128 on rows of 16-byte boundaries run on
kernels of their own: appending both dtypes with pages of up to 128 tokens, scores in bfloat16 with groups of up to 16 heads, attention in
bfloat16 with pages of 16, 32, 64 or 128 tokens and groups of up to 128 heads, in float32 with pages of a multiple of 8 tokens and groups of up
to 8.  The choice has its own up to 16384 pages.  What is left, 32-bit scores among it, runs on kernels for any sizes, many times
slower.  Tensors lie on the current device; the calls run on its current stream.
"""
from __future__ import annotations

import struct
from ctypes import c_char_p, c_int, c_int64
from typing import Optional

import torch

from . import gemm_ops
from .lib import DTYPE_CODE, KernelError, check, library, num_sms, require_cuda
from .ops import _fn

_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16

# A decode step of few tokens is as long as its calls take the host.  So the arguments of a call go as one packed struct (24 of them one
# by one cost ctypes 2.8 us, packed 0.5), the stream last, and the checks ask each tensor once for each thing.
_PACK = {
    "dinfer_page_append": struct.Struct("5qd18q").pack,
    "dinfer_page_scores": struct.Struct("22q").pack,
    "dinfer_choose_pages": struct.Struct("13q").pack,
    "dinfer_attention_pages": struct.Struct("18qd3q").pack,
    "dinfer_attention_pages_umma": struct.Struct("18qd4q").pack,
}
_BOUND = {}
_SMS = {}                               # multiprocessors by device


def _call(libname: str, fname: str, what: str, *args) -> None:
    """The library's function on the current stream."""
    bound = _BOUND.get(fname)
    if bound is None:
        bound = _BOUND[fname] = _fn(libname, fname, [c_char_p]) + (_PACK[fname],)
    lib, f, pack = bound
    check(lib, f(pack(*args, _stream())), what)


_raw_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _device() -> int:
    return _raw_device() if _raw_device is not None else torch.cuda.current_device()


def _multiprocessors() -> int:
    at = _device()
    n = _SMS.get(at)
    if n is None:
        n = _SMS[at] = num_sms()
    return n


def _stream() -> int:
    return _raw_stream(_device()) if _raw_stream is not None else torch.cuda.current_stream().cuda_stream


# Steps of fewer tokens, and of single tokens alone, are not asked about: token by token is the shorter way for them, where the tensor-core
# kernel for tokens takes the call (groups of up to 16 heads, up to 1024 chosen pages)
PORTION_TOKENS = 24
TOKEN_GROUP, TOKEN_TOP = 16, 1024


def _portions(head, always: bool = False) -> int:
    """Bytes of workspace of the kernel in which neighbouring tokens walk the pages they chose together, where it takes this call (rows that
    TMA can address, some pages, a scale that is positive in 32 bits) and is the shorter way (or ``always``); else 0."""
    q, ldq, out, ldo, cache, num_pages, _, width, _, B, _, _, top, T, H, Hkv, D, page_size, scale = head
    if not scale > 2.0 ** -150 or num_pages == 0 or ldq % 8 or ldo % 8 or (q | out | cache) % 16 or num_pages * 2 * Hkv * page_size > 0x7fffffff:
        return 0
    f = library("attention_pages_umma").dinfer_attention_pages_umma_workspace
    f.argtypes, f.restype = [c_int] * 9, c_int64
    return f(B, width, top, T, H, Hkv, D, page_size, 0 if always else _multiprocessors())


def _here(what: str, *tensors) -> None:
    """On CUDA, all on the current device (the kernels run there, whatever the tensors say)."""
    at = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != at:
            require_cuda(*tensors)
            raise KernelError(f"{what}: tensors on devices {at} and {t.get_device()}")
    if at < 0 or at != _device():
        require_cuda(*tensors)
        raise KernelError(f"{what}: tensors on device {at}, the current device is {_device()}")


def _ints(what: str, names: str, *tensors) -> None:
    for t in tensors:
        if t.dtype != _I32 or not t.is_contiguous():
            raise KernelError(f"{what}: {names} must be contiguous int32")


def _batch(what: str, T: int, block_table, cu_seqlens, positions):
    """(requests, table width)"""
    shape = block_table.shape
    if len(shape) != 2 or cu_seqlens.shape != (shape[0] + 1,) or positions.numel() != T or shape[0] == 0:
        raise KernelError(f"{what}: block_table [B, width] with B > 0, cu_seqlens [B + 1], positions [T]")
    if block_table.dtype != _I32 or cu_seqlens.dtype != _I32 or positions.dtype != _I32 or not block_table.is_contiguous() \
            or not cu_seqlens.is_contiguous() or not positions.is_contiguous():
        raise KernelError(f"{what}: block_table, cu_seqlens and positions must be contiguous int32")
    return shape


def _rows(what: str, name: str, t, width: int):
    """(rows, row stride) of rows [T, width] with a contiguous last axis"""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or stride[1] != 1 or shape[1] != width:
        raise KernelError(f"{what}: {name} rows [T, {width}] with a contiguous last axis, not {tuple(shape)}")
    return shape[0], stride[0]


def _meet(a: int, lda: int, b: int, ldb: int, rows: int, width: int, size: int) -> bool:
    """Whether rows of ``width`` elements at address ``a`` and others at ``b``, strides in elements, have memory in common (or lie among one
    another with strides that differ, which is taken for the same)."""
    wide, last = width * size, (rows - 1) * size
    if a + last * lda + wide <= b or b + last * ldb + wide <= a:
        return False
    step = lda * size
    return lda != ldb or step == 0 or (b - a) % step < wide or (a - b) % step < wide


def _heads(what: str, num_heads: int, num_kv_heads: int, head_dim: int) -> None:
    if num_heads <= 0 or num_kv_heads <= 0 or num_heads % num_kv_heads or not 0 < head_dim <= 512:
        raise KernelError(f"{what}: {num_heads} heads of {head_dim} over {num_kv_heads} key/value heads")


def _paged(what: str, cache):
    """(pages, 2, key/value heads, page size, head size) of a paged cache"""
    shape = cache.shape
    if len(shape) != 5 or shape[1] != 2 or shape[3] == 0 or not cache.is_contiguous():
        raise KernelError(f"{what}: cache shape {tuple(shape)} is not [pages, 2, Hkv, page, D], contiguous")
    return shape


def _code(what: str, dtype) -> int:
    code = DTYPE_CODE.get(dtype)
    if code is None:
        raise KernelError(f"{what}: dtype {dtype} is not one the kernels take (float32, bfloat16)")
    return code


def append(qkv: torch.Tensor, positions: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, eps: float,
           q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
           q_out: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, means: torch.Tensor,
           interleaved: bool = False) -> torch.Tensor:
    """From the projection's rows ``qkv`` [T, (H + 2 Hkv) D] (q heads | k heads | v heads; only read): q, normed and turned, into
    ``q_out`` [T, H * D]; k, normed and turned, and v into ``cache`` [pages, 2, Hkv, page, D] at ``slots`` (int32 [T], page *
    page_size + offset; -1: a row that is not kept; the batch may have a page's tokens in any order); and the mean of the keys, as cached, of every page whose last offset this
    step writes into ``means`` [pages, Hkv, D].  Other pages' means are left as they are.  ``q_weight`` / ``k_weight`` [D]: head norm
    ``x / sqrt(mean(x^2) + eps) * w``, or None for both; ``cos_sin`` f32 [positions, rot]: the angle table (``cos | sin``) of the
    first ``rot`` elements, pairs (i, i + rot/2) or with ``interleaved`` (2i, 2i + 1), which reaches every position; None: no
    rotation.  A slot is written by one token of the step at most.  Returns ``q_out``."""
    what = "page_append"
    _here(what, qkv, positions, q_weight, k_weight, cos_sin, q_out, cache, slots, means)
    _heads(what, num_heads, num_kv_heads, head_dim)
    T, ld = _rows(what, "qkv", qkv, (num_heads + 2 * num_kv_heads) * head_dim)
    rows, ldq = _rows(what, "q_out", q_out, num_heads * head_dim)
    num_pages, _, Hkv, page_size, D = _paged(what, cache)
    dt = qkv.dtype
    if rows != T or q_out.dtype != dt or cache.dtype != dt or means.dtype != dt or Hkv != num_kv_heads or D != head_dim:
        raise KernelError(f"{what}: q_out [T, H * D], cache [pages, 2, {num_kv_heads}, page, {head_dim}] and means of the rows' dtype")
    if means.shape != (num_pages, Hkv, D) or not means.is_contiguous():
        raise KernelError(f"{what}: means [pages, Hkv, D], contiguous, not {tuple(means.shape)}")
    _ints(what, "positions and slots", positions, slots)
    if positions.numel() != T or slots.numel() != T:
        raise KernelError(f"{what}: positions and slots int32 [T]")
    w_dt, qw, kw = dt, 0, 0
    if q_weight is not None and k_weight is not None:
        w_dt = q_weight.dtype
        if q_weight.numel() != D or k_weight.numel() != D or k_weight.dtype != w_dt or not q_weight.is_contiguous() \
                or not k_weight.is_contiguous():
            raise KernelError(f"{what}: norm weights [head_dim], contiguous, of one dtype")
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    elif q_weight is not None or k_weight is not None:
        raise KernelError(f"{what}: q and k norm weights come together")
    rot = table_rows = angles = 0
    if cos_sin is not None:
        if cos_sin.dtype != _F32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
            raise KernelError(f"{what}: angle table must be contiguous float32 [positions, rot]")
        table_rows, rot = cos_sin.shape
        angles = cos_sin.data_ptr()
    _call("page_append", "dinfer_page_append", what, qkv.data_ptr(), ld, positions.data_ptr(), qw, kw, eps, angles, table_rows, rot,
          1 if interleaved else 0, q_out.data_ptr(), ldq, cache.data_ptr(), means.data_ptr(), slots.data_ptr(), num_pages, page_size,
          T, num_heads, Hkv, D, _code(what, dt), _code(what, w_dt))
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
    shape = means.shape
    if len(shape) != 3 or not means.is_contiguous() or means.dtype != q.dtype:
        raise KernelError(f"{what}: means [pages, Hkv, D], contiguous, of q's dtype")
    num_pages, Hkv, D = shape
    _heads(what, num_heads, Hkv, D)
    T, ldq = _rows(what, "q", q, num_heads * D)
    B, width = _batch(what, T, block_table, cu_seqlens, positions)
    pages = width if pages is None else pages
    if not 0 <= pages <= width or page_size <= 0:
        raise KernelError(f"{what}: {pages} pages of {page_size} tokens, the table holds {width}")
    if out is None:
        out = torch.empty(T, Hkv, pages, dtype=_F32, device=q.device)
        ldt, ldg = Hkv * pages, pages
    else:
        if out.dtype != _F32 or out.shape != (T, Hkv, pages) or (pages > 1 and out.stride(2) != 1):
            raise KernelError(f"{what}: out float32 [T, Hkv, pages] with a contiguous last axis")
        ldt, ldg, _ = out.stride()
    _call("page_choice", "dinfer_page_scores", what, q.data_ptr(), ldq, means.data_ptr(), num_pages, block_table.data_ptr(), width,
          cu_seqlens.data_ptr(), B, positions.data_ptr(), out.data_ptr(), ldt, ldg, T, num_heads, Hkv, D, page_size, pages,
          _code(what, q.dtype), *((_multiprocessors(), gemm_ops._state(q.device)["status"].data_ptr()) if T >= 16 else (0, 0)))
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
    shape, stride = scores.shape, scores.stride()
    if len(shape) != 3 or scores.dtype != _F32 or (shape[2] > 1 and stride[2] != 1) or shape[2] == 0:
        raise KernelError(f"{what}: scores float32 [T, Hkv, pages] with a contiguous last axis and at least one page")
    T, Hkv, pages = shape
    _ints(what, "positions", positions)
    if positions.numel() != T:
        raise KernelError(f"{what}: positions int32 [T]")
    if page_size <= 0 or first < 0 or recent < 1 or top < first + recent:
        raise KernelError(f"{what}: {first} first and {recent} recent pages of {top}, pages of {page_size} tokens")
    if out is None:
        out = torch.empty(T, Hkv, top, dtype=_I32, device=scores.device)
    elif out.dtype != _I32 or out.shape != (T, Hkv, top) or not out.is_contiguous():
        raise KernelError(f"{what}: out int32 [T, Hkv, top], contiguous")
    _call("page_choice", "dinfer_choose_pages", what, scores.data_ptr(), stride[0], stride[1], positions.data_ptr(), page_size, first,
          recent, top, pages, out.data_ptr(), T, Hkv)
    return out


def attention_pages(q: torch.Tensor, out: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, positions: torch.Tensor, chosen: torch.Tensor, num_heads: int,
                    scale: float) -> torch.Tensor:
    """``out[t, h] = softmax over the seen keys (scale * q[t, h] . k) v``: token t sees the keys of its request's pages
    ``chosen[t, g]`` (int32 [T, Hkv, top]; g the head's key/value head) at positions up to ``positions[t]``.  Numbers outside the
    table's columns and pages the table does not hold are no pages, a page named twice counts twice, and a token that sees
    nothing gets zeros; one that sees keys whose scores are all -inf gets what is not a number, as the softmax does.  ``q`` and
    ``out`` [T, H * D] may be strided rows, of memory of their own; ``cache`` [pages, 2, Hkv, page, D].  Rows behind the last request's
    tokens are left as they are.  Returns ``out``."""
    what = "attention_pages"
    _here(what, q, out, cache, block_table, cu_seqlens, positions, chosen)
    dt = q.dtype
    if out.dtype != dt or cache.dtype != dt:
        raise KernelError(f"{what}: q, out and cache of one dtype")
    code = _code(what, dt)
    num_pages, _, Hkv, page_size, D = _paged(what, cache)
    _heads(what, num_heads, Hkv, D)
    T, ldq = _rows(what, "q", q, num_heads * D)
    rows, ldo = _rows(what, "out", out, num_heads * D)
    if rows != T:
        raise KernelError(f"{what}: out [T, H * D] of q's shape")
    q_at, out_at = q.data_ptr(), out.data_ptr()
    if T and _meet(q_at, ldq, out_at, ldo, T, num_heads * D, q.element_size()):
        raise KernelError(f"{what}: out must not be q's memory (a row may be made twice)")
    B, width = _batch(what, T, block_table, cu_seqlens, positions)
    _ints(what, "chosen", chosen)
    shape = chosen.shape
    if len(shape) != 3 or shape[0] != T or shape[1] != Hkv or shape[2] == 0:
        raise KernelError(f"{what}: chosen int32 [T, Hkv, top] with top > 0")
    top = shape[2]
    head = (q_at, ldq, out_at, ldo, cache.data_ptr(), num_pages, block_table.data_ptr(), width, cu_seqlens.data_ptr(), B,
            positions.data_ptr(), chosen.data_ptr(), top, T, num_heads, Hkv, D, page_size, scale)
    if dt == _BF16 and T and (T >= PORTION_TOKENS and T > B or num_heads > TOKEN_GROUP * Hkv or top > TOKEN_TOP):
        size = _portions(head)
        if size:
            work = torch.empty(size, dtype=torch.uint8, device=q.device)
            _call("attention_pages_umma", "dinfer_attention_pages_umma", "attention_pages_umma", *head, work.data_ptr(), size,
                  gemm_ops._state(q.device)["status"].data_ptr())
            return out
    _call("attention_pages", "dinfer_attention_pages", what, *head, _multiprocessors(), code)
    return out
