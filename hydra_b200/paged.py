"""Serving on a paged key-value cache: requests of any lengths in one batch, their keys and values in pages that lie anywhere
in two tensors.  One step of a server is

    plan = paged_plan(context_lens, new_lens, block_tables, free_pages, page_size, max_new_tokens)   # pages and slots
    q = paged_append(q, k, v, k_cache, v_cache, plan.slots, cos, sin, plan.positions, ...)           # per layer
    o = paged_decode_attention(q, k_cache, v_cache, block_tables, plan.kv_lens)                      # per layer

all on the device: nothing here reads a length on the host, so a step can be captured into a CUDA graph and replayed while the
tensors' contents change (padded batches: requests of length 0, rows with slot and position -1).  The log probabilities of
the answer's tokens are ``hydra_b200.sampling.token_logprobs``.

The reference has no cache (its generation helper re-runs the whole forward, diagnostics/eval_checkpoint.py:127-160), so
nothing here has a counterpart in it.  The calls are plain functions, not registered torch ops: they write into the caller's
cache.  They are inference only: they refuse tensors that autograd would record, tensors that they write count as changed, and
under ``torch.compile`` they break the graph.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib, kernels

Tensor = torch.Tensor
_MAX = kernels._INT32_MAX


class PagedPlan(NamedTuple):
    """What :func:`paged_plan` writes for a step of ``B`` requests."""
    kv_lens: Tensor      # int32 [B]      tokens in the cache once the new ones are there
    cu_new: Tensor       # int32 [B + 1]  new tokens before each request: request b's are rows cu_new[b] .. cu_new[b + 1] - 1
    positions: Tensor    # int32 [max_new_tokens]  -1 behind the last token
    slots: Tensor        # int64 [max_new_tokens]  page * page_size + row; -1 behind the last token or without a page
    free_start: Tensor   # int32 [1]      where the free list goes on: the next call's ``free_start``
    status: Tensor       # int32 [1]      0, or bits of ``PLAN_OUT_OF_PAGES`` and so on


PLAN_OUT_OF_PAGES = _lib.PLAN_OUT_OF_PAGES
PLAN_TABLE_FULL = _lib.PLAN_TABLE_FULL
PLAN_OUT_OF_ROOM = _lib.PLAN_OUT_OF_ROOM
PLAN_BAD_LENGTH = _lib.PLAN_BAD_LENGTH


def _ints(what: str, t: Tensor, dtype: torch.dtype, dim: int) -> Tensor:
    if t.dtype != dtype or t.dim() != dim:
        raise ValueError(f"{what} must be a {dim}-dimensional {str(dtype).split('.')[1]} tensor, got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def paged_plan(context_lens: Tensor, new_lens: Tensor, block_tables: Tensor, free_pages: Tensor, page_size: int,
               max_new_tokens: int, free_start: Optional[Tensor] = None) -> PagedPlan:
    """Pages, slots and positions of a step from the requests' lengths (``hb200_paged_plan``), in one launch.

    ``context_lens`` and ``new_lens`` int32 [B] (up to 4096 requests): tokens that request b has in the cache and tokens that it
    adds.  ``block_tables`` int32 [B, width]: its pages; the entries that it needs beyond ``ceil(context / page_size)`` are
    taken from ``free_pages`` int32 [F], request after request, from ``free_start`` int32 [1] on (default 0), and written in
    place.  The other inputs are left as they are, so repeating a call repeats its result; none of them may lie between the
    tables' first and last entry.  ``max_new_tokens``: rows of
    ``slots`` and ``positions`` (the new tokens of all requests, packed; a fixed number serves a captured graph).

    Where pages, table columns or rows run out the entries concerned are -1 and ``status`` says so (one int32 on the device:
    reading it is the caller's choice); nothing is written out of range.  To recycle a finished request's pages, build the
    next free list with them: ``torch.cat([free_pages[start:], block_tables[b, :n]])``."""
    dev = kernels._require_cuda(context_lens, new_lens, block_tables, free_pages)
    context_lens = _ints("paged_plan: context_lens", context_lens, torch.int32, 1)
    new_lens = _ints("paged_plan: new_lens", new_lens, torch.int32, 1)
    free_pages = _ints("paged_plan: free_pages", free_pages, torch.int32, 1)
    B, shape = context_lens.shape[0], block_tables.shape
    if new_lens.shape[0] != B or len(shape) != 2 or shape[0] != B or block_tables.dtype != torch.int32:
        raise ValueError(f"paged_plan: {B} context lengths, {new_lens.shape[0]} new lengths and int32 block tables [{B}, width] "
                         f"are wanted, got {block_tables.dtype} {tuple(shape)}")
    width, (ld, unit) = shape[1], block_tables.stride()
    if (width > 1 and unit != 1) or (B > 1 and ld < width):
        raise ValueError("paged_plan: the rows of block_tables must be contiguous and apart (they are written in place)")
    page_size, room = int(page_size), int(max_new_tokens)
    if page_size < 1 or room < 0:
        raise ValueError(f"paged_plan: page_size {page_size} and max_new_tokens {room} must be positive")
    if B > _MAX or width > _MAX or page_size > _MAX or room > _MAX:
        raise kernels._past_int32("paged_plan", B, width, page_size, room)
    if free_start is not None:
        if free_start.get_device() != dev.index or free_start.dtype != torch.int32 or free_start.numel() != 1:
            raise ValueError("paged_plan: free_start must be one int32 on the tables' device")
    i32, one = torch.int32, (1,)
    with kernels._on(dev):
        new = kernels._empty_strided
        plan = PagedPlan(new((B,), one, i32), new((B + 1,), one, i32), new((room,), one, i32), new((room,), one, torch.int64), new(one, one, i32),
                         new(one, one, i32))
        kv_lens, cu_new, positions, slots, start_out, status = plan
        _lib.check(_lib.lib().hb200_paged_plan(
            context_lens.data_ptr(), new_lens.data_ptr(), B, block_tables.data_ptr(), ld if B > 1 else width, width,
            page_size, free_pages.data_ptr(), free_pages.shape[0], free_start.data_ptr() if free_start is not None else None,
            kv_lens.data_ptr(), cu_new.data_ptr(), positions.data_ptr(), slots.data_ptr(), room, start_out.data_ptr(),
            status.data_ptr(), kernels._stream(dev)), "paged_plan")
    increment_version(block_tables)   # (written behind torch's back: a graph that kept the old entries has to know)
    return plan


def _cache(what: str, k_cache: Tensor, v_cache: Tensor) -> _lib.PagedCache:
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"{what}: k_cache and v_cache must be [num_pages, kv_heads, page_size, head_dim] of one shape and dtype, "
                         f"got {tuple(shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}")
    pages, heads, rows, hd = shape
    if pages > _MAX or heads > _MAX or rows > _MAX or hd > _MAX:
        raise kernels._past_int32(what, *shape)
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and hd > 1:
        raise ValueError(f"{what}: a head's row in the cache must be contiguous")
    if pages * heads * rows * hd == 0:
        raise ValueError(f"{what}: an empty cache {tuple(shape)}")
    return _lib.PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages, rows, heads, hd,
                           kernels._dtype_code(k_cache))   # in the order of the struct


def paged_append(q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slots: Tensor, cos: Tensor, sin: Tensor,
                 positions: Tensor, *, q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
                 norm: Optional[str] = "rms", eps: float = 1e-6, q_scale: float = 1.0, k_scale: float = 1.0,
                 layout: str = "interleaved") -> Tensor:
    """:func:`hydra_b200.kernels.fused_qk_norm_rope` of packed tokens whose keys go straight into the cache, and their values
    with them (``hb200_qk_norm_rope``): one pass over the projection's rows.

    q [T, Hq, hd], k and v [T, Hkv, hd] (views of one projection are read in place), ``slots`` int64 and ``positions`` int32 or
    int64 [T] as :func:`paged_plan` writes them, caches [num_pages, Hkv, page_size, hd] in q's dtype by any strides with
    contiguous rows (token-major pages: pass ``cache.transpose(1, 2)``) that do not overlap: not one another, k's not v's (they may
    lie side by side in one tensor), and neither any other argument (which is refused).  hd up to 256 in any of the three types;
    :func:`paged_decode_attention` reads bf16 and f16 caches with hd a multiple of 8.  Returns the normed and rotated queries
    [T, Hq, hd]; cache rows without a slot here stay as they are.  A row with a negative position is padding (zeros
    returned, nothing stored), one with a negative slot is computed but not stored; a position beyond the tables or a slot
    beyond the cache gives NaN.  Of two rows with the same slot either's values may stay, or some of each's."""
    dev = kernels._require_cuda(q, k, v, k_cache, v_cache, slots, cos, sin, positions)
    a, b = q.shape, k.shape
    if len(a) != 3 or len(b) != 3 or v.shape != b or a[0] != b[0] or a[2] != b[2]:
        raise ValueError(f"paged_append: q [T, Hq, hd], k and v [T, Hkv, hd] are wanted, got {tuple(a)}, {tuple(b)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype == k_cache.dtype):
        raise ValueError("paged_append: q, k, v and the caches must share a dtype")
    cache = _cache("paged_append", k_cache, v_cache)
    if cache.n_kv_heads != b[1] or cache.head_dim != b[2]:
        raise ValueError(f"paged_append: keys {tuple(b)} do not fit the cache {tuple(k_cache.shape)}")
    slots = _ints("paged_append: slots", slots, torch.int64, 1)
    if slots.shape[0] != a[0]:
        raise ValueError(f"paged_append: {slots.shape[0]} slots for {a[0]} tokens")
    if k_cache.requires_grad or v_cache.requires_grad:
        raise RuntimeError("paged_append: the caches are written in place and cannot require grad")
    if forward_ad._current_level >= 0:
        kernels._refuse_tangents("paged_append", k_cache, v_cache)
    q_out, _ = kernels._qk_norm_rope("paged_append", dev, q, k, cos, sin, positions, q_weight, k_weight, norm, eps, q_scale, k_scale,
                                     layout, v=v, slots=slots, cache=cache)
    increment_version((k_cache, v_cache))
    return q_out


_workspace_bytes: dict = {}     # (device, requests, query heads, kv heads, head size) -> bytes


def paged_decode_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_tables: Tensor, kv_lens: Tensor, *,
                           scale: Optional[float] = None, return_lse: bool = False,
                           out: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Attention of one new token per request over the paged cache (``hb200_paged_decode_attention``): request b's query heads
    q[b] [Hq, hd] against its first ``kv_lens[b]`` cached tokens, grouped-query heads in order (query head h reads kv head
    ``h // (Hq // Hkv)``), softmax of ``scale * q . k`` (default ``hd ** -0.5``).

    q [B, Hq, hd] bf16 or f16 (up to 4096 requests, 1024 heads; hd a multiple of 8 up to 256), caches as in
    :func:`paged_append`, ``block_tables`` int32 [B, width], ``kv_lens`` int32 [B].  Returns [B, Hq, hd] (in ``out``
    if given, which must not lie within the memory that an input reaches over) and, if asked, the fp32 logarithm of each softmax's
    sum [B, Hq].  Scores and weights in 32 bits, for any finite scale.  A request of length 0 gives zeros and -inf; one whose
    table names a page outside the cache, or whose length passes its table, gives NaN.  What lies behind a
    request's length in its last page is not looked at; an infinite value among the attended ones gives NaN or infinity in
    its column.  Requests may share pages.  Equal inputs give equal bits."""
    dev = kernels._require_cuda(q, k_cache, v_cache, block_tables, kv_lens)
    kernels._refuse_autograd("paged_decode_attention", q, k_cache, v_cache, out)
    dtype = q.dtype
    if q.dim() != 3 or dtype != k_cache.dtype or (dtype != torch.bfloat16 and dtype != torch.float16):
        raise ValueError(f"paged_decode_attention: q must be [B, Hq, hd] in the caches' dtype, bfloat16 or float16, got {tuple(q.shape)} {q.dtype}")
    cache = _cache("paged_decode_attention", k_cache, v_cache)
    B, Hq, hd = q.shape
    if cache.head_dim != hd or Hq < 1 or Hq % cache.n_kv_heads:
        raise ValueError(f"paged_decode_attention: queries {tuple(q.shape)} do not fit the cache {tuple(k_cache.shape)}")
    kv_lens = _ints("paged_decode_attention: kv_lens", kv_lens, torch.int32, 1)
    block_tables = _ints("paged_decode_attention: block_tables", block_tables, torch.int32, 2)
    rows, width = block_tables.shape
    if B > _MAX or Hq > _MAX or width > _MAX:
        raise kernels._past_int32("paged_decode_attention", B, Hq, width)
    if kv_lens.shape[0] != B or rows != B:
        raise ValueError(f"paged_decode_attention: {B} queries, {kv_lens.shape[0]} lengths, {rows} table rows")
    if (cache.k_stride_page | cache.k_stride_head | cache.k_stride_row | cache.v_stride_page | cache.v_stride_head | cache.v_stride_row) % 8 \
            or (cache.k | cache.v) % 16:
        raise ValueError("paged_decode_attention: the rows of the caches must begin on 16-byte boundaries")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"paged_decode_attention: scale {scale}")
    sb, sh, unit = q.stride()
    if unit != 1 or sb % 8 or sh % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        q = q.clone() if q.data_ptr() % 16 else q
        sb, sh, _ = q.stride()
    given = out is not None
    if given:
        if out.shape != q.shape or out.dtype != dtype or out.device != dev or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("paged_decode_attention: out must be a contiguous, 16-byte aligned tensor of q's shape and dtype")
        for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables), ("kv_lens", kv_lens)):
            if kernels._overlap(out, t):
                raise ValueError(f"paged_decode_attention: out must not overlap {name}, which is read while results are stored")
    with kernels._on(dev):
        new = kernels._empty_strided
        if out is None:
            out = new((B, Hq, hd), (Hq * hd, hd, 1), dtype)
        lse = new((B, Hq), (Hq, 1), torch.float32) if return_lse else None
        if B > 0:
            L = _lib.lib()
            key = (dev.index, B, Hq, cache.n_kv_heads, hd)
            n = _workspace_bytes.get(key)
            if n is None:
                n = _workspace_bytes[key] = L.hb200_paged_attention_workspace_bytes(B, Hq, cache.n_kv_heads, hd)
            ws = new((n,), (1,), torch.uint8)
            _lib.check(L.hb200_paged_decode_attention(
                cache, q.data_ptr(), sb, sh, out.data_ptr(), lse.data_ptr() if return_lse else None,
                block_tables.data_ptr(), width, width, kv_lens.data_ptr(), B, Hq, scale,
                ws.data_ptr(), n, kernels._stream(dev)), "paged_decode_attention")
    if given:
        increment_version(out)
    return (out, lse) if return_lse else out


__all__ = ["PagedPlan", "paged_plan", "paged_append", "paged_decode_attention", "PLAN_OUT_OF_PAGES", "PLAN_TABLE_FULL",
           "PLAN_OUT_OF_ROOM", "PLAN_BAD_LENGTH"]
