"""Paged fixed-rate E8 KV cache (CUDA, sm_100a): append, attention, page operations.

The chunk caches (codec, llm.compressed_attention) hold a batch of one length
per layer, as the reference's does (llm/compressed_kv_cache.py:342-395).  A
page pool holds sequences of any length that share, fork and free their
pages, at 4 bits per dimension and one fp32 scale per token, head and side:

  codes   int32 (layers, n_pages, 2, n_heads, page_tokens, head_dim / 8)
  scales  fp32  (layers, n_pages, 2, n_heads, page_tokens)     2: K, V
  table   int32 (rows, width)  the pages of a row's tokens, -1: none
  lens    int32 (rows,)        tokens held
  refs    int32 (n_pages,)     table entries naming a page, 0: free

``append`` and ``tree_attention`` take one layer of the pool, the page
operations all layers.  The page operations return new tables and leave their
inputs as they are.  Nothing here synchronises with the host: data errors (an
index outside the pool, too few free pages, a non-finite vector) are OR-ed
into ``err``, a (1,) int32 device tensor, for ``_lib.raise_flags``.
``llm.paged_cache.PagedKVCache`` keeps the tensors together.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import call, lib

_I32, _F32 = torch.int32, torch.float32


def empty_pool(n_layers: int, n_pages: int, n_heads: int, head_dim: int, page_tokens: int = 64, device=None):
    """(codes, scales, refs) of an empty pool."""
    _lib.require_cuda()
    dev = torch.device("cuda") if device is None else device
    if head_dim not in (64, 128) or page_tokens not in (16, 32, 64, 128, 256):
        raise ValueError("a page pool takes head_dim 64 or 128 and pages of 16, 32, 64, 128 or 256 tokens")
    shape = (n_layers, n_pages, 2, n_heads, page_tokens)
    return (torch.zeros(*shape, head_dim // 8, dtype=_I32, device=dev), torch.ones(shape, dtype=_F32, device=dev),
            torch.zeros(n_pages, dtype=_I32, device=dev))


def _pool(codes: torch.Tensor, scales: torch.Tensor, dims: int):
    """(device index, n_pages, heads, page_tokens, head_dim) of a pool or one of its layers, checked."""
    if not codes.is_cuda:
        _lib.require_cuda(codes)
    shape, index = codes.shape, codes.get_device()
    if len(shape) != dims or shape[-4] != 2 or codes.dtype is not _I32 or not codes.is_contiguous() or \
            _wrong(scales, _F32, shape[:-1], index):
        raise ValueError("a page pool is contiguous int32 codes " + ("(layers, " if dims == 6 else "(") +
                         "n_pages, 2, heads, page_tokens, head_dim / 8) with fp32 scales of the same leading shape")
    if shape[-1] not in (8, 16) or shape[-2] not in (16, 32, 64, 128, 256):
        raise ValueError("a page pool takes head_dim 64 or 128 and pages of 16, 32, 64, 128 or 256 tokens")
    return index, shape[-5], shape[-3], shape[-2], shape[-1] * 8


def _wrong(t: torch.Tensor, dtype, shape, index: int) -> bool:
    return t.dtype is not dtype or t.shape != shape or t.get_device() != index or not t.is_contiguous()


def _need(t: torch.Tensor, dtype, shape, name: str, index: int) -> int:
    """The address of t, which must be contiguous, of this dtype, shape and device."""
    if _wrong(t, dtype, shape, index):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{index}")
    return t.data_ptr()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last dimension, 16-byte aligned, its other strides multiples of 8 elements."""
    s = t.stride()  # of three or four dimensions
    if s[-1] == 1 and not (t.data_ptr() & 15 or (s[0] | s[1] | s[-2]) & 7):
        return t
    if t.is_contiguous() and not t.data_ptr() & 15:  # (a dimension of one element may have any stride)
        return t.reshape(-1).view(t.shape)
    return t.clone(memory_format=torch.contiguous_format)


def append(codes: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
           dequantised: bool = False, err: Optional[torch.Tensor] = None):
    """Quantise tokens into their slots of one layer (lq_paged_append).

    k, v (n, heads, head_dim), float32 / float16 / bfloat16, any strides; slots
    int64 (n,): page * page_tokens + row, distinct, negative: not stored.  With
    ``dequantised`` returns the stored values (k, v) in the inputs' dtype, as
    CompressedKVCache.update() does, else None."""
    index, n_pages, H, P, D = _pool(codes, scales, 5)
    shape = k.shape
    if len(shape) != 3 or shape[1] != H or shape[2] != D or v.shape != shape or k.dtype is not v.dtype or \
            k.get_device() != index or v.get_device() != index:
        raise ValueError(f"k and v must be (n, {H}, {D}) tensors of one dtype on the pool's device")
    n = shape[0]
    slots_p, dt = _need(slots, torch.int64, (n,), "slots", index), _lib.dtype_code(k.dtype)
    k, v = _rows(k), _rows(v)
    ko = vo = None
    if dequantised:
        ko = torch.empty_like(k) if k.is_contiguous() else torch.empty_like(k, memory_format=torch.contiguous_format)
        vo = torch.empty_like(ko)
    call("lq_paged_append", index, k.data_ptr(), v.data_ptr(), dt, n, H, D, *k.stride()[:2], *v.stride()[:2], slots_p,
         n_pages, P, codes.data_ptr(), scales.data_ptr(), _ptr(ko), _ptr(vo), _ptr(err))
    return (ko, vo) if dequantised else None


def tree_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor,
                   lens: torch.Tensor, mask: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                   max_len: Optional[int] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                   err: Optional[torch.Tensor] = None):
    """Attention of T positions a sequence over one layer's pages (lq_paged_attention).

    q (B, Hq, T, D) float16 / bfloat16, Hq a multiple of the pool's heads.  The
    last T of a sequence's ``lens`` tokens are the positions' own (drafts of a
    tree, a chunk of a prompt, or the one token of a decode step): position t
    sees all tokens before them, and draft j where mask[t, j] -- bool (T, T) or
    (B, T, T), e.g. each draft's ancestors and itself -- or, without a mask,
    j <= t.  ``max_len``: an upper bound on ``lens`` known to the host (default:
    the table's width), which sets the split; longer rows are right, but slower.  Returns o (B, Hq, T, D) in q's
    dtype (and the fp32 (B, Hq, T) log-sum-exp if return_lse); a position that
    sees nothing gives 0 and -inf."""
    index, n_pages, H, P, D = _pool(codes, scales, 5)
    if q.dim() != 4 or q.get_device() != index:
        raise ValueError(f"q must be (B, Hq, T, {D}) on the pool's device")
    B, Hq, T, d = q.shape
    if d != D or Hq % H or Hq == 0 or T == 0:
        raise ValueError(f"q must be (B, Hq, T, {D}) with Hq a multiple of {H} and T at least 1")
    dtype = q.dtype
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError(f"tree_attention takes float16 or bfloat16 queries, not {dtype}")
    width = table.shape[1] if table.dim() == 2 else -1
    table_p, lens_p = _need(table, _I32, (B, width), "table", index), _need(lens, _I32, (B,), "lens", index)
    mask_p, mask_stride = None, 0
    if mask is not None:
        per_row = mask.dim() == 3
        mask_p = _need(mask, torch.bool, (B, T, T) if per_row else (T, T), "mask", index)
        mask_stride = T * T if per_row else 0
    q = _rows(q)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        if _need(out, dtype, (B, Hq, T, D), "out", index) % (D // 16):
            raise ValueError(f"out must be aligned to {D // 16} bytes")
    lse = lens.new_empty((B, Hq, T), dtype=_F32) if return_lse else None
    bound = width * P if max_len is None else min(int(max_len), width * P)
    need = _attention_workspace(B, H, Hq // H, T, D, bound)
    ws = codes.new_empty(need // 4) if need else None
    call("lq_paged_attention", index, q.data_ptr(), _lib.dtype_code(dtype), *q.stride()[:3], codes.data_ptr(),
         scales.data_ptr(), n_pages, P, table_p, width, width, lens_p, bound, mask_p, mask_stride, B, H, Hq // H, T, D,
         1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), out.data_ptr(), _ptr(lse), _ptr(ws), need,
         _ptr(err))
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _attention_workspace(*shape: int) -> int:
    return lib().lq_paged_attention_workspace(*shape)


def fork_pages(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
               parents: torch.Tensor, reserve: int = 0, err: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """New (table, lens, refs) whose row i continues old row parents[i] (int64; -1:
    an empty row), with pages for ``reserve`` more tokens (lq_pages_fork).

    Full pages are shared; the page a row writes to next stays with the row's
    first child if nobody else names it (refs 1), the others get a copy of its
    live rows in a fresh page.  Rows that no child names are freed.  parents = arange reserves, parents with -1
    entries free rows, repeated parents fork: beam search's reordering is
    parents = the selected beams."""
    index, n_pages, H, P, D = _pool(codes, scales, 6)
    if table.dim() != 2 or parents.dim() != 1:
        raise ValueError("table is (rows, width) and parents (children,)")
    (rows, width), n = table.shape, parents.shape[0]
    table_p, lens_p = _need(table, _I32, (rows, width), "table", index), _need(lens, _I32, (rows,), "lens", index)
    refs_p, parents_p = _need(refs, _I32, (n_pages,), "refs", index), _need(parents, torch.int64, (n,), "parents", index)
    # (empty_like is the cheaper call)
    new_table = torch.empty_like(table) if n == rows else table.new_empty((n, width))
    new_lens = torch.empty_like(lens) if n == rows else lens.new_empty(n)
    new_refs = torch.empty_like(refs)
    need = 4 * (rows + n + n_pages)  # lq_pages_fork_workspace
    ws = refs.new_empty(need // 4)
    call("lq_pages_fork", index, table_p, rows, width, lens_p, refs_p, parents_p, n, int(reserve), new_table.data_ptr(),
         new_lens.data_ptr(), new_refs.data_ptr(), codes.data_ptr(), scales.data_ptr(), codes.shape[0], n_pages, H, P, D,
         ws.data_ptr(), need, _ptr(err))
    return new_table, new_lens, new_refs


def compact_pages(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, refs: torch.Tensor,
                  err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the live pages to the front of the pool (lq_pages_compact): (table,
    refs, n_live), n_live a (1,) int32 device tensor.  ``table`` holds every
    entry that names a page (any shape)."""
    index, n_pages, H, P, D = _pool(codes, scales, 6)
    table_p, refs_p = _need(table, _I32, table.shape, "table", index), _need(refs, _I32, (n_pages,), "refs", index)
    new_table, new_refs, n_live = torch.empty_like(table), torch.empty_like(refs), refs.new_empty(1)
    need = 12 * n_pages + 4  # lq_pages_compact_workspace
    ws = refs.new_empty(need // 4)
    call("lq_pages_compact", index, table_p, table.numel(), refs_p, new_table.data_ptr(), new_refs.data_ptr(),
         n_live.data_ptr(), codes.data_ptr(), scales.data_ptr(), codes.shape[0], n_pages, H, P, D, ws.data_ptr(), need,
         _ptr(err))
    return new_table, new_refs, n_live


def copy_pages(codes: torch.Tensor, scales: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               count: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> None:
    """Copy pages src[i] to dst[i] in all layers (lq_pages_copy); no page is both
    a source and a destination, and no destination is named twice.  ``count``, a
    (1,) int32 device tensor, limits the pairs."""
    index, n_pages, H, P, D = _pool(codes, scales, 6)
    n = src.numel()
    src_p, dst_p = _need(src, _I32, (n,), "src", index), _need(dst, _I32, (n,), "dst", index)
    if count is None:
        count = torch.full((1,), n, dtype=_I32, device=src.device)
    call("lq_pages_copy", index, src_p, dst_p, _need(count, _I32, (1,), "count", index), n, codes.data_ptr(),
         scales.data_ptr(), codes.shape[0], n_pages, H, P, D, _ptr(err))


def accept_tokens(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, n_draft: int,
                  accepted: torch.Tensor, err: Optional[torch.Tensor] = None,
                  refs: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keep the accepted ones of each row's last ``n_draft`` tokens (lq_pages_accept).

    accepted int32 (rows, most): draft indices, strictly ascending (a path of
    the tree from its root), padded with -1.  Their rows move to the front of
    the drafts' slots in all layers.  Returns the new lens.

    The pages that drafts move into must be their row's own.  A fork after the
    drafts came in may have shared one; with ``refs`` a row that would move a
    draft into such a page is left as it is and reported (EF_PAGE)."""
    index, n_pages, H, P, D = _pool(codes, scales, 6)
    if table.dim() != 2 or accepted.dim() != 2:
        raise ValueError("table is (rows, width) and accepted (rows, most)")
    (rows, width), most = table.shape, accepted.shape[1]
    table_p, lens_p = _need(table, _I32, (rows, width), "table", index), _need(lens, _I32, (rows,), "lens", index)
    accepted_p = _need(accepted, _I32, (rows, most), "accepted", index)
    new_lens = torch.empty_like(lens)
    rest = (int(n_draft), accepted_p, most, new_lens.data_ptr(), codes.data_ptr(), scales.data_ptr(), codes.shape[0],
            n_pages, H, P, D, _ptr(err))
    if refs is None:
        call("lq_pages_accept", index, table_p, rows, width, lens_p, *rest)
    else:
        call("lq_pages_accept_shared", index, table_p, rows, width, lens_p, _need(refs, _I32, (n_pages,), "refs", index),
             *rest)
    return new_lens
