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

import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, lib, ptr, stream_handle

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
    """The pool's shape after its layer dimension, checked."""
    _lib.require_cuda(codes)
    shape = codes.shape
    if len(shape) != dims or codes.dtype != _I32 or scales.dtype != _F32 or scales.shape != shape[:-1] or \
            shape[-4] != 2 or not (codes.is_contiguous() and scales.is_contiguous()) or scales.device != codes.device:
        raise ValueError("a page pool is contiguous int32 codes " + ("(layers, " if dims == 6 else "(") +
                         "n_pages, 2, heads, page_tokens, head_dim / 8) with fp32 scales of the same leading shape")
    if shape[-1] not in (8, 16) or shape[-2] not in (16, 32, 64, 128, 256):
        raise ValueError("a page pool takes head_dim 64 or 128 and pages of 16, 32, 64, 128 or 256 tokens")
    return shape[-5], shape[-3], shape[-2], shape[-1] * 8


def _index(t: torch.Tensor, dtype, shape, name: str, device):
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last dimension, 16-byte aligned, its other strides multiples of 8 elements."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def append(codes: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
           dequantised: bool = False, err: Optional[torch.Tensor] = None):
    """Quantise tokens into their slots of one layer (lq_paged_append).

    k, v (n, heads, head_dim), float32 / float16 / bfloat16, any strides; slots
    int64 (n,): page * page_tokens + row, distinct, negative: not stored.  With
    ``dequantised`` returns the stored values (k, v) in the inputs' dtype, as
    CompressedKVCache.update() does, else None."""
    n_pages, H, P, D = _pool(codes, scales, 5)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (H, D) or k.dtype != v.dtype or \
            k.device != codes.device or v.device != codes.device:
        raise ValueError(f"k and v must be (n, {H}, {D}) tensors of one dtype on the pool's device")
    n = k.shape[0]
    _index(slots, torch.int64, (n,), "slots", codes.device)
    dt = _lib.dtype_code(k.dtype)
    k, v = _rows(k), _rows(v)
    ko = vo = None
    if dequantised:
        ko, vo = torch.empty((n, H, D), dtype=k.dtype, device=k.device), torch.empty((n, H, D), dtype=k.dtype,
                                                                                   device=k.device)
    with torch.cuda.device(codes.device):
        check(lib().lq_paged_append(ptr(k), ptr(v), dt, n, H, D, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                    ptr(slots), n_pages, P, ptr(codes), ptr(scales), ptr(ko), ptr(vo), ptr(err),
                                    stream_handle(codes.device)), "lq_paged_append")
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
    the table's width), which sets the split.  Returns o (B, Hq, T, D) in q's
    dtype (and the fp32 (B, Hq, T) log-sum-exp if return_lse); a position that
    sees nothing gives 0 and -inf."""
    n_pages, H, P, D = _pool(codes, scales, 5)
    dev = codes.device
    if q.dim() != 4 or q.shape[3] != D or q.shape[1] % H or q.shape[1] == 0 or q.shape[2] == 0 or q.device != dev:
        raise ValueError(f"q must be (B, Hq, T, {D}) with Hq a multiple of {H}, on the pool's device")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"tree_attention takes float16 or bfloat16 queries, not {q.dtype}")
    B, Hq, T, _ = q.shape
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table must hold {B} rows")
    _index(table, _I32, table.shape, "table", dev)
    _index(lens, _I32, (B,), "lens", dev)
    mask_stride = 0
    if mask is not None:
        _index(mask, torch.bool, (B, T, T) if mask.dim() == 3 else (T, T), "mask", dev)
        mask_stride = T * T if mask.dim() == 3 else 0
    q = _rows(q)
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=dev)
    else:
        _index(out, q.dtype, (B, Hq, T, D), "out", dev)
    lse = torch.empty((B, Hq, T), dtype=_F32, device=dev) if return_lse else None
    width = table.shape[1]
    bound = width * P if max_len is None else min(int(max_len), width * P)
    with torch.cuda.device(dev):
        need = lib().lq_paged_attention_workspace(B, H, Hq // H, T, D, bound)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(lib().lq_paged_attention(ptr(q), _lib.dtype_code(q.dtype), q.stride(0), q.stride(1), q.stride(2),
                                       ptr(codes), ptr(scales), n_pages, P, ptr(table), width, width, ptr(lens), bound,
                                       ptr(mask), mask_stride, B, H, Hq // H, T, D,
                                       1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), ptr(out), ptr(lse),
                                       ptr(ws), need, ptr(err), stream_handle(dev)), "lq_paged_attention")
    return (out, lse) if return_lse else out


def fork_pages(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
               parents: torch.Tensor, reserve: int = 0, err: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """New (table, lens, refs) whose row i continues old row parents[i] (int64; -1:
    an empty row), with pages for ``reserve`` more tokens (lq_pages_fork).

    Full pages are shared; the page a row writes to next stays with the row's
    first child, the others get a copy of its live rows in a fresh page.  Rows
    that no child names are freed.  parents = arange reserves, parents with -1
    entries free rows, repeated parents fork: beam search's reordering is
    parents = the selected beams."""
    n_pages, H, P, D = _pool(codes, scales, 6)
    dev = codes.device
    if table.dim() != 2 or parents.dim() != 1:
        raise ValueError("table is (rows, width) and parents (children,)")
    (rows, width), n = table.shape, parents.shape[0]
    _index(table, _I32, (rows, width), "table", dev)
    _index(lens, _I32, (rows,), "lens", dev)
    _index(refs, _I32, (n_pages,), "refs", dev)
    _index(parents, torch.int64, (n,), "parents", dev)
    new = (torch.empty((n, width), dtype=_I32, device=dev), torch.empty(n, dtype=_I32, device=dev),
           torch.empty(n_pages, dtype=_I32, device=dev))
    with torch.cuda.device(dev):
        need = lib().lq_pages_fork_workspace(rows, n, n_pages)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        check(lib().lq_pages_fork(ptr(table), rows, width, ptr(lens), ptr(refs), ptr(parents), n, int(reserve),
                                  *(ptr(t) for t in new), ptr(codes), ptr(scales), codes.shape[0], n_pages, H, P, D,
                                  ptr(ws), need, ptr(err), stream_handle(dev)), "lq_pages_fork")
    return new


def compact_pages(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, refs: torch.Tensor,
                  err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the live pages to the front of the pool (lq_pages_compact): (table,
    refs, n_live), n_live a (1,) int32 device tensor.  ``table`` holds every
    entry that names a page (any shape)."""
    n_pages, H, P, D = _pool(codes, scales, 6)
    dev = codes.device
    _index(table, _I32, table.shape, "table", dev)
    _index(refs, _I32, (n_pages,), "refs", dev)
    new_table, new_refs = torch.empty_like(table), torch.empty_like(refs)
    n_live = torch.empty(1, dtype=_I32, device=dev)
    with torch.cuda.device(dev):
        need = lib().lq_pages_compact_workspace(n_pages)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        check(lib().lq_pages_compact(ptr(table), table.numel(), ptr(refs), ptr(new_table), ptr(new_refs), ptr(n_live),
                                     ptr(codes), ptr(scales), codes.shape[0], n_pages, H, P, D, ptr(ws), need, ptr(err),
                                     stream_handle(dev)), "lq_pages_compact")
    return new_table, new_refs, n_live


def copy_pages(codes: torch.Tensor, scales: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               count: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> None:
    """Copy pages src[i] to dst[i] in all layers (lq_pages_copy); no page is both
    a source and a destination, and no destination is named twice.  ``count``, a
    (1,) int32 device tensor, limits the pairs."""
    n_pages, H, P, D = _pool(codes, scales, 6)
    dev = codes.device
    n = src.numel()
    _index(src, _I32, (n,), "src", dev)
    _index(dst, _I32, (n,), "dst", dev)
    if count is None:
        count = torch.full((1,), n, dtype=_I32, device=dev)
    _index(count, _I32, (1,), "count", dev)
    with torch.cuda.device(dev):
        check(lib().lq_pages_copy(ptr(src), ptr(dst), ptr(count), n, ptr(codes), ptr(scales), codes.shape[0], n_pages, H,
                                  P, D, ptr(err), stream_handle(dev)), "lq_pages_copy")


def accept_tokens(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, n_draft: int,
                  accepted: torch.Tensor, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keep the accepted ones of each row's last ``n_draft`` tokens (lq_pages_accept).

    accepted int32 (rows, most): draft indices, strictly ascending (a path of
    the tree from its root), padded with -1.  Their rows move to the front of
    the drafts' slots in all layers.  Returns the new lens."""
    n_pages, H, P, D = _pool(codes, scales, 6)
    dev = codes.device
    if table.dim() != 2 or accepted.dim() != 2:
        raise ValueError("table is (rows, width) and accepted (rows, most)")
    (rows, width), most = table.shape, accepted.shape[1]
    _index(table, _I32, (rows, width), "table", dev)
    _index(lens, _I32, (rows,), "lens", dev)
    _index(accepted, _I32, (rows, most), "accepted", dev)
    new_lens = torch.empty_like(lens)
    with torch.cuda.device(dev):
        check(lib().lq_pages_accept(ptr(table), rows, width, ptr(lens), int(n_draft), ptr(accepted), most,
                                    ptr(new_lens), ptr(codes), ptr(scales), codes.shape[0], n_pages, H, P, D, ptr(err),
                                    stream_handle(dev)), "lq_pages_accept")
    return new_lens
