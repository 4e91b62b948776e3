"""A paged E8 KV cache for search decoding: ragged batches, trees of drafts, beams.

``PagedKVCache`` keeps a page pool (paged.py) with the tables of its rows.  A
step of ``n`` new tokens a row is

    cache.begin(n)                      # pages and slots for the n tokens
    for layer in ...:
        cache.append(layer, k, v)       # (B, Hkv, n, D): quantised into the pages
        o = cache.attend(layer, q, mask)

after which the rows hold the n tokens.  For a tree of drafted tokens ``mask``
names each draft's ancestors and itself, and ``accept`` then keeps the drafts
that the model confirmed; for beams ``fork`` reorders the rows
(beam.beam_select's beams).  The reference's cache grows one dense buffer per
layer and has none of these (llm/compressed_kv_cache.py:342-395).

Nothing synchronises with the host: the host keeps an upper bound of the
lengths (``max_len``, which sets how attention splits its work and nothing
else; a caller that knows better after freeing rows may lower it), and
``flags()`` reads the error word.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import paged


class PagedKVCache:
    """A pool of n_pages pages of page_tokens tokens for n_layers layers.

    rows: sequences at the start, all empty; max_tokens: the longest a row may
    grow (the width of its table)."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, rows: int, max_tokens: int,
                 page_tokens: int = 64, device=None):
        self.codes, self.scales, self.refs = paged.empty_pool(n_layers, n_pages, n_kv_heads, head_dim, page_tokens,
                                                              device)
        dev = self.codes.device
        self.page_tokens = int(page_tokens)
        width = -(-int(max_tokens) // self.page_tokens)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self.max_len = 0  # no row is longer (but those whose list accept() refused)
        self._n_new = 0
        self._slots: Optional[torch.Tensor] = None

    @property
    def rows(self) -> int:
        return self.table.shape[0]

    # ---- a step -------------------------------------------------------------
    def begin(self, n: int) -> None:
        """Make room for n tokens a row and count them in.

        Rows of different lengths (prompts) take the longest's n, and accept()
        then keeps each row's own tokens, 0, 1, ... with -1 for the padding.
        Attention and accept() take up to 4,096 tokens a row."""
        self.fork(torch.arange(self.rows, device=self.table.device), reserve=n)
        self.lens = self.lens + n
        self.max_len += n
        self._n_new = n
        self._slots = self._slots_of_last(n)

    def _slots_of_last(self, n: int) -> torch.Tensor:
        """Where each row's last n tokens go, (rows * n,) int64."""
        p, width = self.page_tokens, self.table.shape[1]
        at = self.lens.long()[:, None] + torch.arange(-n, 0, device=self.table.device)
        page = self.table.gather(1, (at // p).clamp_(max=width - 1)).long()
        # not stored (flags() says so): tokens without a page, whose slot is negative, and those past the table
        return torch.where(at < width * p, page * p + at % p, -1).reshape(-1)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, dequantised: bool = False
               ) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """Store the step's keys and values (B, Hkv, n, D) of a layer; with
        ``dequantised`` returns the stored values in the same shape."""
        B, H, n, D = k.shape
        if self._slots is None or n != self._n_new or B != self.rows:
            raise ValueError(f"append takes the {self._n_new} tokens of each of {self.rows} rows that begin() made room for")
        kv = paged.append(self.codes[layer], self.scales[layer], k.transpose(1, 2).reshape(B * n, H, D),
                          v.transpose(1, 2).reshape(B * n, H, D), self._slots, dequantised, self.err)
        return None if kv is None else tuple(t.view(B, n, H, D).transpose(1, 2) for t in kv)

    def attend(self, layer: int, q: torch.Tensor, mask: Optional[torch.Tensor] = None,
               sm_scale: Optional[float] = None) -> torch.Tensor:
        """Attention of the step's positions: q (B, Hq, n, D) -> the same shape."""
        return paged.tree_attention(q, self.codes[layer], self.scales[layer], self.table, self.lens, mask, sm_scale,
                                    self.max_len, err=self.err)

    # ---- between steps --------------------------------------------------------
    def accept(self, accepted: torch.Tensor) -> None:
        """Keep the accepted drafts of the last step (paged.accept_tokens); the rest go.

        Accept before a fork: drafts that a fork shared between rows cannot move
        any more, and a row that would need it is left as it is (flags())."""
        if self._n_new == 0:
            raise ValueError("accept takes the drafts of one begin(), once")
        self.lens = paged.accept_tokens(self.codes, self.scales, self.table, self.lens, self._n_new, accepted, self.err,
                                        self.refs)
        self.max_len += accepted.shape[1] - self._n_new
        self._n_new = 0  # what is left are tokens
        self._slots = None

    def fork(self, parents: torch.Tensor, reserve: int = 0) -> None:
        """Row i becomes a continuation of row parents[i] (-1: empty); rows not named are freed."""
        self.table, self.lens, self.refs = paged.fork_pages(self.codes, self.scales, self.table, self.lens, self.refs,
                                                            parents, reserve, self.err)
        self._slots = None

    def free(self, rows: torch.Tensor) -> None:
        """Empty the rows (int64 indices) and give their pages back."""
        parents = torch.arange(self.rows, device=self.table.device)
        parents[rows] = -1
        self.fork(parents)

    def compact(self) -> torch.Tensor:
        """Move the pages in use to the front of the pool; their number, (1,) int32 on the device."""
        self.table, self.refs, n_live = paged.compact_pages(self.codes, self.scales, self.table, self.refs, self.err)
        if self._slots is not None:  # in a step: the rest of its tokens go where the pages are now
            self._slots = self._slots_of_last(self._n_new)
        return n_live

    def flags(self) -> int:
        """The LQ_EF_* bits raised so far (synchronises); see _lib.raise_flags."""
        return int(self.err.item()) & 0xFFFFFFFF
