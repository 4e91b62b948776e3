"""Beam search's selection over beams and vocabulary (CUDA, sm_100a).

The reference decodes greedily (llm/e2e_eval.py:212).  ``beam_select`` reads a
step's logits once and returns the best continuations; its beams are the
``parents`` of ``paged.fork_pages``, which reorders the cache.
"""
from __future__ import annotations

import functools
from typing import Tuple

import torch

from . import _lib
from ._lib import call, lib


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The n best of scores[b, k] + log_softmax(logits[b, k])[v] for each b (lq_beam_select).

    logits (B, K, V) float32 / float16 / bfloat16 with a contiguous last
    dimension; scores fp32 (B, K).  Returns (scores fp32, beams int64, words
    int64), each (B, n), best first; equal totals go to the lower beam, then the
    larger logit, then the lower word.  Banned words (logits of -inf, NaN) and
    dead beams (scores of -inf) are never chosen; places left without a
    candidate hold -inf, -1, -1.  n up to 128, K up to 256."""
    if not logits.is_cuda:
        _lib.require_cuda(logits)
    index = logits.get_device()
    if logits.dim() != 3 or scores.shape != logits.shape[:2] or scores.dtype is not torch.float32 or \
            scores.get_device() != index:
        raise ValueError("beam_select takes logits (B, K, V) and fp32 scores (B, K) on one device")
    B, K, V = logits.shape
    if V == 0 or K == 0 or not 1 <= n <= 128 or K > 256 or V > 1 << 24:
        raise ValueError("beam_select takes 1..256 beams, 1..2^24 words and n in 1..128")
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    top = scores.new_empty((B, n))
    beams = scores.new_empty((B, n), dtype=torch.int64)
    words = torch.empty_like(beams)
    dtype = _lib.dtype_code(logits.dtype)
    need = _workspace(dtype, B, K, V, n)
    ws = beams.new_empty(need // 8 + 1)
    call("lq_beam_select", index, logits.data_ptr(), dtype, B, K, V, *logits.stride()[:2], scores.data_ptr(), n,
         top.data_ptr(), beams.data_ptr(), words.data_ptr(), ws.data_ptr(), need)
    return top, beams, words


@functools.lru_cache(maxsize=4096)
def _workspace(*shape: int) -> int:
    return lib().lq_beam_select_workspace(*shape)
