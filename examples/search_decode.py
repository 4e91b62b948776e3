"""Search decoding over the paged E8 cache: greedy, a tree of drafts, beams.

    python examples/search_decode.py [--tokens 24] [--device cuda:0]

A small randomly initialised decoder (no weights are needed) runs the three
loops that a server runs over ``llm.paged_cache.PagedKVCache``:

* greedy decoding, one token a step;
* greedy decoding from trees of drafts: each step checks a tree and keeps the
  longest path the model confirms (half of the drafts here are right, so the
  loop takes fewer steps).  A tree's sums run in another order than a single
  token's, so where two logits of this bfloat16 model are closer than its
  rounding, either may win and the two loops part;
* beam search: beam_select picks the continuations, fork reorders the cache.

Prints the steps each took and whether the tree's tokens are the greedy ones.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from latticequant_b200 import _lib  # noqa: E402
from latticequant_b200.beam import beam_select  # noqa: E402
from latticequant_b200.llm.paged_cache import PagedKVCache  # noqa: E402

LAYERS, HEADS, KV_HEADS, DIM, VOCAB = 3, 8, 2, 64, 512
WIDTH = HEADS * DIM


class TinyLM:
    """A pre-norm decoder with rotary positions; attention comes from the cache."""

    def __init__(self, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) / shape[0] ** 0.5).to(torch.bfloat16)

        self.embed = torch.randn(VOCAB, WIDTH, generator=g, device=device).to(torch.bfloat16)
        self.layers = [dict(q=w(WIDTH, HEADS * DIM), k=w(WIDTH, KV_HEADS * DIM), v=w(WIDTH, KV_HEADS * DIM),
                            o=w(HEADS * DIM, WIDTH), up=w(WIDTH, 2 * WIDTH), down=w(2 * WIDTH, WIDTH))
                       for _ in range(LAYERS)]
        self.head = w(WIDTH, VOCAB) * 4
        self.freq = 10000.0 ** (-torch.arange(0, DIM, 2, device=device) / DIM)

    def _rotate(self, x, pos):
        a = pos[:, None, :, None] * self.freq
        c, s = a.cos(), a.sin()
        x0, x1 = x.float().chunk(2, -1)
        return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], -1).to(x.dtype)

    def __call__(self, ids, pos, cache, mask=None):
        """Logits (B, n, VOCAB) of n tokens a row at positions pos (B, n); their K/V go into the cache."""
        B, n = ids.shape
        norm = torch.nn.functional.rms_norm
        x = self.embed[ids]
        cache.begin(n)
        for i, p in enumerate(self.layers):
            h = norm(x, (WIDTH,))
            q, k, v = ((h @ p[m]).view(B, n, -1, DIM).transpose(1, 2) for m in "qkv")
            cache.append(i, self._rotate(k, pos), v)
            o = cache.attend(i, self._rotate(q, pos), mask)
            x = x + o.transpose(1, 2).reshape(B, n, -1) @ p["o"]
            x = x + torch.nn.functional.silu(norm(x, (WIDTH,)) @ p["up"]) @ p["down"]
        return norm(x, (WIDTH,)).float() @ self.head.float()


def new_cache(rows, device, tokens):
    return PagedKVCache(LAYERS, KV_HEADS, DIM, n_pages=rows * (-(-tokens // 16) + 2), rows=rows, max_tokens=tokens,
                        page_tokens=16, device=device)


def prefill(model, prompt, cache):
    pos = torch.arange(prompt.shape[1], device=prompt.device).expand_as(prompt)
    return model(prompt, pos, cache)[:, -1]


def greedy(model, prompt, tokens):
    cache = new_cache(prompt.shape[0], prompt.device, prompt.shape[1] + tokens + 1)
    out = [prefill(model, prompt, cache).argmax(-1)]
    for i in range(tokens - 1):
        pos = torch.full_like(out[-1], prompt.shape[1] + i)[:, None]
        out.append(model(out[-1][:, None], pos, cache)[:, -1].argmax(-1))
    _lib.raise_flags(cache.flags(), "greedy")
    return torch.stack(out, 1), tokens


def tree_decode(model, prompt, tokens, guesses):
    """Greedy decoding of one row through trees: node 0 is the last token, then two chains of two
    drafts each, one of them guesses (B, tokens + 4) -- what a draft model would propose."""
    dev, depth = prompt.device, 2
    cache = new_cache(1, dev, prompt.shape[1] + tokens + 16)
    out = [int(prefill(model, prompt, cache).argmax(-1))]
    parent = [-1, 0, 1, 0, 3]
    mask = torch.zeros(5, 5, dtype=torch.bool, device=dev)
    for j, p in enumerate(parent):
        if p >= 0:
            mask[j] = mask[p]
        mask[j, j] = True
    steps = 1
    while len(out) < tokens:
        at = len(out)
        chain = [int(t) for t in guesses[0, at: at + depth]]
        ids = torch.tensor([[out[-1], *[(t + 1) % VOCAB for t in chain], *chain]], device=dev)
        base = prompt.shape[1] + at - 1
        pos = torch.tensor([[base, base + 1, base + 2, base + 1, base + 2]], device=dev)
        best = model(ids, pos, cache, mask)[0].argmax(-1).tolist()
        steps += 1
        path, grown = [0], True
        while grown:  # follow the child that the model itself would have produced
            grown = False
            for j in range(1, 5):
                if parent[j] == path[-1] and int(ids[0, j]) == best[path[-1]]:
                    path.append(j)
                    grown = True
                    break
        out += [best[j] for j in path]
        cache.accept(torch.tensor([path + [-1] * (depth + 1 - len(path))], dtype=torch.int32, device=dev))
    _lib.raise_flags(cache.flags(), "tree_decode")
    return torch.tensor([out[:tokens]], device=dev), steps


def beam_search(model, prompt, tokens, beams):
    """The best sequences (1, beams, tokens) and their scores for one prompt."""
    dev = prompt.device
    cache = new_cache(1, dev, prompt.shape[1] + tokens + 1)
    cache_rows = torch.zeros(beams, dtype=torch.int64, device=dev)
    logits = prefill(model, prompt, cache)
    # one prompt, one prefill: its pages are shared by the beams
    wide = new_cache(beams, dev, prompt.shape[1] + tokens + 1)
    wide.codes[:, : cache.codes.shape[1]] = cache.codes
    wide.scales[:, : cache.scales.shape[1]] = cache.scales
    wide.refs[: cache.refs.shape[0]] = cache.refs
    wide.table, wide.lens, wide.max_len = cache.table, cache.lens, cache.max_len
    wide.fork(cache_rows)
    scores, _, words = beam_select(logits[None], torch.zeros(1, 1, device=dev), beams)
    out = words.view(beams, 1)
    for i in range(tokens - 1):
        pos = torch.full((beams, 1), prompt.shape[1] + i, device=dev)
        logits = model(out[:, -1:], pos, wide)[:, -1]
        scores, parents, words = beam_select(logits.view(1, beams, VOCAB), scores, beams)
        wide.fork(parents[0])
        out = torch.cat([out[parents[0]], words.view(beams, 1)], 1)
    _lib.raise_flags(wide.flags(), "beam_search")
    return out[None], scores


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--device", default="cuda:0")
    a = ap.parse_args()
    dev = torch.device(a.device)
    model = TinyLM(dev)
    prompt = torch.randint(0, VOCAB, (1, 37), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    want, n = greedy(model, prompt, a.tokens + 4)
    guesses = torch.where(torch.arange(a.tokens + 4, device=dev) % 4 < 2, want, 0)
    got, steps = tree_decode(model, prompt, a.tokens, guesses)
    print(f"greedy: {a.tokens} steps; tree: {steps} steps, same tokens: {bool((got == want[:, :a.tokens]).all())}")
    best, scores = beam_search(model, prompt, a.tokens, 4)
    print("beams:", [f"{s:.3f}" for s in scores[0].tolist()], "best:", best[0, 0].tolist()[:8], "...")


if __name__ == "__main__":
    main()
