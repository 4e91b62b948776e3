"""PagedKVCache and the search-decoding example run together as they would be used.

The caches hold the same tokens whichever way they came in, so a path's
attention over a tree, over beams and token by token is the same up to the
attention's own tolerance (tests/test_gpu_paged.py); beam search is checked
against a search that recomputes every prefix from the start.
"""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("search_decode", os.path.join(ROOT, "examples", "search_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _cache(rows=2, **kw):
    from latticequant_b200.llm.paged_cache import PagedKVCache

    return PagedKVCache(2, 2, 64, n_pages=40, rows=rows, max_tokens=160, page_tokens=16, **kw)


def _close(a, b):
    # two attentions of the same keys: each within 1e-3 of the row's largest value, bf16 roundings of 2^-8
    top = b.float().abs().amax(-1, keepdim=True)
    return bool(((a.float() - b.float()).abs() <= 2e-3 * top + 2 ** -7 * b.float().abs()).all())


def test_tree_paths_equal_token_by_token():
    g = torch.Generator(device="cuda").manual_seed(0)
    B, n = 2, 5
    ctx = [torch.randn(B, 2, 45, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    new = [torch.randn(B, 2, n, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    q = torch.randn(B, 6, n, 64, device="cuda", generator=g).to(torch.bfloat16)
    tree = _cache()
    tree.begin(45)
    kd, vd = tree.append(0, *ctx, dequantised=True)
    assert kd.shape == ctx[0].shape and float((kd - ctx[0]).float().abs().max()) < 1.0
    tree.begin(n)
    tree.append(0, *new)
    parent = [-1, 0, 1, 0, 3]
    mask = torch.zeros(n, n, dtype=torch.bool, device="cuda")
    for j, p in enumerate(parent):
        if p >= 0:
            mask[j] = mask[p]
        mask[j, j] = True
    o = tree.attend(0, q, mask)
    path = [0, 3, 4]
    line = _cache()
    line.begin(45)
    line.append(0, *ctx)
    for j in path:
        line.begin(1)
        line.append(0, new[0][:, :, j:j + 1], new[1][:, :, j:j + 1])
        assert _close(line.attend(0, q[:, :, j:j + 1]), o[:, :, j:j + 1])
    # accepting the path leaves the same cache as decoding it
    tree.accept(torch.tensor([path] * B, dtype=torch.int32, device="cuda"))
    assert tree.lens.tolist() == line.lens.tolist() == [48, 48] and tree.max_len == 48
    tree.begin(1)
    line.begin(1)
    for c in (tree, line):
        c.append(0, new[0][:, :, :1], new[1][:, :, :1])
    assert torch.equal(tree.attend(0, q[:, :, :1]), line.attend(0, q[:, :, :1]))
    assert tree.flags() == 0 and line.flags() == 0


def test_fork_free_and_compact_keep_rows():
    g = torch.Generator(device="cuda").manual_seed(1)
    c = _cache(rows=3)
    kv = [torch.randn(3, 2, 37, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    q = torch.randn(3, 4, 1, 64, device="cuda", generator=g).to(torch.bfloat16)
    c.begin(37)
    c.append(0, *kv)
    before = c.attend(0, q[:, :, :1])
    c.fork(torch.tensor([2, 0, 2, 2], device="cuda"))
    after = c.attend(0, q[[2, 0, 2, 2]])
    assert torch.equal(after, before[[2, 0, 2, 2]])
    assert int((c.refs > 0).sum()) == 3 + 2 + 3 - 0 and c.refs.max() == 3  # two shared pages, one open page each
    c.free(torch.tensor([1, 2], device="cuda"))
    assert c.lens.tolist() == [37, 0, 0, 37] and int((c.refs > 0).sum()) == 4
    n = c.compact()
    assert n.tolist() == [4] and int(c.table.max()) == 3
    again = c.attend(0, q[[2, 2, 2, 2]])
    assert torch.equal(again[[0, 3]], before[[2, 2]]) and not again[1:3].any()
    assert c.flags() == 0


def test_full_pool_is_reported():
    from latticequant_b200 import _lib

    c = _cache(rows=4)
    c.begin(160)
    c.fork(torch.zeros(4, dtype=torch.int64, device="cuda"))
    assert c.flags() == 0
    d = _cache(rows=5)
    d.begin(160)
    assert d.flags() == _lib.EF_CAPACITY
    with pytest.raises(_lib.LatticeQuantError):
        _lib.raise_flags(d.flags(), "begin")
    with pytest.raises(ValueError):
        d.append(0, *[torch.zeros(5, 2, 3, 64, device="cuda")] * 2)


def test_example_tree_equals_greedy(ex):
    dev = torch.device("cuda")
    model = ex.TinyLM(dev)
    prompt = torch.randint(0, ex.VOCAB, (1, 37), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    want, _ = ex.greedy(model, prompt, 20)
    guesses = torch.where(torch.arange(20, device=dev) % 4 < 2, want, 0)
    got, steps = ex.tree_decode(model, prompt, 16, guesses)
    assert torch.equal(got, want[:, :16]) and steps < 16


def test_example_beams_equal_recomputed_prefixes(ex):
    dev = torch.device("cuda")
    model = ex.TinyLM(dev)
    prompt = torch.randint(0, ex.VOCAB, (1, 21), device=dev, generator=torch.Generator(device=dev).manual_seed(2))
    best, scores = ex.beam_search(model, prompt, 6, 3)
    # every prefix again from the start in its own cache, the same selection in float64
    seqs, tot = [[]], torch.zeros(1, dtype=torch.float64, device=dev)
    for _ in range(6):
        cand = []
        for i, s in enumerate(seqs):
            ids = torch.cat([prompt, torch.tensor([s], device=dev, dtype=torch.int64)], 1)
            lp = torch.log_softmax(ex.prefill(model, ids, ex.new_cache(1, dev, 64))[0].double(), -1)
            top = lp.topk(3)
            cand += [(float(tot[i] + v), s + [int(w)]) for v, w in zip(*top)]
        cand.sort(key=lambda c: -c[0])
        seqs = [c[1] for c in cand[:3]]
        tot = torch.tensor([c[0] for c in cand[:3]], dtype=torch.float64, device=dev)
    assert best[0].tolist() == seqs
    # logits of bf16 layers differ between a prompt's chunk and single tokens by bf16 roundings
    assert math.isclose(float(scores[0, 0]), float(tot[0]), abs_tol=0.5)
