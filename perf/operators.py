"""Measured cases of search decoding over the paged E8 cache.

Four operators: the append that quantises tokens into pages, attention of a
block of query positions (one token, or a tree of drafted ones) over the
pages, the page operations (fork, compact, accept), and beam search's
selection.  ``own`` False computes them with elementary torch operations in
32 bits; True calls the framework.

Pool layout: codes int32 (..., n_pages, 2, H, P, D/8), scales fp32
(..., n_pages, 2, H, P); index 0 of the pair is K, 1 is V.  A word holds one
E8 block as [coset | u0..u6 (4 bits each) | u7 >> 1], u = floor coordinate + 8,
u7's low bit being the parity of u0..u6.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BOUND = 7 - 1 / 64  # largest |x| / scale: the nearest E8 point then stays within [-8, 7.5]


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a 32-sequence Llama-3.1-8B-shaped batch: latency
        dict(name="append_step_b32", kind="append", dtype="bf16", n=32, heads=8, dim=128, page=64, pages=64),
        # a ragged prefill, Qwen2.5-7B-shaped heads, with padded slots
        dict(name="append_prefill_16411", kind="append", dtype="f16", n=16411, heads=4, dim=128, page=64, pages=320),
        # one user, one token, a short odd context: latency
        dict(name="attend_1x777", kind="attend", dtype="bf16", batch=1, heads=8, group=4, dim=128, t=1, ctx=777, page=64,
             ragged=False),
        # the framework's batch-32 decode step at 16,384 tokens
        dict(name="attend_32x16384", kind="attend", dtype="bf16", batch=32, heads=8, group=4, dim=128, t=1, ctx=16384,
             page=64, ragged=False),
        # a small tree for each sequence of a ragged batch
        dict(name="tree13_16x8190", kind="attend", dtype="bf16", batch=16, heads=8, group=4, dim=128, t=13, ctx=8190,
             page=64, ragged=True),
        # a wide tree over a long context, Qwen2.5-7B-shaped (7 query heads a KV head)
        dict(name="tree64_4x32768_g7", kind="attend", dtype="f16", batch=4, heads=4, group=7, dim=128, t=64, ctx=32768,
             page=64, ragged=False),
        # head_dim 64, small pages, a middling tree
        dict(name="tree31_8x4099_d64", kind="attend", dtype="bf16", batch=8, heads=4, group=8, dim=64, t=31, ctx=4099,
             page=16, ragged=True),
        # beams reordered after a step: shared prefixes, the open pages copied, all 32 layers
        dict(name="fork_32_beams", kind="fork", layers=32, heads=8, dim=128, page=64, rows=32, beams=4, ctx=4000),
        # a fragmented pool pulled together
        dict(name="compact_pool_512", kind="compact", layers=16, heads=8, dim=128, page=64, pages=512, live=0.5),
        # accepted drafts of 32 sequences moved to the front, all layers
        dict(name="accept_32x13", kind="accept", layers=32, heads=8, dim=128, page=64, rows=32, t=13, take=5, ctx=900),
        # one user's 4 beams over a 32,000-word vocabulary: latency
        dict(name="beam_1x4_32000", kind="beam", dtype="f32", batch=1, beams=4, vocab=32000, n=8, banned=False),
        # a serving batch of beams over Llama's vocabulary, some words banned
        dict(name="beam_32x8_128256", kind="beam", dtype="bf16", batch=32, beams=8, vocab=128256, n=16, banned=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "fork", "compact", "accept", "beam", "beam"])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    heads = rng.randint(1, 8)
    if kind == "append":
        n = _log(rng, 1, 16000)
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), n=n, heads=heads, dim=dim, page=page,
                    pages=n // page + rng.randint(2, 40))
    if kind == "attend":
        batch, t, group = _log(rng, 1, 32), rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64)]), rng.randint(1, 8)
        most = min(65536, 2_000_000 // (batch * heads), 400_000_000 // (batch * heads * group * t))
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), batch=batch, heads=heads, group=group, dim=dim, t=t,
                    ctx=max(t, _log(rng, 64, max(65, most))), page=page, ragged=rng.random() < 0.5)
    if kind == "fork":
        beams = rng.randint(2, 8)
        return dict(kind=kind, layers=rng.randint(1, 32), heads=heads, dim=dim, page=page, rows=beams * rng.randint(1, 4),
                    beams=beams, ctx=_log(rng, 1, 4000))
    if kind == "compact":
        return dict(kind=kind, layers=rng.randint(1, 16), heads=heads, dim=dim, page=page,
                    pages=_log(rng, 8, 40000 // page), live=rng.uniform(0.1, 0.9))
    if kind == "accept":
        t = rng.randint(2, 64)
        return dict(kind=kind, layers=rng.randint(1, 32), heads=heads, dim=dim, page=page, rows=_log(rng, 1, 32), t=t,
                    take=rng.randint(1, max(1, t // 2)), ctx=_log(rng, 1, 1000))
    beams = rng.randint(1, 16)
    return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), batch=_log(rng, 1, 16), beams=beams,
                vocab=_log(rng, 1000, 128256), n=rng.choice([beams, 2 * beams]), banned=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(g, n, heads, dim, dtype):
    """K or V vectors: Gaussian channels, a few of them large, token norms that vary."""
    x = torch.randn(n, heads, dim, device="cuda", generator=g)
    gain = torch.where(torch.rand(1, heads, dim, device="cuda", generator=g) < 0.03, 4.0, 1.0)
    return (x * gain * torch.exp(0.3 * torch.randn(n, heads, 1, device="cuda", generator=g))).to(dtype)


def _lens(g, case):
    b, ctx, t = case["batch"], case["ctx"], case["t"]
    if not case["ragged"]:
        return torch.full((b,), ctx, dtype=torch.int32, device="cuda")
    r = torch.rand(b, device="cuda", generator=g)
    lens = (t + r * (ctx - t)).to(torch.int32)
    lens[0] = ctx
    return lens


def _tree(g, b, t):
    """Ancestor masks of random trees: node j's parent is an earlier node, node 0 the root."""
    depth_pick = torch.rand(b, t, device="cuda", generator=g)
    parent = (depth_pick * torch.arange(t, device="cuda")).long().clamp(min=0)
    mask = torch.zeros(b, t, t, dtype=torch.bool, device="cuda")
    rows = torch.arange(b, device="cuda")
    for j in range(t):
        if j:
            mask[:, j] = mask[rows, parent[:, j]]
        mask[:, j, j] = True
    return mask


def _table(g, rows, width, n_pages):
    ids = torch.randperm(n_pages, device="cuda", generator=g)[: rows * width]
    return ids.view(rows, width).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "beam":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        x = 2.0 * torch.randn(b, k, v, device="cuda", generator=g)
        hot = torch.randint(0, v, (b, k, 12), device="cuda", generator=g)
        x.scatter_add_(2, hot, 6 + 3 * torch.rand(b, k, 12, device="cuda", generator=g))
        if case["banned"]:
            x.masked_fill_(torch.rand(b, 1, v, device="cuda", generator=g) < 0.1, float("-inf"))
        scores = -20 * torch.rand(b, k, device="cuda", generator=g)
        return dict(case=case, logits=x.to(DTYPES[case["dtype"]]), scores=scores)
    h, d, p = case["heads"], case["dim"], case["page"]
    if kind == "append":
        n, pages = case["n"], case["pages"]
        dt = DTYPES[case["dtype"]]
        slots = torch.randperm(pages * p, device="cuda", generator=g)[:n]
        if n > 64:
            slots[n - 3:] = -1  # padding of the batch
        return dict(case=case, k=_tokens(g, n, h, d, dt), v=_tokens(g, n, h, d, dt), slots=slots,
                    codes=torch.zeros(pages, 2, h, p, d // 8, dtype=torch.int32, device="cuda"),
                    scales=torch.ones(pages, 2, h, p, device="cuda"))
    if kind == "attend":
        b, t = case["batch"], case["t"]
        dt = DTYPES[case["dtype"]]
        width = -(-case["ctx"] // p)
        n_pages = b * width
        table = _table(g, b, width, n_pages)
        codes = torch.empty(n_pages, 2, h, p, d // 8, dtype=torch.int32, device="cuda")
        scales = torch.empty(n_pages, 2, h, p, device="cuda")
        step = max(1, (1 << 17) // (p * h))
        for at in range(0, n_pages, step):  # a bounded piece of the pool at a time
            m = min(step, n_pages - at)
            x = torch.stack([_tokens(g, m * p, h, d, dt), _tokens(g, m * p, h, d, dt)], 1)  # (m*p, 2, h, d)
            words, s, _ = _quantise(x)
            codes[at:at + m] = words.view(m, p, 2, h, d // 8).permute(0, 2, 3, 1, 4)
            scales[at:at + m] = s.view(m, p, 2, h).permute(0, 2, 3, 1)
        q = torch.randn(b, h * case["group"], t, d, device="cuda", generator=g).to(dt)
        return dict(case=case, q=q, codes=codes, scales=scales, table=table, lens=_lens(g, case),
                    mask=_tree(g, b, t) if t > 1 else None)
    layers = case["layers"]
    if kind == "fork":
        # prompts shared by their beams, a last page of each beam's own
        rows, beams, ctx = case["rows"], case["beams"], case["ctx"]
        width = ctx // p + 2
        groups = rows // beams
        full = ctx // p
        n_pages = groups * full + 4 * rows + 8
        perm = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
        table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        table[:, :full] = perm[: groups * full].view(groups, full).repeat_interleave(beams, 0)
        table[:, full] = perm[groups * full: groups * full + rows]
        lens = torch.full((rows,), ctx, dtype=torch.int32, device="cuda")
        refs = torch.bincount(table[table >= 0].long(), minlength=n_pages).to(torch.int32)
        parents = (torch.arange(rows, device="cuda") // beams) * beams + \
            torch.randint(0, beams, (rows,), device="cuda", generator=g)
        more = dict(table=table, lens=lens, refs=refs, parents=parents)
    elif kind == "compact":
        n_pages = case["pages"]
        n_live = max(1, int(n_pages * case["live"]))
        live = torch.randperm(n_pages, device="cuda", generator=g)[:n_live].to(torch.int32)
        rows = max(1, n_live // 32)
        width = n_live // rows
        table = live[: rows * width].view(rows, width).contiguous()
        refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        refs[table.view(-1).long()] = 1
        more = dict(table=table, refs=refs)
    else:
        rows, t, ctx, take = case["rows"], case["t"], case["ctx"], case["take"]
        width = -(-(ctx + t) // p)
        n_pages = rows * width
        table = _table(g, rows, width, n_pages)
        lens = torch.full((rows,), ctx + t, dtype=torch.int32, device="cuda")
        # accepted paths from the root: node 0, then nodes past the path's own slots
        accepted = torch.full((rows, take), -1, dtype=torch.int32, device="cuda")
        pick = torch.argsort(torch.rand(rows, t - take, device="cuda", generator=g), 1)[:, : take - 1].sort(1).values
        accepted[:, 0] = 0
        accepted[:, 1: 1 + pick.shape[1]] = (pick + take).to(torch.int32)
        more = dict(table=table, lens=lens, accepted=accepted)
    codes = torch.randint(-2**31, 2**31 - 1, (layers, n_pages, 2, h, p, d // 8), dtype=torch.int32, device="cuda",
                          generator=g)
    scales = torch.rand(layers, n_pages, 2, h, p, device="cuda", generator=g) + 0.1
    return dict(case=case, codes=codes, scales=scales, **more)


# ---------------------------------------------------------------- plain forms
def _d8(x):
    """Nearest point of D8 (the last axis holds 8): round, and where the sum is odd move the
    coordinate that rounding moved most the other way."""
    r = torch.round(x)
    res = x - r
    cost = (1.0 - 2.0 * res.abs()) + torch.arange(8, dtype=torch.float32, device=x.device) * 1e-7
    flip = torch.where(res >= 0, 1.0, -1.0)
    hit = torch.arange(8, device=x.device) == cost.argmin(-1, keepdim=True)
    odd = r.sum(-1, keepdim=True) % 2 != 0
    return torch.where(odd & hit, r + flip, r)


def _sum8(e):
    """Left-to-right sum of the 8 squares."""
    s = e * e
    return ((((((s[..., 0] + s[..., 1]) + s[..., 2]) + s[..., 3]) + s[..., 4]) + s[..., 5]) + s[..., 6]) + s[..., 7]


def _quantise(x):
    """(..., D) -> code words (..., D/8) int32, scales (...), values (..., D) in x's dtype."""
    xf = x.float()
    amax = xf.abs().amax(-1)
    s = torch.where(amax < 1e-6, 1.0, amax * (1 / BOUND))
    y = (xf / s[..., None]).unflatten(-1, (-1, 8))
    whole = _d8(y)
    half = _d8(y - 0.5) + 0.5
    coset = _sum8(y - whole) > _sum8(y - half)
    point = torch.where(coset[..., None], half, whole)
    u = torch.floor(point).to(torch.int64) + 8
    u[..., 7] >>= 1
    shift = torch.tensor([27, 23, 19, 15, 11, 7, 3, 0], device=x.device)
    word = (u << shift).sum(-1) + (coset.to(torch.int64) << 31)
    word = torch.where(word >= 2**31, word - 2**32, word).to(torch.int32)
    return word, s, (point.flatten(-2) * s[..., None]).to(x.dtype)


def _values(words, scales):
    """Code words (..., D/8) and scales (...) -> fp32 values (..., D)."""
    shift = torch.tensor([27, 23, 19, 15, 11, 7, 3, 0], dtype=torch.int32, device=words.device)
    low = torch.tensor([15] * 7 + [7], dtype=torch.int32, device=words.device)
    u = (words[..., None] >> shift) & low
    odd = u[..., :7].sum(-1, dtype=torch.int32) & 1
    u[..., 7] = 2 * u[..., 7] + odd
    point = (u - 8).float() + 0.5 * (words < 0)[..., None].float()
    return point.flatten(-2) * scales[..., None]


def _plain_append(s):
    words, scale, values = _quantise(torch.stack([s["k"], s["v"]], 1))  # (n, 2, h, ..)
    fine = s["slots"] >= 0
    page, off = s["slots"][fine] // s["case"]["page"], s["slots"][fine] % s["case"]["page"]
    s["codes"][page, :, :, off] = words[fine]
    s["scales"][page, :, :, off] = scale[fine]
    return dict(k=values[:, 0].contiguous(), v=values[:, 1].contiguous(), scales=s["scales"])


def _plain_attend(s):
    c, q = s["case"], s["q"]
    b, h, t, d = c["batch"], c["heads"], c["t"], c["dim"]
    page = s["table"].long()
    kv = _values(s["codes"][page], s["scales"][page])  # (b, width, 2, h, p, d)
    n = kv.shape[1] * kv.shape[4]
    k = kv[:, :, 0].transpose(1, 2).reshape(b, h, n, d)
    v = kv[:, :, 1].transpose(1, 2).reshape(b, h, n, d)
    del kv
    at = torch.arange(n, device=q.device)[None, None] - (s["lens"][:, None, None] - t)  # draft index of a slot
    see = (at < 0).expand(b, t, n)
    if s["mask"] is None:
        see = see | (at == 0)
    else:
        see = see | ((at >= 0) & (at < t) & s["mask"].gather(2, at.clamp(0, t - 1).expand(b, t, n)))
    x = q.float().view(b, h, c["group"] * t, d) @ k.transpose(2, 3) * (1 / math.sqrt(d))
    x = x.view(b, h, c["group"], t, n).masked_fill(~see[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    l = e.sum(-1, keepdim=True)
    o = (e.view(b, h, c["group"] * t, n) @ v).view(b, h, c["group"], t, d)
    o = torch.where(l > 0, o / l, 0.0)
    return dict(o=o.reshape(b, h * c["group"], t, d).to(q.dtype), lse=(m + torch.log(l)).reshape(b, h * c["group"], t))


def _count(entries, n):
    return torch.bincount(entries[entries >= 0].long(), minlength=n).to(torch.int32)


def _plain_fork(s):
    p, table, parents, refs = s["case"]["page"], s["table"], s["parents"], s["refs"]
    width = table.shape[1]
    has = parents >= 0
    old = table[parents.clamp(min=0)]
    lens = torch.where(has, s["lens"][parents.clamp(min=0)], 0)
    first = ~(parents[:, None] == parents[None, :]).tril(-1).any(1)
    col = torch.arange(width, device=table.device)[None]
    full = (lens // p)[:, None]
    used = has[:, None] & (col < ((lens + 1 + p - 1) // p)[:, None])  # room for one more token
    keep = used & ((col < full) | (first[:, None] & (old >= 0)))
    fresh = used & ~keep
    free = (refs == 0).nonzero()[:, 0].to(torch.int32)
    rank = (fresh.flatten().cumsum(0) - 1).view_as(old).clamp(0, free.numel() - 1)
    new = torch.where(keep, old, torch.where(fresh, free[rank], -1))
    part = has & ~first & (lens % p > 0)
    src, dst = old.gather(1, full.clamp(max=width - 1))[part, 0].long(), new.gather(1, full.clamp(max=width - 1))[part, 0].long()
    live = torch.arange(p, device=table.device)[None] < (lens % p)[part][:, None]  # (copies, p)
    codes, scales = s["codes"], s["scales"]
    codes[:, dst] = torch.where(live[None, :, None, None, :, None], codes[:, src], codes[:, dst])
    scales[:, dst] = torch.where(live[None, :, None, None, :], scales[:, src], scales[:, dst])
    n = refs.numel()
    return dict(table=new, lens=lens, refs=refs - _count(table, n) + _count(new, n), codes=codes, scales=scales)


def _plain_compact(s):
    live = s["refs"] > 0
    n = live.sum()
    ids = torch.arange(live.numel(), device=live.device)
    src, dst = (live & (ids >= n)).nonzero()[:, 0], (~live & (ids < n)).nonzero()[:, 0]
    to = ids.clone()
    to[src] = dst
    s["codes"][:, dst] = s["codes"][:, src]
    s["scales"][:, dst] = s["scales"][:, src]
    refs = s["refs"].clone()
    refs[dst] = s["refs"][src]
    refs[src] = 0
    table = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].to(torch.int32), -1)
    return dict(table=table, refs=refs, n_live=n.to(torch.int32).view(1), codes=s["codes"], scales=s["scales"])


def _plain_accept(s):
    p, table, acc = s["case"]["page"], s["table"], s["accepted"].long()
    base = (s["lens"] - s["case"]["t"]).long()
    take = acc >= 0
    row, j = take.nonzero(as_tuple=True)
    at, to = base[row] + acc[row, j], base[row] + j
    sp, dp = table[row, at // p].long(), table[row, to // p].long()
    s["codes"][:, dp, :, :, to % p] = s["codes"][:, sp, :, :, at % p]
    s["scales"][:, dp, :, :, to % p] = s["scales"][:, sp, :, :, at % p]
    return dict(lens=(base + take.sum(1)).to(torch.int32), codes=s["codes"], scales=s["scales"])


def _plain_beam(s):
    x = s["logits"].float()
    b, k, v = x.shape
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    # best first within a beam (equal logits by word), then over the beams (equal totals by beam)
    best, word = torch.sort(x, dim=-1, descending=True, stable=True)
    n = s["case"]["n"]
    total = (best[..., :n] - lse) + s["scores"][..., None]
    top, at = torch.sort(total.flatten(1), dim=-1, descending=True, stable=True)
    m = word[..., :n].shape[-1]
    return dict(scores=top[:, :n].contiguous(), beams=at[:, :n] // m, words=word[..., :n].flatten(1).gather(1, at[:, :n]))


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact,
                "accept": _plain_accept, "beam": _plain_beam}[kind](s)
    from latticequant_b200 import beam, paged

    if kind == "append":
        k, v = paged.append(s["codes"], s["scales"], s["k"], s["v"], s["slots"], dequantised=True)
        return dict(k=k, v=v, scales=s["scales"])
    if kind == "attend":
        o, lse = paged.tree_attention(s["q"], s["codes"], s["scales"], s["table"], s["lens"], mask=s["mask"],
                                      return_lse=True)
        return dict(o=o, lse=lse)
    if kind == "fork":
        table, lens, refs = paged.fork_pages(s["codes"], s["scales"], s["table"], s["lens"], s["refs"], s["parents"],
                                             reserve=1)
        return dict(table=table, lens=lens, refs=refs, codes=s["codes"], scales=s["scales"])
    if kind == "compact":
        table, refs, n_live = paged.compact_pages(s["codes"], s["scales"], s["table"], s["refs"])
        return dict(table=table, refs=refs, n_live=n_live, codes=s["codes"], scales=s["scales"])
    if kind == "accept":
        lens = paged.accept_tokens(s["codes"], s["scales"], s["table"], s["lens"], s["case"]["t"], s["accepted"])
        return dict(lens=lens, codes=s["codes"], scales=s["scales"])
    scores, beams, words = beam.beam_select(s["logits"], s["scores"], s["case"]["n"])
    return dict(scores=scores, beams=beams, words=words)


# ---------------------------------------------------------------- floors
def work(case):
    kind = case["kind"]
    if kind == "beam":
        n = case["batch"] * case["beams"] * case["vocab"]
        return dict(bytes=n * DTYPES[case["dtype"]].itemsize + case["batch"] * case["n"] * 20, flops=3 * n)
    h, d, p = case["heads"], case["dim"], case["page"]
    row = d // 2 + 4  # a token's K or V of one head: codes and scale
    if kind == "append":
        n = 2 * case["n"] * h
        return dict(bytes=n * (2 * d * DTYPES[case["dtype"]].itemsize + row) + 8 * case["n"], flops=30 * n * d)
    if kind == "attend":
        b, t, rows = case["batch"], case["t"], case["group"] * case["t"]
        tokens = case["ctx"] * b if not case["ragged"] else case["ctx"] + (b - 1) * (case["ctx"] + t) // 2
        return dict(bytes=tokens * h * 2 * row + b * h * rows * (4 * d + 4) + (b * t * t if t > 1 else 0),
                    flops=4 * tokens * h * rows * d)
    line = case["layers"] * 2 * h * row  # a token's rows in every layer
    if kind == "fork":
        rows, width = case["rows"], case["ctx"] // p + 2
        copies = rows - rows * (1 - (1 - 1 / case["beams"]) ** case["beams"])  # children that are not their parent's first
        return dict(bytes=2 * copies * (case["ctx"] % p) * line + 8 * rows * width, flops=0)
    if kind == "compact":
        return dict(bytes=2 * case["pages"] * case["live"] * (1 - case["live"]) * p * line + 8 * case["pages"], flops=0)
    return dict(bytes=2 * case["rows"] * max(0, case["take"] - 1) * line + 8 * case["rows"], flops=0)


# ---------------------------------------------------------------- 64 bits
def _exact_quantise(x):
    """Values of the nearest E8 points in 64 bits: of the 16 roundings that matter (each coset, with one
    coordinate moved or none), the nearest with an even sum."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    s = torch.where(amax < 1e-6, 1.0, amax / BOUND)
    y = (x / s).unflatten(-1, (-1, 8))
    best, near = None, None
    for off in (0.0, 0.5):
        base = torch.round(y - off)
        side = torch.where(y - off >= base, 1.0, -1.0)
        even = base.sum(-1) % 2 == 0
        d0 = ((y - off - base) ** 2).sum(-1)
        for i in range(-1, 8):
            move = torch.zeros(8, dtype=torch.float64, device=x.device)
            gain = torch.zeros_like(d0)
            if i >= 0:
                move[i] = 1.0
                gain = 1 - 2 * (y - off - base)[..., i].abs()
            dist = torch.where(even if i < 0 else ~even, d0 + gain, float("inf"))
            point = base + side * move + off
            best, near = (point, dist) if best is None else (torch.where((dist < near)[..., None], point, best),
                                                             torch.minimum(dist, near))
    return s[..., 0], best.flatten(-2) * s


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact", "accept"):
        return None  # whole numbers and moved values
    s = prepare(case, seed)
    if kind == "append":
        scale, kv = _exact_quantise(torch.stack([s["k"], s["v"]]))  # (2, n, h, ..)
        scales = s["scales"].double()
        fine = s["slots"] >= 0
        page, off = s["slots"][fine] // case["page"], s["slots"][fine] % case["page"]
        for i in range(2):
            scales[page, i, :, off] = scale[i][fine]
        return dict(k=kv[0], v=kv[1], scales=scales)
    if kind == "beam":
        x = s["logits"].double()
        lse = torch.logsumexp(x, -1, keepdim=True)
        total = (x - lse + s["scores"].double()[..., None]).flatten(1)
        top, at = torch.sort(total, dim=1, descending=True, stable=True)
        top, at = top[:, : case["n"]], at[:, : case["n"]]
        return dict(scores=top, beams=at // case["vocab"], words=at % case["vocab"])
    # attention, one sequence and KV head at a time over its own tokens
    b, h, g, t, d, p = (case[k] for k in ("batch", "heads", "group", "t", "dim", "page"))
    o = torch.zeros(b, h * g, t, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h * g, t), float("-inf"), dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(s["lens"][i])
        if not n:
            continue
        page = s["table"][i, : -(-n // p)].long()
        see = torch.ones(t, n, dtype=torch.bool, device="cuda")
        if s["mask"] is not None:
            see[:, max(0, n - t):] = s["mask"][i][:, max(0, t - n):]
        for j in range(h):
            kv = []
            for side in range(2):
                w = s["codes"][page, side, j].reshape(-1, d // 8)[:n].long() & 0xFFFFFFFF
                half = (w // 2**31).double() / 2
                digits = [((w // 2**(27 - 4 * e)) % 16).double() for e in range(7)]
                digits.append(2 * (w % 8).double() + sum(digits) % 2)
                v = torch.stack([x - 8 + half for x in digits], -1).reshape(n, d)
                kv.append(v * s["scales"][page, side, j].reshape(-1)[:n, None].double())
            x = torch.einsum("gtd,nd->gtn", s["q"][i, j * g:(j + 1) * g].double(), kv[0]) / math.sqrt(d)
            x = x.masked_fill(~see[None], float("-inf"))
            lse[i, j * g:(j + 1) * g] = torch.logsumexp(x, -1)
            o[i, j * g:(j + 1) * g] = torch.einsum("gtn,nd->gtd", torch.softmax(x, -1), kv[1])
    return dict(o=o, lse=lse)
