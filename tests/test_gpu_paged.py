"""The paged E8 cache (paged.py) against plain implementations in 64 bits.

* append: the code words are the framework's own lattice search and 4-bit code
  (encode_e8, pack_e8) of x / s bit for bit, s = amax / (7 - 1/64), and no other
  even-sum point in reach is nearer in 64 bits;
* tree_attention: float64 attention over the values the pages stand for.  The
  kernel's scores are fp32 sums of exact products; a weight is rounded to fp16
  (2^-11) and the output to q's type.  A weight's error enters a channel as
  sum(w e v) / sum(w), at the size of the output itself times 2^-11, so
  |o - ref| <= 1e-3 max|ref| of the row plus one rounding of the output (the unit
  roundoff 2^-p of p significant bits: 2^-8 bf16, 2^-11 fp16, of its value); lse
  within 1e-4 max(1, |lse|), the bar the other attention tests use;
* page operations: whole numbers and moved words, equal to loops on the host.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BOUND = np.float32(7 - 1 / 64)


@pytest.fixture(scope="module")
def P():
    from latticequant_b200 import paged

    return paged


def _values(codes, scales):
    """float64 values of code words (..., W) with scales (...)."""
    w = codes.cpu().numpy().astype(np.int64) & 0xFFFFFFFF
    u = np.stack([(w >> (27 - 4 * i)) & 15 for i in range(7)], -1)
    last = 2 * (w & 7) + u.sum(-1) % 2
    pts = np.concatenate([u, last[..., None]], -1) - 8 + 0.5 * (w >> 31)[..., None]
    return pts.reshape(*w.shape[:-1], -1) * scales.cpu().numpy().astype(np.float64)[..., None]


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,H,D,page", [(1, 1, 64, 16), (3, 5, 128, 32), (257, 8, 128, 64), (40, 3, 64, 256)])
def test_append_codes_are_the_frameworks(P, dtype, n, H, D, page):
    from latticequant_b200.core import compact_storage, e8_quantizer

    g = torch.Generator(device="cuda").manual_seed(n + D)
    pages = n // page + 3
    codes, scales, _ = P.empty_pool(1, pages, H, D, page)
    codes, scales = codes[0], scales[0]
    x = [(torch.randn(n, H, D, device="cuda", generator=g) * torch.exp(torch.randn(n, H, 1, device="cuda", generator=g))
          ).to(dtype) for _ in range(2)]
    x[0][0, 0] = 0  # a zero vector
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n]
    if n > 2:
        slots[1] = -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv = P.append(codes, scales, x[0], x[1], slots, dequantised=True, err=err)
    assert int(err.item()) == 0
    for side in range(2):
        xf = x[side].float()
        amax = xf.abs().amax(-1)
        s = torch.where(amax < 1e-6, torch.ones_like(amax), amax * float(np.float32(1) / BOUND))
        q = e8_quantizer.encode_e8((xf / s[..., None]).reshape(-1, 8))
        assert float(q.min()) >= -8 and float(q.max()) <= 7.5
        by = compact_storage.pack_e8(q, 4).cpu().numpy().astype(np.int64)
        want = ((by[:, 0] << 24) | (by[:, 1] << 16) | (by[:, 2] << 8) | by[:, 3]).reshape(n, H, D // 8)
        for i in range(n):
            if int(slots[i]) < 0:
                continue
            pg, off = int(slots[i]) // page, int(slots[i]) % page
            assert np.array_equal(codes[pg, side, :, off].cpu().numpy().astype(np.int64) & 0xFFFFFFFF, want[i])
            assert torch.equal(scales[pg, side, :, off], s[i])
        assert torch.equal(kv[side], (q.view(n, H, D) * s[..., None]).to(dtype))
    stored = slots[slots >= 0]
    other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    other[stored] = False
    assert not codes.transpose(2, 3).reshape(pages, 2, page, -1).transpose(1, 2).reshape(pages * page, -1)[other].any()


def test_append_points_are_nearest_in_64_bits(P):
    g = torch.Generator(device="cuda").manual_seed(5)
    n, H, D = 64, 2, 64
    codes, scales, _ = P.empty_pool(1, 4, H, D, 16)
    x = torch.randn(n, H, D, device="cuda", generator=g)
    P.append(codes[0], scales[0], x, x, torch.arange(n, device="cuda"))
    v = _values(codes[0, :, 0], scales[0, :, 0])  # (pages, H, P, D)
    v = v.transpose(0, 2, 1, 3).reshape(n, H, D)
    s = scales[0, :, 0].permute(0, 2, 1).reshape(n, H, 1).cpu().numpy().astype(np.float64)
    y, q = x.cpu().numpy().astype(np.float64) / s, v / s
    d = ((y - q).reshape(-1, 8) ** 2).sum(1)
    best = np.full(len(d), np.inf)
    yb = y.reshape(-1, 8)
    for off in (0.0, 0.5):
        base = np.floor(yb - off)
        for bits in range(256):  # every corner of the unit cell with an even sum
            c = base + np.array([(bits >> i) & 1 for i in range(8)])
            dist = ((yb - off - c) ** 2).sum(1)
            best = np.minimum(best, np.where(c.sum(1) % 2 == 0, dist, np.inf))
    # fp32 quotients (|y| < 7, error 2^-22) move a squared distance by less than 8 * 2 * 2^-22
    assert (d <= best + 16 * 2.0 ** -22).all()


def test_append_special_values_strides_and_slots(P):
    from latticequant_b200 import _lib

    H, D, page = 2, 128, 16
    codes, scales, _ = P.empty_pool(1, 2, H, D, page)
    x = torch.randn(6, H, D, device="cuda")
    x[0, 0, 5] = float("nan")
    x[1, 1, 7] = float("inf")
    x[2] = 3e38
    x[3] = 1e-30
    x[4] = x[4] * 1e-3
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, _ = P.append(codes[0], scales[0], x, torch.zeros_like(x), torch.arange(6, device="cuda"), True, err)
    assert int(err.item()) == _lib.EF_NONFINITE
    assert not k[0, 0].any() and not k[1, 1].any() and torch.isfinite(k).all()
    assert float(scales[0, 0, 0, 0, 0]) == 1.0 and not k[3].any() and float(scales[0, 0, 0, 0, 3]) == 1.0
    assert float((k[2] / x[2] - 1).abs().max()) < 0.08
    # views: heads first, and a row offset that breaks the 16-byte alignment
    big = torch.randn(H, 9, D + 3, device="cuda")
    view = big[:, :, 3:].transpose(0, 1)
    a, _ = P.append(codes[0], scales[0], view, view, torch.arange(9, device="cuda"), True)
    b, _ = P.append(codes[0], scales[0], view.contiguous(), view.contiguous(), torch.arange(9, device="cuda"), True)
    assert torch.equal(a, b)
    err.zero_()
    before = codes.clone()
    P.append(codes[0], scales[0], x[4:5], x[4:5], torch.tensor([2 * page], device="cuda"), err=err)
    assert int(err.item()) == _lib.EF_PAGE and torch.equal(codes, before)
    P.append(codes[0], scales[0], x[:0], x[:0], torch.empty(0, dtype=torch.int64, device="cuda"))


# ---------------------------------------------------------------- attention
def _pool(P, g, lens, H, D, page, spread=0.3, n_extra=2, dtype=torch.bfloat16):
    """Pages holding random tokens; the rows past a sequence's length hold NaN scales and random words."""
    B = len(lens)
    width = max(1, max(-(-n // page) for n in lens))
    n_pages = B * width + n_extra
    codes = torch.randint(-2**31, 2**31 - 1, (n_pages, 2, H, page, D // 8), dtype=torch.int32, device="cuda", generator=g)
    scales = torch.full((n_pages, 2, H, page), float("nan"), device="cuda")
    perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(1))
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = perm[at:at + need].int()
        at += need
        if n:
            pos = torch.arange(n)
            slots = (table[b, pos // page].long() * page + pos % page).cuda()
            kv = [torch.randn(n, H, D, device="cuda", generator=g) *
                  torch.exp(spread * torch.randn(n, H, 1, device="cuda", generator=g)) for _ in range(2)]
            P.append(codes, scales, kv[0].to(dtype), kv[1].to(dtype), slots)
    return codes, scales, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def _ref(q, codes, scales, table, lens, mask, scale):
    B, Hq, T, D = q.shape
    H, page = codes.shape[2], codes.shape[3]
    G = Hq // H
    o, lse = np.zeros((B, Hq, T, D)), np.full((B, Hq, T), -np.inf)
    qd = q.double().cpu().numpy()
    m = None if mask is None else mask.cpu().numpy()
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        pg = table[b, : -(-n // page)].long()
        kv = _values(codes[pg], scales[pg])  # (pages, 2, H, page, D)
        kv = kv.transpose(1, 2, 0, 3, 4).reshape(2, H, -1, D)[:, :, :n]
        j = np.arange(n) - (n - T)
        see = np.ones((T, n), bool)
        for t in range(T):
            d = j >= 0
            see[t, d] = (j[d] <= t) if m is None else (m[b] if m.ndim == 3 else m)[t, j[d]]
        for h in range(Hq):
            s = qd[b, h] @ kv[0, h // G].T * scale
            s = np.where(see, s, -np.inf)
            mx = s.max(1, keepdims=True)
            live = np.isfinite(mx[:, 0])
            e = np.exp(s - np.where(np.isfinite(mx), mx, 0))
            l = e.sum(1)
            o[b, h, live] = (e @ kv[1, h // G])[live] / l[live, None]
            lse[b, h, live] = (mx[:, 0] + np.log(np.where(l > 0, l, 1)))[live]
    return o, lse


def _check(o, lse, ro, rl):
    ulp = 2.0 ** -8 if o.dtype == torch.bfloat16 else 2.0 ** -11
    od, ld = o.double().cpu().numpy(), lse.double().cpu().numpy()
    top = np.abs(ro).max(-1, keepdims=True)
    assert (np.abs(od - ro) <= 1e-3 * top + ulp * np.abs(ro) + 1e-30).all(), np.abs(od - ro).max()
    assert np.array_equal(np.isinf(ld), np.isinf(rl))
    fin = np.isfinite(rl)
    assert (np.abs(ld[fin] - rl[fin]) <= 1e-4 * np.maximum(1, np.abs(rl[fin]))).all()


def _tree(T, seed, batch=None):
    rng = np.random.default_rng(seed)
    m = np.zeros((batch or 1, T, T), bool)
    for b in range(batch or 1):
        for t in range(T):
            if t:
                m[b, t] = m[b, rng.integers(0, t)]
            m[b, t, t] = True
    return torch.from_numpy(m if batch else m[0]).cuda()


CASES = [
    # lens, H, G, T, D, page, dtype, mask
    ([1], 1, 1, 1, 64, 16, torch.float16, None),
    ([777], 2, 4, 1, 128, 64, torch.bfloat16, None),
    ([0, 1, 15, 16, 17, 64, 65, 513], 3, 7, 1, 128, 16, torch.float16, None),
    ([5000, 3], 2, 8, 1, 64, 256, torch.bfloat16, None),
    ([13, 200, 1000], 2, 4, 13, 128, 64, torch.bfloat16, "batch"),
    ([64, 2100], 2, 7, 64, 128, 64, torch.float16, "one"),
    ([33, 90], 2, 3, 33, 64, 32, torch.bfloat16, "causal"),
    ([40, 333], 1, 8, 31, 64, 16, torch.float16, "batch"),
    ([7, 2], 2, 2, 5, 128, 16, torch.bfloat16, "one"),     # fewer tokens than positions
    ([300], 1, 1, 129, 128, 128, torch.float16, "causal"),  # a prompt's chunk
    ([70], 2, 16, 3, 128, 64, torch.bfloat16, "one"),
    ([130, 700, 0], 2, 5, 24, 128, 128, torch.bfloat16, "batch"),
]


@pytest.mark.parametrize("lens,H,G,T,D,page,dtype,mask", CASES)
def test_attention_matches_float64(P, lens, H, G, T, D, page, dtype, mask):
    g = torch.Generator(device="cuda").manual_seed(len(lens) * 100 + T)
    codes, scales, table, ln = _pool(P, g, lens, H, D, page)
    q = torch.randn(len(lens), H * G, T, D, device="cuda", generator=g).to(dtype)
    m = None if mask in (None, "causal") else _tree(T, T, len(lens) if mask == "batch" else None)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = P.tree_attention(q, codes, scales, table, ln, m, return_lse=True, err=err)
    assert int(err.item()) == 0
    _check(o, lse, *_ref(q, codes, scales, table, lens, m, 1 / math.sqrt(D)))
    again, _ = P.tree_attention(q, codes, scales, table, ln, m, return_lse=True, max_len=max(max(lens), 1))
    _check(again, lse, o.double().cpu().numpy(), lse.double().cpu().numpy())


def _ref_gpu(q, codes, scales, table, lens, mask, scale):
    """_ref on the GPU in float64, for batches too large for the host: K and V of every sequence at the longest length."""
    B, Hq, T, D = q.shape
    H, page = codes.shape[2], codes.shape[3]
    n = table.shape[1] * page
    shift = torch.tensor([27, 23, 19, 15, 11, 7, 3], device="cuda")
    pg = table.clamp(min=0).long()
    w = codes[pg].long() & 0xFFFFFFFF
    u = (w[..., None] >> shift) & 15
    last = 2 * (w & 7) + u.sum(-1) % 2
    pts = torch.cat([u, last[..., None]], -1).double() - 8 + 0.5 * (w >> 31)[..., None]
    kv = (pts.flatten(-2) * scales[pg].double()[..., None]).nan_to_num(0)  # (B, width, 2, H, page, D)
    k, v = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, B, H, 1, n, D)
    j = torch.arange(n, device="cuda")[None, None] - (lens.long()[:, None, None] - T)
    see = (j < 0).expand(B, T, n).clone()
    t = torch.arange(T, device="cuda")[None, :, None]
    drafts = (j >= 0) & (j < T)
    if mask is None:
        see |= drafts & (j <= t)
    else:
        see |= drafts & mask.expand(B, T, T).gather(2, j.clamp(0, T - 1).expand(B, T, n))
    x = q.double().view(B, H, Hq // H * T, D) @ k.squeeze(2).transpose(2, 3) * scale
    x = x.view(B, H, Hq // H, T, n).masked_fill(~see[:, None, None], float("-inf"))
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    o = (p.view(B, H, -1, n) @ v.squeeze(2)).view(B, Hq, T, D)
    return o.cpu().numpy(), lse.view(B, Hq, T).cpu().numpy()


# enough (sequence, head) pairs that a CTA walks many tiles: every kernel's pipeline goes round its buffers
@pytest.mark.parametrize("G,T,D,page,dtype", [
    (4, 1, 128, 64, torch.bfloat16), (8, 1, 64, 16, torch.float16),                     # up to 8 rows
    (4, 4, 128, 32, torch.float16), (3, 5, 64, 64, torch.bfloat16),                     # 16
    (7, 4, 128, 128, torch.bfloat16), (2, 16, 64, 32, torch.float16),                   # 32
    (4, 13, 128, 16, torch.float16), (8, 8, 64, 256, torch.bfloat16), (4, 13, 128, 256, torch.bfloat16),  # 64
    (5, 33, 128, 64, torch.float16),                                                    # more than one CTA's rows
])
def test_attention_many_tiles(P, G, T, D, page, dtype):
    g = torch.Generator(device="cuda").manual_seed(G * 100 + T)
    B, H = 75, 8
    rng = np.random.default_rng(T)
    lens = [int(x) for x in rng.integers(0, 1700, B)]
    lens[0], lens[1], lens[2], lens[3] = 1700, 0, 1, 1664
    codes, scales, table, ln = _pool(P, g, lens, H, D, page, spread=1.0, dtype=dtype)
    q = (2 * torch.randn(B, H * G, T, D, device="cuda", generator=g)).to(dtype)
    m = _tree(T, T, B) if T > 1 else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = P.tree_attention(q, codes, scales, table, ln, m, return_lse=True, err=err)
    assert int(err.item()) == 0
    ro, rl = _ref_gpu(q, codes, scales, table, ln, m, 1 / math.sqrt(D))
    _check(o, lse, ro, rl)
    for _ in range(3):  # nothing in the result depends on timing
        assert torch.equal(o, P.tree_attention(q, codes, scales, table, ln, m))


@pytest.mark.parametrize("T", [2, 40])
def test_attention_rows_that_see_nothing(P, T):
    """No context and an empty mask row: o = 0, lse = -inf; other rows are unaffected."""
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = [T, T + 20]
    codes, scales, table, ln = _pool(P, g, lens, 2, 128, 16)
    q = torch.randn(2, 8, T, 128, device="cuda", generator=g).to(torch.bfloat16)
    m = _tree(T, 1, 2)
    m[:, 1] = False
    o, lse = P.tree_attention(q, codes, scales, table, ln, m, return_lse=True)
    assert not o[0, :, 1].any() and torch.isinf(lse[0, :, 1]).all() and torch.isfinite(lse[1]).all()
    _check(o, lse, *_ref(q, codes, scales, table, lens, m, 1 / math.sqrt(128)))


@pytest.mark.parametrize("T", [1, 24])
def test_attention_scales_far_apart(P, T):
    """V scales over 2^-40..2^40 and large scores: the fp16 weights stay in range."""
    g = torch.Generator(device="cuda").manual_seed(9)
    lens = [400, 129]
    codes, scales, table, ln = _pool(P, g, lens, 2, 128, 16)
    scales[:, 1] *= torch.exp2(torch.randint(-40, 41, scales[:, 1].shape, device="cuda", generator=g).float())
    q = (8 * torch.randn(2, 8, T, 128, device="cuda", generator=g)).to(torch.bfloat16)
    o, lse = P.tree_attention(q, codes, scales, table, ln, None, return_lse=True)
    _check(o, lse, *_ref(q, codes, scales, table, lens, None, 1 / math.sqrt(128)))


def test_attention_strides_streams_and_out(P):
    g = torch.Generator(device="cuda").manual_seed(2)
    lens = [150, 90]
    codes, scales, table, ln = _pool(P, g, lens, 2, 128, 32)
    base = torch.randn(2, 6, 8, 128, device="cuda", generator=g).to(torch.float16)
    want, wl = _ref(base.transpose(1, 2), codes, scales, table, lens, None, 0.05)
    side = torch.cuda.Stream()
    out = torch.empty(2, 8, 6, 128, dtype=torch.float16, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, lse = P.tree_attention(base.transpose(1, 2), codes, scales, table, ln, sm_scale=0.05, out=out, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    assert o is out
    _check(o, lse, want, wl)
    odd = torch.randn(2, 8, 6, 130, device="cuda", generator=g).to(torch.float16)[..., 1:129]  # 2-byte aligned rows
    a = P.tree_attention(odd, codes, scales, table, ln)
    assert torch.equal(a, P.tree_attention(odd.contiguous(), codes, scales, table, ln))
    graph, cap = torch.cuda.CUDAGraph(), torch.empty_like(out)
    with torch.cuda.graph(graph):
        P.tree_attention(base.transpose(1, 2), codes, scales, table, ln, sm_scale=0.05, out=cap)
    graph.replay()
    assert torch.equal(cap, out)


def test_attention_past_32_bit_offsets(P):
    """Pages whose words lie past 2^31: a pool of 2^31 words and more."""
    H, D, page = 8, 128, 64
    n_pages = 2**31 // (2 * H * page * D // 8) + 40
    codes = torch.empty(n_pages, 2, H, page, D // 8, dtype=torch.int32, device="cuda")
    scales = torch.empty(n_pages, 2, H, page, device="cuda")
    lens = [1000]
    table = (n_pages - 1 - torch.arange(16, device="cuda")).to(torch.int32)[None].contiguous()
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pos = torch.arange(1000, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 1000, H, D, device="cuda", generator=g).to(torch.float16)
    P.append(codes, scales, x[0], x[1], table[0, pos // page].long() * page + pos % page)
    for T in (1, 32):
        q = torch.randn(1, H * 4, T, D, device="cuda", generator=g).to(torch.float16)
        o, lse = P.tree_attention(q, codes, scales, table, ln, return_lse=True)
        _check(o, lse, *_ref(q, codes, scales, table, lens, None, 1 / math.sqrt(D)))


@pytest.mark.parametrize("T", [1, 20])
def test_attention_bad_tables_are_reported(P, T):
    from latticequant_b200 import _lib

    g = torch.Generator(device="cuda").manual_seed(6)
    codes, scales, table, ln = _pool(P, g, [100], 1, 64, 16)
    q = torch.randn(1, 4, T, 64, device="cuda", generator=g).to(torch.float16)
    for entry in (-1, codes.shape[0], 2**31 - 1):
        bad = table.clone()
        bad[0, 2] = entry
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        o = P.tree_attention(q, codes, scales, bad, ln, err=err)
        assert int(err.item()) == _lib.EF_PAGE and torch.isfinite(o).all()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    P.tree_attention(q, codes, scales, table, ln + 100, err=err)
    assert int(err.item()) == _lib.EF_PAGE


def test_refusals(P):
    codes, scales, refs = P.empty_pool(2, 4, 2, 64, 16)
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    ln = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device="cuda")
    bad = [
        lambda: P.empty_pool(1, 4, 2, 96),
        lambda: P.empty_pool(1, 4, 2, 64, 48),
        lambda: P.tree_attention(q.float(), codes[0], scales[0], table, ln),
        lambda: P.tree_attention(q[:, :3], codes[0], scales[0], table, ln),
        lambda: P.tree_attention(q, codes, scales, table, ln),
        lambda: P.tree_attention(q, codes[0], scales[0].half(), table, ln),
        lambda: P.tree_attention(q, codes[0], scales[0], table.long(), ln),
        lambda: P.tree_attention(q, codes[0], scales[0], table, ln.cpu()),
        lambda: P.tree_attention(q, codes[0], scales[0], table, ln, torch.ones(2, 2, dtype=torch.bool, device="cuda")),
        lambda: P.tree_attention(q.cpu(), codes[0], scales[0], table, ln),
        lambda: P.append(codes[0], scales[0], q[0], q[0], ln.long()),
        lambda: P.append(codes[0], scales[0], q[:, :2, 0].double(), q[:, :2, 0].double(), ln.long()),
        lambda: P.append(codes[0], scales[0], q[:, :2, 0], q[:, :2, 0], ln),
        lambda: P.fork_pages(codes, scales, table, ln, refs[:2], ln.long()),
        lambda: P.fork_pages(codes, scales, table, ln, refs, ln),
        lambda: P.compact_pages(codes[0], scales[0], table, refs),
        lambda: P.accept_tokens(codes, scales, table, ln, 1, ln),
        lambda: P.copy_pages(codes, scales, ln, ln[:0]),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(RuntimeError):
        P.accept_tokens(codes, scales, table, ln, 0, ln[:, None].contiguous())


# ---------------------------------------------------------------- page operations
def _fork_ref(table, lens, refs, parents, reserve, page):
    width = table.shape[1]
    free = [i for i, r in enumerate(refs) if r == 0]
    new, nl, copies, seen = np.full((len(parents), width), -1), [], [], set()
    for i, p in enumerate(parents):
        if p < 0:
            nl.append(0)
            continue
        n = int(lens[p])
        nl.append(n)
        full, need = n // page, -(-(n + reserve) // page)
        new[i, :full] = table[p, :full]
        for c in range(full, need):
            if p not in seen and table[p, c] >= 0:
                new[i, c] = table[p, c]
            else:
                new[i, c] = free.pop(0)
                if c == full and n % page:
                    copies.append((table[p, c], new[i, c], n % page))
        seen.add(p)
    nr = refs.copy()
    for x in table[table >= 0]:
        nr[x] -= 1
    for x in new[new >= 0]:
        nr[x] += 1
    return new, np.array(nl), nr, copies


@pytest.mark.parametrize("page,D,H,L", [(16, 64, 1, 1), (32, 128, 3, 2), (64, 128, 8, 3)])
@pytest.mark.parametrize("reserve", [0, 1, 70])
def test_fork_matches_loops(P, page, D, H, L, reserve):
    rng = np.random.default_rng(page + reserve)
    width, n_pages = 12, 200
    lens = [0, 1, page - 1, page, page + 1, 3 * page + 5, 5 * page]
    ids = list(rng.permutation(n_pages))
    table = np.full((len(lens), width), -1, np.int32)
    for b, n in enumerate(lens):
        for c in range(-(-n // page) + (b == 5)):  # one row holds a reserved page already
            table[b, c] = ids.pop()
    table[4, 0] = table[5, 0]  # a shared full page
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    refs[ids[0]] = 1  # held by somebody else
    parents = np.array([5, 5, -1, 2, 4, 5, 2, 0, 3, 3, 1])
    codes = torch.randint(-2**31, 2**31 - 1, (L, n_pages, 2, H, page, D // 8), dtype=torch.int32, device="cuda")
    scales = torch.rand(L, n_pages, 2, H, page, device="cuda")
    c0, s0 = codes.clone(), scales.clone()
    want = _fork_ref(table, lens, refs, parents, reserve, page)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    t, n, r = P.fork_pages(codes, scales, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                           torch.from_numpy(refs).cuda(), torch.from_numpy(parents).cuda(), reserve, err)
    assert int(err.item()) == 0
    assert np.array_equal(t.cpu().numpy(), want[0]) and np.array_equal(n.cpu().numpy(), want[1])
    assert np.array_equal(r.cpu().numpy(), want[2]) and len(want[3]) == 3
    for src, dst, live in want[3]:
        c0[:, dst, :, :, :live] = c0[:, src, :, :, :live]
        s0[:, dst, :, :, :live] = s0[:, src, :, :, :live]
    assert torch.equal(codes, c0) and torch.equal(scales, s0)


def test_fork_without_free_pages_and_bad_parents(P):
    from latticequant_b200 import _lib

    codes, scales, refs = P.empty_pool(1, 3, 1, 64, 16)
    table = torch.tensor([[0, 1, -1]], dtype=torch.int32, device="cuda")
    refs[:2] = 1
    ln = torch.tensor([20], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    t, _, _ = P.fork_pages(codes, scales, table, ln, refs, torch.zeros(4, dtype=torch.int64, device="cuda"), 0, err)
    assert int(err.item()) == _lib.EF_CAPACITY
    assert t.tolist() == [[0, 1, -1], [0, 2, -1], [0, -1, -1], [0, -1, -1]]
    err.zero_()
    t, n, r = P.fork_pages(codes, scales, table, ln, refs, torch.tensor([1], device="cuda"), 0, err)
    assert int(err.item()) == _lib.EF_PAGE and t.tolist() == [[-1, -1, -1]] and r.tolist() == [0, 0, 0]
    err.zero_()
    P.fork_pages(codes, scales, table, ln, refs, torch.tensor([0], device="cuda"), 100, err)  # past the table's width
    assert int(err.item()) & _lib.EF_PAGE
    t, n, r = P.fork_pages(codes, scales, table, ln, refs, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert t.shape == (0, 3) and r.tolist() == [0, 0, 0]


@pytest.mark.parametrize("n_pages,live", [(1, 1.0), (7, 0.5), (300, 0.0), (300, 1.0), (2500, 0.4)])
def test_compact_matches_loops(P, n_pages, live):
    rng = np.random.default_rng(n_pages)
    used = rng.random(n_pages) < live
    refs = np.where(used, rng.integers(1, 4, n_pages), 0).astype(np.int32)
    ids = np.flatnonzero(used)
    table = np.concatenate([rng.permutation(ids), [-1, -1]]).astype(np.int32)[None]
    codes = torch.randint(-2**31, 2**31 - 1, (2, n_pages, 2, 1, 16, 8), dtype=torch.int32, device="cuda")
    scales = torch.rand(2, n_pages, 2, 1, 16, device="cuda")
    c0, s0 = codes.clone(), scales.clone()
    t, r, n = P.compact_pages(codes, scales, torch.from_numpy(table).cuda(), torch.from_numpy(refs).cuda())
    k = len(ids)
    assert n.tolist() == [k]
    to = np.arange(n_pages)
    src, dst = ids[ids >= k], np.flatnonzero(~used[:k])
    to[src] = dst
    assert np.array_equal(t.cpu().numpy(), np.where(table >= 0, to[table], -1))
    want = np.zeros(n_pages, np.int32)
    want[to[ids]] = refs[ids]
    assert np.array_equal(r.cpu().numpy(), want)
    c0[:, dst] = c0[:, src]
    s0[:, dst] = s0[:, src]
    assert torch.equal(codes, c0) and torch.equal(scales, s0)


def test_copy_pages(P):
    codes = torch.randint(-2**31, 2**31 - 1, (3, 9, 2, 2, 16, 16), dtype=torch.int32, device="cuda")
    scales = torch.rand(3, 9, 2, 2, 16, device="cuda")
    c0, s0 = codes.clone(), scales.clone()
    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3, 0, 5], [8, 2, 1]))
    P.copy_pages(codes, scales, src, dst, torch.tensor([2], dtype=torch.int32, device="cuda"))
    c0[:, [8, 2]], s0[:, [8, 2]] = c0[:, [3, 0]], s0[:, [3, 0]]
    assert torch.equal(codes, c0) and torch.equal(scales, s0)
    P.copy_pages(codes, scales, src, dst)
    c0[:, 1], s0[:, 1] = c0[:, 5], s0[:, 5]
    assert torch.equal(codes, c0) and torch.equal(scales, s0)


@pytest.mark.parametrize("page,D,H", [(16, 64, 3), (64, 128, 8)])
def test_accept_matches_loops(P, page, D, H):
    from latticequant_b200 import _lib

    T, L, width = 40, 2, 8
    lens = [T, T + 3, page * 2 + T - 1, 100, 5, 0]
    acc = [[0, 1, 2], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10], list(range(0, 40, 2)), [], [], []]
    accepted = np.full((len(lens), 20), -1, np.int32)
    for b, a in enumerate(acc):
        accepted[b, :len(a)] = a
    n_pages = len(lens) * width
    table = np.random.default_rng(0).permutation(n_pages).reshape(-1, width).astype(np.int32)
    codes = torch.randint(-2**31, 2**31 - 1, (L, n_pages, 2, H, page, D // 8), dtype=torch.int32, device="cuda")
    scales = torch.rand(L, n_pages, 2, H, page, device="cuda")
    c0, s0 = codes.clone(), scales.clone()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = [torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()]
    out = P.accept_tokens(codes, scales, *args, T, torch.from_numpy(accepted).cuda(), err)
    assert int(err.item()) == 0
    assert out.tolist() == [max(n - T, 0) + len(a) for n, a in zip(lens, acc)]
    for b, a in enumerate(acc):
        base = lens[b] - T
        for j, i in enumerate(a):
            (sp, so), (dp, do) = [(int(table[b, x // page]), x % page) for x in (base + i, base + j)]
            c0[:, dp, :, :, do], s0[:, dp, :, :, do] = c0[:, sp, :, :, so].clone(), s0[:, sp, :, :, so].clone()
    assert torch.equal(codes, c0) and torch.equal(scales, s0)
    # lists that are not ascending or out of range leave their rows alone
    for wrong in ([3, 2], [1, 1], [0, T]):
        accepted[:] = -1
        accepted[0, :2] = wrong
        err.zero_()
        out = P.accept_tokens(codes, scales, *args, T, torch.from_numpy(accepted).cuda(), err)
        assert int(err.item()) == _lib.EF_PAGE and int(out[0]) == lens[0]
        assert torch.equal(codes, c0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_equals_the_frameworks_search_at_its_ties(P, dtype):
    """Values on the lattice's decision surfaces (quarter steps of the scale, repeated magnitudes), where the
    search's short form hands over to the long one, and a million blocks of ordinary values."""
    from latticequant_b200.core import e8_quantizer

    g = torch.Generator(device="cuda").manual_seed(11)
    n, H, D = 4096, 2, 128
    # a first channel of 7 - 1/64 makes the scale 1 up to a rounding, so the rest are exact steps of it
    x = torch.randint(-27, 28, (n, H, D), device="cuda", generator=g).float() / 4
    x[..., 0] = 7 - 1 / 64
    y = torch.randn(n, H, D, device="cuda", generator=g)
    y[: n // 2, :, 8:16] = y[: n // 2, :, 8:9] * torch.where(torch.rand(n // 2, H, 8, device="cuda", generator=g) < 0.5, -1, 1)
    for v in (x.to(dtype), y.to(dtype)):
        codes, scales, _ = P.empty_pool(1, n // 64, H, D, 64)
        k, _ = P.append(codes[0], scales[0], v, v, torch.arange(n, device="cuda"), dequantised=True)
        amax = v.float().abs().amax(-1)
        s = amax * float(np.float32(1) / BOUND)
        q = e8_quantizer.encode_e8((v.float() / s[..., None]).reshape(-1, 8)).view(n, H, D)
        assert torch.equal(k, (q * s[..., None]).to(dtype))
        stored = _values(codes[0, :, 0], scales[0, :, 0]).transpose(0, 2, 1, 3).reshape(n, H, D)
        assert np.array_equal(stored, q.double().cpu().numpy() * s[..., None].double().cpu().numpy())


@pytest.mark.parametrize("lens,H,G,T,dtype,mask", [
    ([9, 10, 200, 64], 2, 3, 3, torch.bfloat16, "batch"),     # 9 rows: one in the last tile
    ([1, 2030, 0], 1, 4, 4, torch.float16, "one"),            # 16, fewer tokens than positions
    ([5000, 11], 3, 1, 11, torch.bfloat16, "causal"),
    ([16385], 1, 15, 1, torch.float16, None),
])
def test_attention_two_row_tiles(P, lens, H, G, T, dtype, mask):
    """9 to 16 rows of 64 channels, with rows that see nothing and entries outside the pool."""
    from latticequant_b200 import _lib

    g = torch.Generator(device="cuda").manual_seed(T)
    codes, scales, table, ln = _pool(P, g, lens, H, 64, 16, spread=1.0)
    q = torch.randn(len(lens), H * G, T, 64, device="cuda", generator=g).to(dtype)
    m = None if mask in (None, "causal") else _tree(T, T, len(lens) if mask == "batch" else None)
    if m is not None:
        m[..., 1, :] = False
    o, lse = P.tree_attention(q, codes, scales, table, ln, m, return_lse=True)
    _check(o, lse, *_ref(q, codes, scales, table, lens, m, 1 / 8))
    assert torch.equal(o, P.tree_attention(q, codes, scales, table, ln, m))
    for entry in (-1, codes.shape[0], 2**31 - 1):
        bad = table.clone()
        bad[0, 0] = entry
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        o = P.tree_attention(q, codes, scales, bad, ln, m, err=err)
        assert int(err.item()) == _lib.EF_PAGE and torch.isfinite(o).all()
