"""The paged cache at its limits: what it refuses, reports and survives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    from latticequant_b200 import paged

    return paged


def _filled(P, lens, H, D, page, seed=0, dtype=torch.float16):
    """(codes, scales, table, lens) of one layer: sequence b holds lens[b] random tokens in pages of its own."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, -(-max(lens) // page))
    codes, scales, _ = P.empty_pool(1, len(lens) * width, H, D, page)
    table = torch.arange(len(lens) * width, device="cuda", dtype=torch.int32).view(-1, width)
    for b, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        kv = torch.randn(2, n, H, D, device="cuda", generator=g).to(dtype)
        P.append(codes[0], scales[0], kv[0], kv[1], table[b, pos // page].long() * page + pos % page)
    return codes[0], scales[0], table, torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D,off", [(64, 1), (128, 1), (128, 2)])
def test_misaligned_outputs_are_refused(P, D, off):
    codes, scales, table, ln = _filled(P, [40], 2, D, 16)
    q = torch.randn(1, 4, 1, D, device="cuda").to(torch.float16)
    buf = torch.zeros(4 * D + 8, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="aligned"):
        P.tree_attention(q, codes, scales, table, ln, out=buf[off: off + 4 * D].view(1, 4, 1, D))
    fine = D // 32  # the least that the stores take
    o = P.tree_attention(q, codes, scales, table, ln, out=buf[fine: fine + 4 * D].view(1, 4, 1, D))
    assert torch.equal(o, P.tree_attention(q, codes, scales, table, ln))


def test_copy_reads_no_pair_past_the_lists(P):
    """A count above the lists' length copies the listed pairs and no other."""
    codes = torch.randint(-2**31, 2**31 - 1, (2, 9, 2, 1, 16, 8), dtype=torch.int32, device="cuda")
    scales = torch.rand(2, 9, 2, 1, 16, device="cuda")
    c0, s0 = codes.clone(), scales.clone()
    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3, 0, 5, 6], [8, 2, 1, 7]))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for count in (7, 2**31 - 1, 0, -1):  # the lists end before their memory does
        P.copy_pages(codes, scales, src[:2], dst[:2], torch.tensor([count], dtype=torch.int32, device="cuda"), err)
        if count > 0:
            c0[:, [8, 2]], s0[:, [8, 2]] = c0[:, [3, 0]], s0[:, [3, 0]]
        assert torch.equal(codes, c0) and torch.equal(scales, s0) and int(err.item()) == 0


@pytest.mark.parametrize("G,T,D", [(4, 4, 128), (4, 8, 128), (8, 8, 128), (3, 10, 64), (8, 8, 64)])
def test_short_blocks_leave_nothing_behind(P, G, T, D):
    """One or two tiles a block and many blocks a SM in a row: a block's last arrivals come before it ends, so its
    successor in the same shared memory answers as it does alone."""
    lens = [T + (37 * b) % 230 for b in range(96)]
    codes, scales, table, ln = _filled(P, lens, 4, D, 64)
    q = torch.randn(len(lens), 4 * G, T, D, device="cuda").to(torch.float16)
    alone = torch.cat([P.tree_attention(q[b: b + 1], codes, scales, table[b: b + 1], ln[b: b + 1], max_len=256)
                       for b in range(len(lens))])
    o = P.tree_attention(q, codes, scales, table, ln, max_len=256)
    # (the split, and so the order of the sums, is that of the batch: fp16's unit roundoff and a weight's, twice)
    top = alone.float().abs().amax(-1, keepdim=True)
    assert bool(((o.float() - alone.float()).abs() <= 2e-3 * top + 2 ** -10 * alone.float().abs()).all())
    for _ in range(20):
        assert torch.equal(o, P.tree_attention(q, codes, scales, table, ln, max_len=256))


def _cache(rows, n_pages=24, max_tokens=64, page=16, layers=1):
    from latticequant_b200.llm.paged_cache import PagedKVCache

    return PagedKVCache(layers, 2, 64, n_pages=n_pages, rows=rows, max_tokens=max_tokens, page_tokens=page)


def _kv(g, rows, n):
    return [torch.randn(rows, 2, n, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]


@pytest.mark.parametrize("n", [1, 20, 40])
def test_tokens_past_the_table_are_not_stored(n):
    """Rows that are as long as their table allows keep what they hold, and so do the rows that share their pages."""
    from latticequant_b200 import _lib

    g = torch.Generator(device="cuda").manual_seed(n)
    c = _cache(2)
    c.begin(64)
    c.append(0, *_kv(g, 2, 64))
    c.fork(torch.tensor([0, 0, 1], device="cuda"))
    q = torch.randn(3, 4, 1, 64, device="cuda", generator=g).to(torch.bfloat16)
    before, codes, scales = c.attend(0, q), c.codes.clone(), c.scales.clone()
    assert c.flags() == 0
    c.begin(n)
    k, v = c.append(0, *_kv(g, 3, n), dequantised=True)
    assert c.flags() & _lib.EF_PAGE and k.shape == (3, 2, n, 64)
    assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)
    c.lens = (c.lens - n).clamp_(max=64)
    c.max_len = 64
    assert torch.equal(c.attend(0, q), before)


def test_tokens_up_to_the_tables_end_are_stored():
    """A row one token short of its table stores that token and drops the next; a shorter row beside it stores both."""
    g = torch.Generator(device="cuda").manual_seed(1)
    c, one = _cache(2), _cache(1)
    kv = _kv(g, 2, 63)
    c.begin(63)
    c.append(0, *kv)
    c.fork(torch.tensor([0, 1], device="cuda"))
    c.lens = torch.tensor([63, 30], dtype=torch.int32, device="cuda")
    new = _kv(g, 2, 2)
    c.begin(2)
    c.append(0, *new)
    one.begin(64)
    one.append(0, *[torch.cat([x[:1], y[:1, :, :1]], 2) for x, y in zip(kv, new)])
    page, row = int(c.table[0, 3]), int(one.table[0, 3])
    assert torch.equal(c.codes[0, page], one.codes[0, row]) and torch.equal(c.scales[0, page], one.scales[0, row])
    short = _cache(1)
    short.begin(32)
    short.append(0, *[torch.cat([x[1:, :, :30], y[1:]], 2) for x, y in zip(kv, new)])
    for col in range(2):
        assert torch.equal(c.codes[0, int(c.table[1, col])], short.codes[0, int(short.table[0, col])])


def test_compaction_within_a_step():
    """Pages renamed between begin() and the last layer's append(): the rest of the step follows them."""
    g = torch.Generator(device="cuda").manual_seed(3)
    ctx, new = _kv(g, 4, 30), _kv(g, 4, 5)
    q = torch.randn(4, 4, 5, 64, device="cuda", generator=g).to(torch.bfloat16)
    out = []
    for compact in (False, True):
        c = _cache(4, layers=2)
        c.begin(30)
        c.append(0, *ctx)
        c.append(1, *ctx)
        c.free(torch.tensor([0, 1, 2], device="cuda"))  # holes below the other row's pages
        c.begin(5)
        c.append(0, *new)
        if compact:
            n = c.compact()
            assert int(c.table.max()) == int(n) - 1
        c.append(1, *new)
        out.append([c.attend(layer, q) for layer in range(2)] + [c.lens])
        assert c.flags() == 0
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("reserve", [0, 3, 40])
def test_fork_copies_a_shared_page_that_is_written_next(P, reserve):
    """Rows 0 and 1 both name page 5, of which they hold 9 tokens: neither may write there."""
    L, H, page, D = 2, 3, 16, 64
    codes = torch.randint(-2**31, 2**31 - 1, (L, 20, 2, H, page, D // 8), dtype=torch.int32, device="cuda")
    scales = torch.rand(L, 20, 2, H, page, device="cuda")
    old = [[2, 5, 7, -1, -1], [2, 5, -1, -1, -1], [9, 1, 7, -1, -1]]  # a shared page past the first one to write, too
    table = torch.tensor(old, dtype=torch.int32, device="cuda")
    lens = [25, 25, 32]
    refs = torch.bincount(table[table >= 0].long(), minlength=20).to(torch.int32)
    c0, s0 = codes.clone(), scales.clone()
    parents, err = [0, 1, 2, 0], torch.zeros(1, dtype=torch.int32, device="cuda")
    t, n, r = P.fork_pages(codes, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), refs,
                           torch.tensor(parents, device="cuda"), reserve, err)
    assert int(err.item()) == 0 and n.tolist() == [25, 25, 32, 25]
    free, want = [i for i in range(20) if int(refs[i]) == 0], []
    for p in parents:
        full, need = lens[p] // page, -(-(lens[p] + reserve) // page)
        row = old[p][:full] + [free.pop(0) for _ in range(full, need)]  # no page of theirs is their own
        if lens[p] % page:
            c0[:, row[full], :, :, : lens[p] % page] = c0[:, old[p][full], :, :, : lens[p] % page]
            s0[:, row[full], :, :, : lens[p] % page] = s0[:, old[p][full], :, :, : lens[p] % page]
        want.append(row + [-1] * (5 - len(row)))
    assert t.tolist() == want
    assert torch.equal(r, torch.bincount(t[t >= 0].long(), minlength=20).to(torch.int32))
    assert torch.equal(codes, c0) and torch.equal(scales, s0)


def test_rollback_behind_a_fork():
    """Drafts are rejected after a fork shared the page that they filled: the rows go on apart, as rows of their own would."""
    g = torch.Generator(device="cuda").manual_seed(4)
    ctx, drafts = _kv(g, 1, 14), _kv(g, 1, 5)
    c = _cache(1)
    c.begin(14)
    c.append(0, *ctx)
    c.begin(5)
    c.append(0, *drafts)
    c.fork(torch.tensor([0, 0], device="cuda"))  # 19 tokens: page 0 is full, and shared
    c.accept(torch.full((2, 1), -1, dtype=torch.int32, device="cuda"))
    new = [_kv(g, 2, 1) for _ in range(4)]
    for kv in new:
        c.begin(1)
        c.append(0, *kv)
    assert c.lens.tolist() == [18, 18] and c.flags() == 0
    q = torch.randn(2, 4, 1, 64, device="cuda", generator=g).to(torch.bfloat16)
    o = c.attend(0, q)
    for b in range(2):
        own = _cache(1)
        own.begin(18)
        own.append(0, *[torch.cat([x] + [kv[i][b: b + 1] for kv in new], 2) for i, x in enumerate(ctx)])
        assert torch.equal(o[b: b + 1], own.attend(0, q[b: b + 1]))
    assert torch.equal(c.refs, torch.bincount(c.table[c.table >= 0].long(), minlength=24).to(torch.int32))


def test_accept_moves_nothing_into_a_shared_page():
    """A tree of drafts split by a fork: the drafts that filled the page before it are held by both rows."""
    from latticequant_b200 import _lib

    g = torch.Generator(device="cuda").manual_seed(5)
    ctx, drafts = _kv(g, 1, 14), _kv(g, 1, 5)
    c = _cache(1, layers=2)
    c.begin(14)
    for layer in range(2):
        c.append(layer, *ctx)
    c.begin(5)
    for layer in range(2):
        c.append(layer, *drafts)
    c.fork(torch.tensor([0, 0, 0], device="cuda"))
    codes, scales = c.codes.clone(), c.scales.clone()
    # row 0 keeps drafts that are in place, row 1 would move draft 3 into slot 15, row 2's list moves only in its own page
    c.accept(torch.tensor([[0, 1, 2, -1], [0, 3, 4, -1], [0, 1, 2, 4]], dtype=torch.int32, device="cuda"))
    assert c.flags() == _lib.EF_PAGE
    assert c.lens.tolist() == [17, 19, 18]
    own = int(c.table[2, 1])
    codes[:, own, :, :, 1], scales[:, own, :, :, 1] = codes[:, own, :, :, 2], scales[:, own, :, :, 2]
    assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)


def test_accept_with_counts_equals_accept_where_nothing_is_shared(P):
    L, H, page, D, T = 2, 2, 16, 64, 9
    lens = [T, 40, 33]
    table = torch.randperm(12, device="cuda").to(torch.int32).view(3, 4)
    acc = torch.tensor([[0, 2, 5, 8], [1, 3, -1, -1], [0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    refs = torch.ones(12, dtype=torch.int32, device="cuda")
    refs[table[1, 0]] = 3  # a shared page in front of the drafts
    codes = torch.randint(-2**31, 2**31 - 1, (L, 12, 2, H, page, D // 8), dtype=torch.int32, device="cuda")
    scales = torch.rand(L, 12, 2, H, page, device="cuda")
    c1, s1, err = codes.clone(), scales.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    a = P.accept_tokens(codes, scales, table, ln, T, acc, err)
    b = P.accept_tokens(c1, s1, table, ln, T, acc, err, refs)
    assert a.tolist() == b.tolist() == [4, 33, 28] and int(err.item()) == 0
    assert torch.equal(codes, c1) and torch.equal(scales, s1)
    with pytest.raises(ValueError):
        P.accept_tokens(codes, scales, table, ln, T, acc, err, refs[:3])


def test_a_step_is_accepted_once():
    g = torch.Generator(device="cuda").manual_seed(6)
    c = _cache(2)
    with pytest.raises(ValueError):
        c.accept(torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    c.begin(20)
    c.append(0, *_kv(g, 2, 20))
    c.begin(3)
    c.append(0, *_kv(g, 2, 3))
    keep = torch.tensor([[0, 2], [1, -1]], dtype=torch.int32, device="cuda")
    c.accept(keep)
    for between in (lambda: None, lambda: c.fork(torch.tensor([1, 0], device="cuda"))):
        between()
        with pytest.raises(ValueError):
            c.accept(keep)
    assert c.lens.tolist() == [21, 22] and c.max_len == 22 and c.flags() == 0


@pytest.mark.parametrize("T,G,D", [(1, 4, 128), (3, 4, 64), (13, 4, 128), (16, 8, 64)])
@pytest.mark.parametrize("planned", [0, 1, 130, 700, 2600])
def test_rows_longer_than_planned_are_read_whole(P, T, G, D, planned):
    """max_len sets the split; rows beyond it are attended to their end by either kernel, in a cluster or not."""
    lens = [3000, 131, 40, 2601]
    codes, scales, table, ln = _filled(P, lens, 2, D, 16)
    q = torch.randn(4, 2 * G, T, D, device="cuda").to(torch.float16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, wl = P.tree_attention(q, codes, scales, table, ln, return_lse=True)
    o, lse = P.tree_attention(q, codes, scales, table, ln, return_lse=True, max_len=planned, err=err)
    assert int(err.item()) == 0
    # two orders of the same sums: fp16's unit roundoff and a weight's, twice
    top = want.float().abs().amax(-1, keepdim=True)
    assert bool(((o.float() - want.float()).abs() <= 2e-3 * top + 2 ** -10 * want.float().abs()).all())
    assert bool(((lse - wl).abs() <= 2e-4 * wl.abs().clamp(min=1)).all())


def test_a_refused_row_is_attended_whole():
    """A list that accept() refuses leaves its row all the drafts, and later steps see them."""
    from latticequant_b200 import _lib

    g = torch.Generator(device="cuda").manual_seed(7)
    ctx, drafts, new = _kv(g, 2, 20), _kv(g, 2, 9), _kv(g, 2, 1)
    q = torch.randn(2, 4, 1, 64, device="cuda", generator=g).to(torch.bfloat16)
    c = _cache(2)
    for n, kv in ((20, ctx), (9, drafts)):
        c.begin(n)
        c.append(0, *kv)
    c.accept(torch.tensor([[0], [12]], dtype=torch.int32, device="cuda"))  # 12: no such draft
    assert c.flags() == _lib.EF_PAGE and c.lens.tolist() == [21, 29]
    c.err.zero_()
    c.begin(1)
    c.append(0, *new)
    o = c.attend(0, q)
    assert c.flags() == 0
    for b, n in ((0, 1), (1, 9)):
        own = _cache(1)
        own.begin(20 + n + 1)
        own.append(0, *[torch.cat([x[b: b + 1], d[b: b + 1, :, :n], y[b: b + 1]], 2) for x, d, y in zip(ctx, drafts, new)])
        w = own.attend(0, q[b: b + 1])
        assert bool(((o[b: b + 1] - w).float().abs() <= 2e-3 * w.float().abs().max() + 2 ** -7 * w.float().abs()).all())


@pytest.mark.parametrize("B,H,G,T,D,longest,shorter", [
    (16, 8, 4, 13, 128, 11328, (11200, 5000, 129)), (32, 8, 4, 1, 128, 2944, (2752, 2100, 64)),
    (1, 2, 4, 1, 64, 40000, (39000, 20000, 2049)), (2, 2, 7, 9, 64, 9000, (8990, 4097, 640)),
])
def test_a_workspace_serves_shorter_bounds_and_narrower_tables(B, H, G, T, D, longest, shorter):
    """The C entry with the workspace of the longest context, asked for less by max_len and by the table."""
    from latticequant_b200 import _lib

    lib, page = _lib.lib(), 64
    need = lib.lq_paged_attention_workspace(B, H, G, T, D, longest)
    ws = torch.empty(need // 4 + 4, dtype=torch.int32, device="cuda")
    ws[need // 4:] = 12345
    codes = torch.full((4, 2, H, page, D // 8), 0x44444444, dtype=torch.int32, device="cuda")
    scales = torch.ones(4, 2, H, page, device="cuda")
    width = -(-longest // page)
    table = torch.randint(0, 4, (B, width), dtype=torch.int32, device="cuda")
    q = torch.randn(B, H * G, T, D, device="cuda").to(torch.float16)
    out = torch.empty_like(q)
    for n in (longest, *shorter):
        for max_len, cols in ((n, width), (longest, -(-n // page))):
            lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
            out.fill_(7)
            status = lib.lq_paged_attention(q.data_ptr(), 1, *q.stride()[:3], codes.data_ptr(), scales.data_ptr(), 4, page,
                                            table.data_ptr(), cols, width, lens.data_ptr(), max_len, None, 0, B, H, G, T, D,
                                            1.0, out.data_ptr(), None, ws.data_ptr() if need else None, need, None, None)
            assert status == 0, (n, max_len, cols)
            torch.cuda.synchronize()
            assert not out.any() and (ws[need // 4:] == 12345).all()  # every value is zero


@pytest.mark.parametrize("T,G,D", [(2, 4, 128), (2, 8, 64), (3, 4, 128), (4, 7, 128), (13, 4, 128), (12, 8, 64), (4, 8, 64)])
def test_query_rows_of_any_magnitude_beside_one_another(P, T, G, D):
    """bf16 rows 2^60 above, 2^-12, 2^-30 and 2^-90 of their neighbours, zero, and with infinities or NaN: the others'
    answers are theirs alone.  Bounds as in test_gpu_paged."""
    import math

    import test_gpu_paged as base

    g = torch.Generator(device="cuda").manual_seed(T * 10 + G)
    lens = [300, 150]
    codes, scales, table, ln = base._pool(P, g, lens, 2, D, 16)
    q = torch.randn(2, 2 * G, T, D, device="cuda", generator=g)
    q[0, 0, 0] *= 2.0**60
    q[0, 1, 1] *= 2.0**-12
    q[1, 0, 0] *= 2.0**-30
    q[1, 1, 1] *= 2.0**-90
    q[1, 2, 0] = 0
    q = q.to(torch.bfloat16)
    o, lse = P.tree_attention(q, codes, scales, table, ln, return_lse=True)
    base._check(o, lse, *base._ref(q, codes, scales, table, lens, None, 1 / math.sqrt(D)))
    bad = q.clone()
    bad[0, 2, 0, 3], bad[1, 3, 1, 5] = float("inf"), float("nan")
    o2 = P.tree_attention(bad, codes, scales, table, ln)
    keep = torch.ones(2, 2 * G, T, dtype=torch.bool, device="cuda")
    keep[0, 2, 0] = keep[1, 3, 1] = False
    assert torch.equal(o2[keep], o[keep])


def test_single_tokens_cut_out_of_odd_rows(P):
    """One token of one head, one position: strides that no element uses may be anything."""
    codes, scales, table, ln = _filled(P, [50], 1, 128, 16)
    wide = torch.randn(1, 3 * 128 + 3, device="cuda").to(torch.float16)
    k, v, q = (wide[:, None, i * 128: (i + 1) * 128] for i in range(3))
    assert k.stride(0) % 8 and k.is_contiguous()
    c1, s1 = codes.clone(), scales.clone()
    slot = torch.tensor([50], device="cuda")
    a = P.append(codes, scales, k, v, slot, dequantised=True)
    b = P.append(c1, s1, k.clone().view(-1).view(1, 1, 128), v.clone().view(-1).view(1, 1, 128), slot, dequantised=True)
    assert torch.equal(codes, c1) and torch.equal(scales, s1) and all(torch.equal(x, y) for x, y in zip(a, b))
    ln += 1
    q = q[:, None]
    assert q.shape == (1, 1, 1, 128) and any(s % 8 for s in q.stride()[:-1])
    o = P.tree_attention(q, codes, scales, table, ln)
    assert torch.equal(o, P.tree_attention(q.clone().view(-1).view(1, 1, 1, 128), codes, scales, table, ln))


@pytest.mark.parametrize("lens,H,G,T,D,page,dtype,mask", [
    ([4096], 1, 1, 4096, 64, 64, torch.float16, None),            # a prompt's chunk that is the whole context
    ([2500, 2048], 1, 3, 2048, 128, 64, torch.bfloat16, None),
    ([5000, 700, 701], 2, 4, 700, 128, 16, torch.float16, None),  # a chunk after a context
    ([1900], 1, 2, 700, 128, 256, torch.bfloat16, "tree"),
    ([3000, 90], 1, 64, 1, 128, 32, torch.float16, None),         # the widest group
    ([3000, 90], 2, 33, 2, 64, 64, torch.bfloat16, None),
    ([800, 4], 1, 64, 5, 128, 128, torch.float16, "tree"),
    ([100, 7], 1, 24, 300, 64, 16, torch.bfloat16, None),         # fewer tokens than positions
])
def test_long_chunks_and_wide_groups(P, lens, H, G, T, D, page, dtype, mask):
    """Bounds as in test_gpu_paged."""
    import math

    import test_gpu_paged as base

    g = torch.Generator(device="cuda").manual_seed(T + G)
    codes, scales, table, ln = base._pool(P, g, lens, H, D, page)
    q = torch.randn(len(lens), H * G, T, D, device="cuda", generator=g).to(dtype)
    m = base._tree(T, 3, len(lens)) if mask else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = P.tree_attention(q, codes, scales, table, ln, m, return_lse=True, err=err)
    assert int(err.item()) == 0
    base._check(o, lse, *base._ref_gpu(q, codes, scales, table, ln, m, 1 / math.sqrt(D)))


@pytest.mark.parametrize("T,D", [(1, 64), (1, 128), (3, 64), (4, 128), (12, 64), (24, 128)])
@pytest.mark.parametrize("vmag,boost", [(1.0, 18), (0.03, 14), (0.03, 18), (1e-3, 10), (1e-3, 18)])
def test_a_zero_value_that_holds_most_of_the_weight(P, T, D, vmag, boost):
    """A sink: its V is zero (stored with scale 1) and its score `boost` above the rest; what the others leave in the
    output keeps its digits.  Bounds as in test_gpu_paged."""
    import math

    import test_gpu_paged as base

    g = torch.Generator(device="cuda").manual_seed(1)
    n = 400
    kv = torch.randn(2, n, 1, D, device="cuda", generator=g)
    kv[1] *= vmag
    u = torch.randn(D, device="cuda", generator=g)
    u /= u.norm()
    kv[0] -= (kv[0] @ u)[..., None] * u
    for at in (7, 200):  # two of them, the second 2 below the first
        kv[0, at, 0], kv[1, at] = u * (boost - (at > 7) * 2) * math.sqrt(D) / 8, 0
    kv[1, 300] = 0  # and an ordinary one
    q = torch.randn(1, 4, T, D, device="cuda", generator=g)
    q = (q - (q @ u)[..., None] * u + 8 * u).to(torch.bfloat16)
    codes, scales, _ = P.empty_pool(1, 8, 1, D, 64)
    P.append(codes[0], scales[0], kv[0].to(torch.bfloat16), kv[1].to(torch.bfloat16), torch.arange(n, device="cuda"))
    table = torch.arange(8, device="cuda", dtype=torch.int32)[None].contiguous()
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    o, lse = P.tree_attention(q, codes[0], scales[0], table, ln, return_lse=True)
    base._check(o, lse, *base._ref(q, codes[0], scales[0], table, [n], None, 1 / math.sqrt(D)))


def test_prompts_of_different_lengths_padded_to_one():
    """begin() with the longest, accept() with each row's own tokens: the rows are those of caches of their own."""
    g = torch.Generator(device="cuda").manual_seed(8)
    lens, n = [37, 3, 0, 20], 37
    ctx, new = _kv(g, 4, n), _kv(g, 4, 1)
    q = torch.randn(4, 4, 1, 64, device="cuda", generator=g).to(torch.bfloat16)
    c = _cache(4)
    c.begin(n)
    c.append(0, *ctx)
    at = torch.arange(n, device="cuda", dtype=torch.int32)[None]
    c.accept(torch.where(at < torch.tensor(lens, device="cuda")[:, None], at, -1).to(torch.int32))
    assert c.lens.tolist() == lens and c.max_len == n
    c.begin(1)
    c.append(0, *new)
    o = c.attend(0, q)
    for b, m in enumerate(lens):
        own = _cache(1)
        own.begin(m + 1)
        own.append(0, *[torch.cat([x[b: b + 1, :, :m], y[b: b + 1]], 2) for x, y in zip(ctx, new)])
        assert torch.equal(o[b: b + 1], own.attend(0, q[b: b + 1]))
    assert c.flags() == 0
