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
