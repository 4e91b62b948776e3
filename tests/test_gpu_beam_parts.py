"""beam_select where a CTA streams many tiles of a row, and where totals are hard to compute.

Every returned place is checked for itself: its score against the float64 total
of the (beam, word) that it names, the places unique and in order, and nothing
left out that is better than the last by more than the error.  A total is
(x - max) - ln(sum) + score, so its error is an fp32 rounding or two of the
total's own size and the sum's 2e-6 at most.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def select():
    from latticequant_b200.beam import beam_select

    return beam_select


def _totals(x, s):
    """float64 totals (B, K, V) on the GPU; -inf: no candidate."""
    xd = x.double()
    xd = torch.where(xd.isnan(), -torch.inf, xd)
    mx = xd.amax(-1, keepdim=True)
    safe = torch.where(mx.isinf(), 0.0, mx)
    ls = torch.log(torch.exp(xd - safe).sum(-1, keepdim=True))
    t = (xd - safe) - ls + s.double()[..., None]
    bad = mx.isinf() | ~(s[..., None] > -torch.inf)  # a row with +inf or nothing, a dead beam
    return torch.where(bad | xd.isinf() | t.isnan(), -torch.inf, t)


def _check(got, x, s, n):
    score, beam, word = got
    tot = _totals(x, s)
    B, K, V = tot.shape
    flat = tot.flatten(1)
    have = (flat > -torch.inf).sum(1).clamp(max=n)
    place = torch.arange(n, device=x.device)[None]
    live = place < have[:, None]
    assert torch.equal(score > -torch.inf, live)
    assert ((beam == -1) & (word == -1) | live).all()
    at = torch.where(live, beam * V + word, 0)
    mine = flat.gather(1, at)
    scale = torch.where(live, mine, 0).abs().clamp(min=1)
    err = 2e-6 * scale
    assert torch.where(live, (score.double() - mine).abs() <= err, True).all()
    assert all(len(set(r[:c].tolist())) == int(c) for r, c in zip(at, have))
    assert (torch.where(live, score, -torch.inf).diff(dim=1).nan_to_num(0) <= 0).all()
    # equal scores: the lower beam, then the larger logit, then the lower word
    logit = torch.where(x.isnan(), -torch.inf, x.float()).flatten(1).gather(1, at)
    for b in range(B):
        c = int(have[b])
        keys = [(-float(score[b, i]), int(beam[b, i]), -float(logit[b, i]) + 0.0, int(word[b, i])) for i in range(c)]
        assert keys == sorted(keys)
    # no better candidate was left out
    best = flat.sort(1, descending=True).values[:, :n]
    assert torch.where(live, (best - mine) <= 2 * err, True).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", [(32, 8, 50257, 16), (15, 30, 128256, 30), (64, 8, 32000, 8), (3, 256, 20011, 128)])
def test_rows_of_many_tiles(select, dtype, B, K, V, n):
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (2 * torch.randn(B, K, V, device="cuda", generator=g)).to(dtype)
    s = -5 * torch.rand(B, K, device="cuda", generator=g)
    _check(select(x, s, n), x, s, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1, 5])
def test_rows_that_keep_growing(select, dtype, off):
    """Ascending logits: every load reaches the bound, the lists are cut again and again; rows off the boundary too."""
    V, g = 40000, torch.Generator(device="cuda").manual_seed(off)
    ramp = torch.linspace(-8, 8, V, device="cuda") + 1e-3 * torch.randn(450, 1, V, device="cuda", generator=g)
    big = torch.zeros(450, 1, V + 11, device="cuda").to(dtype)
    big[..., off: off + V] = ramp.to(dtype)
    x = big[..., off: off + V]
    s = -torch.rand(450, 1, device="cuda", generator=g)
    for n in (1, 8, 128):
        _check(select(x, s, n), x, s, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_thousands_of_equal_maxima_in_later_tiles(select, dtype):
    """The lists overflow (or are cut to ties only) after a quiet start, and the row is ranked by rounds."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(460, 1, 60000, device="cuda", generator=g).clamp_(max=1.5).to(dtype)
    x[:, :, 21000:29000] = 2.0
    x[7, 0, 50000:59000] = 2.5
    x[8, 0, ::2] = 2.0
    x[9, 0, 40000:] = 3.0
    x[9, 0, 59999] = 3.5
    s = torch.zeros(460, 1, device="cuda")
    got = select(x, s, 24)
    _check(got, x, s, 24)
    first = list(range(21000, 21024))
    assert got[2][0].tolist() == first and got[2][459].tolist() == first
    assert got[2][7].tolist() == list(range(50000, 50024)) and got[2][8].tolist()[:3] == [0, 2, 4]
    assert got[2][9].tolist() == [59999] + list(range(40000, 40023))


def test_sums_are_rescaled_when_a_later_tile_is_larger(select):
    """The largest logit comes last, far above the rest, and -inf, NaN and +inf in tiles of their own."""
    x = torch.randn(450, 1, 30000, device="cuda")
    x[:, :, 29990] = 60.0
    x[1, :, :20000] = -torch.inf
    x[2, :, 5000:25000] = torch.nan
    x[3, :, 28000] = torch.inf
    x[4, :, 100] = torch.inf
    x[5] = -torch.inf
    s = torch.linspace(-3, 0, 450, device="cuda")[:, None].contiguous()
    got = select(x, s, 6)
    _check(got, x, s, 6)
    assert got[1][3].tolist() == got[1][4].tolist() == got[1][5].tolist() == [-1] * 6


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_masked_with_the_types_lowest_value(select, dtype):
    """All of a row at the lowest finite value is a uniform row; some of it at that value leaves the others' totals alone."""
    low = torch.finfo(dtype).min
    x = torch.randn(3, 4, 5000, device="cuda").to(dtype)
    x[0] = low
    x[1, :, ::2] = low
    x[2, 1:] = low
    s = -torch.rand(3, 4, device="cuda")
    _check(select(x, s, 10), x, s, 10)
    got = select(x[:1, :1].contiguous(), torch.zeros(1, 1, device="cuda"), 5)
    assert got[2].tolist() == [[0, 1, 2, 3, 4]]
    assert torch.allclose(got[0].double(), torch.full((1, 5), -np.log(5000), dtype=torch.float64, device="cuda"), rtol=2e-6)


@pytest.mark.parametrize("offset", [1e3, -3e4, 1e7])
def test_logits_with_a_large_offset(select, offset):
    """Steps of 1/4 stay exact up to 2^22; 1e7 leaves whole numbers.  The totals do not depend on the offset."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-30, 30, (2, 3, 9000), device="cuda", generator=g) * (0.25 if abs(offset) < 1e6 else 1.0)
    s = -4 * torch.rand(2, 3, device="cuda", generator=g)
    moved = (x + offset).contiguous()
    assert torch.equal((moved.double() - offset).float(), x)
    _check(select(moved, s, 12), moved, s, 12)
    for a, b in zip(select(moved, s, 12), select(x, s, 12)):
        assert torch.equal(a, b)
