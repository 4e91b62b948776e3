"""beam_select against a float64 sort of every candidate.

Candidates are ordered by total, then beam, then logit, then word.  Two totals
that differ by less than the fp32 error of theirs may come out in either order,
so chosen places are compared by total (2e-6 of max(1, |total|): a log-sum-exp
of fp32 exponentials, one subtraction and one addition) and exactly where the
totals are exact.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def select():
    from latticequant_b200.beam import beam_select

    return beam_select


def _ref(logits, scores, n):
    x = logits.double().cpu().numpy()
    s = scores.double().cpu().numpy()
    B, K, V = x.shape
    out = []
    with np.errstate(all="ignore"):
        for b in range(B):
            cand = []
            for k in range(K):
                row = np.where(np.isnan(x[b, k]), -np.inf, x[b, k])
                mx = row.max()
                lse = mx + np.log(np.exp(row - mx).sum()) if np.isfinite(mx) else np.nan
                tot = row - lse + s[b, k]
                ok = np.flatnonzero(tot > -np.inf)
                cand += [(-tot[v], k, -row[v], v) for v in ok[np.argsort(-row[ok], kind="stable")][:n]]
            cand.sort()
            cand = cand[:n] + [(np.inf, -1, 0, -1)] * (n - len(cand))
            out.append([(-c[0], c[1], c[3]) for c in cand])
    return np.array(out)  # (B, n, 3)


def _check(got, want, exact=True):
    s, k, v = (t.cpu().numpy() for t in got)
    ws = want[..., 0]
    fin = np.isfinite(ws)
    assert np.array_equal(np.isneginf(s), ~fin)
    assert (np.abs(s[fin] - ws[fin]) <= 2e-6 * np.maximum(1, np.abs(ws[fin]))).all()
    if exact:
        assert np.array_equal(k, want[..., 1]) and np.array_equal(v, want[..., 2])
    else:  # a pick may trade places with one whose total is as near as the error
        for b in range(s.shape[0]):
            near = 1e-5 * max(1, np.abs(ws[b][fin[b]]).max(initial=0))
            mine, theirs = set(zip(k[b], v[b])), set(map(tuple, want[b, :, 1:].astype(int)))
            assert all(abs(s[b, -1] - t) <= near for (kk, vv, t) in zip(k[b], v[b], s[b]) if (kk, vv) not in theirs)
            assert len(mine) == len(theirs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 97, 6), (3, 4, 8192, 8), (2, 5, 8193, 10),
                                     (1, 4, 32000, 8), (2, 16, 50257, 32), (1, 2, 128256, 128), (9, 1, 1000, 1)])
def test_matches_float64(select, dtype, B, K, V, n):
    g = torch.Generator(device="cuda").manual_seed(V + n)
    x = (3 * torch.randn(B, K, V, device="cuda", generator=g)).to(dtype)
    s = -10 * torch.rand(B, K, device="cuda", generator=g)
    _check(select(x, s, n), _ref(x, s, n), exact=False)


def test_ties_go_to_the_lower_beam_and_word(select):
    """Equal logits in every row (more than a slice's buffer holds) and equal scores."""
    for V in (40, 3000, 20000):
        x = torch.zeros(2, 3, V, device="cuda")
        s = torch.tensor([[-1.0, -1.0, -1.0], [-3.0, -1.0, -2.0]], device="cuda")
        sc, k, v = select(x, s, 12)
        assert k.tolist() == [[0] * 12, [1] * 12] and v.tolist() == [list(range(12))] * 2
    x = torch.zeros(1, 4, 16, device="cuda", dtype=torch.bfloat16)
    x[..., 9] = 1
    x[..., 3] = 1
    _, k, v = select(x, torch.zeros(1, 4, device="cuda"), 8)
    assert k[0].tolist() == [0, 0, 1, 1, 2, 2, 3, 3] and v[0].tolist() == [3, 9] * 4
    # negative and positive zero are the same logit
    x = torch.tensor([[[0.0, -0.0, 0.0]]], device="cuda")
    assert select(x, torch.zeros(1, 1, device="cuda"), 3)[2].tolist() == [[0, 1, 2]]


def test_many_equal_largest_logits(select):
    """5,000 words share the largest logit of a row: the fallback ranks by rounds."""
    x = torch.randn(2, 2, 30000, device="cuda").clamp_(max=1.0)
    x[1, 1, 7:5007] = 2.0
    s = torch.tensor([[0.0, -0.5], [-1.0, -0.5]], device="cuda")
    _check(select(x, s, 16), _ref(x, s, 16), exact=False)
    assert select(x, s, 16)[2][1].tolist() == list(range(7, 23))


def test_banned_words_dead_beams_and_nan(select):
    inf = float("inf")
    x = torch.randn(4, 3, 9000, device="cuda")
    x[0, :, 5:] = -inf                 # 5 words left a beam
    x[1, 0], x[1, 1, 4] = -inf, inf    # a row with nothing, a row with +inf
    x[2, :, ::2] = float("nan")
    x[3] = -inf
    s = torch.zeros(4, 3, device="cuda")
    s[0, 1], s[2, 0], s[2, 2] = -inf, float("nan"), -1e9
    got = select(x, s, 20)
    _check(got, _ref(x, s, 20), exact=False)
    assert got[1][0].tolist()[10:] == [-1] * 10 and got[2][3].tolist() == [-1] * 20
    assert set(got[1][1].tolist()) == {2} and set(got[1][2].tolist()) == {1}


def test_rows_off_the_16_byte_boundary_and_strides(select):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        big = torch.randn(2, 4, 8191 + 40, device="cuda").to(dtype)
        s = -torch.rand(2, 4, device="cuda")
        for off in (1, 3, 7):
            view = big[:, 1:3, off:off + 8185 + off]
            # (the slices' sums run in another order when a row starts off the boundary)
            _check(select(view, s[:, 1:3], 9), _ref(view, s[:, 1:3], 9), exact=False)
        wide = big.transpose(1, 2).contiguous().transpose(1, 2)  # words far apart
        assert all(torch.equal(p, q) for p, q in zip(select(wide, s, 5), select(big, s, 5)))


def test_refusals(select):
    x, s = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, device="cuda")
    for f in (lambda: select(x[0], s, 2), lambda: select(x, s.half(), 2), lambda: select(x, s[:, :2], 2),
              lambda: select(x, s, 0), lambda: select(x, s, 129), lambda: select(x.double(), s, 2),
              lambda: select(x[..., :0], s, 2), lambda: select(x, s.cpu(), 2)):
        with pytest.raises(ValueError):
            f()
    assert select(x[:0], s[:0], 2)[0].shape == (0, 2)
