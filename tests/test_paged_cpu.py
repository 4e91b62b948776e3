"""The paged cache's and beam selection's C entry points without a GPU: arguments
are refused before anything is launched, and the workspace sizes add up."""
import pytest

OK, INVALID, CAPACITY = 0, -1, -3
PTR = 4096  # aligned and never dereferenced: every call below is refused or has nothing to do


@pytest.fixture(scope="module")
def lib():
    from latticequant_b200 import _lib

    return _lib.lib()


def _attention(lib, **kw):
    a = dict(q=PTR, dtype=1, sb=64, sh=64, st=64, codes=PTR, scales=PTR, n_pages=4, page=16, table=PTR, width=4, stride=4,
             lens=PTR, max_len=64, mask=None, mask_stride=0, batch=1, heads=1, group=1, n_query=1, dim=64, scale=1.0,
             out=PTR, lse=None, ws=None, ws_bytes=0, err=None, stream=None)
    a.update(kw)
    return lib.lq_paged_attention(*a.values())


def test_attention_refusals(lib):
    for bad in (dict(q=None), dict(codes=None), dict(scales=None), dict(table=None), dict(lens=None), dict(out=None),
                dict(dtype=0), dict(dtype=7), dict(sb=65), dict(sh=4), dict(st=1), dict(q=PTR + 2), dict(codes=PTR + 4),
                dict(scales=PTR + 4), dict(page=48), dict(page=8), dict(page=512), dict(n_pages=0), dict(dim=96),
                dict(group=0), dict(group=65), dict(n_query=0), dict(n_query=4097), dict(heads=0), dict(batch=-1),
                dict(batch=65536), dict(max_len=-1), dict(width=-1), dict(width=(1 << 20) + 1)):
        assert _attention(lib, **bad) == INVALID, bad
    assert _attention(lib, batch=0) == OK
    # long contexts need a workspace: missing, misaligned, too small
    long = dict(max_len=1 << 20, width=1 << 16, stride=1 << 16)
    need = lib.lq_paged_attention_workspace(1, 1, 1, 1, 64, 1 << 20)
    assert need > 0
    assert _attention(lib, **long) == INVALID
    assert _attention(lib, ws=PTR + 8, ws_bytes=need, **long) == INVALID
    assert _attention(lib, ws=PTR, ws_bytes=need - 1, **long) == CAPACITY


def test_attention_workspace(lib):
    f = lib.lq_paged_attention_workspace
    assert f(1, 8, 4, 1, 128, 777) == 0          # a cluster joins its splits
    assert f(512, 8, 4, 16, 128, 4096) == 0      # enough sequences: no split
    assert f(1, 8, 4, 1, 128, 100000) % (8 * 4 * (128 + 4) * 4) == 0
    assert f(1, 8, 4, 1, 96, 100000) == 0        # no such shape


def test_append_refusals(lib):
    def call(**kw):
        a = dict(k=PTR, v=PTR, dtype=2, n=4, heads=2, dim=64, kn=128, kh=64, vn=128, vh=64, slots=PTR, pages=4, page=16,
                 codes=PTR, scales=PTR, ko=None, vo=None, err=None, stream=None)
        a.update(kw)
        return lib.lq_paged_append(*a.values())

    for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(codes=None), dict(scales=None), dict(dtype=3), dict(n=-1),
                dict(heads=0), dict(dim=32), dict(kn=129), dict(vh=4), dict(k=PTR + 8), dict(vo=PTR + 4), dict(page=17),
                dict(pages=-1), dict(n=1 << 30)):
        assert call(**bad) == INVALID, bad
    assert call(n=0) == OK


def test_page_operation_refusals(lib):
    def fork(**kw):
        a = dict(table=PTR, rows=2, width=4, lens=PTR, refs=PTR, parents=PTR, n=2, reserve=0, nt=PTR, nl=PTR, nr=PTR,
                 codes=PTR, scales=PTR, layers=1, pages=8, heads=1, page=16, dim=64, ws=PTR, ws_bytes=1 << 20, err=None,
                 stream=None)
        a.update(kw)
        return lib.lq_pages_fork(*a.values())

    for bad in (dict(table=None), dict(refs=None), dict(nr=None), dict(nt=None), dict(parents=None), dict(codes=None),
                dict(ws=None), dict(width=0), dict(width=(1 << 20) + 1), dict(reserve=-1), dict(layers=0),
                dict(layers=65535), dict(pages=0), dict(page=24), dict(dim=8), dict(codes=PTR + 4), dict(rows=-1)):
        assert fork(**bad) == INVALID, bad
    assert fork(ws_bytes=4 * (2 + 2 + 8) - 1) == CAPACITY
    assert lib.lq_pages_fork_workspace(2, 2, 8) == 4 * (2 + 2 + 8)
    assert lib.lq_pages_compact_workspace(8) == 12 * 8 + 4
    compact = [PTR, 8, PTR, PTR, PTR, PTR, PTR, PTR, 1, 8, 1, 16, 64, PTR, 1 << 20, None, None]
    for i, v in ((0, None), (1, -1), (2, None), (5, None), (8, 0), (11, 40), (13, None)):
        assert lib.lq_pages_compact(*compact[:i], v, *compact[i + 1:]) == INVALID, i
    assert lib.lq_pages_compact(*compact[:14], 12 * 8 + 3, *compact[15:]) == CAPACITY
    copy = [PTR, PTR, PTR, 3, PTR, PTR, 1, 8, 1, 16, 64, None, None]
    for i, v in ((0, None), (2, None), (3, -1), (4, None), (10, 65)):
        assert lib.lq_pages_copy(*copy[:i], v, *copy[i + 1:]) == INVALID, i
    assert lib.lq_pages_copy(*copy[:3], 0, *copy[4:]) == OK
    accept = [PTR, 2, 4, PTR, 5, PTR, 3, PTR, PTR, PTR, 1, 8, 1, 16, 64, None, None]
    for i, v in ((0, None), (2, 0), (3, None), (4, 0), (4, 4097), (5, None), (6, -1), (7, None), (13, 15)):
        assert lib.lq_pages_accept(*accept[:i], v, *accept[i + 1:]) == INVALID, i
    assert lib.lq_pages_accept(PTR, 0, *accept[2:]) == OK


def test_beam_refusals(lib):
    a = [PTR, 0, 2, 3, 100, 300, 100, PTR, 4, PTR, PTR, PTR, PTR, 1 << 20, None]
    for i, v in ((0, None), (1, 5), (2, -1), (3, 0), (3, 257), (4, 0), (4, (1 << 24) + 1), (7, None), (8, 0), (8, 129),
                 (9, None), (12, None)):
        assert lib.lq_beam_select(*a[:i], v, *a[i + 1:]) == INVALID, i
    need = lib.lq_beam_select_workspace(0, 2, 3, 100, 4)
    assert need > 0 and lib.lq_beam_select(*a[:13], need - 1, None) == CAPACITY
    assert lib.lq_beam_select(*a[:2], 0, *a[3:]) == OK
    assert lib.lq_beam_select_workspace(0, 2, 3, 0, 4) == 0


def test_python_refuses_cpu_tensors():
    import torch

    from latticequant_b200 import beam, paged

    codes = torch.zeros(2, 2, 1, 16, 8, dtype=torch.int32)
    with pytest.raises((ValueError, RuntimeError)):
        paged.append(codes, torch.ones(2, 2, 1, 16), torch.zeros(1, 1, 64), torch.zeros(1, 1, 64),
                     torch.zeros(1, dtype=torch.int64))
    with pytest.raises((ValueError, RuntimeError)):
        beam.beam_select(torch.zeros(1, 1, 4), torch.zeros(1, 1), 1)


def test_error_flag_text():
    from latticequant_b200 import _lib

    with pytest.raises(_lib.LatticeQuantError, match="page pool"):
        _lib.raise_flags(_lib.EF_PAGE, "x")
