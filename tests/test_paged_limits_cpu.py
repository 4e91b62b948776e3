"""What the paged cache's C entry points have to refuse, or to size, before anything is launched (no GPU)."""
import pytest

INVALID, CAPACITY = -1, -3
PTR = 4096  # aligned and never dereferenced: every call below is refused


@pytest.fixture(scope="module")
def lib():
    from latticequant_b200 import _lib

    return _lib.lib()


@pytest.mark.parametrize("dim,bytes_", [(64, 4), (128, 8)])
def test_attention_refuses_outputs_that_its_stores_cannot_take(lib, dim, bytes_):
    """A lane stores head_dim / 32 elements of 16 bits at once."""
    for off in range(1, bytes_):
        assert lib.lq_paged_attention(PTR, 1, dim, dim, dim, PTR, PTR, 4, 16, PTR, 4, 4, PTR, 64, None, 0, 1, 1, 1, 1, dim,
                                      1.0, PTR + off, None, None, 0, None, None) == INVALID


def test_page_operations_refuse_misaligned_workspaces(lib):
    """The workspaces hold 32-bit words."""
    for off in (1, 2, 3):
        assert lib.lq_pages_fork(PTR, 2, 4, PTR, PTR, PTR, 2, 0, PTR, PTR, PTR, PTR, PTR, 1, 8, 1, 16, 64, PTR + off, 1 << 20,
                                 None, None) == INVALID
        assert lib.lq_pages_compact(PTR, 8, PTR, PTR, PTR, PTR, PTR, PTR, 1, 8, 1, 16, 64, PTR + off, 1 << 20, None,
                                    None) == INVALID


def test_accept_with_counts_refusals(lib):
    a = [PTR, 2, 4, PTR, PTR, 5, PTR, 3, PTR, PTR, PTR, 1, 8, 1, 16, 64, None, None]
    for i, v in ((0, None), (2, 0), (3, None), (4, None), (5, 0), (5, 4097), (6, None), (7, -1), (8, None), (14, 15)):
        assert lib.lq_pages_accept_shared(*a[:i], v, *a[i + 1:]) == INVALID, i
    assert lib.lq_pages_accept_shared(PTR, 0, *a[2:]) == 0


@pytest.mark.parametrize("batch,heads,group,n_query,dim", [
    (16, 8, 4, 13, 128), (32, 8, 4, 1, 128), (1, 8, 4, 1, 128), (1, 1, 1, 1, 64), (4, 4, 7, 64, 128), (8, 4, 8, 31, 64),
    (3, 2, 5, 3, 64), (1, 4, 7, 2048, 128), (75, 8, 4, 4, 128)])
def test_attention_workspace_is_enough_for_fewer_tokens(lib, batch, heads, group, n_query, dim):
    f = lib.lq_paged_attention_workspace
    lengths = sorted({1, 2, 63, 64, 65, 2048, 2049, 2752, 2944, 11200, 11328, 1 << 20, 1 << 28,
                      *range(0, 40000, 97)})
    sizes = [f(batch, heads, group, n_query, dim, n) for n in lengths]
    assert sizes == sorted(sizes)
