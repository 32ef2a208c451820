"""The orthogonalised updates refuse a call before any part of it runs."""
import pytest

from spilltune_amd import _lib


def _table(*sizes):
    return (_lib.MatrixBatch * len(sizes))(*[
        _lib.MatrixBatch(x=4096, out=8192, count=n, rows=r, cols=c) for n, r, c in sizes])


def _call(*sizes):
    _lib.call("st_orthogonalize", len(sizes), _table(*sizes), 1, 5, 3.4445, -4.775, 2.0315, 1e-7, 4096,
              1 << 60, None)


MANY = ((1 << 24) - 1, 1, 1 << 20)  # more workgroups than a launch numbers


# behind matrices of the same table, of tables of another class of ranks, of more than
# one table holds
@pytest.mark.parametrize("before", [[(1, 4, 8)], [(1, 64, 100), (1, 4, 4096)], [(1, 16, 4096)] * 50,
                                    [(2, 20, 300), (0, 4, 4), (1, 200, 300)]])
def test_a_table_behind_others(before):
    with pytest.raises(ValueError, match="too many"):
        _call(*before, MANY)
    assert _lib.query("st_orthogonalize_workspace_bytes", len(before) + 1, _table(*before, MANY)) == -1
    assert _lib.query("st_orthogonalize_workspace_bytes", len(before), _table(*before)) >= 0


def test_the_query_tells_refused_sizes():
    for sizes in ((1, 1025, 1025), (1, -1, 4), (1, 4, 1 << 30), (1 << 24, 4, 4)):
        assert _lib.query("st_orthogonalize_workspace_bytes", 1, _table(sizes)) == -1


@pytest.mark.parametrize("sizes", [((1 << 22), 17, 20), ((1 << 22), 4, 2100), ((1 << 20), 33, 40)])
def test_many_small_matrices_are_taken(sizes):
    """Only the launches that are made bound the matrices of a call."""
    assert _lib.query("st_orthogonalize_workspace_bytes", 1, _table(sizes)) > 0
