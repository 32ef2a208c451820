"""The workspace query gives what the backward of the norms asks for, and no less."""
import pytest

from spilltune_amd import _lib

P = 4096


def _bwd(rows, H, rows_per, columns, nbytes):
    gate = dict(gate=P, mode=_lib.ST_GATE_COLUMNS) if columns else dict(gate=None, mode=0)
    _lib.call("st_residual_norms_bwd", P, P, P, P, gate["gate"], gate["mode"], 0, rows_per, rows, H, 1.0,
              1e-6, P, P, P, P, P, P, P if columns else None, P, P, P, nbytes, None)


@pytest.mark.parametrize("H", [1, 8, 64, 512, 520, 2048, 4096, 4097, 8192, 16384])
@pytest.mark.parametrize("rows,rows_per", [(1, 1), (2, 1), (3, 3), (8, 8), (8, 2), (2103, 2103),
                                           (30000, 30000), (30000, 100), (65533 * 3, 3), (7, 7)])
def test_a_byte_less_is_refused(rows, H, rows_per):
    columns = rows_per < rows
    need = _lib.query("st_residual_norms_workspace_bytes", rows, H, rows_per)
    assert need >= rows // rows_per * 3 * H * 4
    for short in (need - 1, need // 2, 0):
        with pytest.raises(ValueError, match=f"needs {need} workspace"):
            _bwd(rows, H, rows_per, columns, short)
