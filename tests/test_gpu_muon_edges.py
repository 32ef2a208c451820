"""Orthogonalised updates where the formula has no number of its own, and calls that
are refused before anything is written."""
import pytest
import torch

from spilltune_amd import muon
from tests.test_gpu_muon import check, make

pytestmark = pytest.mark.gpu


# one for each form: registers, one wave's steps, LDS, one launch a step, tiles
@pytest.mark.parametrize("shape", [(4, 64), (1, 1), (16, 4096), (4096, 16), (20, 300), (300, 31),
                                   (40, 300), (300, 100), (200, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zero_matrix_without_eps(shape, dtype):
    """U = 0 stays 0 also with eps = 0, and its neighbours are what they are by themselves."""
    u = torch.stack([make(shape, k, dtype) for k in range(3)])
    u[1] = 0
    out = muon.orthogonalize(u, eps=0.0)
    assert (out[1] == 0).all()
    for k in (0, 2):
        check(out[k], u[k], eps=0.0)
        assert torch.equal(out[k], muon.orthogonalize(u[k].clone(), eps=0.0))
    u[2].view(-1)[-1] = float("nan")
    out = muon.orthogonalize(u, eps=0.0)
    assert (out[1] == 0).all() and out[2].isnan().all() and not out[0].isnan().any()


def test_more_matrices_than_another_rank_could_have():
    """2^21 and a few matrices of rank 17: bounded by the launches they take, whose
    workgroups are one a matrix (matrices of rank 33 take eight)."""
    n = (1 << 21) + 5
    u = torch.zeros(n, 17, 18, device="cuda")
    for at in (0, 1 << 20, n - 3):
        u[at:at + 3] = make((3, 17, 18), at % 100)
    out = muon.orthogonalize(u)
    for at in (0, 1 << 20, n - 3):
        check(out[at:at + 3], u[at:at + 3])
    assert (out[3:1 << 20] == 0).all() and (out[(1 << 20) + 3:n - 3] == 0).all()
    del u, out
    torch.cuda.empty_cache()
