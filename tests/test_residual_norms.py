"""Refusals of the norms around a block part, before any device work."""
import ctypes

import pytest
import torch

from spilltune_amd import _lib, ops

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,kw,match", [
    ((z(2, 8), z(2, 8)), {}, "on the GPU"),
    ((z(2, 8, dtype=torch.float32), z(2, 8)), {}, "bf16"),
    ((z(2, 8), z(1, 8)), {}, "one shape"),
    ((z(2, 16385), z(2, 16385)), {}, "16384"),
    ((z(2, 0), z(2, 0)), {}, "16384"),
    ((z(2, 8), z(2, 8), z(7)), {}, "post"),
    ((z(2, 8), z(2, 8), None, z(8, dtype=torch.float32)), {}, "pre"),
    ((z(2, 8), z(2, 8)), {"gate": z(8, dtype=torch.float16)}, "bf16 or fp32"),
    ((z(2, 8), z(2, 8)), {"gate": z(2)}, "a gate of"),
    ((z(2, 3, 8), z(2, 3, 8)), {"gate": z(1, 3, 8)}, "a gate of"),
    ((z(2, 3, 8), z(2, 3, 8)), {"gate": z(3, 8)}, "a gate of"),
    ((z(2, 8), z(2, 8)), {"scale": float("nan")}, "scale"),
    ((z(2, 8), z(2, 8)), {"eps": -1e-6}, "eps"),
])
def test_arguments(args, kw, match):
    with pytest.raises(ValueError, match=match):
        ops.residual_norms(*args, **kw)


def _fwd(y=4096, post=None, pre=None, gate=None, mode=0, per=4, rows=4, H=64, scale=1.0, normed=None):
    _lib.call("st_residual_norms_fwd", y, 8192, post, pre, gate, mode, 0, per, rows, H, scale, 1e-6,
              12288, normed, None, None, None)


@pytest.mark.parametrize("kw,match", [
    ({"H": 0}, "hidden"), ({"rows": -1}, "rows"), ({"H": 16385}, "16384"), ({"rows": 1 << 40}, "2\\^40"),
    ({"mode": 4}, "gate"), ({"mode": 1}, "differ"), ({"gate": 4096}, "differ"),
    ({"gate": 4096, "mode": 1, "per": 3}, "divide"), ({"gate": 4096, "mode": 1, "per": 0}, "divide"),
    ({"y": None}, "NULL"), ({"y": 4104}, "16-byte"), ({"pre": 4096}, "NULL output"),
    ({"scale": float("inf")}, "scale"),
])
def test_c_forward_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _fwd(**kw)


def _bwd(post=None, pre=None, gate=None, mode=0, per=4, rows=4, r1=None, r2=None, dn=None, dgate=None,
         dpost=None, dpre=None, ws=None, nbytes=0):
    _lib.call("st_residual_norms_bwd", 4096, 8192, post, pre, gate, mode, 0, per, rows, 64, 1.0, 1e-6,
              r1, r2, 4096, dn, 12288, 12288, dgate, dpost, dpre, ws, nbytes, None)


@pytest.mark.parametrize("kw,match", [
    ({"post": 4096}, "statistics"), ({"dn": 4096}, "statistics"),
    ({"dpost": 4096}, "not there"), ({"dpre": 4096}, "not there"), ({"dgate": 4096}, "not there"),
    ({"post": 4096, "r1": 4096, "dpost": 4096}, "workspace"),
    ({"post": 4096, "r1": 4096, "dpost": 4096, "ws": 4100, "nbytes": 1 << 30}, "aligned"),
    ({"gate": 4096, "mode": 1, "per": 1, "rows": 65534, "dgate": 4096, "ws": 4096,
      "nbytes": 1 << 40}, "65534"),
])
def test_c_backward_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _bwd(**kw)


def test_no_rows_need_no_device():
    _fwd(rows=0, y=None)
    _bwd(rows=0)
    assert _lib.query("st_residual_norms_workspace_bytes", 0, 64, 1) == 0
    assert _lib.query("st_residual_norms_workspace_bytes", 8, 64, 3) == 0
    assert _lib.query("st_residual_norms_workspace_bytes", 8, 64, 8) >= 3 * 64 * 4
