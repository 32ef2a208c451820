"""Refusals of the orthogonalised updates, before any device work."""
import ctypes
import math

import pytest
import torch

from spilltune_amd import _lib, muon


def test_arguments():
    x = torch.zeros(4, 5)
    assert muon.orthogonalize([]) == []
    for bad, kw, match in (
            (x, {}, "on the GPU"), ([x, x.to(torch.bfloat16)], {}, "one type"),
            (x.double(), {}, "one type"), (torch.zeros(5), {}, "one type"), ([x, None], {}, "tensors"),
            (x, {"steps": 2.0}, "integer"), (x, {"steps": True}, "integer"),
            (x.clone().requires_grad_(True), {}, "derivative")):
        with pytest.raises(ValueError, match=match):
            muon.orthogonalize(bad, **kw)
    for kw in ({"lr": math.inf}, {"momentum": 1.0}, {"momentum": -0.1}, {"weight_decay": -1.0}):
        with pytest.raises(ValueError, match="unsupported_capability"):
            muon.Muon(**kw)


def _call(shape=(4, 8), count=1, dtype=1, steps=5, abc=(3.4445, -4.775, 2.0315), eps=1e-7, x=4096,
          ws=4096, nbytes=1 << 40):
    t = (_lib.MatrixBatch * 1)(_lib.MatrixBatch(x=x, out=8192, count=count, rows=shape[0],
                                                cols=shape[1]))
    _lib.call("st_orthogonalize", 1, t, dtype, steps, *abc, eps, ctypes.c_void_p(ws), nbytes, None)


@pytest.mark.parametrize("kw,match", [
    ({"shape": (1025, 1025)}, "shorter side"), ({"shape": (-1, 4)}, "negative"),
    ({"count": -1}, "negative"), ({"shape": (4, 1 << 30)}, "2\\^30"), ({"count": 1 << 24}, "2\\^24"),
    ({"dtype": 2}, "dtype"), ({"steps": 0}, "steps"), ({"steps": 13}, "steps"),
    ({"steps": 65, "abc": (1.0, 0.0, 0.0)}, "steps"), ({"abc": (math.nan, 0.0, 0.0)}, "finite"),
    ({"eps": -1.0}, "eps"), ({"x": None}, "NULL"), ({"x": 4097}, "misaligned"),
    ({"shape": (4, 4096), "nbytes": 16}, "workspace"), ({"shape": (4, 4096), "ws": None}, "workspace"),
    ({"shape": (33, 40), "ws": None}, "workspace"),
    # 2^23 matrices of 32 chunks each: more workgroups than a launch numbers
    ({"shape": (1, 1 << 20), "count": (1 << 24) - 1, "nbytes": 1 << 60}, "too many"),
])
def test_c_entry_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _call(**kw)


def test_empty_work_needs_no_device():
    _call(shape=(0, 4))
    _call(count=0)
    _lib.call("st_orthogonalize", 0, None, 1, 5, 1.0, 0.0, 0.0, 0.0, None, 0, None)
    assert _lib.query("st_orthogonalize_workspace_bytes", 0, None) == 0


def test_workspace_of_a_larger_rank():
    def need(*shapes):
        t = (_lib.MatrixBatch * len(shapes))(*[
            _lib.MatrixBatch(x=4096, out=8192, count=1, rows=r, cols=c) for r, c in shapes])
        return _lib.query("st_orthogonalize_workspace_bytes", len(shapes), t)
    assert 0 < need((16, 4096)) < need((64, 4096)) < need((128, 4096)) < need((1024, 4096))
    # tables are used one after the other: the largest counts
    assert need((16, 4096), (1024, 4096)) == need((1024, 4096))
