"""Refusals of the balance loss, before any device work."""
import pytest
import torch

from spilltune_amd import _lib, moe

X, I = torch.zeros(2, 3, 8), torch.zeros(2, 3, 2, dtype=torch.int32)


@pytest.mark.parametrize("args,kw,match", [
    ((X, I), {}, "on the GPU"), ((X.double(), I), {}, "logits"), ((X[0, 0], I[0, 0]), {}, "logits"),
    ((X, I.float()), {}, "indices"), ((X, I[0]), {}, "indices"), ((X, I[:, :2]), {}, "indices"),
    ((torch.zeros(2, 3, 513), I), {}, "512"), ((X, torch.zeros(2, 3, 65, dtype=torch.int32)), {}, "64"),
    ((X, I[..., :0]), {}, "64"), ((X, I), {"score": "relu"}, "score"),
    ((X, I), {"valid": torch.ones(2, 3)}, "valid"),
    ((X, I), {"valid": torch.ones(3, dtype=torch.bool)}, "valid"),
    ((X[0], I[0]), {"per_row": True}, "per_row"), ((X[:0], I[:0]), {}, "token"),
])
def test_arguments(args, kw, match):
    with pytest.raises(ValueError, match=match):
        moe.balance_loss(*args, **kw)


def _fwd(logits=4096, dtype=1, groups=1, per=4, E=8, k=2, ws=4096, nbytes=1 << 40):
    _lib.call("st_balance_fwd", logits, dtype, 4096, 0, None, groups, per, E, k, 0, 4096, 4096, 4096,
              ws, nbytes, None)


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 2}, "dtype"), ({"groups": 0}, "groups"), ({"per": 0}, "groups"), ({"E": 513}, "512"),
    ({"E": 0}, "512"), ({"k": 65}, "64"), ({"k": 0}, "64"), ({"groups": 65536}, "65536"),
    ({"per": 1 << 25}, "2\\^25"), ({"logits": None}, "NULL"), ({"ws": None}, "workspace"),
    ({"nbytes": 4}, "workspace"), ({"ws": 4098}, "aligned"),
])
def test_c_entry_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _fwd(**kw)


def test_c_backward_refuses():
    with pytest.raises(ValueError, match="NULL"):
        _lib.call("st_balance_bwd", 4096, 1, None, 1, 4, 8, 2, 0, None, 4096, 4096, 4096, None)
    with pytest.raises(ValueError, match="512"):
        _lib.call("st_balance_bwd", 4096, 1, None, 1, 4, 600, 2, 0, 4096, 4096, 4096, 4096, None)
