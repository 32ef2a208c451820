"""Refusals of the embedding, before any device work."""
import pytest
import torch

from spilltune_amd import _lib, ops
from spilltune_amd.embedding import TokenEmbedding

IDS = torch.tensor([0, 1])


@pytest.mark.parametrize("args,kw,match", [
    ((torch.zeros(4, 8), IDS), {}, "on the GPU"),
    ((torch.zeros(4, 8).double(), IDS), {}, "table"), ((torch.zeros(8), IDS), {}, "table"),
    ((torch.zeros(0, 8), IDS), {}, "table"), ((torch.zeros(4, 8), IDS.float()), {}, "int64"),
    ((torch.zeros(4, 8), IDS), {"scale": float("inf")}, "scale"),
    ((torch.zeros(4, 8), IDS), {"padding_idx": 4}, "padding_idx"),
    ((torch.zeros(4, 8), IDS), {"padding_idx": -1}, "padding_idx"),
    ((torch.zeros(4, 8), IDS), {"padding_idx": True}, "padding_idx"),
])
def test_arguments(args, kw, match):
    with pytest.raises(ValueError, match=match):
        ops.embedding(*args, **kw)


def test_token_embedding_refuses():
    with pytest.raises(ValueError, match="table"):
        TokenEmbedding(torch.zeros(8), device="cpu")
    with pytest.raises(ValueError, match="table"):
        TokenEmbedding(torch.zeros(4, 8, dtype=torch.int32), device="cpu")
    with pytest.raises(ValueError, match="on the GPU"):
        TokenEmbedding(torch.zeros(4, 8), device="cpu")


def _fwd(table=4096, dtype=1, ids=4096, n=4, V=8, H=16):
    _lib.call("st_embedding_fwd", table, dtype, ids, 0, n, V, H, 1.0, 8192, None)


def _bwd(dout=4096, n=4, V=8, H=16, grad=8192, dtype=1, accumulate=0, ws=4096, nbytes=1 << 40):
    _lib.call("st_embedding_bwd", dout, 4096, 0, n, V, H, 1.0, -1, grad, dtype, accumulate, ws, nbytes,
              None)


@pytest.mark.parametrize("call,kw,match", [
    (_fwd, {"dtype": 3}, "dtype"), (_fwd, {"table": None}, "NULL"), (_fwd, {"n": -1}, "tokens"),
    (_fwd, {"V": 0}, "table"), (_fwd, {"H": 0}, "table"), (_fwd, {"n": 1 << 31}, "2\\^31"),
    (_fwd, {"V": 1 << 31}, "2\\^31"), (_fwd, {"H": 1 << 24}, "2\\^31"),
    (_bwd, {"dtype": 2}, "dtype"), (_bwd, {"dtype": 0, "accumulate": 1}, "fp32"),
    (_bwd, {"grad": None}, "gradient"), (_bwd, {"grad": 8196}, "misaligned"),
    (_bwd, {"dout": None}, "NULL"), (_bwd, {"ws": None}, "workspace"),
    (_bwd, {"nbytes": 8}, "workspace"), (_bwd, {"ws": 4100}, "aligned"),
    (_bwd, {"n": (1 << 31) - 1, "H": 1 << 20, "nbytes": 1 << 62}, "launch"),
])
def test_c_entries_refuse(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


def test_no_tokens_need_no_device():
    _fwd(n=0, table=None)
    assert _lib.query("st_embedding_bwd_workspace_bytes", 0, 8, 16) == 0
    assert _lib.query("st_embedding_bwd_workspace_bytes", 5, 8, 16) > 0
