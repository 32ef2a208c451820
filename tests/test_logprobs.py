"""Token log probabilities on the CPU: refusals before any device work."""
import ctypes
import math

import pytest
import torch

from spilltune_amd import _lib, ops

BF = torch.bfloat16


def test_token_logprobs_refuses():
    h, w, t = torch.zeros(2, 3, 16, dtype=BF), torch.zeros(40, 16, dtype=BF), torch.zeros(2, 3).long()
    f = ops.token_logprobs
    for a, b in ((h.float(), w), (h, w.float()), (h, w[0]), (h[..., :8], w)):
        with pytest.raises(ValueError, match="expects bf16"):
            f(a, b, t)
    with pytest.raises(ValueError, match="frozen"):
        f(h, w.clone().requires_grad_(True), t)
    with pytest.raises(ValueError, match="multiples of 8"):
        f(h[..., :12].contiguous(), w[:, :12].contiguous(), t)
    for bad in (t.int(), t[:1], t[0]):
        with pytest.raises(ValueError, match="tokens must be int64"):
            f(h, w, bad)
    for top in (-1, 65, 2.0, True):
        with pytest.raises(ValueError, match="top must be"):
            f(h, w, t, top=top)
    with pytest.raises(ValueError, match="top must be 0..5"):
        f(h, w[:5], t, top=6)
    for kw in ({"temperature": 0.0}, {"temperature": -1.0}, {"temperature": math.nan}, {"cap": -1.0},
               {"cap": math.inf}):
        with pytest.raises(ValueError, match="temperature must be positive"):
            f(h, w, t, **kw)
    with pytest.raises(ValueError, match="GPU"):
        f(h, w, t)


def test_abi_refuses_before_the_device():
    p, n = ctypes.c_void_p(16), ctypes.c_void_p(None)

    def fwd(rows=4, H=16, V=40, ldh=16, ldw=16, T=1.0, cap=0.0, top=0, hidden=p, ws=p, wb=1 << 40,
            lp=p, tt=p):
        _lib.call("st_token_logprobs_fwd", hidden, rows, H, ldh, p, V, ldw, p, -100, T, cap, top, lp, p,
                  p, p, tt, None, ws, wb, None)
    for kw, msg in (({"H": 12}, "16-byte"), ({"ldw": 8}, "16-byte"), ({"ldh": 20}, "16-byte"),
                    ({"T": 0.0}, "temperature"), ({"cap": -1.0}, "cap"), ({"top": 41}, "within"),
                    ({"V": 400, "top": 65}, "too large"), ({"V": 1 << 23}, "too large"),
                    ({"V": (1 << 20) + 1, "top": 1}, "too large"), ({"hidden": n}, "NULL"),
                    ({"hidden": ctypes.c_void_p(8)}, "unaligned"), ({"lp": n}, "NULL"),
                    ({"tt": n, "top": 2}, "NULL"), ({"wb": 10}, "workspace"), ({"ws": n}, "workspace")):
        with pytest.raises(ValueError, match=msg):
            fwd(**kw)
    fwd(rows=0)

    def bwd(ldd=16, dh=p, wb=1 << 40):
        _lib.call("st_token_logprobs_bwd", p, 4, 16, 16, p, 40, 16, p, -100, 1.0, 0.0, 0, p, p, p, n, n,
                  n, p, n, n, dh, ldd, p, wb, None)
    for kw, msg in (({"ldd": 8}, "NULL or"), ({"dh": n}, "NULL"), ({"wb": 10}, "workspace")):
        with pytest.raises(ValueError, match=msg):
            bwd(**kw)
    q = lambda *a: _lib.query("st_token_logprobs_workspace_bytes", *a)  # noqa: E731
    assert q(0, 16, 40, 16, 0, 0, 0) == 0 and q(4, 16, 40, 8, 0, 0, 0) == 0
    assert q(1000, 64, 5000, 64, 5, 0, 0) - q(1000, 64, 5000, 64, 0, 0, 0) == 1000 * 5000 * 4
    assert q(1000, 64, 5000, 64, 5, 1, 0) == q(1000, 64, 5000, 64, 0, 0, 0)
    assert q(1000, 64, 5000, 64, 0, 0, 1) >= 1000 * 5000 * 2


def test_abi_refuses_numbers_and_sizes_out_of_range():
    """Temperatures and caps whose reciprocals leave fp32; a vocabulary whose
    gradient rows leave 32-bit offsets."""
    p = ctypes.c_void_p(16)

    def fwd(V=40, T=1.0, cap=0.0):
        _lib.call("st_token_logprobs_fwd", p, 4, 16, 16, p, V, 16, p, -100, T, cap, 0, p, p, p, p, p,
                  None, p, 1 << 40, None)
    for kw in ({"T": 1e-31}, {"T": 1e31}, {"cap": 1e-31}, {"cap": 1e31}):
        with pytest.raises(ValueError, match="out of range"):
            fwd(**kw)
    with pytest.raises(ValueError, match="too large"):
        fwd(V=(1 << 21) + 1)


def test_row_chunks_stay_within_a_call():
    for rows, per in ((5, 1 << 40), (1 << 24, 21), (100000, 1 << 20)):
        chunks = ops._row_chunks(rows, per)
        assert chunks[0][0] == 0 and chunks[-1][1] == rows
        assert all(0 < z - a <= 1 << 22 for a, z in chunks)
        assert all(z == a for (_, z), (a, _) in zip(chunks, chunks[1:]))


@pytest.mark.parametrize("rows,H,V", [(100000, 8192, 512), (1 << 20, 16384, 32), (3000, 4096, 151936), (7, 64, 40),
                                      (200, 16384, 200000)])
def test_backward_scratch_counts_the_partial_sums(rows, H, V):
    """A small vocabulary under a wide model: the fp32 partial sums are the larger
    part of the backward's scratch."""
    def need(n):
        return _lib.query("st_token_logprobs_workspace_bytes", n, H, V, H, 0, 0, 1)
    chunks = ops._scratch_chunks(rows, 2 * V, need)
    assert chunks[0][0] == 0 and chunks[-1][1] == rows
    assert all(z == a for (_, z, _), (a, _, _) in zip(chunks, chunks[1:]))
    for a, z, nbytes in chunks:
        assert nbytes == need(z - a) and (nbytes <= ops.LOGPROB_SCRATCH or z - a <= 256)
    assert not ops._scratch_chunks(0, 2 * V, need)
    # no more ranges than they take
    assert len(chunks) == 1 or need(2 * (chunks[0][1] + 256)) > ops.LOGPROB_SCRATCH
