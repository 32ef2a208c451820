"""Calls whose launches would not fit a grid are refused on the host, before any
kernel (fake pointers never reach one)."""
import ctypes

import pytest

from spilltune_amd import _lib

P, BIG = ctypes.c_void_p(1 << 20), 1 << 62


def test_plans_and_attention():
    for B, S in ((1 << 13, 1 << 20), ((1 << 24) - 1, 1 << 11)):  # blocks of 32; tiles of 128
        with pytest.raises(ValueError, match="too large a launch"):
            _lib.call("st_span_plan", P, P, B, S, P, BIG, None)
    for B, S, H in ((1 << 20, 1, 16), (1 << 14, 128 * 256, 4)):
        with pytest.raises(ValueError, match="too large a launch"):
            _lib.call("st_span_attn_fwd", P, P, P, B, S, H, H, 64, 64, 1.0, 0.0, None, P, P, P, P, P, None)
    for B, S, H, KV in ((1 << 20, 1, 16, 16), (1 << 19, 1, 16, 16), (1, 1 << 20, 1024, 1)):
        with pytest.raises(ValueError, match="too large a launch"):
            _lib.call("st_span_attn_bwd", P, P, P, P, P, P, B, S, H, KV, 64, 64, 1.0, 0.0, None, P, P, P,
                      P, P, P, P, BIG, None)


def test_token_logprobs():
    def fwd(rows, V):
        _lib.call("st_token_logprobs_fwd", P, rows, 16, 16, P, V, 16, P, -100, 1.0, 0.0, 0, P, P, P, P, P,
                  None, P, BIG, None)

    def bwd(rows, V, H=16, logits=None):
        _lib.call("st_token_logprobs_bwd", P, rows, H, H, P, V, H, P, -100, 1.0, 0.0, 0, P, P, P, P, P,
                  logits, P, P, P, P, H, P, BIG, None)
    for rows, V in ((1 << 22, 1 << 21), (1 << 22, 1 << 18)):
        with pytest.raises(ValueError, match="too many tiles"):
            fwd(rows, V)
        with pytest.raises(ValueError, match="too many tiles"):
            bwd(rows, V)
    with pytest.raises(ValueError, match="too many tiles"):  # of the hidden states' gradient
        bwd(1 << 22, 1 << 10, H=1 << 20, logits=P)
