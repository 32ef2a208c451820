"""Operators without a forward-mode derivative refuse dual tensors instead of
dropping their tangents (refused on the host, before any device work)."""
import pytest
import torch
from torch.autograd import forward_ad

from spilltune_amd import ops, packed

BF = torch.bfloat16


def _calls():
    q, z = torch.zeros(1, 2, 4, 64, dtype=BF), torch.zeros(1, 4, dtype=torch.int32)
    mask = packed.SpanMask(1, 4, z, z, z, z)  # no plan is read before the checks
    slopes = torch.zeros(2)
    spans = lambda q, k, v, s: packed.span_attention(q, k, v, 1.0, mask, slopes=s)  # noqa: E731
    rotary, pos = packed.Rotary(64, 1e4, device="cpu"), torch.zeros(2, 3, dtype=torch.int32)
    y, w = torch.zeros(6, 256, dtype=BF), torch.ones(64, dtype=BF)
    turn = lambda y, a, b: packed.rope_positions(y, pos, rotary, 2, 1, norms=(a, b))  # noqa: E731
    h, head, t = torch.zeros(2, 16, dtype=BF), torch.zeros(40, 16, dtype=BF), torch.zeros(2).long()
    return {"spans": (spans, [q, q, q, slopes]), "turn": (turn, [y, w, w]),
            "logprobs": (lambda h, w: ops.token_logprobs(h, w, t), [h, head])}


@pytest.mark.parametrize("name", ["spans", "turn", "logprobs"])
def test_dual_tensors_are_refused(name):
    call, tensors = _calls()[name]
    with forward_ad.dual_level():
        for i, t in enumerate(tensors):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            args = tensors[:i] + [dual] + tensors[i + 1:]
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError,
                                                                 match="forward-mode"):
                    call(*args)
        with pytest.raises(ValueError, match="GPU"):  # no tangent: as outside the level
            call(*tensors)
    with pytest.raises(ValueError, match="GPU"):
        call(*tensors)
