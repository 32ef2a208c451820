"""Masks and positions of one size are not one and the same."""
import torch

from spilltune_amd import packed


def test_masks_and_positions_are_equal_to_themselves_alone():
    a, b = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, 4, dtype=torch.int32)
    x, y = packed.SpanMask(1, 4, a, a, a, a), packed.SpanMask(1, 4, b, b, b, b)
    assert x == x and x != y and len({x, y}) == 2
    r, s = (packed.Rotary(64, t, device="cpu") for t in (1e4, 1e6))
    p, q, t = packed.Positions(a, r), packed.Positions(b, r), packed.Positions(a, s)
    assert p == p and p != q and p != t and len({p, q, t}) == 3
