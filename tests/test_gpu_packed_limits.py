"""Attention over runs of keys at the ends of its documented ranges, against
64-bit restatements (bounds: see _packed_ref.span_ref)."""
import random

import pytest
import torch

from spilltune_amd import packed
from tests._packed_ref import span_ref
from tests.test_gpu_packed import _check, _documents, _randn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("scale,cap", [(1e30, 1e27), (1e30, 1e30), (1e20, 1e16), (1e17, 1e30), (1e-30, 3.0),
                                       (1e-30, 1e-26), (1e-30, 1e30), (1e30, None), (1e-30, None)])
def test_scales_and_caps_at_their_limits(dims, scale, cap):
    """Ordinary scores of very small or large products: the capped score's
    polynomial lost them to an overflow.  Some queries are 0."""
    (DQ, DV), B, S, H, KV = dims, 1, 150, 4, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    # scale * q.k of deviation about 1.5 (or 1.5 caps, where the cap is small)
    part = (1.5 * min(1.0, cap or 1.0) / scale) ** 0.5 * DQ ** -0.25
    q, k = ((_randn(g, B, n, S, DQ) * part).to(BF) for n in (H, KV))
    q[:, :, ::7] = 0
    v, dout = _randn(g, B, KV, S, DV).to(BF), _randn(g, B, S, H * DV).to(BF)
    mask = packed.document_mask(_documents(random.Random(3), B, S, 10, 100, 6).cuda())
    want, bound = span_ref(q, k, v, scale, mask.key_start, mask.key_end, cap, None, dout)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = packed.span_attention(*leaves, scale, mask, cap=cap)
    _check((out, *torch.autograd.grad(out, leaves, dout)), want, bound)


def test_rotation_of_more_tokens_than_one_grid_dimension():
    """2^24 and more tokens (2^32 threads) in one call, against slices of it."""
    T, D = (1 << 24) + 11, 8
    g = torch.Generator(device="cuda").manual_seed(6)
    rotary = packed.Rotary(D, 1e4, device="cuda")
    y = _randn(g, T, 3 * D).to(BF).requires_grad_(True)
    pos = (torch.arange(T, device="cuda") % 4099)[None]
    ups = [_randn(g, 1, 1, T, D).to(BF) for _ in range(3)]
    got = packed.rope_positions(y, pos, rotary, 1, 1)
    (dy,) = torch.autograd.grad(got, y, ups)
    for a in (0, (1 << 22) - 5, (1 << 23) - 5, (1 << 23) + 7000, (1 << 24) - 5):
        part = slice(a, a + 16)
        x = y.detach()[part].clone().requires_grad_(True)
        want = packed.rope_positions(x, pos[:, part].contiguous(), rotary, 1, 1)
        (dx,) = torch.autograd.grad(want, x, [u[:, :, part] for u in ups])
        assert all(torch.equal(o[:, :, part], w) for o, w in zip(got, want))
        assert torch.equal(dy[part], dx)
