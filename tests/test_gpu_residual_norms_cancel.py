"""Norms around a part where the residual and what is added nearly cancel: the backward's
h is the forward's to the bit, so that a row's h and its norm fit together."""
import pytest
import torch

from spilltune_amd import ops

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("learn", [False, True])
def test_rows_of_one_value(gated, learn):
    """H = 1, no norm after the part: with u = dnormed pre and h = residual + scale gate y,
    d h = u r (1 - h^2 r^2), r = (h^2 + eps)^-1/2, is u eps r^3: a difference of two
    numbers that are equal but for eps.  In fp32 each is rounded a few times, at most
    2^-24 of u r a time (below eight steps); h is off by half a step of the residual and of
    the product, which moves u eps r^3 by at most 3 |off| r of itself."""
    g = torch.Generator().manual_seed(12)
    M = 40000
    y = torch.randn(M, 1, generator=g).to(BF).cuda()
    gate = (0.5 + 0.4 * torch.randn(M, 1, generator=g)).cuda() if gated else None
    scale = 0.7
    added = scale * y.double() * (gate.double() if gated else 1)
    res = (-added.cpu() * (1 + 0.02 * torch.randn(M, 1, generator=g))).to(BF).cuda()
    pre = torch.tensor([1.25], dtype=BF, device="cuda").requires_grad_(learn)
    dn = torch.randn(M, 1, generator=g).to(BF).cuda()
    leaf = res.clone().requires_grad_(True)
    leaves = [leaf] + ([gate.requires_grad_(True)] if gated else []) + ([pre] if learn else [])
    _, normed = ops.residual_norms(y, leaf, None, pre, gate=gate, scale=scale, eps=EPS)
    got = torch.autograd.grad(normed, leaves, dn)
    # fp32's scale is what the kernel multiplies by
    added = torch.tensor(scale, dtype=F32).double().cuda() * y.double() * (
        gate.detach().double() if gated else 1)
    h = res.double() + added
    r = (h * h + EPS).rsqrt()
    u = dn.double() * 1.25
    want = u * EPS * r**3
    off = 2**-24 * 2 * (res.double().abs() + added.abs())
    room = 2**-21 * (u * r).abs() + 4 * want.abs() * off * r
    assert ((got[0].double() - want).abs() <= 2**-8 * want.abs() + room).all()
    if gated:
        by = (scale * y.double()).abs()
        ref = scale * y.double() * want
        assert ((got[1].double() - ref).abs() <= 2**-22 * ref.abs() + by * room * (1 + 2**-20)).all()


@pytest.mark.parametrize("H", [2, 8, 40, 520, 2056, 4104, 8200])
def test_exact_cancellation(H):
    """h = residual + scale gate y is 0 but for its rounding, which eps = 0 would show: with
    products that fp32 holds, it is 0 in both directions and the norm's gradients too."""
    g = torch.Generator().manual_seed(H)
    y = torch.randint(-8, 9, (30, H), generator=g).to(BF).cuda()
    res = -0.5 * y
    res[:, 0] += 1  # not a row of zeros
    leaf, dn = res.clone().requires_grad_(True), torch.randn(30, H, generator=g).to(BF).cuda()
    h, normed = ops.residual_norms(y, leaf, None, torch.ones(H, dtype=BF, device="cuda"), scale=0.5,
                                   eps=0.0)
    (d,) = torch.autograd.grad(normed, [leaf], dn)
    one = torch.zeros(30, H, dtype=F64, device="cuda")
    one[:, 0] = 1
    assert torch.equal(h.double(), one)
    root = H**0.5
    want = root * dn.double() * (1 - one)
    assert ((d.double() - want).abs() <= 2**-8 * want.abs() + 2**-20 * root * dn.double().abs()).all()
