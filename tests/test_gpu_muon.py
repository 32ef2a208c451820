"""Orthogonalised updates against the formula in 64 bits, and the optimizer on them."""
import math

import pytest
import torch

from spilltune_amd import engine, lora, moe, muon

pytestmark = pytest.mark.gpu

ABC = muon.COEFFICIENTS


def formula(u, steps=5, abc=ABC, eps=1e-7):
    a, b, c = abc
    x = u.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def check(out, u, **kw):
    """Rounded once: half a step of the type, and what 64 bits leave: 2^-53 of the
    largest, times 1e3 terms of a sum, times the steps' growth of at most 1e5 here."""
    ref = formula(u, **kw)
    assert out.shape == u.shape and out.dtype == u.dtype
    if not ref.numel():
        return
    bound = torch.finfo(u.dtype).eps / 2 * ref.abs() + 1.2e-8 * ref.abs().max()
    if u.dtype == torch.float32:  # values near the smallest normal keep fewer bits
        bound = bound + 1e-38
    worst = ((out.double() - ref).abs() - bound).max()
    assert worst <= 0, float(worst)


def make(shape, seed=0, dtype=torch.float32, fall=30.0):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(*shape, generator=g)
    r = min(shape[-2:])
    d = torch.logspace(0, -math.log10(fall), r)
    return (1e-3 * u * (d[:, None] if shape[-2] == r else d)).to(dtype).cuda()


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 3), (4, 256), (688, 4), (5, 301), (301, 5), (16, 4096),
          (4096, 16), (15, 1000), (1023, 17), (17, 33), (32, 2103), (2103, 32), (33, 130), (130, 47),
          (64, 64), (64, 1025), (999, 64), (65, 65), (65, 300), (301, 66), (100, 2049), (128, 4096),
          (4096, 128), (130, 129), (200, 201), (257, 300), (2, 70001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    u = make(shape, sum(shape), dtype)
    check(muon.orthogonalize(u), u)


def test_shorter_side_of_1024():
    u = make((1024, 1030), 3)
    check(muon.orthogonalize(u, steps=3), u, steps=3)


@pytest.mark.parametrize("steps,abc", [(1, ABC), (2, ABC), (7, ABC), (12, ABC),
                                       (20, (1.875, -1.25, 0.375)), (3, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize("shape", [(16, 500), (500, 40), (70, 90)])
def test_steps_and_coefficients(shape, steps, abc):
    u = make(shape, 5, fall=3.0)
    check(muon.orthogonalize(u, steps=steps, coefficients=abc), u, steps=steps, abc=abc)


def test_classical_steps_reach_an_orthogonal_matrix():
    """(15, -10, 3) / 8 converges to the polar factor: XX' = 1 to 32 bits."""
    x = muon.orthogonalize(make((24, 700), 9, fall=4.0), steps=16, coefficients=(1.875, -1.25, 0.375))
    g = x.double() @ x.double().mT
    assert (g - torch.eye(24, device=g.device)).abs().max() < 1e-5


def test_many_matrices_of_many_shapes_in_one_call():
    """More matrices than a launch's table holds, classes mixed, empty ones among them."""
    shapes = [SHAPES[i % len(SHAPES)] for i in range(75)] + [(0, 5), (5, 0), (0, 3, 4)]
    shapes += [(3, 8, 100), (2, 3, 60, 6), (4, 70, 80)]
    us = [make(s, i) if 0 not in s else torch.empty(s, device="cuda") for i, s in enumerate(shapes)]
    kept = [u.clone() for u in us]
    out = muon.orthogonalize(us)
    for u, k, o in zip(us, kept, out):
        assert torch.equal(u, k)
        check(o, u)
    # the matrices of a batch do not know of each other
    assert all(torch.equal(a, b) for a, b in zip(muon.orthogonalize(us), out))


@pytest.mark.parametrize("shapes", [
    [(70, 40, 300), (5, 700, 64), (64, 33), (2, 48, 4097)],       # short sides of one block
    [(3, 128, 5000), (90, 200, 72), (100, 131), (5000, 96), (7, 127, 1001)],  # of two
    [(2, 200, 3000), (3000, 150), (5, 129, 260), (193, 194)],     # of more
    [(700, 64, 65), (4, 64, 2000)]])                              # more units than workgroups
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shares_that_end_inside_matrices(shapes, dtype):
    us = [make(s, i, dtype) for i, s in enumerate(shapes)]
    for u, o in zip(us, muon.orthogonalize(us)):
        check(o, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("r", [1, 3, 12, 16])
def test_matrices_held_whole(r, dtype):
    """Long sides that eight, four, two and one wave hold, one more, and odd counts of them;
    with a longer one in the call, none is."""
    us = [make((3 + K % 7, *((r, K) if K % 3 else (K, r))), K, dtype)
          for K in (16, 64, 65, 255, 256, 257, 511, 512, 516, 1023, 1024, 1025, 2044, 2047, 2048)]
    for group in (us, us + [make((r, 2049), 1, dtype)]):
        for u, o in zip(group, muon.orthogonalize(group)):
            check(o, u)


@pytest.mark.parametrize("shape", [(3, 7, 600), (3, 300, 12), (3, 40, 300), (3, 300, 72), (3, 100, 1000), (3, 150, 400)])
def test_one_matrix_that_is_not_finite_among_others(shape):
    """Also in the last row of a short side that ends inside a tile."""
    u = make(shape, 4)
    u[1, -1, -1] = math.inf
    out = muon.orthogonalize(u)
    assert torch.isnan(out[1]).all()
    check(out[::2], u[::2])


def test_small_singular_values_keep_their_digits():
    """Directions 1e-5 of the largest: their squares are below 32 bits' resolution."""
    g = torch.Generator().manual_seed(1)
    q, _ = torch.linalg.qr(torch.randn(8, 8, generator=g, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(600, 8, generator=g, dtype=torch.float64))
    s = torch.tensor([1.0, 1.0, 0.1, 0.01, 1e-3, 1e-4, 1e-5, 1e-5], dtype=torch.float64)
    u = ((q * s) @ v.T).float().cuda()
    check(muon.orthogonalize(u), u)


def test_zero_and_non_finite_matrices():
    u = make((4, 12, 200), 2)
    u[1] = 0.0
    u[2, 3, 7] = math.inf
    u[3, 0, 0] = math.nan
    out = muon.orthogonalize(u)
    check(out[:1], u[:1])
    assert (out[1] == 0).all() and out[2:].isnan().all()
    tiny = 1e-30 * torch.ones(3, 5, device="cuda")
    huge = 1e30 * make((3, 50), 4)
    check(muon.orthogonalize(tiny), tiny)
    check(muon.orthogonalize(huge), huge)


def test_layouts():
    base = make((40, 600), 8)
    for u in (base.t(), base[:, 1:], base[3:19, 5:105], base.view(-1)[1:1 + 16 * 100].view(16, 100),
              make((6, 12, 90), 1).transpose(0, 1), base.expand(2, 40, 600)):
        check(muon.orthogonalize(u), u)
    b = make((40, 601), 8, torch.bfloat16).view(-1)[1:1 + 16 * 100].view(16, 100)
    check(muon.orthogonalize(b), b)


def test_offsets_past_32_bits():
    """More than 2^31 elements in one batch: the last matrices as by themselves."""
    u = torch.zeros(2100, 16, 65536, device="cuda")
    u[-2:] = make((2, 16, 65536), 4)
    out = muon.orthogonalize(u)
    check(out[-2:], u[-2:])
    assert (out[:2] == 0).all() and (out[1024:1026] == 0).all()


def test_streams_and_graphs():
    us = [make((16, 4096), 1), make((4096, 16), 2), make((100, 333), 3)]
    ref = muon.orthogonalize(us)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = muon.orthogonalize(us)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(muon.orthogonalize(us))
        graphs.append(g)
    for k in range(4):
        for u in us:
            u.mul_(1.0 + k).add_(1e-4 * torch.randn_like(u))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = muon.orthogonalize(us)
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, eager))


# ----------------------------------------------------------------- optimizer
def _projections():
    g = torch.Generator().manual_seed(3)
    shapes = {"self_attn.q_proj": (96, 64), "self_attn.k_proj": (32, 64), "self_attn.v_proj": (32, 64),
              "mlp.down_proj": (64, 176)}
    ps = lora.create_lora_for_block(0, "full_attention", shapes, rank=4, alpha=8.0, device="cuda",
                                    targets=tuple(shapes), generator=g)
    ps["experts"] = moe.make_expert_lora("experts", 6, 64, 48, rank=3, alpha=6.0, device="cuda",
                                         segments=2, generator=g, b_std=0.1)
    for p in ps.values():
        for t in (p.grad_A, p.grad_B, p.m_A, p.m_B):
            t.copy_(torch.randn(t.shape, generator=g) * 1e-3)
    return ps


@pytest.mark.parametrize("nesterov,decay,rms", [(True, 0.0, 0.2), (False, 0.1, None)])
def test_optimizer_step(nesterov, decay, rms):
    ps = _projections()
    before = {(k, n): getattr(p, n).detach().double().clone() for k, p in ps.items()
              for n in ("A", "B", "grad_A", "grad_B", "m_A", "m_B", "v_A")}
    opt = muon.Muon(lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=decay, match_rms=rms)
    opt.step(ps)
    assert opt.step_count == 1
    for k, p in ps.items():
        assert torch.equal(p.v_A.double(), before[k, "v_A"])
        for f in "AB":
            g, m = before[k, "grad_" + f], before[k, "m_" + f]
            m = 0.9 * m + 0.1 * g
            u = 0.9 * m + 0.1 * g if nesterov else m
            n = getattr(p, "segments", 1)
            mats = u.view(-1, u.shape[-2] // n, u.shape[-1])
            o = formula(mats).reshape(u.shape)
            rows, cols = mats.shape[-2:]
            scale = rms * math.sqrt(max(rows, cols)) if rms else math.sqrt(max(1.0, rows / cols))
            want = (1.0 - 0.02 * decay) * before[k, f] - 0.02 * scale * o
            now = getattr(p, f).detach().double()
            # the momenta's roundings (2^-24 each, a few of them) grow with the steps
            assert (getattr(p, "m_" + f).double() - m).abs().max() <= 4 * 2**-24 * m.abs().max()
            assert (now - want).abs().max() <= 2e-5 * 0.02 * scale * o.abs().max() \
                + 2**-22 * want.abs().max()
            assert getattr(p, f).is_leaf and getattr(p, f).requires_grad


def test_optimizer_needs_one_for_tables():
    class Table:
        pass
    with pytest.raises(ValueError, match="no optimizer"):
        muon.Muon().step({"embedding": Table()})


def test_optimizer_in_a_stack_with_adamw():
    """Same call surface as AdamW."""
    ps = _projections()
    for opt in (engine.AdamW(lr=1e-3), muon.Muon(lr=1e-3)):
        opt.step(ps)
        opt.zero_grad(ps)
        assert all(float(p.grad_A.abs().max()) == 0.0 for p in ps.values())
