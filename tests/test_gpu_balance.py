"""Balance loss, per-expert counts and their gradient against 64 bits."""
import pytest
import torch
from torch.autograd import forward_ad

from spilltune_amd import moe

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def formula(logits, indices, score, valid, per_row):
    """(loss, counts) of logits [B, S, E] in 64 bits, row by row as written down."""
    E, k = logits.shape[-1], indices.shape[-1]
    rows = [slice(b, b + 1) for b in range(logits.shape[0])] if per_row else [slice(None)]
    losses, counts = [], []
    for r in rows:
        x, i = logits[r].reshape(-1, E), indices[r].reshape(-1, k)
        if valid is not None:
            v = valid[r].reshape(-1)
            x, i = x[v], i[v]
        i = i.flatten().long()
        c = torch.bincount(i[(i >= 0) & (i < E)], minlength=E)
        counts.append(c)
        if not len(x):
            continue
        p = x.softmax(-1)
        if score == "sigmoid":
            p = x.sigmoid() / (x.sigmoid().sum(-1, keepdim=True) + 1e-20)
        losses.append(E * (c.double() / (k * len(x)) * p.mean(0)).sum())
    loss = torch.stack(losses).mean() if losses else torch.zeros((), dtype=F64, device=logits.device)
    return loss, torch.stack(counts)


def make(B, S, E, k, dtype, seed=0, sure=1.0):
    g = torch.Generator().manual_seed(seed)
    x = sure * (torch.randn(B, S, E, generator=g) + 0.7 * torch.randn(E, generator=g))
    x = x.to(dtype)
    return x.cuda(), x.float().topk(k, -1).indices.to(torch.int32).cuda()


def check(x, i, score="softmax", valid=None, per_row=False, dloss=0.7):
    leaf = x.detach().clone().requires_grad_(True)
    loss, counts = moe.balance_loss(leaf, i, score=score, valid=valid, per_row=per_row)
    ref = x.double().requires_grad_(True)
    want, want_counts = formula(ref, i, score, valid, per_row)
    assert loss.dtype == F32 and loss.shape == () and counts.dtype == torch.int64
    assert torch.equal(counts, want_counts)
    # exponentials and sums of positive terms: 2^-24 a step, fewer than 2^10 in a row
    # (16 tokens a lane and more only where there are many: their sum is a mean)
    assert abs(float(loss.detach()) - float(want.detach())) <= 2**-14 * float(want.detach().abs()) + 1e-30
    (g,) = torch.autograd.grad(loss, [leaf], torch.tensor(dloss, device="cuda"))
    if want.requires_grad:
        (r,) = torch.autograd.grad(want, [ref], torch.tensor(dloss, device="cuda", dtype=F64))
    else:
        r = torch.zeros_like(ref)
    assert g.dtype == x.dtype and g.shape == x.shape
    # p (a - sum a p): both parts are rounded at 2^-24 times a few steps of p times the
    # largest a, which is at least the largest |r| / p
    ok = torch.ones(x.shape[:-1], dtype=torch.bool, device="cuda") if valid is None else valid
    E, k = x.shape[-1], i.shape[-1]
    rows = counts.double().amax(-1)
    n = ok.sum(-1).double() if per_row else ok.sum().double().reshape(1)
    a = dloss * E * rows / (k * n.clamp(min=1) ** 2) / max(1, int((n > 0).sum()))
    a = a[:, None, None] if per_row else a[None, :, None]
    with torch.no_grad():
        p = x.double().softmax(-1)
        if score == "sigmoid":
            p = x.double().sigmoid() / (x.double().sigmoid().sum(-1, keepdim=True) + 1e-20)
        bound = torch.finfo(x.dtype).eps / 2 * r.abs() + 2**-17 * a * p + 1e-37
    assert ((g.double() - r).abs() <= bound)[ok].all()
    assert (g[~ok] == 0).all()
    return loss, counts, g


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("B,S,E,k", [(1, 1, 1, 1), (1, 1, 8, 2), (2, 3, 5, 5), (1, 77, 60, 4),
                                     (3, 77, 128, 8), (2, 500, 64, 1), (2, 65, 63, 3), (1, 9, 65, 64),
                                     (4, 1030, 256, 8), (1, 2049, 512, 8), (1, 5000, 16, 2)])
def test_sizes(B, S, E, k, score, dtype):
    x, i = make(B, S, E, k, dtype, seed=S + E)
    for per_row in (False, True):
        check(x, i, score, per_row=per_row)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("per_row", [False, True])
def test_padded_rows(score, per_row):
    x, i = make(5, 90, 48, 6, F32, seed=2)
    n = torch.tensor([90, 41, 1, 0, 77], device="cuda")
    valid = torch.arange(90, device="cuda") < n[:, None]
    want = check(x, i, score, valid, per_row)
    dirty, picks = x.clone(), i.clone()
    dirty[~valid] = float("nan")
    dirty[1, 60] = float("inf")
    picks[~valid] = 1 << 30
    got = check_same(dirty, picks, score, valid, per_row)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hole = valid.clone()
    hole[0, 5], hole[4, 0] = False, False  # not only right padding
    check(x, i, score, hole, per_row)


def check_same(x, i, score, valid, per_row):
    leaf = x.detach().clone().requires_grad_(True)
    loss, counts = moe.balance_loss(leaf, i, score=score, valid=valid, per_row=per_row)
    return loss, counts, torch.autograd.grad(loss, [leaf], torch.tensor(0.7, device="cuda"))[0]


def test_nothing_valid():
    x, i = make(2, 6, 16, 2, F32)
    for per_row in (False, True):
        loss, counts, g = check(x, i, valid=torch.zeros(2, 6, dtype=torch.bool, device="cuda"),
                                per_row=per_row)
        assert float(loss.detach()) == 0.0 and int(counts.sum()) == 0 and (g == 0).all()


def test_picks_outside_and_twice():
    x, i = make(2, 40, 32, 4, F32, seed=5)
    i[0, :7, 0], i[1, 3, 2], i[1, 4, 1] = -1, 32, -(1 << 31)
    i[0, 10] = 3  # one expert four times
    check(x, i)
    wide = i.long()
    wide[1, 5:9, 0] += 1 << 32  # whose lower halves are experts
    wide[0, 11, 1] = -(1 << 63)
    check(x, wide, per_row=True)


def test_sure_routers():
    """Logits of +-1e4, masked experts of -inf, equal ones: 1 when balanced."""
    x, i = make(2, 50, 24, 2, F32, seed=6, sure=3e3)
    check(x, i)
    check(x, i, "sigmoid")
    x, i = make(2, 50, 24, 2, F32, seed=6)
    x[..., 3::5] = -float("inf")
    check(x, x.topk(2, -1).indices)
    check(x, x.topk(2, -1).indices, "sigmoid")
    low = torch.full((1, 4, 8), -3e38, device="cuda")  # sigmoids of 0: no share for any
    check(low, i[:1, :4] % 8, "sigmoid")
    even = torch.zeros(1, 12, 6, device="cuda")
    picks = torch.arange(24, device="cuda").view(1, 12, 2) % 6
    loss, counts, g = check(even, picks)
    assert abs(float(loss) - 1.0) < 1e-6 and (counts == 4).all()


def test_against_differences():
    x, i = make(2, 9, 12, 3, F32, seed=8)
    for score in ("softmax", "sigmoid"):
        _, _, g = check(x, i, score, dloss=1.0)
        d = torch.randn(x.shape, device="cuda", dtype=F64)
        ends = [formula(x.double() + s * 1e-4 * d, i, score, None, False)[0] for s in (1, -1)]
        slope = float(ends[0] - ends[1]) / 2e-4
        assert abs(float((g.double() * d).sum()) - slope) <= 1e-5 * float((g.double() * d).abs().sum())


def test_layouts_streams_and_graphs():
    x, i = make(3, 64, 40, 4, F32, seed=9)
    want = check_same(x, i, "softmax", None, True)
    wide = torch.zeros(3, 64, 50, device="cuda")
    wide[..., 5:45] = x
    turned = i.transpose(0, 1).contiguous().transpose(0, 1)
    leaf = wide[..., 5:45].detach().requires_grad_(True)
    loss, counts = moe.balance_loss(leaf, turned, per_row=True)
    g = torch.autograd.grad(loss, [leaf], torch.tensor(0.7, device="cuda"))[0]
    assert torch.equal(loss, want[0]) and torch.equal(counts, want[1]) and torch.equal(g, want[2])
    flat = moe.balance_loss(x.view(-1, 40), i.view(-1, 4))
    assert torch.equal(flat.counts, moe.balance_loss(x, i).counts) and flat.counts.shape == (1, 40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = check_same(x, i, "softmax", None, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    leaf, up = x.clone().requires_grad_(True), torch.tensor(0.7, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts = moe.balance_loss(leaf, i, per_row=True)
        (g,) = torch.autograd.grad(loss, [leaf], up)
    for k in range(3):
        with torch.no_grad():
            leaf.mul_(0.9).add_(0.1 * torch.randn_like(leaf))
        i.copy_((i + 1) % 40)
        graph.replay()
        torch.cuda.synchronize()
        eager = check_same(leaf, i, "softmax", None, True)
        assert torch.equal(loss, eager[0]) and torch.equal(counts, eager[1]) and torch.equal(g, eager[2])


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last row's gradient as by itself (each row its own)."""
    B, S, E = 3, 1400000, 512
    x = torch.zeros(B, S, E, dtype=BF, device="cuda")
    i = torch.zeros(B, S, 1, dtype=torch.int32, device="cuda")
    x[-1, -2000:] = torch.randn(2000, E, device="cuda", generator=torch.Generator("cuda").manual_seed(1)
                                ).to(BF)
    i[-1, -2000:, 0] = torch.arange(2000, device="cuda", dtype=torch.int32) % E
    valid = torch.zeros(B, S, dtype=torch.bool, device="cuda")
    valid[-1, -2000:] = True
    x.requires_grad_(True)
    loss, counts = moe.balance_loss(x, i, valid=valid, per_row=True)
    (g,) = torch.autograd.grad(loss, [x])
    assert int(counts[-1].sum()) == 2000 and int(counts[:2].sum()) == 0
    few = x.detach()[-1:, -2000:].clone()
    want, _, _ = check(few, i[-1:, -2000:], dloss=1.0)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-4
    check_few = few.clone().requires_grad_(True)
    (fg,) = torch.autograd.grad(moe.balance_loss(check_few, i[-1:, -2000:]).loss, [check_few])
    assert torch.equal(g[-1, -2000:], fg[0]) and (g[0, :9] == 0).all() and (g[-1, :9] == 0).all()


def test_refused_derivatives():
    x, i = make(1, 4, 8, 2, F32)
    leaf = x.requires_grad_(True)
    loss, _ = moe.balance_loss(leaf, i)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, [leaf], create_graph=True)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        moe.balance_loss(forward_ad.make_dual(x.detach(), torch.ones_like(x)), i)
