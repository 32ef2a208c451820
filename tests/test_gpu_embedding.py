"""Scaled embedding lookup and the table's gradient by sorted tokens, against 64 bits."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from spilltune_amd import engine, ops
from spilltune_amd.embedding import TokenEmbedding

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def make(n, V, H, dtype=F32, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed)
    table = (0.1 * torch.randn(V, H, generator=g)).to(dtype).cuda()
    if ids is None:  # frequencies that fall with the rank
        ids = (torch.exp(torch.rand(n, generator=g, dtype=F64) * math.log(V)).long() - 1) * 7919 % V
    dout = torch.randn(*ids.shape, H, generator=g).to(BF).cuda()
    return table, ids.cuda(), dout


def reference(ids, dout, V, scale, padding=None):
    """(gradient, sums of the terms' sizes, how many) in 64 bits."""
    d = dout.double().reshape(-1, dout.shape[-1])
    flat = ids.reshape(-1).long()
    keep = (flat >= 0) & (flat < V)
    if padding is not None:
        keep &= flat != padding
    flat, d = flat[keep], d[keep]
    out = torch.zeros(2, V, d.shape[1], dtype=F64, device=d.device)
    out[0].index_add_(0, flat, d)
    out[1].index_add_(0, flat, d.abs())
    return scale * out[0], abs(scale) * out[1], torch.bincount(flat, minlength=V)[:, None]


def check_grad(grad, ids, dout, scale, padding=None, before=None):
    ref, size, many = reference(ids, dout, grad.shape[0], scale, padding)
    # additions of 2^-24 of the sum so far, at most the sizes' sum; the scale's rounding
    room = 2**-24 * (many + 2) * size
    if before is not None:
        ref, room = ref + before.double(), room + 2**-24 * (ref.abs() + before.double().abs())
    bound = torch.finfo(grad.dtype).eps / 2 * ref.abs() + room
    worst = float(((grad.double() - ref).abs() - bound).max())
    assert worst <= 0, worst
    if before is None:
        assert (grad[many[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (1, 1000, 64), (2, 3, 8), (15, 7, 40), (16, 511, 24),
                                   (17, 512, 33), (77, 513, 1024), (1000, 32000, 264),
                                   (1023, 300000, 8), (1025, 262143, 72), (4097, 262144, 16),
                                   (16384, 32000, 16), (16385, 32000, 16), (33000, 50257, 9),
                                   (70001, 2, 64), (40000, 128256, 40), (5, 40, 5000)])
def test_lookup_and_gradient(n, V, H, dtype):
    table, ids, dout = make(n, V, H, dtype, seed=n)
    t = table.clone().requires_grad_(True)
    out = ops.embedding(t, ids, scale=1.7)
    want = (table[ids].double() * 1.7)
    # one product in fp32 (and the scale's own rounding), then bf16
    assert ((out.double() - want).abs() <= (2**-8 + 2**-22) * want.abs()).all()
    (grad,) = torch.autograd.grad(out, [t], dout)
    assert grad.dtype == dtype
    check_grad(grad, ids, dout, 1.7)
    again = torch.autograd.grad(ops.embedding(t, ids, scale=1.7), [t], dout)[0]
    assert torch.equal(grad, again)


@pytest.mark.parametrize("n", [1, 16, 31, 33, 400, 20000])
@pytest.mark.parametrize("pattern", ["one", "two", "blocks", "last"])
def test_runs_over_chunk_ends(n, pattern):
    """Long runs of one token: inside, over and on the ends of chunks."""
    at = torch.arange(n)
    ids = {"one": torch.zeros(n, dtype=torch.long), "two": at % 2, "blocks": at // 16,
           "last": torch.where(at < n // 3, 5, 9)}[pattern]
    V = int(ids.max()) + 1
    table, ids, dout = make(n, V, 136, seed=n, ids=ids)
    t = table.requires_grad_(True)
    (grad,) = torch.autograd.grad(ops.embedding(t, ids), [t], dout)
    check_grad(grad, ids, dout, 1.0)


def test_sums_in_the_order_of_positions():
    """Two positions' sum does not depend on where they stand: with 2^24 and 1 the
    rounding shows the order of three."""
    dout = torch.tensor([[2.0**24], [1.0], [1.0], [-2.0**24]], device="cuda").to(BF).repeat(1, 8)
    t = torch.zeros(3, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(ops.embedding(t, torch.tensor([1, 1, 1, 1], device="cuda")), [t], dout)
    assert float(g[1, 0]) == 0.0  # ((2^24 + 1) + 1) - 2^24 in fp32
    (g,) = torch.autograd.grad(ops.embedding(t, torch.tensor([1, 1, 1, 1], device="cuda")), [t],
                               dout[[1, 2, 0, 3]])
    assert float(g[1, 0]) == 2.0


@pytest.mark.parametrize("n", [50, 20000])
def test_padding_and_tokens_outside_the_table(n):
    table, ids, dout = make(n, 90, 64, seed=3)
    ids[::3] = 7
    ids[1::11], ids[2::13] = -1, 90
    ids[4::17] = 2**40 + 5
    dout[ids == 7] = float("nan")  # padded rows may hold anything
    t = table.clone().requires_grad_(True)
    out = ops.embedding(t, ids, scale=2.0, padding_idx=7)
    bad = (ids < 0) | (ids >= 90)
    assert out[bad].isnan().all() and torch.equal(out[~bad], (2.0 * table)[ids[~bad]].to(BF))
    (grad,) = torch.autograd.grad(out, [t], dout)
    keep = ids != 7
    check_grad(grad, ids[keep], dout[keep], 2.0)
    assert (grad[7] == 0).all()
    none = torch.full((n,), 7, device="cuda")
    (grad,) = torch.autograd.grad(ops.embedding(t, none, padding_idx=7), [t], dout)
    assert (grad == 0).all()


def test_shapes_types_and_layouts():
    table, ids, dout = make(24, 40, 48, seed=5)
    want = table[ids].to(BF)
    assert torch.equal(ops.embedding(table, ids.view(2, 3, 4)), want.view(2, 3, 4, 48))
    assert torch.equal(ops.embedding(table, ids.int()), want)
    assert torch.equal(ops.embedding(table, ids.cpu()), want)
    assert torch.equal(ops.embedding(table, ids[3]), want[3])
    assert torch.equal(ops.embedding(table, ids.view(4, 6).t()), want.view(4, 6, 48).transpose(0, 1))
    assert ops.embedding(table, ids[:0]).shape == (0, 48)
    wide = torch.zeros(40, 49, device="cuda")
    wide[:, 1:] = table
    assert torch.equal(ops.embedding(wide[:, 1:], ids), want)
    t = table.clone().requires_grad_(True)
    g = torch.autograd.grad(ops.embedding(t, ids), [t], dout)[0]
    turned = dout.t().contiguous().t()
    assert torch.equal(g, torch.autograd.grad(ops.embedding(t, ids.int()), [t], turned)[0])
    (g,) = torch.autograd.grad(ops.embedding(t, ids[:0]), [t], dout[:0])
    assert (g == 0).all()


def test_against_differences():
    table, ids, dout = make(200, 30, 16, seed=6)
    t = table.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.embedding(t, ids, scale=3.0), [t], dout)
    d = torch.randn(30, 16, device="cuda", dtype=F64)
    ends = [(3.0 * (table.double() + s * 1e-3 * d)[ids] * dout.double()).sum() for s in (1, -1)]
    assert abs(float((g.double() * d).sum() - (ends[0] - ends[1]) / 2e-3)) <= \
        2**-20 * float((g.double() * d).abs().sum()) + 1e-6


def test_streams_and_graphs():
    table, ids, dout = make(3000, 500, 128, seed=7)
    many = make(20000, 500, 128, seed=8)[1:]
    t = table.clone().requires_grad_(True)

    def grads():
        return [torch.autograd.grad(ops.embedding(t, i, scale=0.5), [t], d)[0]
                for i, d in ((ids, dout), many)]
    want = grads()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = grads()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = grads()
    for k in range(3):
        for i in (ids, many[0]):
            i.copy_((i * 3 + k) % 500)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, grads())), k


def test_refused_derivatives():
    table, ids, dout = make(5, 6, 8)
    t = table.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.embedding(t, ids), [t], dout, create_graph=True)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        ops.embedding(forward_ad.make_dual(table.detach(), torch.ones_like(table)), ids)


# ----------------------------------------------------------------- the trained table
@pytest.mark.parametrize("n", [300, 20000])
def test_token_embedding_adds_and_replaces(n):
    table, ids, dout = make(n, 700, 40, BF, seed=9)
    e = TokenEmbedding(table.cpu(), device="cuda", scale=6.0, padding_idx=0)
    assert e.weight.dtype == F32 and torch.equal(e(ids), ops.embedding(table.float(), ids, scale=6.0))
    before = torch.randn_like(e.grad)
    e.grad.copy_(before)
    e.add_grad(ids, dout)
    check_grad(e.grad, ids, dout, 6.0, 0, before)
    quiet = torch.bincount(ids, minlength=700) == 0
    quiet[0] = True
    assert torch.equal(e.grad[quiet], before[quiet])
    e.add_grad(ids.cpu(), dout, accumulate=False)
    check_grad(e.grad, ids, dout, 6.0, 0)
    with pytest.raises(ValueError, match="shaped like"):
        e.add_grad(ids, dout[:1])
    e.zero_grad()
    assert (e.grad == 0).all()


@pytest.mark.parametrize("n", [300, 20000])
@pytest.mark.parametrize("H", [4, 9, 12, 15, 33, 1001, 1027])
def test_columns_that_end_inside_a_chunk(H, n):
    """Rows of no whole chunks: looked up, summed and added to a gradient once each."""
    for dtype in (F32, BF):
        table, ids, dout = make(n, 50, H, dtype, seed=H)
        t = table.clone().requires_grad_(True)
        out = ops.embedding(t, ids, scale=1.7)
        want = table[ids].double() * 1.7
        assert ((out.double() - want).abs() <= (2**-8 + 2**-22) * want.abs()).all()
        (grad,) = torch.autograd.grad(out, [t], dout)
        check_grad(grad, ids, dout, 1.7)
    e = TokenEmbedding(table, device="cuda", scale=1.7)
    before = torch.randn_like(e.grad)
    e.grad.copy_(before)
    e.add_grad(ids, dout)
    check_grad(e.grad, ids, dout, 1.7, before=before)


def test_adamw_updates_a_table():
    table, ids, dout = make(50, 60, 16, seed=10)
    e = TokenEmbedding(table, device="cuda")
    p = table.clone().requires_grad_(True)
    ref = torch.optim.AdamW([p], lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1, foreach=False)
    own = engine.AdamW(lr=1e-2, weight_decay=0.1)
    for k in range(3):
        own.zero_grad({"embedding": e})
        e.add_grad(ids, dout * (k + 1))
        p.grad = e.grad.clone()
        ref.step()
        own.step({"embedding": e})
        assert torch.equal(e.weight, p.detach()), k


def test_offsets_past_32_bits():
    """A table of more than 2^32 bytes and elements: rows at its end."""
    V, H = 300000, 16384
    t = torch.zeros(V, H, dtype=BF, device="cuda")
    t[-1] = 3.0
    ids = torch.tensor([V - 1, 5, V - 1, V - 2], device="cuda")
    t.requires_grad_(True)
    out = ops.embedding(t, ids)
    assert (out[0] == 3.0).all() and (out[1] == 0).all()
    (g,) = torch.autograd.grad(out, [t], torch.ones_like(out))
    assert (g[-1] == 2.0).all() and (g[-2] == 1.0).all() and (g[5] == 1.0).all()
    assert int((g != 0).any(-1).sum()) == 3
