"""An ExpertBalance through an MoE layer: captured and replayed."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from spilltune_amd import moe

pytestmark = pytest.mark.gpu
BF, H, E, B, S = torch.bfloat16, 256, 16, 3, 50


def _layer(sigmoid, dev):
    g = torch.Generator().manual_seed(8)
    router = torch.randn(E, H, generator=g) * H**-0.5
    w = {"mlp.gate.weight": (router if sigmoid else router.to(BF)).to(dev),
         "mlp.gate.e_score_correction_bias": torch.zeros(E, device=dev),
         "mlp.experts.gate_up_proj": moe.quantize_experts(0.03 * torch.randn(E, 256, H, generator=g),
                                                          "nf4-g128", dev),
         "mlp.experts.down_proj": moe.quantize_experts(0.03 * torch.randn(E, H, 128, generator=g),
                                                       "nf4-g128", dev)}

    def layer(x, balance, valid):
        if sigmoid:
            return moe.deepseek_moe_feed_forward(x, w, num_experts=E, top_k=4, groups=4, group_k=2,
                                                 normalize=True, scale=2.5, balance=balance, valid=valid)
        return moe.moe_feed_forward(x, w, num_experts=E, top_k=4, norm_topk_prob=True, balance=balance,
                                    valid=valid)
    return layer


@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_sums_of_replayed_passes(sigmoid, per_row):
    """Eager passes, then two layers' passes in a graph: after each replay the sums are
    the eager ones' and the last replay's, whatever the program did in between."""
    dev = torch.device("cuda:0")
    layer = _layer(sigmoid, dev)
    g = torch.Generator("cuda").manual_seed(3)
    new = lambda: torch.randn(B, S, H, device=dev, generator=g).to(BF)  # noqa: E731
    valid = torch.arange(S, device=dev) < torch.tensor([[50], [31], [7]], device=dev)
    up = new()
    balance = moe.ExpertBalance(0.25, per_row=per_row)

    def passes(x, balance):
        out = layer(layer(x, balance, valid), balance, valid)
        return out, torch.autograd.grad(out, [x], up)[0]

    def eager(x):
        once = moe.ExpertBalance(0.25, per_row=per_row)
        out, grad = passes(x.detach().clone().requires_grad_(True), once)
        return out.detach(), grad, once
    x = new().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(x, balance)
    torch.cuda.current_stream().wait_stream(side)
    loss, counts = balance.loss.clone(), balance.counts.clone()
    assert balance.passes == 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = passes(x, balance)
    assert balance.passes == 4
    for _ in range(3):
        with torch.no_grad():
            x.copy_(new())
        graph.replay()
        torch.cuda.synchronize()
        noise = [torch.full((n,), 2**40, dtype=torch.int64, device=dev) for n in (1, E, B * E)]
        want_out, want_grad, once = eager(x)
        assert torch.equal(out, want_out) and torch.equal(grad, want_grad)
        assert torch.equal(balance.counts, counts + once.counts)
        # a sum of four numbers in another order: three roundings of at most their sum
        total = float(loss) + float(once.loss)
        assert abs(float(balance.loss) - total) <= 6 * 2**-24 * total
        del noise
    balance.reset()
    assert balance.loss is None and balance.counts is None and balance.passes == 0


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_passes_count_once(reentrant):
    """A layer that torch's checkpoint forms again: the plain pass's sums and gradients."""
    dev = torch.device("cuda:0")
    layer = _layer(False, dev)
    g = torch.Generator("cuda").manual_seed(5)
    x, up = (torch.randn(B, S, H, device=dev, generator=g).to(BF) for _ in range(2))
    got = []
    for again in (False, True):
        balance, leaf = moe.ExpertBalance(2.0), x.clone().requires_grad_(True)
        f = lambda t: layer(t, balance, None)  # noqa: B023,E731
        out = checkpoint(f, leaf, use_reentrant=reentrant) if again else f(leaf)
        out.backward(up)
        got.append((leaf.grad, balance.loss, balance.counts, balance.passes))
    assert got[0][3] == got[1][3] == 1
    assert all(torch.equal(a, b) for a, b in zip(got[0][:3], got[1][:3]))
