"""What an ExpertBalance keeps of the passes (the loss itself: test_gpu_balance.py)."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from spilltune_amd import moe


def _pass(seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand((), generator=g), torch.randint(0, 9, (3, 8), generator=g)


def test_sums_of_eager_passes():
    balance, want = moe.ExpertBalance(0.1), (0.0, torch.zeros(8, dtype=torch.int64))
    assert balance.loss is None and balance.counts is None and balance.passes == 0
    for seed in range(3):
        loss, counts = _pass(seed)
        want = want[0] + float(loss), want[1] + counts.sum(0)
        balance.record(loss, counts)
        loss.zero_(), counts.zero_()  # a pass's tensors are its own again
    assert balance.passes == 3 and torch.equal(balance.counts, want[1])
    assert abs(float(balance.loss) - want[0]) < 1e-6  # three roundings of numbers below 4
    balance.reset()
    assert balance.loss is None and balance.counts is None and balance.passes == 0


def test_captured_passes_count_with_their_last_replay(monkeypatch):
    """A replay writes a captured pass's tensors anew: here, in place."""
    balance = moe.ExpertBalance(0.1)
    eager, passes = _pass(0), [_pass(1), _pass(2)]
    first = eager[0].clone(), eager[1].clone()
    balance.record(*eager)
    monkeypatch.setattr(moe, "_capturing", lambda t: True, raising=False)
    for p in passes:
        balance.record(*p)
    monkeypatch.undo()
    for replay in range(3):
        for k, (loss, counts) in enumerate(passes):
            new = _pass(10 * replay + k + 3)
            loss.copy_(new[0]), counts.copy_(new[1])
        eager[0].zero_(), eager[1].zero_()
        assert balance.passes == 3
        want = first[1].sum(0) + passes[0][1].sum(0) + passes[1][1].sum(0)
        assert torch.equal(balance.counts, want)
        total = float(first[0]) + float(passes[0][0]) + float(passes[1][0])
        assert abs(float(balance.loss) - total) < 1e-6
    balance.reset()
    assert balance.loss is None and balance.passes == 0


def _plain_balance_loss(logits, indices, *, score, valid, per_row):
    """The loss of one group in plain torch, on the host."""
    E = logits.shape[-1]
    counts = torch.bincount(indices.reshape(-1).long(), minlength=E)
    p = logits.float().softmax(-1).reshape(-1, E).mean(0)
    return moe.BalanceLoss(E * (counts / counts.sum() * p).sum(), counts[None])


def _engine(f, x):
    """A block formed again in its backward, as the engine does."""
    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.save_for_backward(x)
            with torch.no_grad():
                return f(x)

        @staticmethod
        def backward(ctx, dy):
            x = ctx.saved_tensors[0].detach().requires_grad_(True)
            with torch.enable_grad():
                y = f(x)
            return torch.autograd.grad(y, [x], dy)[0]
    return Again.apply(x)


@pytest.mark.parametrize("how", [
    lambda f, x: f(x), lambda f, x: checkpoint(f, x, use_reentrant=False),
    lambda f, x: checkpoint(f, x, use_reentrant=True), _engine],
    ids=["plain", "checkpoint", "reentrant", "engine"])
def test_a_pass_counts_once_however_it_is_formed(monkeypatch, how):
    monkeypatch.setattr(moe, "balance_loss", _plain_balance_loss)
    g = torch.Generator().manual_seed(4)
    w, x = torch.randn(6, 8, generator=g), torch.randn(2, 5, 6, generator=g).requires_grad_(True)
    balance = moe.ExpertBalance(0.5)

    def layer(x):
        logits = x.reshape(-1, 6) @ w
        out = moe._balanced(torch.tanh(x.reshape(-1, 6)), logits, logits.topk(2)[1], "softmax", balance,
                            None, x.shape)
        return out.reshape(x.shape).sin()
    up = torch.randn(x.shape, generator=g)
    how(layer, x).backward(up)  # (torch's reentrant checkpoint takes no autograd.grad)
    assert balance.passes == 1 and int(balance.counts.sum()) == 20
    logits = x.reshape(-1, 6) @ w
    loss, _ = _plain_balance_loss(logits, logits.topk(2)[1], score="softmax", valid=None, per_row=False)
    (want,) = torch.autograd.grad((torch.tanh(x).sin() * up).sum() + 0.5 * loss, [x])
    assert torch.allclose(x.grad, want, rtol=1e-5, atol=1e-6)  # sums of eight fp32 terms up to 4
    assert abs(float(balance.loss) - float(loss.detach())) < 1e-5
    with torch.no_grad():
        layer(x)
    assert balance.passes == 1


def test_a_pass_is_there_after_its_forward(monkeypatch):
    monkeypatch.setattr(moe, "balance_loss", _plain_balance_loss)
    balance, x = moe.ExpertBalance(0.5), torch.rand(5, 8).requires_grad_(True)
    out = moe._balanced(x * 2, x * 3, x.topk(2)[1], "softmax", balance, None, x.shape)
    assert balance.passes == 1 and int(balance.counts.sum()) == 10
    for _ in range(2):
        out.sum().backward(retain_graph=True)
    assert balance.passes == 1
