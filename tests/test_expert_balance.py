"""What an ExpertBalance keeps of the passes (the loss itself: test_gpu_balance.py)."""
import torch

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
