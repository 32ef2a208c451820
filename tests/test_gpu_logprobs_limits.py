"""Token log probabilities (HIP) at the ends of their documented ranges; bounds as
in test_gpu_logprobs."""
import pytest
import torch

from spilltune_amd import ops
from tests.test_gpu_logprobs import _close, _inputs, _reference

pytestmark = pytest.mark.gpu


def test_backward_of_a_small_vocabulary_stays_within_its_scratch(monkeypatch):
    rows, H, V = 20000, 4096, 256
    monkeypatch.setattr(ops, "LOGPROB_SCRATCH", 64 << 20)
    h, w, t, g = _inputs(rows, H, V)
    g_lp = torch.randn(rows, generator=g, device="cuda")
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    (dh,) = torch.autograd.grad(r.logprobs, h, g_lp)
    peak = torch.cuda.max_memory_allocated() - before
    assert peak <= dh.numel() * 2 + (64 << 20) + (4 << 20), peak
    want, err, _, _ = _reference(h.detach(), w, t, grads=(g_lp, None, None))
    _close("dh", dh, want[2], err[2])
