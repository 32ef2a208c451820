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


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("temperature,cap", [(1e6, 1.0), (1e5, 30.0), (1e30, 3.0), (0.01, 0.5)])
def test_temperatures_far_above_the_cap(monkeypatch, temperature, cap, kept):
    """The picked entries' share of the gradient passes through the cap's slope,
    whatever the temperature."""
    if not kept:
        monkeypatch.setattr(ops, "LOGPROB_KEEP", 0)
    rows, H, V = 70, 264, 3001
    h, w, t, g = _inputs(rows, H, V)
    g_lp, g_ent = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    g_top = torch.randn(rows, 3, generator=g, device="cuda")
    t[5] = -100
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t, top=3, temperature=temperature, cap=cap)
    (dh,) = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], h, [g_lp, g_ent, g_top])
    want, err, _, _ = _reference(h.detach(), w, t, temperature, cap, (g_lp, g_ent, g_top), r.top_tokens)
    _close("logprobs", r.logprobs, want[0], err[0])
    _close("dh", dh, want[2], err[2])
