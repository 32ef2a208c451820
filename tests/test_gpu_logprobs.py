"""Token log probabilities (HIP) against their 64-bit definition, element by
element within the bounds of their sums and roundings."""
import math

import pytest
import torch

from spilltune_amd import ops

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64
U = 2.0 ** -8   # half a step of bf16
E = 2.0 ** -24  # of fp32


def _inputs(rows, H, V, seed=0, grid=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    h, w = r(rows, H), r(V, H) * (2.0 / math.sqrt(H))
    if grid:  # products and their sums exact in fp32: logits that tie do so exactly
        h, w = (h * 4).round().clamp(-31, 31) / 4, (w * 64).round().clamp(-127, 127) / 64
    t = torch.randint(0, V, (rows,), generator=g, device="cuda")
    return h.to(BF), w.to(BF), t, g


def _reference(h, w, t, temperature=1.0, cap=None, grads=(None, None, None), top_idx=None):
    """((lp, entropy, logits) and, given upstream gradients, dh), bounds alike."""
    h, w = h.double(), w.double()
    l = h @ w.T
    # fp32 sums of H exact products, cap and temperature at 8 roundings
    dl_in = (h.shape[1] * E * (h.abs() @ w.T.abs())).amax(1)
    th = torch.tanh(l / cap) if cap else None
    x = (cap * th if cap else l) / temperature
    dx = (dl_in + 8 * E * (cap or float(l.abs().max()))) / temperature
    lp = x.log_softmax(-1)
    p = lp.exp()
    ent = -(p * lp).sum(-1)
    V = l.shape[1]
    rows = torch.arange(len(t), device=t.device)
    kept = (t >= 0) & (t < V)
    given = t.clamp(0, V - 1)
    out = torch.where(kept, lp[rows, given], 0.0)
    # x moves by dx everywhere; e^x, its sum and its logarithm round (the
    # exponent's argument is up to 100 off its maximum: 128 E)
    e_lp = 2 * dx + 300 * E + 4 * E * out.abs()
    e_ent = (2 * dx + 300 * E) * (2 + math.log(max(V, 3)))
    res, err = [out, ent], [e_lp, e_ent]
    if any(g is not None for g in grads):
        z = torch.zeros_like(ent)
        g_lp, g_ent, g_top = grads
        g_lp = torch.where(kept, g_lp.double(), 0.0) if g_lp is not None else z
        g_ent = g_ent.double() if g_ent is not None else z
        own = torch.zeros_like(l)
        own[rows, given] += g_lp
        if g_top is not None:
            own.scatter_add_(1, top_idx, g_top.double())
        d = own - p * own.sum(1, keepdim=True) - g_ent[:, None] * p * (lp + ent[:, None])
        size = own.abs() + p * (own.abs().sum(1, keepdim=True)
                                + g_ent.abs()[:, None] * (lp + ent[:, None]).abs())
        k = ((1 - th * th) if cap else 1.0) / temperature
        dh = (d * k) @ w
        # dl rounds to bf16 (its terms' fp32 errors: a tenth of that), dh once
        res.append(dh)
        err.append(1.1 * U * ((size * k) @ w.abs()) + U * dh.abs())
    return res, err, l, lp


def _close(name, got, want, bound):
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (name, float(err.max()), float((err / (bound + 1e-30)).max()))


# rows around the 64/128/256-row tiles, vocabularies around the 256-column
# tiles and off the multiples of 8, hidden sizes off the 64-deep steps
SIZES = [(1, 8, 1), (1, 64, 7), (5, 72, 255), (61, 264, 257), (64, 128, 1000), (65, 1024, 4104),
         (129, 200, 256), (200, 64, 33001), (257, 520, 777), (300, 96, 8192), (700, 128, 2050)]


@pytest.mark.parametrize("rows,H,V", SIZES)
@pytest.mark.parametrize("temperature,cap", [(1.0, None), (0.7, 5.0), (2.0, None)])
@pytest.mark.parametrize("kept", [True, False])
def test_values_and_gradient(monkeypatch, rows, H, V, temperature, cap, kept):
    if not kept:  # the backward forms the logits again
        monkeypatch.setattr(ops, "LOGPROB_KEEP", 0)
    h, w, t, g = _inputs(rows, H, V, seed=rows)
    t[::7] = -100
    g_lp, g_ent = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t, temperature=temperature, cap=cap)
    (dh,) = torch.autograd.grad([r.logprobs, r.entropy], h, [g_lp, g_ent])
    want, err, _, _ = _reference(h.detach(), w, t, temperature, cap, (g_lp, g_ent, None))
    for name, a, b, e in zip(("logprobs", "entropy", "dh"), (r.logprobs, r.entropy, dh), want, err):
        _close(name, a, b, e)
    assert bool((r.logprobs[::7] == 0).all())
    assert r.top_logprobs.shape == (rows, 0) and r.top_tokens.shape == (rows, 0)


@pytest.mark.parametrize("rows,V,top", [(1, 64, 64), (5, 300, 1), (70, 5000, 20), (260, 2049, 5),
                                        (3, 2, 2), (130, 1000, 8)])
@pytest.mark.parametrize("kept", [True, False])
def test_alternatives(monkeypatch, rows, V, top, kept):
    """Falling values, ties to the lowest index, and their gradient."""
    if not kept:
        monkeypatch.setattr(ops, "LOGPROB_KEEP", 0)
    h, w, t, g = _inputs(rows, 64, V, seed=V, grid=True)
    w[V // 2:] = w[:V - V // 2].clone()  # every logit of the second half ties with one of the first
    t[1::5] = -100
    g_lp = torch.randn(rows, generator=g, device="cuda")
    g_top = torch.randn(rows, top, generator=g, device="cuda")
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t, top=top, temperature=0.5, cap=6.0)
    (dh,) = torch.autograd.grad([r.logprobs, r.top_logprobs], h, [g_lp, g_top])
    _, _, l, lp = _reference(h.detach(), w, t, 0.5, 6.0)
    idx = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_tokens, idx)
    want, err, _, _ = _reference(h.detach(), w, t, 0.5, 6.0, (g_lp, None, g_top), idx)
    _close("logprobs", r.logprobs, want[0], err[0])
    _close("top", r.top_logprobs, lp.gather(1, idx), err[0][:, None] + 0 * lp.gather(1, idx)
           + 4 * E * lp.gather(1, idx).abs())
    _close("dh", dh, want[2], err[2])


def test_sure_tokens_and_small_entropies():
    """Distributions with all but a millionth on one token: nothing cancels."""
    V, H = 5000, 64
    w = torch.zeros(V, H, device="cuda", dtype=BF)
    w[17, 0] = 1.0
    h = torch.zeros(3, H, device="cuda", dtype=BF)
    h[:, 0] = torch.tensor([10.0, 20.0, 80.0])
    r = ops.token_logprobs(h, w, torch.tensor([17, 17, 3], device="cuda"), top=2)
    want, err, _, lp = _reference(h, w, torch.tensor([17, 17, 3], device="cuda"))
    _close("logprobs", r.logprobs, want[0], 4 * E * (1 + want[0].abs()))
    # terms e^d d of d = -10, -20, -80: the exponential's relative error is 100 E
    _close("entropy", r.entropy, want[1], 200 * E * want[1] + 2 * E)
    assert r.top_tokens.tolist() == [[17, 0]] * 3


def test_rows_of_garbage():
    """NaN and infinite rows keep to themselves; a row without an upstream
    gradient gets zeros whatever it holds; bad device tokens give NaN."""
    h, w, t, g = _inputs(9, 64, 700)
    h[2], h[5, 3] = float("nan"), float("inf")
    t[7], t[8] = 700, -3
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t, top=3)
    g_lp = torch.randn(9, generator=g, device="cuda")
    g_lp[2] = 0
    good = torch.tensor([0, 1, 3, 4, 6], device="cuda")
    (dh,) = torch.autograd.grad(r.logprobs, h, g_lp)
    want, err, l, _ = _reference(h.detach()[good], w, t[good], grads=(g_lp[good], None, None))
    _close("logprobs", r.logprobs[good], want[0], err[0])
    _close("dh", dh[good], want[2], err[2])
    assert bool((dh[2] == 0).all())
    assert bool(torch.isnan(r.logprobs[torch.tensor([2, 5, 7, 8], device="cuda")]).all())
    assert bool(torch.isnan(r.entropy[2])) and r.top_tokens[2].tolist() == [-1, -1, -1]
    assert bool(torch.isfinite(r.entropy[7:]).all())
    assert bool((r.top_tokens < 700).all())


def test_the_same_token_given_and_among_the_alternatives():
    """An entry picked twice counts once; gradients of the alternatives alone."""
    h, w, _, g = _inputs(40, 64, 900, seed=5, grid=True)
    l = h.double() @ w.double().T
    idx = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :3]
    t = idx[:, 1].contiguous()
    g_lp, g_top = torch.randn(40, generator=g, device="cuda"), torch.randn(40, 3, generator=g,
                                                                           device="cuda")
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t, top=3)
    assert torch.equal(r.logprobs, r.top_logprobs[:, 1])
    for grads in ((g_lp, g_top), (None, g_top), (g_lp, None)):
        outs = [o for o, x in zip((r.logprobs, r.top_logprobs), grads) if x is not None]
        (dh,) = torch.autograd.grad(outs, h, [x for x in grads if x is not None], retain_graph=True)
        want, err, _, _ = _reference(h.detach(), w, t, grads=(grads[0], None, grads[1]), top_idx=idx)
        _close("dh", dh, want[2], err[2])


def test_no_second_derivative():
    h, w, t, _ = _inputs(4, 64, 300)
    h.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.token_logprobs(h, w, t).logprobs.sum(), h, create_graph=True)


def test_host_tokens_and_shapes():
    h, w, t, _ = _inputs(12, 64, 300)
    a = ops.token_logprobs(h.view(3, 4, 64), w, t.cpu().view(3, 4), top=2)
    b = ops.token_logprobs(h, w, t, top=2)
    assert a.logprobs.shape == (3, 4) and a.top_tokens.shape == (3, 4, 2)
    assert torch.equal(a.logprobs.view(-1), b.logprobs) and torch.equal(a.entropy.view(-1), b.entropy)
    with pytest.raises(ValueError, match="ignore_index"):
        ops.token_logprobs(h, w, torch.full((12,), 300))
    e = ops.token_logprobs(h[:0], w, t[:0], top=2)
    assert e.logprobs.shape == (0,) and e.top_tokens.shape == (0, 2)
    one = ops.token_logprobs(h[0], w, t[0])
    assert one.logprobs.shape == () and torch.equal(one.logprobs, ops.token_logprobs(
        h[:1], w, t[:1]).logprobs[0])


@pytest.mark.parametrize("keep", [0, 1 << 30])
def test_row_chunks(monkeypatch, keep):
    h, w, t, g = _inputs(600, 64, 3000, grid=True)
    g_lp = torch.randn(600, generator=g, device="cuda")
    h.requires_grad_(True)
    want, err, l, _ = _reference(h.detach(), w, t, grads=(g_lp, None, None))
    monkeypatch.setattr(ops, "LOGPROB_SCRATCH", 1 << 20)
    monkeypatch.setattr(ops, "LOGPROB_KEEP", keep)
    r = ops.token_logprobs(h, w, t, top=4)
    (dh,) = torch.autograd.grad(r.logprobs, h, g_lp)
    _close("logprobs", r.logprobs, want[0], err[0])
    _close("dh", dh, want[2], err[2])
    assert torch.equal(r.top_tokens, torch.sort(l, dim=1, descending=True, stable=True).indices[:, :4])


def test_head_beyond_two_gib():
    rows, H, V = 3, 8192, 140000
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(rows, H, generator=g, device="cuda").to(BF).requires_grad_(True)
    w = torch.empty(V, H, device="cuda", dtype=BF).normal_(0, 0.02, generator=g)
    t = torch.tensor([V - 1, 0, 131072], device="cuda")
    g_lp = torch.tensor([1.0, -2.0, 0.5], device="cuda")
    r = ops.token_logprobs(h, w, t)
    (dh,) = torch.autograd.grad(r.logprobs, h, g_lp)
    want, err, _, _ = _reference(h.detach(), w, t, grads=(g_lp, None, None))
    _close("logprobs", r.logprobs, want[0], err[0])
    _close("dh", dh, want[2], err[2])


def test_operands_of_any_layout_streams_and_graphs():
    h0, w0, t, g = _inputs(70, 128, 900, seed=3)
    wide = torch.zeros(70, 2, 128, device="cuda", dtype=BF)
    wide[:, 1] = h0
    flat = torch.zeros(900 * 128 + 1, device="cuda", dtype=BF)
    flat[1:] = w0.view(-1)
    g_lp, g_ent = (torch.randn(70, generator=g, device="cuda") for _ in range(2))

    def go(h, w):
        h = h.detach().requires_grad_(True)
        r = ops.token_logprobs(h, w, t, top=3)
        (dh,) = torch.autograd.grad([r.logprobs, r.entropy], h, [g_lp, g_ent])
        return [r.logprobs.detach(), r.entropy.detach(), r.top_logprobs.detach(), r.top_tokens, dh]
    a = go(h0, w0)
    for x, y in zip(a, go(wide[:, 1], flat[1:].view(900, 128))):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = go(h0, w0)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    leaf = h0.clone().requires_grad_(True)

    def step():
        r = ops.token_logprobs(leaf, w0, t, top=3)
        (dh,) = torch.autograd.grad([r.logprobs, r.entropy], leaf, [g_lp, g_ent])
        return [r.logprobs.detach(), r.entropy.detach(), r.top_logprobs.detach(), r.top_tokens, dh]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            leaf.copy_(torch.randn(70, 128, generator=g, device="cuda"))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        for x, y in zip(held, eager):
            assert torch.equal(x, y)


def test_saved_tensors_that_a_hook_moved_and_any_shape():
    """Saved tensors kept on the host come back elsewhere; one token, no token and
    rows of tokens."""
    g = torch.Generator(device="cuda").manual_seed(31)
    w = torch.randn(500, 64, generator=g, device="cuda").bfloat16()
    for shape in ((), (0,), (2, 3)):
        h = torch.randn(*shape, 64, generator=g, device="cuda").bfloat16().requires_grad_(True)
        t = torch.randint(500, shape, generator=g, device="cuda")
        grads = []
        for moved in (False, True):
            pack = (lambda x: x.cpu()) if moved else (lambda x: x)
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x.cuda()):
                r = ops.token_logprobs(h * 1, w, t, top=3)
            junk = [torch.full((4, 64), float("nan"), device="cuda") for _ in range(8)]
            assert r.logprobs.shape == r.entropy.shape == shape
            assert r.top_logprobs.shape == r.top_tokens.shape == (*shape, 3)
            grads += torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum(), h)
            del junk
        assert grads[0].shape == h.shape and torch.equal(*grads)
