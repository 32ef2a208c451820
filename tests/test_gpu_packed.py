"""Attention over runs of keys and rotation by positions (HIP) against 64-bit
restatements, element by element within the bounds of their roundings."""
import random

import pytest
import torch

from spilltune_amd import _lib, ops, packed
from tests._packed_ref import U, rope_ref, runs_brute, span_ref, span_scores

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _documents(rng, B, S, lo, hi, pad=0):
    d = torch.full((B, S), -1, dtype=torch.int32)
    for b in range(B):
        i, n = 0, 0
        while i < S - (pad if b % 2 == 0 else 0):
            size = rng.randint(lo, hi)
            d[b, i:min(i + size, S - (pad if b % 2 == 0 else 0))] = n
            i, n = i + size, n + 1
    return d


def _close(name, got, want, bound):
    err = (got.double() - want).abs()
    over = err > bound + 1e-30
    assert not bool(over.any()) and bool(torch.isfinite(got).all()), (
        name, float(err.max()), float((err / (bound + 1e-30)).max()), int(over.sum()))


def _run(B, S, H, KV, DQ, DV, mask, cap=None, slopes=None, seed=0, edit=None):
    """One forward and backward with its 64-bit values; ``edit`` changes the
    operands (q, k, v, dout) after the values are taken."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k = _randn(g, B, H, S, DQ).to(BF), _randn(g, B, KV, S, DQ).to(BF)
    v, dout = _randn(g, B, KV, S, DV).to(BF), _randn(g, B, S, H * DV).to(BF)
    scale = DQ ** -0.5 * 1.5
    want, bound = span_ref(q, k, v, scale, mask.key_start, mask.key_end, cap, slopes, dout)
    if edit:
        edit(q, k, v, dout)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = packed.span_attention(*leaves, scale, mask, cap=cap, slopes=slopes)
    grads = torch.autograd.grad(out, leaves, dout)
    return (out, *grads), want, bound


def _check(got, want, bound, keep=None):
    for i, name in enumerate(("out", "dq", "dk", "dv")):
        sel = (lambda t: t) if keep is None else keep[i]  # noqa: E731
        _close(name, sel(got[i]), sel(want[i]), sel(bound[i]))


# lengths around the 32-query blocks, 64-key steps and 128-row tiles; groups of
# 1, 2, 3, 4; the three head shapes
SHAPES = [(1, 1, 2, 1, 64, 64), (3, 2, 2, 2, 128, 128), (2, 31, 4, 2, 64, 64),
          (1, 33, 3, 1, 128, 128), (2, 64, 2, 2, 192, 128), (1, 65, 8, 2, 128, 128),
          (2, 127, 4, 4, 64, 64), (1, 129, 6, 2, 64, 64), (2, 200, 2, 1, 128, 128),
          (1, 333, 4, 4, 192, 128), (1, 257, 16, 8, 64, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["documents", "padded_window", "bidirectional"])
def test_documents(shape, kind):
    B, S, H, KV, DQ, DV = shape
    rng = random.Random(S * 31 + len(kind))
    pad = S // 4 if kind == "padded_window" else 0
    docs = _documents(rng, B, S, 1, max(1, S // 2), pad)
    marks = torch.tensor([[rng.random() < 0.7 for _ in range(S)] for _ in range(B)])
    kw = {"documents": {}, "padded_window": {"window": max(1, S // 5)},
          "bidirectional": {"bidirectional": marks.cuda()}}[kind]
    mask = packed.document_mask(docs.cuda(), **kw)
    lo, hi, pos = runs_brute(docs, marks if kind == "bidirectional" else None, kw.get("window"))
    assert torch.equal(mask.key_start.cpu(), lo) and torch.equal(mask.key_end.cpu(), hi)
    assert torch.equal(mask.positions.cpu(), pos)
    _check(*_run(*shape, mask, seed=S))


@pytest.mark.parametrize("shape", [(2, 70, 4, 2, 64, 64), (1, 150, 4, 1, 128, 128),
                                   (1, 140, 2, 2, 192, 128)])
@pytest.mark.parametrize("cap,bias", [(3.0, False), (None, True), (20.0, True)])
def test_cap_and_distance(shape, cap, bias):
    B, S, H = shape[:3]
    docs = _documents(random.Random(S), B, S, 10, S, 5)
    mask = packed.document_mask(docs.cuda())
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device="cuda") if bias else None
    _check(*_run(*shape, mask, cap=cap, slopes=slopes, seed=S))


@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (192, 128)])
def test_single_keys_pass_no_score_gradient(dims):
    """A softmax over one key is 1: dq and dk are exactly 0, out and dv are the
    values' and the gradients' own."""
    B, S, H = 2, 140, 4
    KV = H if dims[0] == 192 else 2
    mask = packed.document_mask(torch.zeros(B, S, dtype=torch.int32, device="cuda"), window=1)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (_randn(g, B, h, S, d).to(BF).requires_grad_(True)
               for h, d in ((H, dims[0]), (KV, dims[0]), (KV, dims[1])))
    dout = _randn(g, B, S, H * dims[1]).to(BF)
    out = packed.span_attention(q, k, v, 0.3, mask)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    assert bool((dq == 0).all()) and bool((dk == 0).all())
    heads = v.detach().repeat_interleave(H // KV, 1).transpose(1, 2).reshape(B, S, -1)
    assert torch.equal(out.detach(), heads)
    want = dout.double().view(B, S, KV, H // KV, dims[1]).sum(3).transpose(1, 2)
    _close("dv", dv, want, U * want.abs() + 2.0 ** -20)


def _random_runs(rng, B, S):
    """Runs in no order: empty ones, bounds outside the row, single keys."""
    lo, hi = torch.zeros(B, S, dtype=torch.int32), torch.zeros(B, S, dtype=torch.int32)
    for b in range(B):
        for i in range(S):
            a = rng.randint(-5, S + 3)
            lo[b, i], hi[b, i] = a, a + rng.choice([-3, 0, 1, 2, S // 3, 2 * S, 1 << 29])
    return lo.cuda(), hi.cuda()


@pytest.mark.parametrize("shape", [(2, 45, 4, 2, 64, 64), (1, 300, 4, 2, 128, 128),
                                   (1, 210, 2, 2, 192, 128)])
def test_any_runs(shape):
    lo, hi = _random_runs(random.Random(shape[1]), *shape[:2])
    mask = packed.span_mask(lo, hi)
    assert torch.equal(mask.positions[0].cpu(), torch.arange(shape[1], dtype=torch.int32))
    got, want, bound = _run(*shape, mask, seed=9)
    _check(got, want, bound)
    none = (hi.clamp(0, shape[1]) <= lo.clamp(0, shape[1]))
    assert bool(none.any()) and bool((got[0][none] == 0).all())


def test_groups_split_over_workgroups():
    """dK/dV: a whole group in one workgroup, halves of one, single heads."""
    for shape in ((4, 1100, 16, 8, 64, 64), (2, 1000, 32, 8, 64, 64), (1, 150, 8, 2, 64, 64)):
        docs = _documents(random.Random(1), shape[0], shape[1], 20, 400)
        _check(*_run(*shape, packed.document_mask(docs.cuda()), seed=2))


def test_one_document_is_causal_attention():
    B, S, H, KV, D = 2, 300, 8, 2, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (_randn(g, B, h, S, D).to(BF).requires_grad_(True) for h in (H, KV, KV))
    dout = _randn(g, B, S, H * D).to(BF)
    mask = packed.document_mask(torch.zeros(B, S, dtype=torch.int32, device="cuda"))
    a, b = packed.span_attention(q, k, v, 0.1, mask), ops.causal_attention(q, k, v, 0.1)
    ga, gb = (torch.autograd.grad(t, (q, k, v), dout) for t in (a, b))
    args = (q.detach(), k.detach(), v.detach(), 0.1, mask.key_start, mask.key_end)
    bounds = [span_ref(*args, dout=dout, rounded_ds=r)[1] for r in (False, True)]
    for x, y, e, f in zip((a, *ga), (b, *gb), *bounds):  # each within its bound of the exact value
        assert bool(((x.double() - y.double()).abs() <= e + f).all())


@pytest.mark.parametrize("shape", [(1, 200, 4, 2, 128, 128), (2, 97, 2, 1, 64, 64),
                                   (1, 160, 2, 2, 192, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -3e38])
def test_masked_places_reach_nothing(shape, bad):
    """Infinities and NaN in the rows of one document and of padding leave every
    other document's values as they were; padded rows get zeros."""
    B, S, H, KV = shape[:4]
    docs = torch.zeros(B, S, dtype=torch.int32)
    docs[:, 40:75] = 1
    docs[:, S - 9:] = -1
    hit = docs != 0

    def edit(q, k, v, dout):
        for t in (q, k, v):
            t.transpose(1, 2)[hit.cuda()] = bad
        dout[hit.cuda()] = bad
    mask = packed.document_mask(docs.cuda())
    got, want, bound = _run(*shape, mask, seed=4, edit=edit)
    good = (~hit).cuda()
    rows = [lambda t: t[good]] + [lambda t: t.transpose(1, 2)[good]] * 3
    _check(got, want, bound, rows)
    pad = (docs < 0).cuda()
    assert bool((got[0][pad] == 0).all())
    for t in got[1:]:
        assert bool((t.transpose(1, 2)[pad] == 0).all())


def test_future_keys_with_infinities():
    """A key that only later queries see leaves the earlier ones exact."""
    shape = (1, 90, 2, 1, 64, 64)
    mask = packed.document_mask(torch.zeros(1, 90, dtype=torch.int32, device="cuda"))

    def edit(q, k, v, dout):
        v[:, :, 50] = float("inf")
        k[:, :, 50] = float("nan")
    got, want, bound = _run(*shape, mask, seed=8, edit=edit)
    _close("out", got[0][:, :50], want[0][:, :50], bound[0][:, :50])
    _close("dq", got[1][:, :, :50], want[1][:, :, :50], bound[1][:, :, :50])
    assert bool(torch.isnan(got[0][:, 50:]).all())


def test_nothing_seen_at_all():
    docs = torch.full((2, 70), -1, dtype=torch.int32, device="cuda")
    got, _, _ = _run(2, 70, 4, 2, 128, 128, packed.document_mask(docs))
    for t in got:
        assert bool((t == 0).all())


def test_lse_and_neighbouring_memory():
    """lse of an empty run is +inf, of the others log2 of the sum; nothing is
    written outside the outputs."""
    B, S, H, D = 1, 77, 2, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (_randn(g, B, H, S, D).to(BF) for _ in range(3))
    docs = torch.zeros(B, S, dtype=torch.int32, device="cuda")
    docs[:, 70:] = -1
    mask = packed.document_mask(docs)
    n = B * S * H * D
    out = torch.full((n + 512,), 7.0, dtype=BF, device="cuda")
    lse = torch.full((B * H * S + 64,), 7.0, device="cuda")
    _lib.call("st_span_attn_fwd", _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), B, S, H, H, D, D, 0.125, 0.0,
              None, _lib.ptr(mask.key_start), _lib.ptr(mask.key_end), _lib.ptr(mask.plan),
              _lib.ptr(out), _lib.ptr(lse), _lib.stream_handle("cuda"))
    assert bool((out[n:] == 7).all()) and bool((lse[B * H * S:] == 7).all())
    x = (q.double() @ k.double().transpose(-1, -2)) * 0.125
    x = x.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
    want = torch.logsumexp(x, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
    got = lse[:B * H * S].view(B, H, S)
    assert bool(torch.isinf(got[:, :, 70:]).all()) and bool((got[:, :, 70:] > 0).all())
    # fp32 scores of magnitude below 16 and their sums: 64 and 77 roundings
    assert float((got[:, :, :70].double() - want[:, :, :70]).abs().max()) < 16 * 150 * 2.0 ** -24


def test_operands_of_any_layout_and_repeatable():
    """Strided and shifted operands, another stream, the same bits each time."""
    B, S, H, KV, D = 1, 140, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(6)
    flat = _randn(g, 1 + B * H * S * D).to(BF)
    q0 = flat[1:].view(B, H, S, D)                      # off the 16-byte boundary
    k0 = _randn(g, B, S, KV, D).to(BF).transpose(1, 2)  # token-major storage
    v0 = _randn(g, B, KV, S, 2 * D).to(BF)[..., :D]     # a column slice
    dout0 = _randn(g, B, S, 2, H * D).to(BF)[:, :, 1]
    mask = packed.document_mask(_documents(random.Random(4), B, S, 20, 60).cuda())

    def go(q, k, v, dout):
        ls = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed.span_attention(*ls, 0.2, mask)
        return [out.detach(), *torch.autograd.grad(out, ls, dout)]
    a = go(q0.clone(), k0.contiguous(), v0.contiguous(), dout0.contiguous())
    for x, y in zip(a, go(q0, k0, v0, dout0)):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = go(q0, k0, v0, dout0)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_no_second_derivative():
    g = torch.Generator(device="cuda").manual_seed(6)
    q = _randn(g, 1, 1, 8, 64).to(BF).requires_grad_(True)
    mask = packed.document_mask(torch.zeros(1, 8, dtype=torch.int32, device="cuda"))
    out = packed.span_attention(q, q.detach(), q.detach(), 0.125, mask)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), q, create_graph=True)
    y = _randn(g, 8, 3 * 64).to(BF).requires_grad_(True)
    pos = torch.arange(8, device="cuda").view(1, 8)
    out = packed.rope_positions(y, pos, packed.Rotary(64, 1e4, device="cuda"), 1, 1)[0]
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), y, create_graph=True)


def test_graph_replays():
    """Forward and backward captured; replays after eager work with new operands."""
    B, S, H, KV, D = 1, 260, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (_randn(g, B, h, S, D).to(BF).requires_grad_(True) for h in (H, KV, KV))
    dout = _randn(g, B, S, H * D).to(BF)
    mask = packed.document_mask(_documents(random.Random(5), B, S, 30, 120).cuda())

    def step():
        out = packed.span_attention(q, k, v, 0.125, mask)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), dout)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            for t in (q, k, v, dout):
                t.copy_(_randn(g, *t.shape))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        for x, y in zip(held, eager):
            assert torch.equal(x, y)


# ----------------------------------------------------------------- rotation
LAYOUTS = [(64, 64, False), (64, 64, True), (128, 128, False), (128, 32, True), (128, 64, False),
           (256, 256, False), (80, 20, False), (80, 40, True), (96, 24, False), (128, 2, True),
           (8, 6, True), (16, 10, False)]


@pytest.mark.parametrize("norm,D,rot,inter",
                         [(n, *x) for n in (False, True) for x in LAYOUTS
                          if not n or x[0] in (64, 128, 256)])
@pytest.mark.parametrize("B,S", [(1, 1), (16, 1), (2, 5), (1, 130), (3, 700)])
def test_rope_positions(norm, D, rot, inter, B, S):
    heads, kv = 4, 2
    g = torch.Generator(device="cuda").manual_seed(D + S)
    W = (heads + 2 * kv) * D
    wide = _randn(g, B * S, W + 8).to(BF)
    y = wide[:, 8:] if S % 2 == 0 else wide[:, :W]  # rows of a wider buffer
    pos = torch.randint(0, 200000, (B, S), generator=g, device="cuda",
                        dtype=torch.int64 if S > 100 else torch.int32)
    scaling = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096}
    r = packed.Rotary(D, 10000.0, rotary_dim=rot, interleaved=inter, scaling=scaling, device="cuda")
    norms = tuple((1 + 0.3 * _randn(g, D)).to(BF) for _ in range(2)) if norm else None
    y = y.detach().requires_grad_(True)
    outs = packed.rope_positions(y, pos, r, heads, kv, norms=norms, eps=1e-5)
    grads = [_randn(g, *o.shape).to(BF) for o in outs]
    (dy,) = torch.autograd.grad(outs, y, grads)

    inv, amp = packed.rotary_frequencies(rot, 10000.0, scaling)
    y64 = y.detach().double().requires_grad_(True)
    want = rope_ref(y64, pos, inv, amp, heads, kv, D, rot, inter, norms, 1e-5)
    (dy64,) = torch.autograd.grad(want, y64, [t.double() for t in grads])
    # one rounding to bf16; before it about ten fp32 operations (with norms a sum
    # of D squares: D/16 more) on values of at most the head's largest `top`,
    # two of which are added
    fp32 = (10 + D / 16) * 2.0 ** -23
    for o, w in zip(outs, want):
        top = w.detach().abs().amax(-1, keepdim=True)
        _close("out", o, w.detach(), U * w.detach().abs() + fp32 * 2 * amp * top)
    top = dy64.abs().view(B * S, -1, D).amax(-1, keepdim=True).expand(-1, -1, D).reshape(B * S, W)
    _close("dy", dy, dy64, U * dy64.abs() + fp32 * 4 * amp * top)


def test_rope_far_positions():
    """Angles of positions near 2^31 keep their digits; int64 equals int32."""
    g = torch.Generator(device="cuda").manual_seed(2)
    pos = torch.tensor([[0, 1, 4095, 65537, 999983, 2 ** 30 + 1, 2 ** 31 - 1]], device="cuda")
    y = _randn(g, 7, 6 * 64).to(BF)
    r = packed.Rotary(64, 500000.0, device="cuda")
    a = packed.rope_positions(y, pos, r, 4, 1)
    b = packed.rope_positions(y, pos.int(), r, 4, 1)
    want = rope_ref(y.double(), pos, packed.rotary_frequencies(64, 500000.0)[0], 1.0, 4, 1, 64, 64,
                    False)
    for x, z, w in zip(a, b, want):
        assert torch.equal(x, z)
        # fp64 angles of up to 2^31 are off by 2^-22, theirs and ours
        top = w.abs().amax(-1, keepdim=True)
        _close("far", x, w, U * w.abs() + 2.0 ** -19 * top)


def test_rope_gradient_of_some_outputs():
    """A missing output gradient counts as zeros; values pass straight through."""
    g = torch.Generator(device="cuda").manual_seed(3)
    y = _randn(g, 9, 6 * 64).to(BF).requires_grad_(True)
    pos = torch.arange(9, device="cuda").view(1, 9)
    r = packed.Rotary(64, 10000.0, device="cuda")
    q, k, v = packed.rope_positions(y, pos, r, 4, 1)
    gv = _randn(g, *v.shape).to(BF)
    (dy,) = torch.autograd.grad(v, y, gv)
    assert bool((dy[:, :5 * 64] == 0).all())
    assert torch.equal(dy[:, 5 * 64:].view(1, 9, 1, 64).transpose(1, 2), gv)


def test_rope_graph_and_stream():
    g = torch.Generator(device="cuda").manual_seed(4)
    y = _randn(g, 40, 6 * 128).to(BF).requires_grad_(True)
    pos = torch.arange(20, device="cuda").repeat(2, 1)
    r = packed.Rotary(128, 10000.0, device="cuda")
    w = tuple((1 + 0.1 * _randn(g, 128)).to(BF) for _ in range(2))
    gs = [_randn(g, 2, h, 20, 128).to(BF) for h in (4, 1, 1)]

    def step():
        outs = packed.rope_positions(y, pos, r, 4, 1, norms=w)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, y, gs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            y.copy_(_randn(g, *y.shape))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)


def _moved(f, inputs):
    """Gradients of ``f`` over copies of ``inputs`` whose saved tensors are kept
    on the host and come back elsewhere, the places they had overwritten."""
    leaves = [t.detach().clone().requires_grad_() for t in inputs]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = f(*(t * 1 for t in leaves))
    junk = [torch.full_like(t, float("nan")) for t in leaves for _ in range(8)]
    outs = out if isinstance(out, tuple) else (out,)
    g = torch.Generator(device="cuda").manual_seed(3)
    ups = [torch.randn(o.shape, generator=g, device="cuda").to(o.dtype) for o in outs]
    grads = torch.autograd.grad(outs, leaves, ups)
    del junk
    return grads, ups


@pytest.mark.parametrize("kind", ["spans", "turned", "normed"])
def test_saved_tensors_that_a_hook_moved(kind):
    g = torch.Generator(device="cuda").manual_seed(11)
    B, S, H, KV, D = 2, 150, 4, 2, 64
    documents = torch.zeros(B, S, dtype=torch.int64).cuda()
    mask = packed.document_mask(documents)
    if kind == "spans":
        inputs = [_randn(g, B, h, S, D).to(BF) for h in (H, KV, KV)]
        slopes = torch.rand(H, generator=g, device="cuda")
        f = lambda q, k, v: packed.span_attention(q, k, v, 0.125, mask, slopes=slopes)  # noqa: E731
    else:
        inputs = [_randn(g, B * S, (H + 2 * KV) * D).to(BF)]
        norms = (_randn(g, D).to(BF), _randn(g, D).to(BF)) if kind == "normed" else None
        rotary = packed.Rotary(D, 1e4, device="cuda")
        f = lambda y: packed.rope_positions(y, mask.positions.clone(), rotary, H, KV,  # noqa: E731
                                            norms=norms)
    got, ups = _moved(f, inputs)
    leaves = [t.detach().clone().requires_grad_() for t in inputs]
    outs = f(*leaves)
    want = torch.autograd.grad(outs if isinstance(outs, tuple) else (outs,), leaves, ups)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_checkpointed_attention():
    """Recomputed operands take the place of the saved ones."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator(device="cuda").manual_seed(12)
    B, S, H, KV, D = 1, 200, 4, 2, 128
    mask = packed.document_mask((torch.arange(S)[None] // 70).cuda())
    rotary = packed.Rotary(D, 1e4, device="cuda")
    x, up = _randn(g, B * S, (H + 2 * KV) * D).to(BF), _randn(g, B, S, H * D).to(BF)

    def layer(y):
        q, k, v = packed.rope_positions(y * 1, mask.positions, rotary, H, KV)
        return packed.span_attention(q, k, v, D ** -0.5, mask)

    grads = []
    for run in (layer, lambda y: checkpoint(layer, y, use_reentrant=False)):
        y = x.clone().requires_grad_()
        grads += torch.autograd.grad(run(y), [y], up)
    assert torch.equal(*grads)


@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("cap", [1e3, 1e6, 1e20])
def test_caps_far_above_the_scores(dims, cap):
    """As good as no cap: what a tanh near 1 is off by must not be multiplied."""
    B, S, H = 1, 150, 2
    mask = packed.document_mask(torch.zeros(B, S, dtype=torch.int32, device="cuda"))
    _check(*_run(B, S, H, 2, *dims, mask, cap=cap, seed=7))


def test_scores_on_both_sides_of_a_cap():
    """Blocks whose scores lie in the linear part and well beyond the cap."""
    B, S, H, D, cap, scale = 1, 180, 2, 128, 2.0, 1.5 * 128 ** -0.5
    mask = packed.document_mask(torch.zeros(B, S, dtype=torch.int32, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (_randn(g, B, H, S, D) for _ in range(3))
    q[:, :, ::3] *= 3.0
    k[:, :, 64:] *= 0.05
    q, k, v, dout = q.to(BF), k.to(BF), v.to(BF), _randn(g, B, S, H * D).to(BF)
    want, bound = span_ref(q, k, v, scale, mask.key_start, mask.key_end, cap, None, dout)
    # 1 - tanh^2 is off by up to 2^-21 (four rounded fp32 steps around 1), whatever it is
    x, _, sees = span_scores(q.double(), k.double(), scale, mask.key_start, mask.key_end, cap, None)
    p = torch.softmax(torch.where(sees, x, -1e300), -1)
    do = dout.double().view(B, S, H, D).transpose(1, 2)
    dp = (do @ v.double().transpose(-1, -2)).abs()
    err = 2.0 ** -21 * p * (dp + (p * dp).sum(-1, keepdim=True)) * scale
    bound[1] = bound[1] + err @ k.double().abs()
    bound[2] = bound[2] + err.transpose(-1, -2) @ q.double().abs()
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = packed.span_attention(*leaves, scale, mask, cap=cap)
    _check((out, *torch.autograd.grad(out, leaves, dout)), want, bound)


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last document of the last heads."""
    S, H, KV, D, n, scale = 257 * 256, 264, 8, 128, 256, 128 ** -0.5
    G = H // KV
    assert S * H * D > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(21)
    mask = packed.document_mask((torch.arange(S, device="cuda")[None] // n).int())
    q, k, v, dout = (torch.zeros(s, dtype=BF, device="cuda")
                     for s in ((1, H, S, D), (1, KV, S, D), (1, KV, S, D), (1, S, H * D)))
    ends = [q[:, -G:, -n:], k[:, -1:, -n:], v[:, -1:, -n:], dout[:, -n:, -G * D:]]
    for t in ends:
        t.copy_(_randn(g, *t.shape))
    lo, hi = (t[:, -n:] - (S - n) for t in (mask.key_start, mask.key_end))
    want, bound = span_ref(*(t.contiguous() for t in ends[:3]), scale, lo, hi, None, None,
                           ends[3].contiguous())
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = packed.span_attention(*leaves, scale, mask)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    _check((out[:, -n:, -G * D:], dq[:, -G:, -n:], dk[:, -1:, -n:], dv[:, -1:, -n:]), want, bound)
    # everything else is made of zeros
    assert not bool(out[:, :-n].any()) and not bool(dq[:, :, :-n].any())


def test_rope_offsets_past_32_bits():
    """The last tokens of more than 2^31 elements, against those tokens alone."""
    T, H, KV, D, n = 360001, 32, 8, 128, 5
    W = (H + 2 * KV) * D
    assert T * W > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(22)
    rotary = packed.Rotary(D, 1e4, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")[None]
    y = torch.zeros(T, W, dtype=BF, device="cuda")
    y[-n:] = _randn(g, n, W).to(BF)
    last = y[-n:].clone().requires_grad_(True)
    outs = packed.rope_positions(last, pos[:, -n:].contiguous(), rotary, H, KV)
    ups = [_randn(g, *o.shape).to(BF) for o in outs]
    (want,) = torch.autograd.grad(outs, last, ups)
    y.requires_grad_(True)
    got = packed.rope_positions(y, pos, rotary, H, KV)
    for a, b in zip(got, outs):
        assert torch.equal(a[:, :, -n:], b)
    full = [torch.zeros_like(o) for o in got]
    for f, u in zip(full, ups):
        f[:, :, -n:] = u
    (dy,) = torch.autograd.grad(got, y, full)
    assert torch.equal(dy[-n:], want) and not bool(dy[:-n].any())


def test_one_mask_on_two_streams_at_once():
    """Passes on two streams over one mask, interleaved, against one after the other."""
    g = torch.Generator(device="cuda").manual_seed(23)
    B, S, H, KV, D = 2, 700, 8, 2, 128
    mask = packed.document_mask(_documents(random.Random(5), B, S, 20, 300, 7).cuda())
    sets = [[_randn(g, *s).to(BF) for s in ((B, H, S, D), (B, KV, S, D), (B, KV, S, D), (B, S, H * D))]
            for _ in range(2)]

    def one(q, k, v, dout):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed.span_attention(*leaves, 0.1, mask, cap=5.0)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    want = [one(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(one(*s))
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(res, want[i % 2]))
