"""Norms after and before a block part with gate and residual scale, against the
formula in 64 bits, its gradients through autograd and against differences."""
import pytest
import torch
from torch.autograd import forward_ad

from spilltune_amd import ops

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
NAMES = ("y", "residual", "post", "pre", "gate")


def formula(t, scale, eps):
    def rms(x, w):
        return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    z = t["y"] if t["post"] is None else rms(t["y"], t["post"])
    h = t["residual"] + scale * (z if t["gate"] is None else t["gate"] * z)
    return (h,) if t["pre"] is None else (h, rms(h, t["pre"]))


def inputs(shape, post=True, pre=True, gate=None, gate_dtype=BF, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    H = shape[-1]
    gates = {None: None, "channel": (H,), "row": (shape[0], 1, H), "token": shape[:-1] + (1,),
             "full": shape}
    t = {"y": r(*shape) * (0.1 + r(*shape[:-1], 1).abs()), "residual": 2 * r(*shape),
         "post": 1 + 0.3 * r(H) if post else None, "pre": 1 + 0.3 * r(H) if pre else None,
         "gate": None if gate is None else 0.5 + 0.4 * r(*gates[gate])}
    t = {n: None if v is None else v.to(gate_dtype if n == "gate" else BF).cuda()
         for n, v in t.items()}
    up = [r(*shape).to(BF).cuda() for _ in range(2 if pre else 1)]
    return t, up


def near(out, ref, what, sums=None, terms=0, parts=0.0):
    """Half a step of the output's type; 2^-17 of the row's largest for what fp32 rounds
    within a row (2^-24 a step, sums of at most 32 values a lane and 10 joins, a few
    products: below 2^7 steps); for sums over rows 2^-24 a step of the sum of the
    terms' sizes, and theirs.  ``parts``: the size of what a result is the difference
    of.  A norm's gradient is r (w - x mean(x w) r^2), whose two parts are equal but for
    eps in rows of one value: each is rounded at 2^-24 of r |w|, whatever is left."""
    assert out.shape == ref.shape, what
    ref = ref.double()
    bound = torch.finfo(out.dtype).eps / 2 * ref.abs()
    if sums is None:
        bound = bound + 2**-17 * (ref.abs().amax(-1, keepdim=True) + parts)
    else:
        bound = bound + (2**-17 + 2**-24 * terms) * sums
    worst = float(((out.double() - ref).abs() - bound).max())
    assert worst <= 0, (what, worst)


def check(t, up, scale=1.0, eps=1e-6):
    leaves = [n for n in NAMES if t[n] is not None]
    own = {n: None if v is None else v.detach().clone().requires_grad_(True) for n, v in t.items()}
    out = ops.residual_norms(own["y"], own["residual"], own["post"], own["pre"], gate=own["gate"],
                             scale=scale, eps=eps)
    out = (out,) if t["pre"] is None else out
    grads = torch.autograd.grad(out, [own[n] for n in leaves], up)
    ref = {n: None if v is None else v.detach().double().requires_grad_(True) for n, v in t.items()}
    want = formula(ref, scale, eps)
    ref_grads = dict(zip(leaves, torch.autograd.grad(want, [ref[n] for n in leaves],
                                                     [u.double() for u in up])))
    with torch.no_grad():
        for o, w, n in zip(out, want, ("h", "normed")):
            assert o.dtype == BF
            near(o, w, n)
        # sizes of the terms of the sums over rows
        H = t["y"].shape[-1]
        dH = ref_grads["residual"]
        yn = ref["y"] / (ref["y"].square().mean(-1, keepdim=True) + eps).sqrt() \
            if t["post"] is not None else ref["y"]
        z = yn if t["post"] is None else yn * ref["post"]
        gate = scale if t["gate"] is None else scale * ref["gate"]
        # fp32 errors of dH come from both of its parts
        parts = torch.zeros_like(dH[..., :1])
        if t["pre"] is not None:
            h = want[0]
            parts = (up[1].double() * ref["pre"] / (h.square().mean(-1, keepdim=True) + eps).sqrt()
                     ).abs().amax(-1, keepdim=True)
        big = dH.abs() + dH.abs().amax(-1, keepdim=True) + parts
        room = {"residual": parts, "y": (gate * big).abs().amax(-1, keepdim=True)}
        if t["post"] is not None:
            room["y"] = (gate * big * ref["post"] / (ref["y"].square().mean(-1, keepdim=True) + eps)
                         .sqrt()).abs().amax(-1, keepdim=True)
        size = {"post": (gate * big * yn).abs(), "gate": (scale * big * z).abs()}
        if t["pre"] is not None:
            size["pre"] = (up[1].double() * h / (h.square().mean(-1, keepdim=True) + eps).sqrt()).abs()
        rows = dH.numel() // H
        for n, g in zip(leaves, grads):
            assert g.dtype == t[n].dtype
            if n in ("y", "residual"):
                near(g, ref_grads[n], "d" + n, parts=room[n])
                continue
            s, shape = size[n], t[n].shape
            terms = rows
            if shape == s.shape:
                near(g, ref_grads[n], "d" + n, parts=s.amax(-1, keepdim=True))
                continue
            if n == "gate" and shape[-1] == 1 and H > 1:
                s, terms = s.sum(-1, keepdim=True), 64
            elif n == "gate" and len(shape) == 3:
                s = s.sum(1, keepdim=True)
            else:
                s = s.reshape(-1, H).sum(0)
            near(g, ref_grads[n], "d" + n, s.reshape(shape), terms)


@pytest.mark.parametrize("H", [1, 3, 8, 64, 100, 255, 257, 512, 520, 1000, 1001, 1024, 1032, 2048,
                               2056, 4095, 4096, 4097, 4104, 7168, 8192, 8200, 16383, 16384])
def test_sizes(H):
    check(*inputs((2, 5, H), seed=H), scale=0.22)


@pytest.mark.parametrize("gate_dtype", [BF, F32])
@pytest.mark.parametrize("gate", [None, "channel", "row", "token", "full"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("H", [72, 2049])
def test_forms(H, post, pre, gate, gate_dtype):
    check(*inputs((3, 7, H), post, pre, gate, gate_dtype, seed=H), scale=1.7)


@pytest.mark.parametrize("gate", [None, "channel", "row", "full"])
@pytest.mark.parametrize("H", [9, 1001, 8193, 12296, 16383])
def test_ragged_and_wide_rows(H, gate):
    check(*inputs((2, 9, H), gate=gate, gate_dtype=F32, seed=H), scale=0.7)


@pytest.mark.parametrize("shape,gate", [((1, 1, 4096), "channel"), ((700, 64), "channel"),
                                        ((5000, 3, 16), "row"), ((2, 1500, 136), "row"),
                                        ((3, 1, 40), "row"), ((4096,), None), ((4, 128), "token"),
                                        ((2, 3, 4, 5, 48), "full"), ((1300, 4096), "channel")])
def test_shapes_of_rows(shape, gate):
    check(*inputs(shape, gate=gate, seed=1))


def test_against_differences():
    """<gradient, direction> against central differences of the formula in 64 bits."""
    for gate in ("channel", "row", "token", "full"):
        t, up = inputs((2, 3, 40), gate=gate, gate_dtype=F32, seed=7)
        own = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        out = ops.residual_norms(own["y"], own["residual"], own["post"], own["pre"],
                                 gate=own["gate"], scale=0.7)
        grads = torch.autograd.grad(out, [own[n] for n in NAMES], up)
        for n, g in zip(NAMES, grads):
            d = torch.randn(t[n].shape, device="cuda", dtype=F64,
                            generator=torch.Generator("cuda").manual_seed(1))
            ends = []
            for sign in (1, -1):
                at = {m: v.double() for m, v in t.items()}
                at[n] = at[n] + sign * 1e-5 * d
                ends.append(sum((o * u.double()).sum() for o, u in zip(formula(at, 0.7, 1e-6), up)))
            slope = float(ends[0] - ends[1]) / 2e-5
            # each entry is off by half a step of its type, at most
            room = float((g.double() * d).abs().sum()) * 2**-8 + 1e-4
            assert abs(float((g.double() * d).sum()) - slope) <= room, (gate, n)


def test_one_of_two_results():
    t, up = inputs((4, 96), gate="channel", seed=2)
    for k in (0, 1):
        own = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        out = ops.residual_norms(own["y"], own["residual"], own["post"], own["pre"], gate=own["gate"])
        g = torch.autograd.grad(out[k], [own[n] for n in NAMES], up[k], allow_unused=True)
        ref = {n: v.double().requires_grad_(True) for n, v in t.items()}
        r = torch.autograd.grad(formula(ref, 1.0, 1e-6)[k], [ref[n] for n in NAMES], up[k].double(),
                                allow_unused=True)
        for n, a, b in zip(NAMES, g, r):
            assert (a is None) == (b is None), n
            if a is not None:
                assert ((a.double() - b).abs() <= 2**-8 * b.abs() + 2**-15 * b.abs().max()).all(), n


def test_some_leaves():
    """Only what requires a gradient gets one, and the same bits as with the others."""
    t, up = inputs((3, 200, 136), gate="channel", seed=3)
    full = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    out = ops.residual_norms(full["y"], full["residual"], full["post"], full["pre"],
                             gate=full["gate"])
    every = dict(zip(NAMES, torch.autograd.grad(out, list(full.values()), up)))
    for n in NAMES:
        own = {m: v.detach().requires_grad_(m == n) for m, v in t.items()}
        some = ops.residual_norms(own["y"], own["residual"], own["post"], own["pre"],
                                  gate=own["gate"])
        assert all(torch.equal(a, b) for a, b in zip(some, out))
        (g,) = torch.autograd.grad(some, [own[n]], up)
        assert torch.equal(g, every[n]), n
    with torch.no_grad():
        plain = ops.residual_norms(full["y"], full["residual"], full["post"], full["pre"],
                                   gate=full["gate"])
    assert all(not o.requires_grad and torch.equal(a, o) for a, o in zip(out, plain))


def test_values_that_are_not_finite_stay_in_their_row():
    t, up = inputs((4, 6, 80), gate="token", seed=4)
    clean = ops.residual_norms(t["y"], t["residual"], t["post"], t["pre"], gate=t["gate"])
    t["y"][1, 2, 3] = float("inf")
    t["residual"][2, 0, 5] = float("nan")
    t["y"][3, 1] = 0.0
    t["residual"][3, 1] = 0.0
    out = ops.residual_norms(t["y"], t["residual"], t["post"], t["pre"], gate=t["gate"])
    bad = torch.zeros(4, 6, dtype=torch.bool)
    bad[1, 2] = bad[2, 0] = True
    for o, c in zip(out, clean):
        assert o[1, 2].isnan().any() and o[2, 0].isnan().any() and (o[3, 1] == 0).all()
        same = ~bad.cuda()
        same[3, 1] = False
        assert torch.equal(o[same], c[same])


def test_layouts_and_streams():
    t, up = inputs((6, 5, 96), seed=5)
    want = ops.residual_norms(t["y"], t["residual"], t["post"], t["pre"])
    wide = torch.empty(6, 5, 200, dtype=BF, device="cuda")
    wide[..., 3:99] = t["y"]
    turned = t["residual"].transpose(0, 1).contiguous().transpose(0, 1)
    w = torch.empty(97, dtype=BF, device="cuda")
    w[1:] = t["post"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.residual_norms(wide[..., 3:99], turned, w[1:], t["pre"])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert ops.residual_norms(t["y"][:0], t["residual"][:0], t["post"]).shape == (0, 5, 96)
    e = t["y"][:0].clone().requires_grad_(True)
    p = t["post"].clone().requires_grad_(True)
    g = torch.autograd.grad(ops.residual_norms(e, e.detach(), p).sum(), [e, p])
    assert g[0].shape == e.shape and (g[1] == 0).all()


def test_captured_passes():
    t, up = inputs((3, 300, 264), gate="channel", seed=6)
    own = {n: v.detach().requires_grad_(True) for n, v in t.items()}

    def both():
        out = ops.residual_norms(own["y"], own["residual"], own["post"], own["pre"],
                                 gate=own["gate"], scale=0.3)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, list(own.values()), up))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = both()
    for k in range(3):
        with torch.no_grad():
            for v in own.values():
                v.add_(0.1 * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, both())), k


def test_refused_derivatives():
    t, up = inputs((2, 3, 16))
    y = t["y"].requires_grad_(True)
    h = ops.residual_norms(y, t["residual"])
    (g,) = torch.autograd.grad(h, [y], up[0], retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(h, [y], up[0], create_graph=True)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t["y"].detach(), up[0])
        with pytest.raises(NotImplementedError):
            ops.residual_norms(dual, t["residual"])


def test_offsets_past_32_bits():
    """More than 2^31 entries: the last rows as by themselves."""
    rows, H = 131100, 16384
    y = torch.zeros(rows, H, dtype=BF, device="cuda")
    res = torch.zeros_like(y)
    g = torch.Generator("cuda").manual_seed(1)
    y[-3:], res[-3:] = (torch.randn(3, H, generator=g, device="cuda").to(BF) for _ in range(2))
    w = torch.ones(H, dtype=BF, device="cuda")
    y.requires_grad_(True)
    h, n = ops.residual_norms(y, res, w, w)
    (dy,) = torch.autograd.grad([h, n], [y], [h.detach(), n.detach()])
    few = y.detach()[-3:].clone().requires_grad_(True)
    fh, fn = ops.residual_norms(few, res[-3:], w, w)
    (fd,) = torch.autograd.grad([fh, fn], [few], [fh.detach(), fn.detach()])
    assert torch.equal(h[-3:], fh) and torch.equal(n[-3:], fn) and torch.equal(dy[-3:], fd)
    assert (h[:5] == 0).all() and (dy[:5] == 0).all() and (h[65536:65541] == 0).all()
