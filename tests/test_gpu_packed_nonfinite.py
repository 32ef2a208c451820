"""Attention over runs of keys whose operands hold infinities and NaN: what a
query sees reaches it, what it does not see does not, and a pass over them takes a
bounded number of times the usual time."""
import random

import pytest
import torch

from spilltune_amd import packed
from tests._packed_ref import span_ref, span_scores
from tests.test_gpu_packed import _documents, _randn

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
INF, NAN = float("inf"), float("nan")


def _same_kind(name, got, want, bound):
    """NaN and infinities where the exact sum has them, finite values within the
    bound elsewhere."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (name, "NaN")
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)), (name, "inf")
    assert torch.equal(torch.isneginf(got), torch.isneginf(want)), (name, "-inf")
    ok = torch.isfinite(want)
    err = (got - want)[ok].abs()
    assert bool((err <= bound[ok] + 1e-30).all()), (name, float(err.max()))


def _seen_sums(weights, sees, rows):
    """sum over the seen j of weights[i,j] rows[j] (an unseen row adds nothing,
    whatever it holds), float64 [..., i, d]."""
    terms = torch.where(sees[..., None], weights[..., None] * rows[..., None, :, :], 0.0)
    return terms.sum(-2)


@pytest.mark.parametrize("dims,group", [((64, 64), 2), ((128, 128), 4), ((192, 128), 1), ((192, 128), 2)])
@pytest.mark.parametrize("cap,bias", [(None, False), (5.0, False), (None, True), (5.0, True)])
@pytest.mark.parametrize("window", [None, 9])
def test_kinds_of_sums(dims, group, cap, bias, window):
    """Values and output gradients with a few infinities and NaN (weights are all
    above 0): outputs and the values' gradients are the sums over the seen pairs."""
    (DQ, DV), B, S, KV = dims, 2, 83, 2
    H = KV * group
    g = torch.Generator(device="cuda").manual_seed(DQ + group)
    rng = random.Random(DQ + group)
    q, k, v = (_randn(g, B, n, S, d).to(BF) for n, d in ((H, DQ), (KV, DQ), (KV, DV)))
    dout = _randn(g, B, S, H * DV).to(BF)
    mask = packed.document_mask(_documents(rng, B, S, 5, 50, 4).cuda(), window=window)
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device="cuda") if bias else None
    scale, runs = DQ ** -0.5, (mask.key_start, mask.key_end)
    _, bound = span_ref(q, k, v, scale, *runs, cap, slopes, dout)
    for t, rows in ((v, (B, KV, S)), (dout, (B, S))):
        for _ in range(12):
            at = tuple(rng.randrange(n) for n in rows)
            t[at][rng.randrange(t.shape[-1])] = rng.choice([INF, -INF, NAN])
    x, _, sees = span_scores(q.double(), k.double().repeat_interleave(group, 1), scale, *runs, cap, slopes)
    p = torch.where(sees, torch.softmax(x, -1), 0.0)  # an empty row's NaN too
    sees = sees.expand_as(p)
    want = _seen_sums(p, sees, v.double().repeat_interleave(group, 1))
    do = dout.double().view(B, S, H, DV).transpose(1, 2)
    want_dv = _seen_sums(p.transpose(-1, -2), sees.transpose(-1, -2), do).view(B, KV, group, S, DV).sum(2)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = packed.span_attention(*leaves, scale, mask, cap=cap, slopes=slopes)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    # a finite sum sees none of the edited places: the bound before the edit holds
    _same_kind("out", out, want.transpose(1, 2).reshape(B, S, -1), bound[0])
    _same_kind("dv", dv, want_dv, bound[3])
    # a query's score gradients are finite where its keys' values and its own gradient are
    bad_v = (~torch.isfinite(v.detach())).any(-1).repeat_interleave(group, 1)          # [B,H,S]
    bad_o = (~torch.isfinite(dout.view(B, S, H, DV))).any(-1).transpose(1, 2)
    hit = bad_o | (sees & bad_v[:, :, None, :]).any(-1)                                # [B,H,S] queries
    hit &= (mask.key_end - mask.key_start > 1)[:, None]                                # dS of one key is 0
    assert torch.equal(torch.isfinite(dq).all(-1), ~hit)
    reached = (sees & hit[..., None]).any(-2).view(B, KV, group, S).any(2)
    assert torch.equal(torch.isfinite(dk).all(-1), ~reached)


def _pass_ms(q, k, v, dout, mask, scale):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def go():
        out = packed.span_attention(*leaves, scale, mask)
        return (out, *torch.autograd.grad(out, leaves, dout))
    times = []
    for _ in range(3):
        a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        res = go()
        z.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(z))
    return min(times), res


@pytest.mark.parametrize("dims,H,KV", [((64, 64), 8, 8), ((128, 128), 8, 2), ((192, 128), 8, 8)])
@pytest.mark.parametrize("what", ["all values", "one key", "one value", "everything"])
def test_time_of_a_diverged_pass_is_bounded(dims, H, KV, what):
    """One causal document whose NaN every query, or every later one, sees: the
    answer is NaN, after one more walk of the same tiles (of half more products,
    and their operands sorted by kind: five to eight times the usual time)."""
    (DQ, DV), S = dims, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (_randn(g, 1, n, S, d).to(BF) for n, d in ((H, DQ), (KV, DQ), (KV, DV)))
    dout = _randn(g, 1, S, H * DV).to(BF)
    mask = packed.document_mask(torch.zeros(1, S, dtype=torch.int32, device="cuda"))
    usual, _ = _pass_ms(q, k, v, dout, mask, DQ ** -0.5)
    if what == "all values":
        v.fill_(NAN)
    elif what == "one key":
        k[:, :, 3] = NAN
    elif what == "one value":
        v[:, :, 3, 5] = NAN
    else:
        for t in (q, k, v, dout):
            t.fill_(NAN)
    took, (out, dq, dk, dv) = _pass_ms(q, k, v, dout, mask, DQ ** -0.5)
    print(f"{what} {dims}: {usual:.3f} ms, with NaN {took:.3f} ms")
    heads = out.view(S, H, DV)
    if what == "one value":
        assert bool(torch.isnan(heads[3:, :, 5]).all())
        assert bool(torch.isfinite(heads[:3]).all()) and bool(torch.isfinite(heads[..., :5]).all())
    else:
        first = 3 if what == "one key" else 0
        assert bool(torch.isnan(heads[first:]).all()) and bool(torch.isfinite(heads[:first]).all())
    # (pair by pair it would be some thousand times, and grow with the length)
    assert bool(torch.isnan(dk).any()) and took <= 40 * usual
