"""Norms around a part with gates of many rows."""
import pytest
import torch

from spilltune_amd import ops
from tests.test_gpu_residual_norms import check, formula, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [65534, 65600])
def test_more_frozen_gate_rows_than_are_trained(groups):
    """Learnt norms beside a frozen gate a row: the same as with the gate of every entry.
    Forty rows have a gradient, among them the last ones."""
    H = 16
    t, up = inputs((groups, 2, H), gate="row")
    some = torch.zeros(groups, 1, 1, dtype=torch.bool, device="cuda")
    some[[0, 1, 255, 4096, *range(20000, 20010), *range(groups - 6, groups)]] = True
    up = [u * some for u in up]
    res = []
    for gate in (t["gate"], t["gate"].expand(groups, 2, H).contiguous()):
        own = [t[n].clone().requires_grad_(True) for n in ("y", "residual", "post", "pre")]
        out = ops.residual_norms(own[0], own[1], own[2], own[3], gate=gate, scale=0.7)
        res.append((out, torch.autograd.grad(out, own, up)))
    for a, b in zip(res[0][0] + res[0][1][:2], res[1][0] + res[1][1][:2]):
        assert torch.equal(a, b)
    # the rows' terms, formed alike by both, in 64 bits
    ref = {n: v.double() for n, v in t.items()}
    for n in ("post", "pre"):
        ref[n] = ref[n].expand(groups, 2, H).contiguous().requires_grad_(True)
    terms = torch.autograd.grad(formula(ref, 0.7, 1e-6), [ref["post"], ref["pre"]],
                                [u.double() for u in up])
    for a, b, term in zip(res[0][1][2:], res[1][1][2:], terms):
        # fp32 sums of forty terms (the others are zeros) in two orders, each rounded to bf16
        size = term.abs().sum((0, 1))
        assert ((a.double() - b.double()).abs() <= 2**-7 * b.double().abs() + 2 * 40 * 2**-24 * size
                ).all()
        # a row's terms are within 2^-14 of its largest: see near() there
        room = 2**-14 * 4 * term.abs().amax(-1).sum()
        want = term.sum((0, 1))
        assert ((a.double() - want).abs() <= 2**-8 * want.abs() + room).all()
    with pytest.raises(ValueError, match="65534"):
        gate = t["gate"].clone().requires_grad_(True)
        torch.autograd.grad(ops.residual_norms(t["y"], t["residual"], t["post"], t["pre"], gate=gate),
                            [gate], up)


def test_most_trained_gate_rows():
    t, up = inputs((65533, 2, 8), gate="row")
    check(t, up, scale=0.5)
