"""A trained table under weight decay: the padding token's row is not trained."""
import math
from types import SimpleNamespace

import pytest
import torch

from spilltune_amd import engine, muon


@pytest.mark.parametrize("row", [None, 0, 3, 6])
@pytest.mark.parametrize("through", ["adamw", "muon"])
def test_padding_row_keeps_its_values(row, through):
    g = torch.Generator().manual_seed(1)
    w, grad = torch.randn(7, 5, generator=g), torch.randn(7, 5, generator=g)
    if row is not None:
        grad[row] = 0  # as its gradient is formed
    table = SimpleNamespace(weight=w.clone(), grad=grad, m=torch.zeros(7, 5), v=torch.zeros(7, 5),
                            padding_idx=row)
    adamw = engine.AdamW(lr=0.1, weight_decay=0.5)
    step = adamw.step if through == "adamw" else muon.Muon(table=adamw).step
    want, m, v = w.double(), 0.0, 0.0
    for n in range(1, 4):
        step({"embedding": table})
        m, v = 0.9 * m + 0.1 * grad.double(), 0.999 * v + 0.001 * grad.double().square()
        root = (v / (1 - 0.999**n)).sqrt()
        want = want * (1 - 0.1 * 0.5) - 0.1 * (m / (1 - 0.9**n)) / (root + 1e-8)
    if row is not None:
        want[row] = w[row].double()
        assert torch.equal(table.weight[row], w[row])
    # three steps of some ten fp32 operations on values below 4
    assert (table.weight.double() - want).abs().max() < 30 * 4 * 2**-24
    assert adamw.step_count == 3 and math.isfinite(float(table.weight.sum()))
