"""A trained embedding's padding row through training with weight decay."""
import pytest
import torch

from spilltune_amd import engine, muon, slots
from tests.test_gpu_adapted_step import _model, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_muon", [False, True])
def test_training_with_decay_leaves_the_padding_row(with_muon):
    dev = torch.device("cuda:0")
    model = _model(dev)
    before = model.embedding.weight.clone()
    session = slots.Q4SlotSession(model.blocks, dev, host_budget_bytes=1 << 34,
                                  device_budget_bytes=1 << 34, slots=2)
    table = engine.AdamW(lr=1e-3, weight_decay=0.1)
    engine.train(model, session, _rows(), steps=3, accumulation=2,
                 optimizer=muon.Muon(lr=1e-3, weight_decay=0.1, table=table) if with_muon else table)
    session.close()
    after = model.embedding.weight
    assert torch.equal(after[0], before[0]) and before[0].abs().max() > 0
    seen = torch.cat([r[0].reshape(-1) for r in _rows()]).unique()
    never = [i for i in range(1, 304) if i not in set(seen.tolist())]
    # rows that never occur decay alone: three products of fp32 numbers
    assert never and torch.allclose(after[never], before[never] * (1 - 1e-4)**3, rtol=1e-6, atol=0)
