"""Objectives on token log probabilities know their labels, the window's count of
them and their row: terms on the entropy can leave out padding and the places
between documents."""
import numpy as np
import pytest
import torch

from spilltune_amd import engine, ops, packed, slots


def test_objective_is_told_labels_normalization_and_item(monkeypatch):
    def values(hidden, head, tokens, **kw):
        z = torch.zeros(tokens.shape)
        return ops.TokenLogProbs(z, z + 1, z[..., None][..., :0], z.long()[..., None][..., :0])
    monkeypatch.setattr(ops, "token_logprobs", values)
    documents = torch.tensor([[0, 0, 0, 1, 1, -1]])
    labels = packed.document_labels(torch.tensor([[5, -100, 7, 8, 9, 0]], dtype=torch.int32), documents)
    seen = []

    def objective(r):
        seen.append(r)
        assert isinstance(r, ops.TokenLogProbs) and len(r) == 4
        return (r.entropy * (r.labels != -100)).sum() / r.normalization
    model = type("M", (), {"head": None})
    loss = engine._terminal(model, torch.zeros(1, 6, 8), labels, normalization=4, token_chunk=64,
                            objective=objective, item="row 3")
    assert seen[0].labels.tolist() == [[-100, 7, -100, 9, -100]]
    assert seen[0].labels.dtype == torch.int64 and seen[0].item == "row 3"
    assert float(loss) == 2 / 4


def test_names_of_a_window_fit():
    model = type("M", (), {"device": torch.device("cpu")})
    with pytest.raises(ValueError, match="3 names for 2"):
        engine.window_layer_major(model, None, [(None, None)] * 2, normalization=1, token_chunk=64,
                                  objective=lambda r: 0, names=[0, 1, 2])


@pytest.mark.gpu
@pytest.mark.parametrize("layer_major", [False, True])
def test_entropy_term_of_a_packed_row_is_its_documents(layer_major):
    """Training on log probabilities and an entropy bonus: one padded packed row a
    step against its documents as an accumulation window, in another order of the
    rows too; loss curves of 10 steps to within 1e-2, as for the cross-entropy."""
    from tests.test_gpu_packed_train import _model, _packed_row
    from tests.test_gpu_train import CFG
    dev = torch.device("cuda:0")
    docs, ids, documents = _packed_row(CFG["vocab"])
    rows = [(d, d.clone()) for d in docs if d.shape[1] > 1]
    # a weight of each document, found by its row's number
    weight = [0.5, 2.0, 1.0, 1.5]

    def term(r, w):
        keep = r.labels != -100
        return (w * ((0.3 * r.entropy - r.logprobs) * keep)).sum() / r.normalization
    items = []

    def alone(r):
        items.append(r.item)
        return term(r, weight[r.item])
    w = torch.zeros(ids.shape, device=dev)
    for n, i in enumerate(i for i, d in enumerate(docs) if d.shape[1] > 1):
        w[(documents == i).to(dev)] = weight[n]

    def together(r):
        assert r.item == 0 and r.normalization == sum(d.shape[1] - 1 for d, _ in rows)
        return term(r, w[:, 1:])
    curves = []
    for data, objective, accumulation in (([(ids, ids.clone(), documents)], together, 1),
                                          (rows, alone, len(rows))):
        model, _, _ = _model(dev)
        session = slots.ResidentSession(model.blocks, dev)
        curves.append(engine.train(model, session, data, steps=10, lr=2e-3, token_chunk=64,
                                   accumulation=accumulation, layer_major=layer_major,
                                   objective=objective))
        session.close()
    assert items == [0, 1, 2, 3] * 10
    diff = np.abs(np.array(curves[0]) - np.array(curves[1])).max()
    print(curves[0][0], curves[0][-1], diff)
    assert diff <= 1e-2, curves
