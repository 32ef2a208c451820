"""A model turns plain and packed rows by one rotary embedding."""
import pytest
import torch

from spilltune_amd import dense, engine, packed, slots

BF = torch.bfloat16


def _plain(rotary, device="cpu"):
    z = torch.zeros(8, 16, dtype=BF)
    return engine.DenseModel(embedding=z, norm=z[0], head=z, blocks=[], heads=2, kv_heads=1,
                             head_dim=64, eps=1e-6, theta=1e4, rank=1, alpha=1.0, targets=(),
                             device=device, rotary=rotary)


def test_plain_rows_take_the_models_rotary():
    valid = torch.ones(2, 5, dtype=torch.bool)
    valid[1, 3:] = False
    rotary = packed.Rotary(64, 1e4, rotary_dim=32, device="cpu")
    positions, masks = _plain(rotary).positions_and_masks(valid)
    assert isinstance(positions, packed.Positions) and positions.rotary is rotary
    assert positions.positions.is_contiguous()
    assert positions.positions.tolist() == [[0, 1, 2, 3, 4]] * 2
    assert masks["full_attention"].lengths.tolist() == [5, 3]
    (cos, sin), _ = _plain(None).positions_and_masks(valid)
    want, _ = dense.positions_and_masks(valid, head_dim=64, theta=1e4, device="cpu")
    assert torch.equal(cos, want[0]) and torch.equal(sin, want[1])


SCALED = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 64}


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{"rotary_dim": 16}, {"scaling": SCALED}, {"interleaved": True}])
def test_a_plain_row_scores_as_one_document(kw):
    """The same row without documents and as one document.  The two attention
    kernels round their bf16 outputs apart: half a step, 2^-8, of logits below 8,
    in the logit and in the log-sum-exp; on the average 1e-2, as in training."""
    from tests.test_gpu_packed_train import _model
    from tests.test_gpu_train import CFG
    dev = torch.device("cuda:0")
    model, _, _ = _model(dev, packed.Rotary(CFG["D"], CFG["theta"], device=dev, **kw))
    ids = torch.randint(0, CFG["vocab"], (2, 90), generator=torch.Generator().manual_seed(4))
    session = slots.ResidentSession(model.blocks, dev)
    with session.run():
        plain = engine.score(model, session, ids).logprobs.double()
        packed_row = engine.score(model, session, ids,
                                  documents=torch.zeros_like(ids)).logprobs.double()
        loss, _ = engine.microbatch(model, session, ids, ids, normalization=178, token_chunk=64)
    session.close()
    print("mean difference", float((plain - packed_row).mean()),
          "rms", float((plain - packed_row).square().mean().sqrt()))
    assert abs(float((plain - packed_row).mean())) <= 1e-2
    assert float((plain - packed_row).square().mean().sqrt()) <= 2 * 8 * 2.0 ** -8
    assert abs(loss + float(packed_row.mean())) <= 2 * 8 * 2.0 ** -8


@pytest.mark.gpu
def test_packed_rows_leave_a_plain_models_tables():
    """A model without a rotary of its own turns plain rows by its bf16 tables,
    also after it has seen packed rows."""
    from tests.test_gpu_packed_train import _model
    dev = torch.device("cuda:0")
    model, _, _ = _model(dev)
    model.packed_positions_and_masks(torch.zeros(1, 8, dtype=torch.int64))
    rot, _ = model.positions_and_masks(torch.ones(1, 8, dtype=torch.bool))
    assert isinstance(rot, tuple)


def test_an_adapters_context_bounds_documents_not_rows():
    from spilltune_amd.adapter import ArchiveDenseAdapter
    adapter = object.__new__(ArchiveDenseAdapter)  # nothing below needs an archive or a GPU
    adapter.config = {"max_positions": 8, "head_dim": 64, "theta": 1e4}
    adapter.device, adapter._rotary = torch.device("cpu"), None
    docs = torch.tensor([[0] * 8 + [1] * 5 + [-1] * 4])
    with pytest.raises(ValueError, match="must be on the GPU"):  # past the context check
        adapter.packed_positions_and_masks(docs)
    for bad in (torch.tensor([[0] * 9 + [1] * 3]), torch.zeros(9, dtype=torch.int64)):
        with pytest.raises(ValueError, match="beyond configured context"):
            adapter.packed_positions_and_masks(bad)


def test_a_rotary_given_later_turns_both(monkeypatch):
    model = _plain(None)
    monkeypatch.setattr(packed, "positions_and_masks", lambda documents, rotary, **kw: (rotary, None))
    docs, valid = torch.zeros(1, 4, dtype=torch.int64), torch.ones(1, 4, dtype=torch.bool)
    first, _ = model.packed_positions_and_masks(docs)
    assert first.rotary_dim == 64 and model.packed_positions_and_masks(docs)[0] is first
    assert isinstance(model.positions_and_masks(valid)[0], tuple)
    model.rotary = packed.Rotary(64, 1e4, rotary_dim=32, device="cpu")
    assert model.packed_positions_and_masks(docs)[0] is model.rotary
    assert model.positions_and_masks(valid)[0].rotary is model.rotary
