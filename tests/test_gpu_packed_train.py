"""Packed rows through decoder layers, training and scoring: layer steps against
the CPU oracle with the documents' additive mask and restarted positions, a
packed row's training against its documents trained one by one."""
import random

import numpy as np
import pytest
import torch

from oracle import layer as OL
from oracle import mla as OMLA
from spilltune_amd import deepseek, engine, packed, slots
from spilltune_amd.recompute import streaming_block
from tests import test_gpu_layer as TL
from tests import test_gpu_mla as TM
from tests import test_gpu_train as TT

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _documents(B, S, seed):
    rng = random.Random(seed)
    d = torch.full((B, S), -1, dtype=torch.int64)
    for b in range(B):
        i, n = 0, 0
        while i < S - 7 * b:  # later rows end in padding
            d[b, i:min(i + rng.randint(3, S // 2), S - 7 * b)] = n
            n += 1
            i = int((d[b] >= 0).sum())
    return d


def _additive(documents):
    """[B,1,S,S] bf16: finfo.min where a token of another document, a later one
    or padding stands; a padded token sees itself (its row is not compared)."""
    S = documents.shape[1]
    at = torch.arange(S)
    sees = (documents[:, :, None] == documents[:, None, :]) & (documents >= 0)[:, :, None]
    sees = (sees & (at[:, None] >= at)) | torch.eye(S, dtype=torch.bool)
    return torch.where(sees, 0.0, torch.finfo(BF).min).to(BF)[:, None]


def _restarted(tables, positions):
    return tuple(torch.stack([t[0][p] for p in positions.long()]) for t in tables)


def _step(block, functional_args, hidden, dy, device):
    session = slots.ResidentSession([block], device)
    h = hidden.to(device).requires_grad_(True)
    with session.run():
        out = streaming_block(h, *functional_args, block.functional, block.kwargs,
                              session.reloader(block), block.adapters, block.index)
        out.backward(dy.to(device))
    torch.cuda.synchronize()
    session.close()
    return out.detach(), h.grad


def _compare(rel, cosine, block, lor, out, out_ref, dh, dh_ref, real):
    res = {"out": rel(out.cpu()[real], out_ref[real]), "dh": cosine(dh.cpu()[real], dh_ref[real])}
    for n, p in block.adapters.items():
        res[n + ".A"] = cosine(p.grad_A, lor[n].grad_A)
        res[n + ".B"] = cosine(p.grad_B, lor[n].grad_B)
    TL._assert(res)  # the layer steps' own criteria


@pytest.mark.parametrize("cfg,qk_norm,targets", [
    (TL.TINY, False, TL.PROJ),
    (TL.GQA, True, TL.PROJ),
    (dict(TL.GQA, r=32, alpha=64.0), True, TL.PROJ),  # q, k and v run one by one
    (TL.TINY, False, ("self_attn.q_proj", "self_attn.v_proj", "self_attn.o_proj"))])
def test_packed_dense_layer_step_vs_oracle(oracle_codec, cfg, qk_norm, targets):
    dev = torch.device("cuda:0")
    block, _ = TL.make_layer(cfg, 71, "nf4-g128", targets=targets, qk_norm=qk_norm)
    g = torch.Generator().manual_seed(72)
    B, S, H = cfg["B"], cfg["S"], cfg["H"]
    documents = _documents(B, S, 5)
    real = documents >= 0
    hidden, dy = (torch.randn(B, S, H, generator=g).to(BF) for _ in range(2))
    dy[~real] = 0
    rotary = packed.Rotary(cfg["D"], 500000.0, device=dev)
    positions, mask = packed.positions_and_masks(documents, rotary)
    lor = {n: OL.Lora(n, p.A.detach().cpu(), p.B.detach().cpu(), p.alpha)
           for n, p in block.adapters.items()}
    kw = dict(heads=cfg["heads"], kv_heads=cfg["kv"], head_dim=cfg["D"], eps=cfg["eps"],
              qk_norm=qk_norm)
    tables = _restarted(OL.rotary(1, S, cfg["D"], 500000.0, BF), mask.positions.cpu())
    out_ref, dh_ref = OL.streaming_step(hidden, tables, _additive(documents), dy,
                                        weights=TL.oracle_weights(block, oracle_codec), loras=lor,
                                        cfg=kw)
    out, dh = _step(block, (positions, mask), hidden, dy, dev)
    _compare(TL.rel, TL.cosine, block, lor, out, out_ref, dh, dh_ref, real)


def test_packed_mla_layer_step_vs_oracle(oracle_codec):
    dev = torch.device("cuda:0")
    c = TM._params(heads=4, nope=128, rope=64, vdim=128, kv_rank=128, q_rank=128, interleave=True,
                   moe=False, rope_cfg=TM.YARN)
    g = torch.Generator().manual_seed(81)
    B, S, H = 2, 96, 256
    block = deepseek.make_deepseek_block(0, TM._layer_weights(g, c, H, 128, 256, 16), codec="nf4-g128",
                                         parameters=c, rank=8, alpha=16.0, device=dev, generator=g)
    with torch.no_grad():
        for p in block.adapters.values():
            p.B.copy_(torch.randn(p.B.shape, generator=g) * 0.02)
    documents = _documents(B, S, 6)
    real = documents >= 0
    hidden, dy = (torch.randn(B, S, H, generator=g).to(BF) for _ in range(2))
    dy[~real] = 0
    _, mask = deepseek.packed_positions_and_masks(documents, rope=c["rope_cfg"], rope_dim=64,
                                                  device=dev)
    tables = _restarted(OMLA.rotary(1, S, c["rope_cfg"], 64, BF), mask.positions.cpu())
    lor = {n: OL.Lora(n, p.A.detach().cpu(), p.B.detach().cpu(), p.alpha)
           for n, p in block.adapters.items()}
    out_ref, dh_ref = OMLA.streaming_step(hidden, tables, _additive(documents), dy, parameters=c,
                                          weights=TM._oracle_weights(block, oracle_codec), loras=lor)
    out, dh = _step(block, (tuple(t.to(dev) for t in tables), mask), hidden, dy, dev)
    _compare(TM._rel, TM._cos, block, lor, out, out_ref, dh, dh_ref, real)


def _model(dev, rotary=None):
    layers, emb, norm, head = TT.tiny_weights(99)
    c = TT.CFG
    model = engine.DenseModel(embedding=emb, norm=norm, head=head, layers=layers, heads=c["heads"],
                              kv_heads=c["kv"], head_dim=c["D"], eps=c["eps"], theta=c["theta"],
                              rank=c["r"], alpha=c["alpha"], targets=TT.TARGETS, device=dev,
                              rotary=rotary)
    g = torch.Generator().manual_seed(3)
    loras = []
    for block in model.blocks:
        lo = {}
        for name in sorted(block.adapters):
            p = block.adapters[name]
            A, B = torch.randn(p.A.shape, generator=g) * 0.05, torch.randn(p.B.shape, generator=g) * 0.05
            with torch.no_grad():
                p.A.copy_(A)
                p.B.copy_(B)
            lo[name] = OL.Lora(name, A, B, p.alpha)
        loras.append(lo)
    return model, loras, (emb, norm, head)


def _packed_row(vocab):
    g = torch.Generator().manual_seed(7)
    sizes = (40, 3, 65, 1, 17)
    docs = [torch.randint(0, vocab, (1, n), generator=g) for n in sizes]
    ids = torch.cat(docs + [torch.zeros(1, 6, dtype=torch.int64)], 1)
    documents = torch.cat([torch.full((1, n), i) for i, n in enumerate(sizes)]
                          + [torch.full((1, 6), -1)], 1)
    return docs, ids, documents


@pytest.mark.parametrize("how", ["microbatch", "layer_major", "objective"])
def test_packed_training_equals_training_its_documents(oracle_codec, how):
    """One packed row a step against the oracle training the documents one by one
    as an accumulation window: the loss curves of 10 steps to within 1e-2."""
    dev = torch.device("cuda:0")
    model, loras, (emb, norm, head) = _model(dev)
    docs, ids, documents = _packed_row(TT.CFG["vocab"])
    weights = [TT.decoded(b, oracle_codec) for b in model.blocks]
    session = slots.ResidentSession(model.blocks, dev)
    n = sum(d.shape[1] - 1 for d in docs)

    def objective(r):
        return -r.logprobs.sum() / n
    # the row's labels run across the documents' starts and the padding
    gpu = engine.train(model, session, [(ids, ids.clone(), documents)], steps=10, lr=2e-3,
                       token_chunk=64, layer_major=how == "layer_major",
                       objective=objective if how == "objective" else None)
    c = TT.CFG
    rows = [(d, d.clone()) for d in docs if d.shape[1] > 1]
    cpu = OL.train_reference(emb, norm, head, weights, loras, rows,
                             cfg=dict(heads=c["heads"], kv_heads=c["kv"], head_dim=c["D"],
                                      eps=c["eps"]),
                             theta=c["theta"], steps=10, lr=2e-3, token_chunk=64,
                             accumulation=len(rows))
    diff = np.abs(np.array(gpu) - np.array(cpu)).max()
    print(f"loss {gpu[0]:.4f}->{gpu[-1]:.4f}, oracle {cpu[0]:.4f}->{cpu[-1]:.4f}, {diff:.2e}")
    assert diff <= 1e-2, (diff, gpu, cpu)
    session.close()


def test_scores_of_packed_documents(oracle_codec):
    """A document's scores do not move with its neighbours' tokens (the same
    bits) and agree with the oracle's loss on it alone; -100 places are 0."""
    dev = torch.device("cuda:0")
    rotary = packed.Rotary(TT.CFG["D"], TT.CFG["theta"], device=dev)
    model, loras, (emb, norm, head) = _model(dev, rotary)
    docs, ids, documents = _packed_row(TT.CFG["vocab"])
    session = slots.ResidentSession(model.blocks, dev)
    with session.run():
        a = engine.score(model, session, ids, documents=documents, top=3)
        other = ids.clone()
        other[:, 43:108] = (other[:, 43:108] + 1) % TT.CFG["vocab"]  # document 2
        b = engine.score(model, session, other, documents=documents, top=3)
    keep = torch.ones(ids.shape[1] - 1, dtype=torch.bool)
    keep[42:108] = False  # places whose token or context is of document 2
    for x, y in zip(a, b):
        assert torch.equal(x[:, keep], y[:, keep])
    assert not torch.equal(a.logprobs[:, 44:107], b.logprobs[:, 44:107])
    starts = [39, 42, 107, 108] + list(range(125, 131))
    assert bool((a.logprobs[0, starts] == 0).all())
    weights = [TT.decoded(x, oracle_codec) for x in model.blocks]
    c, at = TT.CFG, 0
    for d in docs:
        n = d.shape[1]
        if n > 1:
            want = OL.train_reference(emb, norm, head, weights, loras, [(d, d.clone())],
                                      cfg=dict(heads=c["heads"], kv_heads=c["kv"], head_dim=c["D"],
                                               eps=c["eps"]), theta=c["theta"], steps=1, lr=0.0)[0]
            got = -float(a.logprobs[0, at:at + n - 1].mean())
            assert abs(got - want) <= 1e-2, (n, got, want)
        at += n
    session.close()


def test_score_of_plain_rows_is_the_loss():
    """Without documents score() sums to the training loss of the same rows."""
    dev = torch.device("cuda:0")
    model, _, _ = _model(dev)
    ids = torch.randint(0, TT.CFG["vocab"], (2, 50), generator=torch.Generator().manual_seed(1))
    session = slots.ResidentSession(model.blocks, dev)
    with session.run():
        r = engine.score(model, session, ids)
        loss, _ = engine.microbatch(model, session, ids, ids, normalization=98, token_chunk=64)
    # the loss reads logits rounded to bf16: |logit| < 8, half a step 2^-8 of it,
    # in both terms of each of the averaged differences
    assert abs(-float(r.logprobs.sum()) / 98 - loss) <= 2 * 8 * 2.0 ** -8
    session.close()
