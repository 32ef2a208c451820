"""A training step with everything around the projections: a trained, scaled
embedding, norms on both sides of a block's parts, balanced experts and
orthogonalised updates -- layer by layer against plain torch, and together
through the engine."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from spilltune_amd import dense, engine, lora, moe, muon, packed, slots
from spilltune_amd.embedding import TokenEmbedding
from spilltune_amd.recompute import streaming_block

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
H, HEADS, KV, D, I, E, K, EPS = 256, 4, 2, 64, 384, 8, 2, 1e-6
ATTENTION = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj")


def weights(g, experts=False, post=True, gates=False):
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w = {n + ".weight": 0.03 * r(*s) for n, s in zip(ATTENTION, (
        (HEADS * D, H), (KV * D, H), (KV * D, H), (H, HEADS * D)))}
    if experts:
        w["mlp.gate.weight"] = r(E, H) * 2 * H**-0.5
        w["mlp.experts.gate_up_proj"] = 0.03 * r(E, 2 * 128, H)
        w["mlp.experts.down_proj"] = 0.03 * r(E, H, 128)
    else:
        for n, s in (("gate", (I, H)), ("up", (I, H)), ("down", (H, I))):
            w[f"mlp.{n}_proj.weight"] = 0.03 * r(*s)
    names = ["input_layernorm", "post_attention_layernorm"]
    if post:
        names += ["pre_feedforward_layernorm", "post_feedforward_layernorm"]
    for n in names:
        w[n + ".weight"] = 1 + 0.2 * r(H)
    if gates:
        for n in ("self_attn.output_gate", "mlp.output_gate"):
            w[n] = 0.5 + 0.3 * r(H)
    return w


def plain_block(x, w, loras, post, scale, gates):
    """The block in 32 bits: x [B, S, H], decoded weights, {name: (A, B, scale)}."""
    B, S, _ = x.shape

    def norm(v, name):
        return v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * w[name + ".weight"]

    def proj(v, name):
        y = F.linear(v, w[name + ".weight"])
        if name in loras:
            a, b, s = loras[name]
            y = y + s * F.linear(F.linear(v, a), b)
        return y

    def turn(t):
        inv = 1.0 / 10000.0 ** (torch.arange(0, D, 2) / D)
        angle = torch.arange(S)[:, None] * inv
        c, s = (torch.cat((f, f), -1) for f in (angle.cos().to(BF).float(), angle.sin().to(BF).float()))
        half = torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1)
        return t * c + half * s
    n = norm(x, "input_layernorm")
    q, k, v = (proj(n, f"self_attn.{p}_proj").view(B, S, -1, D).transpose(1, 2) for p in "qkv")
    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
    score = (q @ k.mT) * D**-0.5
    score = score.masked_fill(torch.ones(S, S).triu(1).bool(), -math.inf)
    att = (score.softmax(-1) @ v).transpose(1, 2).reshape(B, S, -1)

    def add(res, y, name, gate):
        y = norm(y, name) if post else y
        return res + scale * (y * w[gate] if gates else y)
    h = add(x, proj(att, "self_attn.o_proj"), "post_attention_layernorm", "self_attn.output_gate")
    n = norm(h, "pre_feedforward_layernorm" if post else "post_attention_layernorm")
    y = proj(F.silu(proj(n, "mlp.gate_proj")) * proj(n, "mlp.up_proj"), "mlp.down_proj")
    return add(h, y, "post_feedforward_layernorm", "mlp.output_gate")


def decoded(block, oracle_codec):
    out = {}
    for name, entry in block.storage_specs.items():
        spec = entry["spec"]
        bits = oracle_codec.decode4(block.host_weights[entry["parts"]["payload"]].numpy(),
                                    block.host_weights[entry["parts"]["scales"]].numpy(),
                                    spec["numel"], lut=oracle_codec.NF4_LUT)
        out[name] = torch.from_numpy(np.asarray(bits).astype(np.int16)).view(BF).view(spec["shape"])
    out.update({k: v for k, v in block.host_weights.items() if not k.startswith("@")})
    return {k: v.float() for k, v in out.items()}


def _cos(a, b):
    return float(F.cosine_similarity(a.double().cpu().flatten(), b.double().cpu().flatten(), dim=0))


@pytest.mark.parametrize("post,scale,gates,targets", [
    (True, 1.0, False, lora.ALL_DENSE_TARGETS), (True, 0.5, True, lora.DEFAULT_DENSE_TARGETS),
    (False, 0.22, False, lora.ALL_DENSE_TARGETS), (False, 1.0, True, lora.DEFAULT_DENSE_TARGETS)])
def test_block_with_norms_around_its_parts(oracle_codec, post, scale, gates, targets):
    """The layer steps' own criteria: outputs to 2e-2, gradients to a cosine of 0.999."""
    dev = torch.device("cuda:0")
    g = torch.Generator().manual_seed(11)
    block = slots.make_dense_block(0, weights(g, post=post, gates=gates), codec="nf4-g128", heads=HEADS,
                                   kv_heads=KV, head_dim=D, eps=EPS, rank=8, alpha=16.0,
                                   targets=targets, device=dev, generator=g, post_norms=post,
                                   residual_scale=scale)
    loras = {}
    for n, p in block.adapters.items():
        with torch.no_grad():
            p.B.copy_(0.02 * torch.randn(p.B.shape, generator=g))
        loras[n] = (*(t.detach().cpu().requires_grad_(True) for t in (p.A, p.B)), p.scale)
    x, dy = (torch.randn(2, 70, H, generator=g).to(BF) for _ in range(2))
    ref_x = x.float().requires_grad_(True)
    ref = plain_block(ref_x, decoded(block, oracle_codec), loras, post, scale, gates)
    ref.backward(dy.float())
    rot, mask = dense.positions_and_masks(torch.ones(2, 70, dtype=torch.bool), head_dim=D,
                                          theta=10000.0, device=dev)
    session = slots.ResidentSession([block], dev)
    own = x.to(dev).requires_grad_(True)
    with session.run():
        out = streaming_block(own, rot, mask, block.functional, block.kwargs, session.reloader(block),
                              block.adapters, 0)
        out.backward(dy.to(dev))
    session.close()
    assert float((out.detach().cpu().float() - ref.detach()).norm() / ref.detach().norm()) < 2e-2
    assert _cos(own.grad, ref_x.grad) > 0.999
    for n, p in block.adapters.items():
        assert _cos(p.grad_A, loras[n][0].grad) > 0.999, n
        assert _cos(p.grad_B, loras[n][1].grad) > 0.999, n


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("per_row", [False, True])
def test_balance_term_of_a_layer(sigmoid, per_row):
    """With no gradient from above, what comes back is the term's alone: the router's
    matrix times the gradient of its logits."""
    dev = torch.device("cuda:0")
    g = torch.Generator().manual_seed(5)
    router = torch.randn(16, H, generator=g) * H**-0.5
    w = {"mlp.gate.weight": (router if sigmoid else router.to(BF)).to(dev),
         "mlp.gate.e_score_correction_bias": torch.zeros(16, device=dev),
         "mlp.experts.gate_up_proj": moe.quantize_experts(0.03 * torch.randn(16, 256, H, generator=g),
                                                          "nf4-g128", dev),
         "mlp.experts.down_proj": moe.quantize_experts(0.03 * torch.randn(16, H, 128, generator=g),
                                                       "nf4-g128", dev)}
    x = torch.randn(3, 50, H, generator=g).to(BF).to(dev).requires_grad_(True)
    valid = torch.arange(50, device=dev) < torch.tensor([[50], [31], [7]], device=dev)
    balance = moe.ExpertBalance(0.25, per_row=per_row)

    def layer(**kw):
        if sigmoid:
            return moe.deepseek_moe_feed_forward(x, w, num_experts=16, top_k=4, groups=4, group_k=2,
                                                 normalize=True, scale=2.5, return_routing=True, **kw)
        return moe.moe_feed_forward(x, w, num_experts=16, top_k=4, norm_topk_prob=True,
                                    return_routing=True, **kw)
    up = torch.randn(x.shape, device=dev, dtype=BF)
    out, _, idx = layer(balance=balance, valid=valid)
    plain, _, _ = layer()
    assert torch.equal(out, plain)
    (alone,) = torch.autograd.grad(out, [x], torch.zeros_like(up), retain_graph=True)
    # the same by hand, in 64 bits from the logits as the layer forms them
    W = w["mlp.gate.weight"].double()
    logits = x.detach().double() @ W.T
    if not sigmoid:
        logits = logits.float().to(BF).double()
    from tests.test_gpu_balance import formula
    logits.requires_grad_(True)
    loss, counts = formula(logits, idx.view(3, 50, 4), "sigmoid" if sigmoid else "softmax", valid,
                           per_row)
    (dl,) = torch.autograd.grad(0.25 * loss, [logits])
    want = dl @ W
    # logits and their gradient are rounded to bf16 before the product (softmax), which
    # is rounded to bf16: 2^-8 each of the terms; a logit's 2^-8 of up to 4 moves its
    # probability by 2^-6 and the gradient with it
    size = (dl.abs() @ W.abs())
    assert ((alone.double() - want).abs() <= 2**-8 * want.abs() + (2**-5 if not sigmoid else 2**-15)
            * size + 1e-12).all()
    assert (alone[~valid] == 0).all()
    assert balance.passes == 1 and torch.equal(balance.counts, counts.sum(0))
    assert abs(float(balance.loss) - float(loss.detach())) < (2e-2 if not sigmoid else 1e-5)
    # both gradients together: the bf16 sum of two
    (both,) = torch.autograd.grad(out, [x], up, retain_graph=True)
    (rest,) = torch.autograd.grad(plain, [x], up)
    room = 2**-7 * (rest.double().abs() + alone.double().abs()) + 2**-7 * rest.double().abs().amax()
    assert ((both.double() - rest.double() - alone.double()).abs() <= room).all()
    with torch.no_grad():
        layer(balance=balance)
    assert balance.passes == 1  # a pass without gradients adds nothing
    balance.reset()
    assert balance.counts is None
    with pytest.raises(ValueError, match="coefficient"):
        moe.ExpertBalance(math.nan)


def _model(dev, balance=None, trained=True):
    g = torch.Generator().manual_seed(21)
    blocks = []
    for i in range(2):
        blocks.append(slots.make_dense_block(
            i, weights(g, experts=True), codec="nf4-g128", heads=HEADS, kv_heads=KV, head_dim=D,
            eps=EPS, rank=4, alpha=8.0, targets=ATTENTION, device=dev, generator=g,
            moe={"num_experts": E, "top_k": K, "norm_topk_prob": True, "balance": balance},
            expert_lora_rank=4, post_norms=True, residual_scale=0.7))
        for p in blocks[-1].adapters.values():
            with torch.no_grad():
                p.B.copy_(0.02 * torch.randn(p.B.shape, generator=g))
    table = 0.05 * torch.randn(304, H, generator=g)
    return engine.DenseModel(
        embedding=TokenEmbedding(table, device=dev, scale=H**0.5, padding_idx=0) if trained else table,
        norm=torch.ones(H), head=0.05 * torch.randn(304, H, generator=g), blocks=blocks, heads=HEADS,
        kv_heads=KV, head_dim=D, eps=EPS, theta=10000.0, rank=4, alpha=8.0, targets=ATTENTION,
        device=dev)


def _rows(n=4):
    g = torch.Generator().manual_seed(6)
    rows = []
    for k in range(n):
        ids = torch.randint(1, 304, (2, 60), generator=g)
        docs = torch.arange(60).expand(2, 60) // 23
        docs = torch.where(torch.arange(60) < 60 - 9 * k, docs, -1)
        rows.append((torch.where(docs < 0, 0, ids), ids, docs))
    return rows


def _state(model):
    return [t.detach().clone() for b in model.blocks for p in b.adapters.values() for t in (p.A, p.B)] \
        + [model.embedding.weight.clone()]


def test_training_steps_together():
    """Microbatch by microbatch and layer by layer: the same bits; every part moves."""
    dev = torch.device("cuda:0")
    results = []
    for layer_major in (False, True):
        balance = moe.ExpertBalance(0.01, per_row=True)
        model = _model(dev, balance)
        before = _state(model)
        session = slots.Q4SlotSession(model.blocks, dev, host_budget_bytes=1 << 34,
                                      device_budget_bytes=1 << 34, slots=2)
        opt = muon.Muon(lr=2e-3, table=engine.AdamW(lr=1e-3))
        losses = engine.train(model, session, _rows(), steps=2, accumulation=2, optimizer=opt,
                              layer_major=layer_major)
        session.close()
        after = _state(model)
        assert all(math.isfinite(v) for v in losses) and opt.step_count == 2
        assert opt.table.step_count == 2
        assert all(not torch.equal(a, b) and b.isfinite().all() for a, b in zip(before, after))
        assert balance.passes == 2 * 2 * 2 and balance.counts.shape == (E,)
        picked = sum(int((d >= 0).sum()) for _, _, d in _rows()) * K * 2
        assert int(balance.counts.sum()) == picked  # padding is not counted
        assert torch.equal(model.embedding.weight[0], before[-1][0])  # the padding row
        results.append((losses, after, balance.counts, balance.loss))
    assert results[0][0] == results[1][0]
    assert all(torch.equal(a, b) for a, b in zip(results[0][1], results[1][1]))
    assert torch.equal(results[0][2], results[1][2])


def test_embedding_gradient_of_a_microbatch():
    dev = torch.device("cuda:0")
    model = _model(dev)
    session = slots.ResidentSession(model.blocks, dev)
    rows = _rows(2)
    want = torch.zeros(304, H, dtype=torch.float64, device=dev)
    size = torch.zeros_like(want)
    with session.run():
        for k, (ids, labels, docs) in enumerate(rows):
            _, grad = engine.microbatch(model, session, ids, labels, normalization=100, token_chunk=32,
                                        accumulate=k > 0, documents=docs)
            flat = ids.flatten().to(dev)
            rows64 = H**0.5 * grad.double().view(-1, H) * (flat != 0)[:, None]
            want.index_add_(0, flat, rows64)
            size.index_add_(0, flat, rows64.abs())
    session.close()
    # at most 120 positions a token and microbatch, 2^-24 of the sum's size each
    assert ((model.embedding.grad.double() - want).abs() <= 2**-24 * 130 * size).all()
    assert float(want.abs().max()) > 0


def test_scores_of_a_trained_embedding():
    """A table that is looked up on the device scores as the host's."""
    dev = torch.device("cuda:0")
    trained, host = _model(dev), _model(dev, trained=False)
    table = trained.embedding.weight.cpu()
    trained.embedding.scale = 1.0
    trained.embedding.weight.copy_(table.to(BF))
    host.embedding = table.to(BF)
    res = []
    for model in (trained, host):
        session = slots.ResidentSession(model.blocks, dev)
        ids, _, docs = _rows(2)[1]
        with session.run():
            res.append(engine.score(model, session, ids, documents=docs).logprobs)
        session.close()
    assert torch.equal(*res)


def test_valid_tokens_of_masks():
    dev = torch.device("cuda:0")
    docs = torch.tensor([[0, 0, 1, -1], [-1, -1, -1, -1]], device=dev)
    assert torch.equal(dense.valid_tokens(packed.document_mask(docs)), docs >= 0)
    assert dense.valid_tokens(None) is None and dense.valid_tokens(dense.CausalMask(2, 4)) is None
    mask = dense.CausalMask(2, 4, torch.tensor([4, 1], dtype=torch.int32, device=dev))
    assert dense.valid_tokens(mask).tolist() == [[True] * 4, [True, False, False, False]]


def test_embedding_on_the_models_device():
    e = TokenEmbedding(torch.zeros(8, 16), device="cuda")
    with pytest.raises(ValueError, match="model's device"):
        engine.DenseModel(embedding=e, norm=torch.zeros(16), head=torch.zeros(8, 16), blocks=[],
                          heads=2, kv_heads=1, head_dim=8, eps=1e-6, theta=1e4, rank=1, alpha=1.0,
                          targets=(), device="cpu")


def test_balance_through_a_deepseek_block():
    """The block hands its router's term on: other input gradients, the same output, and
    the padded tokens' picks left out."""
    from spilltune_amd import deepseek
    from tests import test_gpu_mla as TM
    dev = torch.device("cuda:0")
    c = TM._params(heads=4, nope=128, rope=64, vdim=128, kv_rank=128, q_rank=None, interleave=False,
                   moe=True, rope_cfg=TM.DEFAULT)
    g = torch.Generator().manual_seed(31)
    w = TM._layer_weights(g, c, 256, 128, 256, 16)
    valid = torch.arange(40) < torch.tensor([[40], [23]])
    hidden, dy = (torch.randn(2, 40, 256, generator=g).to(BF) for _ in range(2))
    dy[~valid] = 0
    res = []
    for coefficient in (None, 5.0):
        balance = None if coefficient is None else moe.ExpertBalance(coefficient)
        block = deepseek.make_deepseek_block(0, w, codec="nf4-g128", parameters=dict(c, balance=balance),
                                             rank=4, alpha=8.0, device=dev,
                                             generator=torch.Generator().manual_seed(1))
        rot, mask = deepseek.positions_and_masks(valid, rope=c["rope_cfg"], rope_dim=c["rope"],
                                                 device=dev)
        session = slots.ResidentSession([block], dev)
        x = hidden.to(dev).requires_grad_(True)
        with session.run():
            out = streaming_block(x, rot, mask, block.functional, block.kwargs,
                                  session.reloader(block), block.adapters, 0)
            out.backward(dy.to(dev))
        session.close()
        res.append((out.detach(), x.grad))
    assert torch.equal(res[0][0], res[1][0]) and not torch.equal(res[0][1], res[1][1])
    assert balance.passes == 1 and int(balance.counts.sum()) == int(valid.sum()) * c["top_k"]
