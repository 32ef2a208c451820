"""Shapes and masks of the packed operators that nothing else reaches: grouped heads
of 192/128 whose key tiles are split over workgroups, more tiles than are sorted,
the widest vocabularies, the MLA block's own tables with windows and bidirectional
runs.  Bounds as in test_gpu_packed and test_gpu_logprobs."""
import random

import pytest
import torch

from oracle import layer as OL
from oracle import mla as OMLA
from spilltune_amd import _lib, deepseek, ops, packed
from tests import test_gpu_logprobs as TP
from tests import test_gpu_mla as TM
from tests.test_gpu_packed import _check, _documents, _run
from tests.test_gpu_packed_train import _compare, _restarted, _step

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _long_first(B, S):
    """One long document, short ones behind it, padding: its key tiles carry most
    of the work and are split."""
    d = torch.full((B, S), -1, dtype=torch.int32)
    d[:, :S * 3 // 4] = 0
    d[:, S * 3 // 4:S - 5] = 1 + (torch.arange(S - 5 - S * 3 // 4) // 9).int()
    return d


@pytest.mark.parametrize("shape", [(1, 300, 8, 2, 192, 128), (1, 700, 16, 2, 192, 128), (2, 515, 12, 1, 192, 128),
                                   (1, 700, 16, 2, 128, 128), (1, 700, 16, 2, 64, 64)])
@pytest.mark.parametrize("cap,bias", [(None, False), (6.0, True)])
def test_grouped_heads_in_parts(shape, cap, bias):
    mask = packed.document_mask(_long_first(*shape[:2]).cuda())
    slopes = torch.tensor([2.0 ** -(h % 7 + 1) for h in range(shape[2])], device="cuda") if bias else None
    _check(*_run(*shape, mask, cap=cap, slopes=slopes, seed=3))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("shape", [(1, 700, 16, 2, 192, 128), (1, 700, 16, 2, 128, 128)])
def test_masked_places_of_tiles_in_parts(shape, bad):
    """Infinities and NaN in the short documents and the padding leave the long
    document's values, whose key tiles are in parts, as they were."""
    docs = _long_first(*shape[:2])
    hit = (docs != 0).cuda()

    def edit(q, k, v, dout):
        for t in (q, k, v):
            t.transpose(1, 2)[hit] = bad
        dout[hit] = bad
    got, want, bound = _run(*shape, packed.document_mask(docs.cuda()), seed=4, edit=edit)
    _check(got, want, bound, [lambda t: t[~hit]] + [lambda t: t.transpose(1, 2)[~hit]] * 3)


def test_more_tiles_than_are_sorted():
    B, S = 16387, 3
    docs = _documents(random.Random(2), B, S, 1, 3, 1)
    _check(*_run(B, S, 2, 1, 64, 64, packed.document_mask(docs.cuda()), seed=5))


@pytest.mark.parametrize("V,top", [(1 << 20, 5), ((1 << 20) - 3, 64), (1 << 21, 0)])
def test_widest_vocabularies(V, top):
    h, w, t, g = TP._inputs(5, 8, V, grid=True)
    t[0], t[1] = V - 1, 0
    g_lp = torch.randn(5, generator=g, device="cuda")
    h.requires_grad_(True)
    r = ops.token_logprobs(h, w, t, top=top)
    (dh,) = torch.autograd.grad(r.logprobs, h, g_lp)
    want, err, l, _ = TP._reference(h.detach(), w, t, grads=(g_lp, None, None))
    TP._close("logprobs", r.logprobs, want[0], err[0])
    TP._close("entropy", r.entropy, want[1], err[1])
    TP._close("dh", dh, want[2], err[2])
    assert torch.equal(r.top_tokens, torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top])


def _additive(mask):
    """[B,1,S,S] bf16 of a mask's runs; a token that sees nothing sees itself (its
    row is not compared)."""
    at = torch.arange(mask.length)
    lo, hi = mask.key_start.cpu(), mask.key_end.cpu()
    sees = (at >= lo[..., None]) & (at < hi[..., None])
    sees = sees | (torch.eye(mask.length, dtype=torch.bool) & (lo >= hi)[..., None])
    return torch.where(sees, 0.0, torch.finfo(BF).min).to(BF)[:, None]


@pytest.mark.parametrize("kind", ["documents", "window", "bidirectional"])
def test_mla_block_with_its_own_packed_tables(oracle_codec, kind):
    dev = torch.device("cuda:0")
    c = TM._params(heads=4, nope=128, rope=64, vdim=128, kv_rank=128, q_rank=128, interleave=True,
                   moe=False, rope_cfg=TM.YARN)
    g = torch.Generator().manual_seed(91)
    B, S, H = 2, 96, 256
    block = deepseek.make_deepseek_block(0, TM._layer_weights(g, c, H, 128, 256, 16), codec="nf4-g128",
                                         parameters=c, rank=8, alpha=16.0, device=dev, generator=g)
    with torch.no_grad():
        for p in block.adapters.values():
            p.B.copy_(torch.randn(p.B.shape, generator=g) * 0.02)
    documents = _documents(random.Random(8), B, S, 7, 50, 9).long()
    real = documents >= 0
    hidden, dy = (torch.randn(B, S, H, generator=g).to(BF) for _ in range(2))
    dy[~real] = 0
    kw = {"documents": {}, "window": {"window": 11},
          "bidirectional": {"bidirectional": torch.rand(B, S, generator=g) < 0.6}}[kind]
    tables, mask = deepseek.packed_positions_and_masks(documents, rope=c["rope_cfg"], rope_dim=64,
                                                       device=dev, **kw)
    want = _restarted(OMLA.rotary(1, S, c["rope_cfg"], 64, BF), mask.positions.cpu())
    for a, b in zip(tables, want):
        # the device's and the host's sines differ by fp32 roundings: half a bf16 step and
        # one more where that crosses a rounding border
        assert a.shape == b.shape
        assert bool(((a.cpu().double() - b.double()).abs() <= 2 * 2.0 ** -8 * b.double().abs() + 2.0 ** -20).all())
    lor = {n: OL.Lora(n, p.A.detach().cpu(), p.B.detach().cpu(), p.alpha)
           for n, p in block.adapters.items()}
    out_ref, dh_ref = OMLA.streaming_step(hidden, want, _additive(mask), dy, parameters=c,
                                          weights=TM._oracle_weights(block, oracle_codec), loras=lor)
    out, dh = _step(block, (tables, mask), hidden, dy, dev)
    _compare(TM._rel, TM._cos, block, lor, out, out_ref, dh, dh_ref, real)


def test_split_tiles_are_split():
    """The shapes above do have tiles in parts: the backward's workspace holds them."""
    for B, S, H, KV, DQ, DV in ((1, 700, 16, 2, 192, 128), (1, 300, 8, 2, 192, 128)):
        q = lambda kv: _lib.query("st_span_attn_workspace_bytes", B, S, H, kv, DQ, DV)  # noqa: E731
        assert q(KV) - q(H) >= B * H * S * (DQ + DV) * 4
