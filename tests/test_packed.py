"""Packed rows on the CPU: runs of documents, frequencies, the references'
gradients against differences, refusals before any device work."""
import ctypes
import math
import random

import pytest
import torch

from spilltune_amd import _lib, deepseek, dense, engine, packed
from tests._packed_ref import rope_ref, runs_brute, span_forward, span_ref


def _documents(rng, B, S):
    d = torch.empty(B, S, dtype=torch.int64)
    for b in range(B):
        i = 0
        while i < S:
            n = rng.choice([1, 1, 2, 5, 13])
            d[b, i:i + n] = rng.choice([-1, -7, 0, 1, 2, 1 << 40])
            i += n
    return d


@pytest.mark.parametrize("S", [1, 2, 7, 40])
@pytest.mark.parametrize("window", [None, 1, 4, 100])
def test_document_runs_match_a_walk(S, window):
    rng = random.Random(S * 1000 + (window or 0))
    for trial in range(20):
        d = _documents(rng, 3, S)
        marks = torch.tensor([[rng.random() < 0.6 for _ in range(S)] for _ in range(3)])
        for bi in (None, marks):
            got = packed.document_runs(d, bidirectional=bi, window=window)
            for g, want in zip(got, runs_brute(d, bi, window)):
                assert g.dtype == torch.int32 and torch.equal(g, want)


def test_document_runs_refuse():
    d = torch.zeros(2, 4, dtype=torch.int32)
    for bad in (d.float(), d[0], d.bool()):
        with pytest.raises(ValueError, match="documents"):
            packed.document_runs(bad)
    with pytest.raises(ValueError, match="bidirectional"):
        packed.document_runs(d, bidirectional=d)
    with pytest.raises(ValueError, match="bidirectional"):
        packed.document_runs(d, bidirectional=torch.zeros(2, 3, dtype=torch.bool))
    for w in (0, -1, 2.0, True):
        with pytest.raises(ValueError, match="window"):
            packed.document_runs(d, window=w)
    with pytest.raises(ValueError, match="GPU"):
        packed.document_mask(d)
    with pytest.raises(ValueError, match="int32"):
        packed.span_mask(d.long(), d)
    with pytest.raises(ValueError, match="int32"):
        packed.span_mask(d, d[:, :2])
    with pytest.raises(ValueError, match="at least one token"):
        packed.span_mask(d[:0], d[:0])
    with pytest.raises(ValueError, match="GPU"):
        packed.span_mask(d, d)


def test_span_attention_refuses():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    z = torch.zeros(1, 4, dtype=torch.int32)
    mask = packed.SpanMask(1, 4, z, z, z, z)  # no plan is read before the checks
    f = packed.span_attention
    with pytest.raises(ValueError, match="SpanMask"):
        f(q, q, q, 1.0, None)
    with pytest.raises(ValueError, match="bf16"):
        f(q.float(), q, q, 1.0, mask)
    with pytest.raises(ValueError, match="do not fit"):
        f(q, q[:, :, :3], q, 1.0, mask)
    with pytest.raises(ValueError, match="do not fit"):
        f(q, torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16), q, 1.0, mask)
    with pytest.raises(ValueError, match="mask of"):
        f(q[:, :, :3], q[:, :, :3], q[:, :, :3], 1.0, mask)
    for scale, cap in ((0.0, None), (-1.0, None), (math.nan, None), (math.inf, None), (1.0, -2.0),
                       (1.0, math.inf)):
        with pytest.raises(ValueError, match="scale must be positive"):
            f(q, q, q, scale, mask, cap=cap)
    for slopes in (torch.zeros(2, dtype=torch.float64), torch.zeros(3),
                   torch.zeros(2, requires_grad=True)):
        with pytest.raises(ValueError, match="slopes"):
            f(q, q, q, 1.0, mask, slopes=slopes)
    with pytest.raises(ValueError, match="GPU"):
        f(q, q, q, 1.0, mask)


def test_abi_refuses_before_the_device():
    """Sizes, dims and pointers are checked on the host (fake pointers never
    reach a kernel)."""
    p, n = ctypes.c_void_p(16), ctypes.c_void_p(None)

    def fwd(B=1, S=4, H=2, KV=1, DQ=64, DV=64, scale=1.0, cap=0.0, q=p, plan=p):
        _lib.call("st_span_attn_fwd", q, p, p, B, S, H, KV, DQ, DV, scale, cap, None, p, p, plan, p,
                  p, None)
    for kw, msg in (({"H": 3, "KV": 2}, "head counts"), ({"DQ": 96, "DV": 96}, "head dims"),
                    ({"scale": 0.0}, "scale"), ({"cap": -1.0}, "cap"), ({"q": n}, "NULL"),
                    ({"plan": ctypes.c_void_p(8)}, "unaligned"), ({"S": 1 << 30}, "too large"),
                    ({"H": 1 << 17}, "too large")):
        with pytest.raises(ValueError, match=msg):
            fwd(**kw)
    fwd(B=0)  # nothing to do

    def bwd(dq=p, ws=p, wb=1 << 40):
        _lib.call("st_span_attn_bwd", p, p, p, p, p, p, 1, 4, 2, 1, 64, 64, 1.0, 0.0, None, p, p, p, dq,
                  p, p, ws, wb, None)
    for kw, msg in (({"dq": n}, "NULL"), ({"wb": 10}, "workspace"), ({"ws": n}, "workspace")):
        with pytest.raises(ValueError, match=msg):
            bwd(**kw)
    with pytest.raises(ValueError, match="needs"):
        _lib.call("st_span_plan", p, p, 2, 100, p, 16, None)
    # blocks, key tiles, two orders, two works, the sum
    assert _lib.query("st_span_plan_bytes", 2, 100) == 4 * (2 * 4 * 4 + 2 * 2 * 1 + 4 * 2 * 1 + 1)
    assert _lib.query("st_span_attn_workspace_bytes", 1, 8, 3, 2, 64, 64) == 0

    def rope(D=64, rot=64, ldx=256, wq=None, wk=None, x=p, B=1, S=4):
        _lib.call("st_rope_pos_fwd", x, ldx, p, 0, p, 1.0, B, S, 2, 1, D, rot, 0, wq, wk, 1e-6, p, p,
                  p, p, None)
    for kw, msg in (({"rot": 63}, "even"), ({"rot": 66}, "even"), ({"D": 60, "rot": 20}, "head_dim"),
                    ({"D": 520, "rot": 64}, "head_dim"), ({"ldx": 248}, "rows below"),
                    ({"ldx": 260}, "rows below"), ({"wq": p}, "together"),
                    ({"D": 96, "wq": p, "wk": p}, "norms with"), ({"x": n}, "NULL"),
                    ({"B": 1 << 20, "S": 1 << 20}, "tokens")):
        with pytest.raises(ValueError, match=msg):
            rope(**kw)
    rope(S=0)


def test_rope_positions_refuses():
    r = packed.Rotary(64, 1e4, device="cpu")
    y, pos = torch.zeros(6, 256, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32)
    f = packed.rope_positions
    with pytest.raises(ValueError, match="Rotary"):
        f(y, pos, None, 2, 1)
    with pytest.raises(ValueError, match="positions"):
        f(y, pos.float(), r, 2, 1)
    for bad in (y.float(), y[:5], y[:, :192]):
        with pytest.raises(ValueError, match="expects bf16"):
            f(bad, pos, r, 2, 1)
    with pytest.raises(ValueError, match="norm weights"):
        f(y, pos, r, 2, 1, norms=(y[0, :64], y[0, :32]))
    with pytest.raises(ValueError, match="GPU"):
        f(y, pos, r, 2, 1)
    for head, kw in ((60, {}), (64, {"rotary_dim": 63}), (64, {"rotary_dim": 80}),
                     (64, {"rotary_dim": 0})):
        with pytest.raises(ValueError, match="rotary part"):
            packed.Rotary(head, 1e4, device="cpu", **kw)


def test_frequencies():
    f = packed.rotary_frequencies
    inv, a = f(64, 10000.0)
    assert a == 1.0 and inv[0] == 1.0 and math.isclose(inv[-1], 10000.0 ** (-62 / 64), rel_tol=1e-15)
    lin, _ = f(64, 10000.0, {"type": "linear", "factor": 4})
    assert all(math.isclose(x, y / 4, rel_tol=1e-15) for x, y in zip(lin, inv))
    sc = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    base, _ = f(128, 500000.0)
    got, _ = f(128, 500000.0, sc)
    for x, y in zip(got, base):
        wave = 2 * math.pi / y
        if wave < 8192 / 4.0:
            assert x == y
        elif wave > 8192 / 1.0:
            assert math.isclose(x, y / 8, rel_tol=1e-14)
        else:
            s = (8192 / wave - 1.0) / 3.0
            assert math.isclose(x, (1 - s) * y / 8 + s * y, rel_tol=1e-14)
    # YaRN: the fp32 table of the MLA path, to its rounding
    for rope in ({"factor": 40.0, "original_max_position_embeddings": 4096, "beta_fast": 32,
                  "beta_slow": 1, "mscale": 1.0, "mscale_all_dim": 1.0},
                 {"factor": 4.0, "original_max_position_embeddings": 32768, "truncate": False}):
        rope = dict(rope, rope_type="yarn", rope_theta=10000.0)
        want, amp = deepseek.rope_parameters(rope, 64)
        got, a = f(64, 10000.0, rope)
        # three fp32 operations and a power of it, cancellation in 1 - (1 - ramp)
        torch.testing.assert_close(torch.tensor(got), want, rtol=1e-5, atol=0)
        assert math.isclose(a, amp, rel_tol=1e-12)
    for bad in ({"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "linear"},
                {"rope_type": "linear", "factor": 0.5}, dict(sc, high_freq_factor=1.0)):
        with pytest.raises(ValueError, match="unsupported_capability"):
            f(64, 10000.0, bad)


@pytest.mark.parametrize("cap,bias", [(None, False), (2.0, False), (None, True), (1.5, True)])
def test_reference_gradients_against_differences(cap, bias):
    """The formulas that the kernels are held to, against central differences."""
    g = torch.Generator().manual_seed(3)
    B, H, S, D, DV = 1, 2, 7, 4, 3
    q, k, v = (torch.randn(B, H, S, d, generator=g, dtype=torch.float64) for d in (D, D, DV))
    lo = torch.tensor([[0, 0, 1, 3, 3, 0, 5]], dtype=torch.int32)
    hi = torch.tensor([[1, 3, 3, 3, 6, 7, 7]], dtype=torch.int32)  # query 3 sees nothing
    slopes = torch.tensor([0.3, 0.05]) if bias else None
    dout = torch.randn(B, S, H * DV, generator=g, dtype=torch.float64)
    _, dq, dk, dv = span_ref(q, k, v, 0.7, lo, hi, cap, slopes, dout)[0]
    do = dout.view(B, S, H, DV).transpose(1, 2)

    def loss(q, k, v):
        return float((span_forward(q, k, v, 0.7, lo, hi, cap, slopes) * do).sum())
    for t, grad in ((0, dq), (1, dk), (2, dv)):
        args = [q, k, v]
        num = torch.zeros_like(args[t])
        for i in range(num.numel()):
            ends = []
            for h in (1e-5, -1e-5):
                moved = [a.clone() for a in args]
                moved[t].view(-1)[i] += h
                ends.append(loss(*moved))
            num.view(-1)[i] = (ends[0] - ends[1]) / 2e-5
        # differences: h^2 of the third derivative, and 2^-53 / h of the loss
        torch.testing.assert_close(grad, num, rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_reference_gradients_against_differences(interleaved):
    g = torch.Generator().manual_seed(5)
    heads, kv, D, rot = 2, 1, 8, 6
    pos = torch.tensor([[0, 5], [70000, 3]])
    inv = [1.0, 0.3, 0.01]
    w = [torch.rand(D, generator=g, dtype=torch.float64) + 0.5 for _ in range(2)]
    y = torch.randn(4, (heads + 2 * kv) * D, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(
        lambda t: rope_ref(t, pos, inv, 1.3, heads, kv, D, rot, interleaved, w), (y,), eps=1e-6,
        atol=1e-7, rtol=1e-6)


def test_block_refuses_positions_of_other_rows():
    z = torch.zeros(1, 4, 256, dtype=torch.bfloat16)
    pos = packed.Positions(torch.zeros(1, 4, dtype=torch.int32), packed.Rotary(64, 1e4, device="cpu"))
    for head_dim, h in ((128, z), (64, z[:, :3])):
        with pytest.raises(ValueError, match="positions of other"):
            dense.dense_block(h, pos, None, heads=4, kv_heads=4, head_dim=head_dim, eps=1e-5)
    with pytest.raises(ValueError, match="causal mask marker and span masks"):
        dense.dense_block(z, pos, "mask", heads=4, kv_heads=4, head_dim=64, eps=1e-5)


def test_engine_refuses():
    model, session = object(), object()
    ids = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="shaped like"):
        engine.score(model, session, ids, documents=ids[:, :3])
    with pytest.raises(ValueError, match="labels and documents"):
        packed.document_labels(ids, ids[0])
    assert packed.document_labels(torch.arange(6).view(1, 6),
                                  torch.tensor([[0, 0, 1, 1, -1, -1]])).tolist() \
        == [[-100, 1, -100, 3, -100, -100]]


def test_abi_refuses_scales_out_of_range():
    """Numbers whose reciprocals or powers leave fp32, and row counts whose
    product leaves 64 bits."""
    p = ctypes.c_void_p(16)

    def fwd(B=1, S=4, H=2, scale=1.0, cap=0.0):
        _lib.call("st_span_attn_fwd", p, p, p, B, S, H, 1, 64, 64, scale, cap, None, p, p, p, p, p,
                  None)
    for kw in ({"scale": 1e-31}, {"scale": 1e31}, {"cap": 1e31}, {"cap": 9e-5}, {"scale": 1e4, "cap": 0.5}):
        with pytest.raises(ValueError, match="out of range"):
            fwd(**kw)
    with pytest.raises(ValueError, match="too large"):
        fwd(B=(1 << 24) - 1, S=(1 << 30) - 1, H=(1 << 16) - 1)


def test_rope_positions_refuses_norms_that_train():
    y, w = torch.zeros(2, 4 * 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    rotary = packed.Rotary(64, 1e4, device="cpu")
    with pytest.raises(ValueError, match="frozen"):
        packed.rope_positions(y, torch.zeros(1, 2, dtype=torch.int32), rotary, 2, 1,
                              norms=(w, w.clone().requires_grad_(True)))
