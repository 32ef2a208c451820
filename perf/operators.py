"""Operator cases: training and scoring on packed documents.

A packed row holds several documents back to back.  Three operators carry a
model over such rows and read its answers out: attention in which every query
sees one run of keys (its document's, up to itself, with bidirectional runs, a
window, capped scores and a distance bias), the rotation of query and key heads
by positions that restart with each document, and the log probabilities of
given tokens under the vocabulary head, with entropy and top alternatives.

``own`` is False: ``run`` computes each operator in elementary torch operations
in 32 bits.  ``own`` is True: ``run`` calls this package.  ``exact`` restates
the operators in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096,
        "beta_fast": 32.0, "beta_slow": 1.0}
LINEAR = {"rope_type": "linear", "factor": 4.0}
SCALINGS = {"default": None, "linear": LINEAR, "llama3": LLAMA3, "yarn": YARN}


def listed():
    return [
        # ---- attention
        # a unit-sized batch of short chat turns (tests, debug runs), a few
        # padded positions at each row's end: launches and host work count
        {"name": "spans_short", "kind": "spans", "B": 3, "S": 77, "heads": 8, "kv": 2, "DQ": 64,
         "DV": 64, "docs": 11, "doc_lo": 5, "doc_hi": 40, "pad": 6, "prefix": False, "window": 0,
         "cap": 0.0, "slopes": False, "train": True},
        # fine-tuning on packed instructions of very unequal length, one
        # decoder layer's grouped-query heads
        {"name": "spans_packed", "kind": "spans", "B": 1, "S": 8192, "heads": 32, "kv": 8,
         "DQ": 128, "DV": 128, "docs": 7, "doc_lo": 60, "doc_hi": 2500, "pad": 0, "prefix": False,
         "window": 0, "cap": 0.0, "slopes": False, "train": True},
        # prompts that see each other whole, answers causal, distance biases, an
        # odd row length, every head with its own key
        {"name": "spans_prefix_bias", "kind": "spans", "B": 2, "S": 2103, "heads": 16, "kv": 16,
         "DQ": 128, "DV": 128, "docs": 3, "doc_lo": 200, "doc_hi": 1500, "pad": 40,
         "prefix": True, "window": 0, "cap": 0.0, "slopes": True, "train": True},
        # scoring one long document through a sliding window with capped scores
        {"name": "spans_window_cap", "kind": "spans", "B": 1, "S": 16384, "heads": 32, "kv": 8,
         "DQ": 128, "DV": 128, "docs": 1, "doc_lo": 16384, "doc_hi": 16384, "pad": 0,
         "prefix": False, "window": 4096, "cap": 50.0, "slopes": False, "train": False},
        # packed rows through multi-head latent attention's 192/128 heads
        {"name": "spans_mla", "kind": "spans", "B": 1, "S": 2048, "heads": 128, "kv": 128,
         "DQ": 192, "DV": 128, "docs": 5, "doc_lo": 100, "doc_hi": 1200, "pad": 0,
         "prefix": False, "window": 0, "cap": 0.0, "slopes": False, "train": True},
        # ---- rotation
        # one token of each of 16 far-apart conversations; interleaved pairs, part of the head
        {"name": "rotary_tokens", "kind": "rotary", "B": 16, "S": 1, "heads": 32, "kv": 8,
         "D": 128, "rotary": 64, "interleaved": True, "norm": False, "scaling": "default",
         "theta": 10000.0, "far": 131072, "train": False},
        # a packed row of the long-context Llama layout, positions from 0 in each document
        {"name": "rotary_packed", "kind": "rotary", "B": 1, "S": 8192, "heads": 32, "kv": 8,
         "D": 128, "rotary": 128, "interleaved": False, "norm": False, "scaling": "llama3",
         "theta": 500000.0, "far": 0, "train": True},
        # Qwen3's normalised heads, odd row length, far positions under YaRN
        {"name": "rotary_norm", "kind": "rotary", "B": 2, "S": 2103, "heads": 32, "kv": 8,
         "D": 128, "rotary": 128, "interleaved": False, "norm": True, "scaling": "yarn",
         "theta": 1000000.0, "far": 100000, "train": True},
        # ---- log probabilities
        # the next token of a handful of prompts with five alternatives
        {"name": "logprobs_few", "kind": "logprobs", "rows": 5, "H": 1024, "V": 32000, "top": 5,
         "temperature": 1.0, "cap": 0.0, "ignored": 0.0, "train": False},
        # evaluation: every answer token of a packed row scored, eight alternatives
        {"name": "logprobs_score", "kind": "logprobs", "rows": 1000, "H": 4096, "V": 128256,
         "top": 8, "temperature": 1.0, "cap": 0.0, "ignored": 0.3, "train": False},
        # a policy or preference step: log probabilities and entropy with gradients
        {"name": "logprobs_train", "kind": "logprobs", "rows": 2048, "H": 4096, "V": 151936,
         "top": 0, "temperature": 1.0, "cap": 0.0, "ignored": 0.2, "train": True},
        # the same for a few decisive tokens of a wide model, sampled at a temperature, capped
        {"name": "logprobs_few_train", "kind": "logprobs", "rows": 61, "H": 7168, "V": 129280,
         "top": 0, "temperature": 0.7, "cap": 30.0, "ignored": 0.0, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["spans", "spans", "rotary", "logprobs"])
    if kind == "spans":
        dq, dv = rng.choice([(64, 64), (128, 128), (128, 128), (192, 128)])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv if dq == 192 else kv * rng.choice([1, 2, 3, 4])
        S = _log(rng, 1, 6000)
        B = rng.choice([1, 2, 3, 4]) if S < 2500 else 1
        lo = _log(rng, 1, max(2, S // 2))
        return {"kind": "spans", "B": B, "S": S, "heads": heads, "kv": kv, "DQ": dq,
                "DV": dv, "docs": rng.randrange(1000), "doc_lo": lo,
                "doc_hi": min(S, lo * rng.choice([1, 4, 30])), "pad": rng.choice([0, 0, S // 9]),
                "prefix": rng.random() < 0.3,
                "window": rng.choice([0, 0, 0, _log(rng, 1, S)]),
                "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "slopes": rng.random() < 0.25,
                "train": rng.random() < 0.7}
    if kind == "rotary":
        D = rng.choice([64, 80, 96, 128, 256])
        norm = D in (64, 128, 256) and rng.random() < 0.4
        kv = rng.choice([1, 2, 4, 8])
        far = rng.choice([0, 0, 30000, 1000000])
        S = _log(rng, 1, 6000)
        return {"kind": "rotary", "B": rng.choice([1, 2]) if S > 300 else rng.choice([1, 3, 16]),
                "S": S, "heads": kv * rng.choice([1, 2, 4]), "kv": kv, "D": D,
                "rotary": rng.choice([D, D, D // 2, D // 4]), "interleaved": rng.random() < 0.5,
                "norm": norm, "scaling": rng.choice(sorted(SCALINGS)),
                "theta": rng.choice([10000.0, 500000.0, 1000000.0]), "far": far,
                "train": rng.random() < 0.7}
    return {"kind": "logprobs", "rows": _log(rng, 1, 2048), "H": 8 * _log(rng, 32, 512),
            "V": 8 * _log(rng, 100, 19000), "top": rng.choice([0, 0, 1, 5, 8, 20]),
            "temperature": rng.choice([1.0, 1.0, 0.6, 1.3]), "cap": rng.choice([0.0, 0.0, 30.0]),
            "ignored": rng.choice([0.0, 0.3]), "train": rng.random() < 0.5}


# ----------------------------------------------------------------- documents
def _documents(case):
    """``[(row, start, end, prefix_end)]`` of the case's documents: lengths from
    the case alone, the last one cut at the row's end less its padding."""
    rng = random.Random(case["docs"])
    lo, hi = case["doc_lo"], max(case["doc_lo"], case["doc_hi"])
    out = []
    for b in range(case["B"]):
        at, limit = 0, case["S"] - (case["pad"] if b % 2 == 0 else case["pad"] // 2)
        while at < limit:
            n = min(_log(rng, lo, hi), limit - at)
            pre = at + int(n * rng.uniform(0.1, 0.6)) if case["prefix"] else at
            out.append((b, at, at + n, pre))
            at += n
    return out


def _key_runs(case):
    """Per document (row, start, and the seen runs [(query, first key, end)])."""
    for b, s, e, pre in _documents(case):
        first = [max(s, i - case["window"] + 1) if case["window"] else s for i in range(s, e)]
        end = [pre if i < pre else i + 1 for i in range(s, e)]
        yield b, s, e, first, end


def _pairs(case):
    return sum(sum(z - a for a, z in zip(first, end))
               for _, _, _, first, end in _key_runs(case))


# ----------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32)


def _spans_inputs(case, seed):
    g = _gen(seed)
    B, S, H, KV = case["B"], case["S"], case["heads"], case["kv"]
    q = _randn(g, B, H, S, case["DQ"])
    k = _randn(g, B, KV, S, case["DQ"])
    # normalised heads with a few outlier columns, as trained keys have them
    q[..., ::16] *= 2.0
    k[..., ::16] *= 2.0
    docs = torch.full((B, S), -1, dtype=torch.int32)
    pre = torch.zeros((B, S), dtype=torch.bool)
    for n, (b, s, e, p) in enumerate(_documents(case)):
        docs[b, s:e] = n
        pre[b, s:p] = True
    slopes = None
    if case["slopes"]:
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=F32,
                              device="cuda")
    dout = _randn(g, B, S, H * case["DV"]).to(BF) if case["train"] else None
    return {"q": q.to(BF), "k": k.to(BF), "v": _randn(g, B, KV, S, case["DV"]).to(BF),
            "docs": docs.cuda(), "prefix": pre.cuda() if case["prefix"] else None,
            "slopes": slopes, "dout": dout, "scale": case["DQ"] ** -0.5}


def _rotary_inputs(case, seed):
    g = _gen(seed)
    B, S, H, KV, D = case["B"], case["S"], case["heads"], case["kv"], case["D"]
    y = _randn(g, B * S, (H + 2 * KV) * D).to(BF)
    if case["far"]:
        base = torch.randint(0, case["far"], (B, 1), generator=g, device="cuda")
        pos = base + torch.arange(S, device="cuda")
    else:  # documents of a few hundred tokens, each from 0
        n = torch.randint(100, 700, (1,), generator=g, device="cuda")
        pos = torch.arange(S, device="cuda").expand(B, S) % n
    st = {"y": y, "pos": pos.to(torch.int32).contiguous(), "eps": 1e-6, "norms": None}
    if case["norm"]:
        st["norms"] = tuple((1.0 + 0.2 * _randn(g, D)).to(BF) for _ in range(2))
    if case["train"]:
        st["dq"] = _randn(g, B, H, S, D).to(BF)
        st["dk"] = _randn(g, B, KV, S, D).to(BF)
        st["dv"] = _randn(g, B, KV, S, D).to(BF)
    return st


def _logprob_inputs(case, seed):
    """Hidden states and head on a grid whose sums are exact in 32 bits, so the
    top tokens are the same whatever the order of a sum; in part of the rows
    the model is sure of the given token, as it is in real text."""
    g = _gen(seed)
    R, H, V = case["rows"], case["H"], case["V"]
    head = _randn(g, V, H).mul_(4096.0 * 1.3 / math.sqrt(H)).round_().clamp_(-255, 255)
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")
    sure = (torch.rand(R, generator=g, device="cuda") < 0.6).to(F32)
    pull = 5.0 * torch.rand(R, generator=g, device="cuda") * sure
    hidden = _randn(g, R, H) + pull[:, None] * head[tokens] / 4096.0
    hidden = hidden.mul_(32.0).round_().clamp_(-127, 127).div_(32.0).to(BF)
    head = head.div_(4096.0).to(BF)
    if case["ignored"]:
        skip = torch.rand(R, generator=g, device="cuda") < case["ignored"]
        tokens = torch.where(skip, torch.full_like(tokens, -100), tokens)
    st = {"hidden": hidden, "head": head, "tokens": tokens}
    if case["train"]:
        st["g_lp"] = _randn(g, R)
        st["g_ent"] = 0.1 * _randn(g, R)
        if case["top"]:
            st["g_top"] = 0.3 * _randn(g, R, case["top"])
    return st


_INPUTS = {"spans": _spans_inputs, "rotary": _rotary_inputs, "logprobs": _logprob_inputs}


def prepare(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    st["case"] = case
    if case["kind"] == "spans":
        if own:
            from spilltune_amd import packed
            # built once for a batch, read by every layer and pass
            st["mask"] = packed.document_mask(st["docs"], bidirectional=st["prefix"],
                                              window=case["window"] or None)
            if case["train"]:
                for n in "qkv":
                    st[n].requires_grad_(True)
    elif case["kind"] == "rotary":
        if own:
            from spilltune_amd import packed
            st["rotary"] = packed.Rotary(case["D"], case["theta"], rotary_dim=case["rotary"],
                                         interleaved=case["interleaved"],
                                         scaling=SCALINGS[case["scaling"]], device="cuda")
            if case["train"]:
                st["y"].requires_grad_(True)
        else:
            inv, st["amplitude"] = _frequencies(case)
            st["inv"] = torch.tensor(inv, dtype=F64, device="cuda")
    elif own and case["train"]:
        st["hidden"].requires_grad_(True)
    return st


# ----------------------------------------------------------------- plain forms
def _spans_plain(st):
    case = st["case"]
    B, H, S, DQ = st["q"].shape
    KV, DV = st["k"].shape[1], st["v"].shape[-1]
    G, cap, scale = H // KV, case["cap"], st["scale"]
    docs = st["docs"].long()
    i = torch.arange(S, device=docs.device)
    dist = i[:, None] - i[None, :]
    out = torch.zeros(B, S, H, DV, dtype=F32, device=docs.device)
    if case["train"]:
        dq, dk, dv = (torch.zeros(st[n].shape, dtype=F32, device=docs.device) for n in "qkv")
    for b in range(B):
        d = docs[b]
        seen = (d[:, None] == d[None, :]) & (d[:, None] >= 0)
        order = dist >= 0
        if st["prefix"] is not None:
            p = st["prefix"][b]
            order = order | (p[:, None] & p[None, :])
        seen = seen & order
        if case["window"]:
            seen = seen & (dist < case["window"])
        some = seen.any(-1)[None, :, None]
        for h in range(KV):
            hs = slice(h * G, (h + 1) * G)
            q, k, v = st["q"][b, hs].float(), st["k"][b, h].float(), st["v"][b, h].float()
            x = torch.matmul(q, k.t().contiguous()) * scale
            if cap:
                t = torch.tanh(x / cap)
                x = t * cap
            if st["slopes"] is not None:
                x = x - st["slopes"][hs][:, None, None] * dist.abs()
            x = torch.where(seen, x, -math.inf)
            top = torch.where(some, x.amax(-1, keepdim=True), 0.0)
            e = torch.exp(x - top)
            p = e / torch.where(some, e.sum(-1, keepdim=True), 1.0)
            del x, e
            out[b, :, hs] = torch.matmul(p, v).transpose(0, 1)
            if not case["train"]:
                continue
            do = st["dout"][b].view(S, H, DV)[:, hs].transpose(0, 1).float().contiguous()
            dp = torch.matmul(do, v.t().contiguous())
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            del dp
            dv[b, h] = torch.matmul(p.view(G * S, S).t().contiguous(), do.view(G * S, DV))
            del p
            if cap:
                ds = ds * (1.0 - t * t)
            ds = ds * scale
            dq[b, hs] = torch.matmul(ds, k)
            dk[b, h] = torch.matmul(ds.view(G * S, S).t().contiguous(),
                                    q.reshape(G * S, DQ))
    out = out.view(B, S, H * DV).to(BF)
    return [out, dq.to(BF), dk.to(BF), dv.to(BF)] if case["train"] else [out]


def _frequencies(case):
    """Inverse frequencies (Python floats) and the amplitude of a rotation."""
    d, theta, sc = case["rotary"], case["theta"], SCALINGS[case["scaling"]]
    inv = [theta ** (-2.0 * j / d) for j in range(d // 2)]
    if sc is None:
        return inv, 1.0
    f = sc["factor"]
    if sc["rope_type"] == "linear":
        return [x / f for x in inv], 1.0
    old = sc["original_max_position_embeddings"]
    if sc["rope_type"] == "llama3":
        lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
        out = []
        for x in inv:
            turns = old * x / (2 * math.pi)  # of this pair over the original context
            mix = min(1.0, max(0.0, (turns - lo) / (hi - lo)))
            out.append(mix * x + (1.0 - mix) * x / f)
        return out, 1.0

    def pair_of(turns):
        return d * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))
    a = max(math.floor(pair_of(sc["beta_fast"])), 0)
    z = min(math.ceil(pair_of(sc["beta_slow"])), d - 1)
    width = z - a if z != a else 0.001
    out = []
    for j, x in enumerate(inv):
        ramp = min(1.0, max(0.0, (j - a) / width))
        out.append(x / f * ramp + x * (1.0 - ramp))
    return out, 0.1 * math.log(f) + 1.0


def _turn(x, cos, sin, interleaved):
    """Rotation of the last axis (all of it rotated) by tables of half its width."""
    n = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :n], x[..., n:])
    c, d = a * cos - b * sin, b * cos + a * sin
    return torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)


def _rotary_plain(st):
    case = st["case"]
    B, S, H, KV, D, rot = (case[n] for n in ("B", "S", "heads", "kv", "D", "rotary"))
    phase = st["pos"].to(F64)[..., None] * st["inv"]
    cos = (phase.cos() * st["amplitude"]).to(F32)[:, :, None]
    sin = (phase.sin() * st["amplitude"]).to(F32)[:, :, None]
    y = st["y"].float().view(B, S, H + 2 * KV, D)
    x = y[:, :, :H + KV]
    if case["norm"]:
        w = torch.cat([st["norms"][0].float().expand(H, D),
                       st["norms"][1].float().expand(KV, D)])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + st["eps"])
        n = x * r
        x = n * w
    z = torch.cat((_turn(x[..., :rot], cos, sin, case["interleaved"]), x[..., rot:]), -1)
    outs = [z[:, :, :H], z[:, :, H:], y[:, :, H + KV:]]
    outs = [o.transpose(1, 2).contiguous().to(BF) for o in outs]
    if case["train"]:
        g = torch.cat((st["dq"], st["dk"]), 1).float().transpose(1, 2)
        g = torch.cat((_turn(g[..., :rot], cos, -sin, case["interleaved"]), g[..., rot:]), -1)
        if case["norm"]:
            g = g * w
            g = r * (g - n * (g * n).mean(-1, keepdim=True))
        dy = torch.cat((g, st["dv"].float().transpose(1, 2)), 2).reshape(B * S, -1)
        outs.append(dy.to(BF))
    return outs


def _logprobs_plain(st):
    case = st["case"]
    tokens = st["tokens"]
    logits = torch.matmul(st["hidden"].float(), st["head"].float().t())
    cols = torch.arange(case["V"], device=tokens.device)
    x, t = logits, None
    if case["cap"]:
        t = torch.tanh(logits / case["cap"])
        x = t * case["cap"]
    x = x / case["temperature"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    p = e / total
    lp = (x - top) - torch.log(total)
    ent = torch.log(total[:, 0]) - (p * (x - top)).sum(-1)
    kept = tokens >= 0
    given = torch.where(kept, tokens, 0)[:, None]
    res = [torch.where(kept, lp.gather(1, given)[:, 0], 0.0), ent]
    idx = []
    if case["top"]:
        rest = logits.clone()
        for _ in range(case["top"]):
            m = rest.amax(-1, keepdim=True)
            idx.append(torch.where(rest == m, cols, case["V"]).amin(-1, keepdim=True))
            rest.scatter_(1, idx[-1], -math.inf)
        idx = torch.cat(idx, 1)
        res += [lp.gather(1, idx), idx]
    if case["train"]:
        g_lp = torch.where(kept, st["g_lp"], 0.0)[:, None]
        total_g = g_lp
        d = torch.zeros_like(x).scatter_add_(1, given, g_lp)
        if case["top"]:
            d.scatter_add_(1, idx, st["g_top"])
            total_g = g_lp + st["g_top"].sum(1, keepdim=True)
        d = d - p * total_g - st["g_ent"][:, None] * p * (lp + ent[:, None])
        d = d / case["temperature"]
        if case["cap"]:
            d = d * (1.0 - t * t)
        res.append(torch.matmul(d, st["head"].float()).to(BF))
    return res


# ----------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return {"spans": _spans_plain, "rotary": _rotary_plain,
                "logprobs": _logprobs_plain}[case["kind"]](state)
    if case["kind"] == "spans":
        from spilltune_amd import packed
        out = packed.span_attention(state["q"], state["k"], state["v"], state["scale"],
                                    state["mask"], cap=case["cap"] or None,
                                    slopes=state["slopes"])
        if not case["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, [state["q"], state["k"], state["v"]],
                                                   state["dout"])]
    if case["kind"] == "rotary":
        from spilltune_amd import packed
        q, k, v = packed.rope_positions(state["y"], state["pos"], state["rotary"], case["heads"],
                                        case["kv"], norms=state["norms"], eps=state["eps"])
        if not case["train"]:
            return [q, k, v]
        (dy,) = torch.autograd.grad([q, k, v], [state["y"]],
                                    [state["dq"], state["dk"], state["dv"]])
        return [q.detach(), k.detach(), v.detach(), dy]
    from spilltune_amd import ops
    r = ops.token_logprobs(state["hidden"], state["head"], state["tokens"], top=case["top"],
                           temperature=case["temperature"], cap=case["cap"] or None)
    res = [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_tokens] if case["top"] else [])
    if case["train"]:
        heads = [r.logprobs, r.entropy] + ([r.top_logprobs] if case["top"] else [])
        grads = [state["g_lp"], state["g_ent"]] + ([state["g_top"]] if case["top"] else [])
        (dh,) = torch.autograd.grad(heads, [state["hidden"]], grads)
        res = [t.detach() for t in res] + [dh]
    return res


# ----------------------------------------------------------------- floors
def work(case):
    if case["kind"] == "spans":
        B, S, H, KV, DQ, DV = (case[n] for n in ("B", "S", "heads", "kv", "DQ", "DV"))
        qb, kb, vb = 2 * B * S * H * DQ, 2 * B * S * KV * DQ, 2 * B * S * KV * DV
        ob = 2 * B * S * H * DV
        flops = 2 * _pairs(case) * H * (DQ + DV)
        moved = qb + kb + vb + ob
        if case["train"]:  # dO in; dQ, dK, dV out; S, dP, dV, dQ, dK
            flops += 2 * _pairs(case) * H * (3 * DQ + 2 * DV)
            moved += ob + qb + kb + vb
        return {"bytes": moved, "flops": flops}
    if case["kind"] == "rotary":
        M, W = case["B"] * case["S"], (case["heads"] + 2 * case["kv"]) * case["D"]
        n = 2 * M * W * (2 if not case["train"] else (5 if case["norm"] else 4))
        return {"bytes": n, "flops": M * W * (3 if not case["train"] else 6)}
    R, H, V = case["rows"], case["H"], case["V"]
    moved = 2 * V * H + 2 * R * H + 8 * R + 8 * R + 12 * R * case["top"]
    flops = 2 * R * V * H
    if case["train"]:
        moved += 2 * R * H + 8 * R
        flops *= 2
    return {"bytes": moved, "flops": flops}


# ----------------------------------------------------------------- 64 bits
def _spans_exact(case, st):
    """Document by document: each query's run of keys as its own softmax."""
    B, H, S, DQ = st["q"].shape
    KV, DV = st["k"].shape[1], st["v"].shape[-1]
    G, scale = H // KV, float(st["scale"])
    q, k, v = (st[n].double() for n in "qkv")
    out = torch.zeros(B, H, S, DV, dtype=F64, device=q.device)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    do = st["dout"].double().view(B, S, H, DV).transpose(1, 2) if case["train"] else None
    for b, s, e, first, end in _key_runs(case):
        a0 = torch.tensor(first, device=q.device)[:, None]
        z0 = torch.tensor(end, device=q.device)[:, None]
        j = torch.arange(s, e, device=q.device)[None, :]
        hidden = (j < a0) | (j >= z0)
        far = (j - j.t()).abs().double()
        # a long document head by head, the heads of a short one together
        n = H if e - s <= 1024 else 1
        for h in range(0, H, n):
            hs, of = slice(h, h + n), [x // G for x in range(h, h + n)]
            kk, vv, qq = k[b, of, s:e], v[b, of, s:e], q[b, hs, s:e]
            score = (qq @ kk.mT) * scale
            slope = 1.0
            if case["cap"]:
                th = (score / case["cap"]).tanh()
                score, slope = case["cap"] * th, 1.0 - th ** 2
            if st["slopes"] is not None:
                score = score - st["slopes"][hs].double()[:, None, None] * far
            prob = score.masked_fill(hidden, -math.inf).softmax(-1)
            out[b, hs, s:e] = prob @ vv
            if case["train"]:
                g = do[b, hs, s:e]
                dp = g @ vv.mT
                ds = prob * (dp - (g * out[b, hs, s:e]).sum(-1, keepdim=True)) * slope * scale
                grads[0][b, hs, s:e] = ds @ kk
                of = torch.tensor(of, device=q.device)
                grads[1][b, :, s:e].index_add_(0, of, ds.mT @ qq)
                grads[2][b, :, s:e].index_add_(0, of, prob.mT @ g)
    out = out.transpose(1, 2).reshape(B, S, H * DV)
    return [out, *grads] if case["train"] else [out]


def _rotary_exact(case, st):
    """Pair by pair as a complex product; gradients through autograd in 64 bits."""
    B, S, H, KV, D, rot = (case[n] for n in ("B", "S", "heads", "kv", "D", "rotary"))
    inv, amplitude = _frequencies(case)
    angle = st["pos"].double()[:, :, None] * torch.tensor(inv, dtype=F64, device=st["pos"].device)
    turn = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    y = st["y"].detach().double().requires_grad_(True)
    heads = y.view(B, S, H + 2 * KV, D).transpose(1, 2)
    q, k, v = heads.split([H, KV, KV], 1)
    res = []
    for n, x in enumerate((q, k)):
        if case["norm"]:
            x = x / (x.square().mean(-1, keepdim=True) + st["eps"]).sqrt() * st["norms"][n].double()
        r = x[..., :rot]
        pairs = r.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else \
            r.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        res.append(torch.cat((z, x[..., rot:]), -1))
    res.append(v)
    if not case["train"]:
        return [t.detach() for t in res]
    (dy,) = torch.autograd.grad(res, y, [st["dq"].double(), st["dk"].double(), st["dv"].double()])
    return [t.detach() for t in res] + [dy]


def _logprobs_exact(case, st):
    head = st["head"].double()
    logits = st["hidden"].detach().double() @ head.T
    x = case["cap"] * (logits / case["cap"]).tanh() if case["cap"] else logits
    lp = (x / case["temperature"]).log_softmax(-1)
    del x
    p = lp.exp()
    ent = -(p * lp).sum(-1)
    kept = st["tokens"] >= 0
    rows = torch.arange(case["rows"], device=kept.device)
    given = st["tokens"].clamp(min=0)
    res = [lp[rows, given] * kept, ent]
    if case["top"]:
        rest, idx = logits.clone(), []
        for _ in range(case["top"]):
            best = rest.max(-1, keepdim=True).values
            idx.append((rest == best).to(torch.uint8).argmax(-1))
            first = torch.where(rest == best, torch.arange(case["V"], device=kept.device),
                                case["V"]).min(-1).values
            idx[-1] = first
            rest[rows, first] = -math.inf
        del rest
        idx = torch.stack(idx, 1)
        res += [lp.gather(1, idx), idx]
    if case["train"]:
        # d lp_c / d x_j = [c = j] - p_j;  d entropy / d x_j = -p_j (lp_j + entropy)
        weight = torch.zeros_like(lp)
        weight[rows, given] += st["g_lp"].double() * kept
        if case["top"]:
            weight.scatter_add_(1, idx, st["g_top"].double())
        d = weight - p * weight.sum(-1, keepdim=True)
        d -= st["g_ent"].double()[:, None] * p * (lp + ent[:, None])
        d /= case["temperature"]
        if case["cap"]:
            d *= 1.0 - (logits / case["cap"]).tanh().square()
        res.append(d @ head)
    return res


def exact(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    return {"spans": _spans_exact, "rotary": _rotary_exact,
            "logprobs": _logprobs_exact}[case["kind"]](case, st)
