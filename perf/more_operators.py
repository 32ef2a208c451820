"""Operator cases: one training step of a decoder that adapts more than its
projections.

Four operators stand around the 4-bit matrix products of such a step: the scaled
lookup of the token embedding with its gradient by sorted tokens, the norms after
and before a part of a block with its gate and residual scale, the balance loss of
a router with its per-expert counts, and the orthogonalised update of the adapters'
factors by Newton-Schulz products.

``own`` is False: ``run`` computes each operator in elementary torch operations in
32 bits.  ``own`` is True: ``run`` calls this package.  ``exact`` restates the
operators in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF, "fp32": F32}

# [out, in] of a decoder layer's seven projections
LAYERS = {
    "llama8b": [(4096, 4096), (1024, 4096), (1024, 4096), (4096, 4096), (14336, 4096),
                (14336, 4096), (4096, 14336)],
    "unit": [(256, 256), (64, 256), (64, 256), (256, 256), (688, 256), (688, 256), (256, 688)],
}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # ---- norms after and before a part of a block
        # one new token of each of four conversations: launches and host work count
        {"name": "norms_tokens", "kind": "norms", "B": 4, "S": 1, "H": 4096, "post": True,
         "pre": True, "gate": "none", "scale": 1.0, "train": False, "learn": False},
        # a training microbatch between attention and MLP, frozen norms, scaled residual
        {"name": "norms_train", "kind": "norms", "B": 4, "S": 2048, "H": 4096, "post": True,
         "pre": True, "gate": "none", "scale": 0.22, "train": True, "learn": False},
        # odd rows of a wide model whose norms and per-channel gate are learnt too
        {"name": "norms_gate", "kind": "norms", "B": 1, "S": 2103, "H": 7168, "post": True,
         "pre": True, "gate": "channel", "scale": 1.0, "train": True, "learn": True},
        # ---- embedding
        # the next token of a handful of rows
        {"name": "embed_tokens", "kind": "embed", "B": 16, "S": 1, "V": 32000, "H": 1024,
         "dtype": "bf16", "scale": 32.0, "padding": False, "train": False},
        # a packed training row over a large vocabulary, the table's gradient with it
        {"name": "embed_train", "kind": "embed", "B": 1, "S": 8192, "V": 128256, "H": 4096,
         "dtype": "fp32", "scale": 1.0, "padding": False, "train": True},
        # padded rows of a smaller model, a large accumulation window, scaled lookup
        {"name": "embed_padded", "kind": "embed", "B": 16, "S": 2103, "V": 32000, "H": 1024,
         "dtype": "bf16", "scale": 32.0, "padding": True, "train": True},
        # ---- balance
        # a microbatch of short chat turns
        {"name": "balance_short", "kind": "balance", "B": 3, "S": 77, "E": 128, "k": 8,
         "score": "softmax", "dtype": "bf16", "per_row": False, "valid": 0.9, "train": True},
        # four rows of a group-limited router's sigmoid scores, each balanced by itself
        {"name": "balance_rows", "kind": "balance", "B": 4, "S": 4096, "E": 256, "k": 8,
         "score": "sigmoid", "dtype": "fp32", "per_row": True, "valid": 0.97, "train": True},
        # ---- orthogonalised updates
        # one layer of a unit-sized model, rank 4
        {"name": "muon_unit", "kind": "muon", "layer": "unit", "layers": 1, "rank": 4,
         "stacked": False, "experts": 0, "H": 0, "I": 0, "steps": 5, "dtype": "fp32"},
        # the whole adapter set of 32 layers at rank 16, the layers' factors of one kind stacked
        {"name": "muon_model", "kind": "muon", "layer": "llama8b", "layers": 32, "rank": 16,
         "stacked": True, "experts": 0, "H": 0, "I": 0, "steps": 5, "dtype": "fp32"},
        # one layer's per-expert adapters of gate|up and down
        {"name": "muon_experts", "kind": "muon", "layer": "", "layers": 1, "rank": 16,
         "stacked": True, "experts": 128, "H": 2048, "I": 768, "steps": 5, "dtype": "fp32"},
        # two layers at a large rank
        {"name": "muon_wide", "kind": "muon", "layer": "llama8b", "layers": 2, "rank": 128,
         "stacked": False, "experts": 0, "H": 0, "I": 0, "steps": 5, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norms", "embed", "balance", "muon"])
    if kind == "norms":
        H = rng.choice([8 * _log(rng, 8, 1024), 8 * _log(rng, 8, 1024), _log(rng, 60, 2000)])
        B = rng.choice([1, 2, 4])
        return {"kind": "norms", "B": B, "S": _log(rng, 1, max(2, (1 << 25) // (H * B))), "H": H,
                "post": rng.random() < 0.8, "pre": rng.random() < 0.8,
                "gate": rng.choice(["none", "channel", "row", "token", "full"]),
                "scale": rng.choice([1.0, 0.22, 1.7]), "train": rng.random() < 0.7,
                "learn": rng.random() < 0.5}
    if kind == "embed":
        H = rng.choice([8 * _log(rng, 8, 512), _log(rng, 30, 1000)])
        V = _log(rng, 100, 150000)
        return {"kind": "embed", "B": rng.choice([1, 2, 7]),
                "S": _log(rng, 1, max(2, min(5000, (1 << 23) // H))), "V": V, "H": H,
                "dtype": rng.choice(["bf16", "fp32"]), "scale": rng.choice([1.0, math.sqrt(H)]),
                "padding": rng.random() < 0.4, "train": rng.random() < 0.7}
    if kind == "balance":
        E = rng.choice([8, 16, 60, 64, 128, 256, 384])
        return {"kind": "balance", "B": rng.choice([1, 2, 4]), "S": _log(rng, 1, 4000), "E": E,
                "k": rng.choice([1, 2, 4, 8]), "score": rng.choice(["softmax", "sigmoid"]),
                "dtype": rng.choice(["bf16", "fp32"]), "per_row": rng.random() < 0.5,
                "valid": rng.choice([1.0, 0.9, 0.3]), "train": rng.random() < 0.8}
    if rng.random() < 0.3:
        return {"kind": "muon", "layer": "", "layers": 1, "rank": rng.choice([4, 8, 12, 16]),
                "stacked": True, "experts": _log(rng, 2, 64), "H": 8 * _log(rng, 32, 256),
                "I": 8 * _log(rng, 8, 96),
                "steps": rng.choice([4, 5, 6]), "dtype": rng.choice(["fp32", "bf16"])}
    rank, stacked = _log(rng, 1, 128), rng.random() < 0.5
    return {"kind": "muon", "layer": rng.choice(["llama8b", "unit"]),
            "layers": max(1, min(8 if stacked else 4, 128 // rank)), "rank": rank,
            "stacked": stacked, "experts": 0, "H": 0, "I": 0,
            "steps": rng.choice([4, 5, 6]), "dtype": rng.choice(["fp32", "bf16"])}


# ----------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 29)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32)


def _norms_inputs(case, seed):
    g = _gen(seed)
    B, S, H = case["B"], case["S"], case["H"]
    y = _randn(g, B, S, H) * (0.2 + _randn(g, B, S, 1).abs())  # rows of unequal size
    res = 2.0 * _randn(g, B, S, H)
    res[..., :: max(1, H // 7)] *= 8.0  # outlier channels of a residual stream
    st = {"y": y.to(BF), "res": res.to(BF), "eps": 1e-6, "post": None, "pre": None, "gate": None}
    for n in ("post", "pre"):
        if case[n]:
            st[n] = (1.0 + 0.3 * _randn(g, H)).to(BF)
    shape = {"none": None, "channel": (H,), "row": (B, 1, H), "token": (B, S, 1),
             "full": (B, S, H)}[case["gate"]]
    if shape:
        st["gate"] = (0.5 + 0.3 * _randn(g, *shape)).to(BF)
    if case["train"]:
        st["dh"] = _randn(g, B, S, H).to(BF)
        if case["pre"]:
            st["dn"] = _randn(g, B, S, H).to(BF)
    return st


def _embed_inputs(case, seed):
    g = _gen(seed)
    B, S, V, H = case["B"], case["S"], case["V"], case["H"]
    # words' frequencies fall with their rank; ranks lie anywhere in the table
    rank = torch.exp(torch.rand(B, S, generator=g, device="cuda", dtype=F64) * math.log(V))
    ids = (rank.long().clamp_(1, V) - 1) * 7919 % V
    if case["padding"]:
        keep = torch.randint(0, S + 1, (B, 1), generator=g, device="cuda")
        ids = torch.where(torch.arange(S, device="cuda") < keep, ids, 0)
    st = {"ids": ids, "table": (0.02 * _randn(g, V, H)).to(DTYPES[case["dtype"]])}
    if case["train"]:
        st["dout"] = _randn(g, B, S, H).to(BF)
    return st


def _balance_inputs(case, seed):
    g = _gen(seed)
    B, S, E, k = case["B"], case["S"], case["E"], case["k"]
    # a router that prefers some experts
    logits = 1.3 * _randn(g, B, S, E) + 0.8 * _randn(g, E)
    st = {"logits": logits.to(DTYPES[case["dtype"]])}
    st["indices"] = st["logits"].float().topk(k, -1).indices.to(torch.int32).contiguous()
    st["valid"] = None
    if case["valid"] < 1.0:  # right padding
        n = (S * (case["valid"] + (1.0 - case["valid"]) *
                  torch.rand(B, 1, generator=g, device="cuda"))).long()
        st["valid"] = torch.arange(S, device="cuda") < n
    st["g"] = 0.5 + torch.rand((), generator=g, device="cuda")
    return st


def _matrices(case):
    """Shapes of the case's updates: a list of 2-D and (experts') 3-D shapes."""
    r = case["rank"]
    if case["experts"]:
        E, H, I = case["experts"], case["H"], case["I"]
        # gate and up, then down: A [r, in], B [out, r] of every expert
        return [(2 * E, r, H), (2 * E, I, r), (E, r, I), (E, H, r)]
    one = [s for n, m in LAYERS[case["layer"]] for s in ((r, m), (n, r))]
    if case["stacked"]:
        return [(case["layers"], *s) for s in one]
    return one * case["layers"]


def _muon_inputs(case, seed):
    g = _gen(seed)
    out = []
    for shape in _matrices(case):
        short = min(shape[-2:])
        # momentum of gradients: a few strong directions, the rest down to 1/30
        fall = torch.logspace(0, -1.5, short, device="cuda", dtype=F32)
        fall = 1e-3 * (0.5 + torch.rand((), generator=g, device="cuda")) * fall
        u = _randn(g, *shape) * (fall[:, None] if shape[-2] == short else fall)
        out.append(u.to(DTYPES[case["dtype"]]))
    out[0].zero_()  # A has no gradient while its B is zero
    return {"updates": out}


_INPUTS = {"norms": _norms_inputs, "embed": _embed_inputs, "balance": _balance_inputs,
           "muon": _muon_inputs}
# inputs that are differentiated, in the order of the outputs
_LEAVES = {"norms": ("y", "res"), "embed": ("table",), "balance": ("logits",), "muon": ()}


def _leaves(case):
    names = _LEAVES[case["kind"]]
    if case["kind"] == "norms" and case["learn"]:
        names += tuple(n for n, has in (("gate", case["gate"] != "none"), ("post", case["post"]),
                                        ("pre", case["pre"])) if has)
    return names if case.get("train") else ()


def prepare(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    st["case"] = case
    if own:
        for n in _leaves(case):
            st[n].requires_grad_(True)
    return st


# ----------------------------------------------------------------- plain forms
def _norms_plain(st):
    case = st["case"]
    y, res = st["y"].float(), st["res"].float()
    H = case["H"]
    gate = 1.0 if st["gate"] is None else st["gate"].float()
    z = y
    if case["post"]:
        r1 = 1.0 / torch.sqrt((y * y).sum(-1, keepdim=True) / H + st["eps"])
        yn = y * r1
        z = yn * st["post"].float()
    h = res + case["scale"] * gate * z
    out = [h]
    if case["pre"]:
        r2 = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / H + st["eps"])
        hn = h * r2
        out.append(hn * st["pre"].float())
    if case["train"]:
        dH = st["dh"].float()
        grads = {}
        if case["pre"]:
            dn = st["dn"].float()
            grads["pre"] = (dn * hn).sum((0, 1))
            g = dn * st["pre"].float()
            dH = dH + r2 * (g - hn * ((g * hn).sum(-1, keepdim=True) / H))
        grads["res"] = dH
        if st["gate"] is not None and case["learn"]:
            d = case["scale"] * dH * z
            over = [i for i, (a, b) in enumerate(zip((1,) * (3 - st["gate"].dim())
                                                     + tuple(st["gate"].shape), d.shape)) if a != b]
            d = d.sum(over, keepdim=True) if over else d
            grads["gate"] = d.reshape(st["gate"].shape)
        q = case["scale"] * gate * dH
        if case["post"]:
            grads["post"] = (q * yn).sum((0, 1))
            w = q * st["post"].float()
            q = r1 * (w - yn * ((w * yn).sum(-1, keepdim=True) / H))
        grads["y"] = q
        out += [grads[n] for n in _leaves(case)]
    return [t.to(BF) for t in out]


def _embed_plain(st):
    case = st["case"]
    table, ids = st["table"], st["ids"]
    out = [(table[ids].float() * case["scale"]).to(BF)]
    if case["train"]:
        flat = ids.reshape(-1)
        d = st["dout"].float().reshape(-1, case["H"])
        if case["padding"]:
            d = d * (flat != 0)[:, None]
        grad = torch.zeros(table.shape, dtype=F32, device=table.device).index_add_(0, flat, d)
        out.append((grad * case["scale"]).to(table.dtype))
    return out


def _balance_plain(st):
    case = st["case"]
    B, S, E, k = (case[n] for n in ("B", "S", "E", "k"))
    G = B if case["per_row"] else 1
    x = st["logits"].float().reshape(G, -1, E)
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        total = e.sum(-1, keepdim=True)
    else:
        e = 1.0 / (1.0 + torch.exp(-x))
        total = e.sum(-1, keepdim=True) + 1e-20
    p = e / total
    valid = torch.ones(B, S, dtype=torch.bool, device=x.device) if st["valid"] is None else st["valid"]
    valid = valid.reshape(G, -1)
    n = valid.sum(-1)
    picks = st["indices"].long().reshape(G, -1)
    counts = torch.zeros(G, E, dtype=torch.int64, device=x.device)
    counts.scatter_add_(1, picks, valid[:, :, None].expand(-1, -1, k).reshape(G, -1).long())
    many = n.clamp(min=1).float()[:, None]
    groups = (n > 0).sum().clamp(min=1).float()
    f = counts.float() * E / (k * many)
    mean = (p * valid[:, :, None]).sum(1) / many
    loss = (f * mean).sum() / groups
    out = [loss, counts]
    if case["train"]:
        a = (f / many / groups * st["g"])[:, None, :]
        dp = a - (a * p).sum(-1, keepdim=True)
        d = p * dp if case["score"] == "softmax" else dp / total * e * (1.0 - e)
        d = d * valid[:, :, None]
        out.append(d.reshape(B, S, E).to(st["logits"].dtype))
    return out


def _newton_schulz(u, steps):
    """[n, rows, columns] in 32 bits, on the shorter side."""
    a, b, c = COEFFICIENTS
    x = u.float()
    if x.shape[-2] > x.shape[-1]:
        x = x.transpose(-2, -1).contiguous()
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + 1e-7)
    for _ in range(steps):
        gram = torch.bmm(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return (x if u.shape[-2] <= u.shape[-1] else x.transpose(-2, -1)).contiguous()


def _muon_plain(st):
    out = []
    for u in st["updates"]:
        o = _newton_schulz(u.reshape(-1, *u.shape[-2:]), st["case"]["steps"])
        out.append(o.reshape(u.shape).to(u.dtype))
    return out


# ----------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return {"norms": _norms_plain, "embed": _embed_plain, "balance": _balance_plain,
                "muon": _muon_plain}[case["kind"]](state)
    leaves = [state[n] for n in _leaves(case)]
    if case["kind"] == "norms":
        from spilltune_amd import ops
        out = ops.residual_norms(state["y"], state["res"], state["post"], state["pre"],
                                 gate=state["gate"], scale=case["scale"], eps=state["eps"])
        out = list(out) if case["pre"] else [out]
        if not leaves:
            return out
        up = [state["dh"]] + ([state["dn"]] if case["pre"] else [])
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, up))
    if case["kind"] == "embed":
        from spilltune_amd import ops
        out = ops.embedding(state["table"], state["ids"], scale=case["scale"],
                            padding_idx=0 if case["padding"] else None)
        if not leaves:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, leaves, state["dout"])]
    if case["kind"] == "balance":
        from spilltune_amd import moe
        loss, counts = moe.balance_loss(state["logits"], state["indices"], score=case["score"],
                                        valid=state["valid"], per_row=case["per_row"])
        if not leaves:
            return [loss, counts]
        return [loss.detach(), counts, *torch.autograd.grad(loss, leaves, state["g"])]
    from spilltune_amd import muon
    return muon.orthogonalize(state["updates"], steps=case["steps"], coefficients=COEFFICIENTS)


# ----------------------------------------------------------------- floors
def work(case):
    if case["kind"] == "norms":
        M, H = case["B"] * case["S"], case["H"]
        full = M * H
        gate = {"none": 0, "channel": H, "row": case["B"] * H, "token": M, "full": full}[case["gate"]]
        n = 3 * full + gate + (full if case["pre"] else 0)
        if case["train"]:
            n += 3 * full + (full if case["pre"] else 0) + (gate if case["learn"] else 0)
        return {"bytes": 2 * n, "flops": (34 if case["train"] else 12) * full}
    if case["kind"] == "embed":
        N, V, H = case["B"] * case["S"], case["V"], case["H"]
        size = 2 if case["dtype"] == "bf16" else 4
        n = N * (8 + 2 * H) + min(N, V) * H * size
        if case["train"]:
            n += 2 * N * H + V * H * size
        return {"bytes": n, "flops": N * H * (2 if case["train"] else 1)}
    if case["kind"] == "balance":
        N, E = case["B"] * case["S"], case["E"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": N * (E * size * (2 if case["train"] else 1) + 4 * case["k"] + 1),
                "flops": N * E * (12 if case["train"] else 5)}
    size = 2 if case["dtype"] == "bf16" else 4
    moved = flops = 0
    for shape in _matrices(case):
        n, (a, b) = (shape[0] if len(shape) == 3 else 1), shape[-2:]
        r, K = min(a, b), max(a, b)
        moved += 2 * size * n * r * K
        # half of the Gram matrix, its polynomial, one product with it
        flops += n * (r * (r + 1) * K + case["steps"] * 4 * r ** 3 + 2 * r * r * K)
    return {"bytes": moved, "flops": flops}


# ----------------------------------------------------------------- 64 bits
def _norms_exact(case, st):
    """Through autograd, in 64 bits."""
    t = {n: None if st[n] is None else st[n].detach().double().requires_grad_(True)
         for n in ("y", "res", "gate", "post", "pre")}

    def norm(x, w):
        return w * (x / (x.square().mean(-1, keepdim=True) + st["eps"]).sqrt())

    z = t["y"] if t["post"] is None else norm(t["y"], t["post"])
    z = z * case["scale"]
    h = t["res"] + (z if t["gate"] is None else t["gate"] * z)
    out = [h] if t["pre"] is None else [h, norm(h, t["pre"])]
    res = [o.detach() for o in out]
    if case["train"]:
        up = [st["dh"].double()] + ([st["dn"].double()] if case["pre"] else [])
        res += torch.autograd.grad(out, [t[n] for n in _leaves(case)], up)
    return res


def _embed_exact(case, st):
    res = [torch.nn.functional.embedding(st["ids"], st["table"].detach().double()) * case["scale"]]
    if case["train"]:
        ids, order = st["ids"].flatten().sort(stable=True)
        d = st["dout"].double().reshape(-1, case["H"])[order]
        if case["padding"]:
            d, ids = d[ids != 0], ids[ids != 0]
        grad = torch.zeros(st["table"].shape, dtype=F64, device=d.device)
        rows, many = torch.unique_consecutive(ids, return_counts=True)
        if len(rows):
            grad[rows] = torch.segment_reduce(d, "sum", lengths=many, axis=0) * case["scale"]
        res.append(grad)
    return res


def _balance_exact(case, st):
    logits = st["logits"].detach().double().requires_grad_(True)
    E, k = case["E"], case["k"]
    valid = st["valid"]
    if valid is None:
        valid = torch.ones(logits.shape[:2], dtype=torch.bool, device=logits.device)
    terms, counts = [], []
    for rows in (range(case["B"]) if case["per_row"] else [slice(None)]):
        x, v, i = logits[rows].reshape(-1, E), valid[rows].reshape(-1), st["indices"][rows]
        x, i = x[v], i.reshape(-1, k)[v]
        counts.append(torch.bincount(i.flatten().long(), minlength=E))
        if len(x):
            p = x.softmax(-1)
            if case["score"] == "sigmoid":
                p = x.sigmoid() / (x.sigmoid().sum(-1, keepdim=True) + 1e-20)
            terms.append(E * (counts[-1].double() / (k * len(x)) * p.mean(0)).sum())
    loss = sum(terms) / max(1, len(terms)) + 0.0 * logits.sum()
    res = [loss.detach(), torch.stack(counts)]
    if case["train"]:
        res += torch.autograd.grad(loss, [logits], st["g"].double())
    return res


def _muon_exact(case, st):
    a, b, c = COEFFICIENTS
    out = []
    for u in st["updates"]:
        x = u.double()
        x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
        tall = x.shape[-2] > x.shape[-1]
        for _ in range(case["steps"]):  # from the side that is short, without turning x
            gram = x.mT @ x if tall else x @ x.mT
            poly = b * gram + c * gram @ gram
            x = a * x + (x @ poly if tall else poly @ x)
        out.append(x)
    return out


def exact(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    return {"norms": _norms_exact, "embed": _embed_exact, "balance": _balance_exact,
            "muon": _muon_exact}[case["kind"]](case, st)
