"""64-bit restatements of the packed-row operators, with bounds on what a
kernel that rounds to bf16 where these do may be off by."""
import math

import torch

U = 2.0 ** -8  # half a step of bf16, relative to the value


def runs_brute(documents, bidirectional=None, window=None):
    """Per token: the first key, the end of the keys, and the position, by walking."""
    B, S = documents.shape
    lo, hi, pos = (torch.zeros(B, S, dtype=torch.int32) for _ in range(3))
    for b in range(B):
        d = documents[b].tolist()
        m = bidirectional[b].tolist() if bidirectional is not None else [False] * S
        for i in range(S):
            if d[i] < 0:
                continue
            s = i
            while s > 0 and d[s - 1] == d[i]:
                s -= 1
            e = i + 1
            while m[i] and e < S and d[e] == d[i] and m[e]:
                e += 1
            pos[b, i] = i - s
            lo[b, i] = max(s, i - window + 1) if window else s
            hi[b, i] = e
    return lo, hi, pos


def span_scores(q, k, scale, lo, hi, cap, slopes):
    """(masked scores, d score / d (scale q.k)) of float64 q, k [B,H,S,D]."""
    S = q.shape[2]
    x = (q @ k.transpose(-1, -2).contiguous()) * scale
    grad = torch.ones_like(x)
    if cap:
        t = torch.tanh(x / cap)
        x, grad = cap * t, 1 - t * t
    at = torch.arange(S, device=q.device)
    if slopes is not None:
        x = x - slopes.double()[None, :, None, None] * (at[:, None] - at[None, :]).abs()
    lo, hi = lo.long().clamp(0, S), hi.long().clamp(0, S)
    sees = (at >= lo[..., None]) & (at < hi[..., None])  # [B,S,S]
    return torch.where(sees[:, None], x, -math.inf), grad, sees[:, None]


def span_forward(q, k, v, scale, lo, hi, cap=None, slopes=None):
    """Output [B,H,S,DV] (float64, every head with its own key rows)."""
    x, _, sees = span_scores(q, k, scale, lo, hi, cap, slopes)
    top = torch.where(sees.any(-1, keepdim=True), x.amax(-1, keepdim=True), 0.0)
    e = torch.where(sees, torch.exp(x - top), 0.0)
    n = e.sum(-1, keepdim=True)
    return (e / torch.where(n > 0, n, 1.0)) @ v


def span_ref(q, k, v, scale, lo, hi, cap=None, slopes=None, dout=None, rounded_ds=False):
    """(values, bounds) of out [B,S,H*DV] and, with dout, dq, dk, dv, by the formulas.

    Bounds: probabilities are rounded to bf16 (U of each value), dS is not; each
    result is rounded once.  delta is summed from the rounded output where a tile's
    queries see more than 256 keys in all (rows longer than that may), from the
    fp32 products otherwise.  fp32 scores of D products, exponentials and sums are
    off by 2^-12 at most, dP by D products of |dO||V|; a tenth covers the first in
    the terms that bf16 rules.  ``rounded_ds``: the bounds of a kernel that rounds
    dS to bf16 and always sums delta from the rounded output."""
    B, H, S, DQ = q.shape
    KV, DV = k.shape[1], v.shape[-1]
    G = H // KV
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    x, grad, sees = span_scores(q, k, scale, lo, hi, cap, slopes)
    top = torch.where(sees.any(-1, keepdim=True), x.amax(-1, keepdim=True), 0.0)
    e = torch.where(sees, torch.exp(x - top), 0.0)
    n = e.sum(-1, keepdim=True)
    p = e / torch.where(n > 0, n, 1.0)
    tok = lambda t: t.transpose(1, 2).reshape(B, S, -1)  # noqa: E731
    o = p @ v
    o_err = 1.1 * U * (p @ v.abs() + o.abs())
    if dout is None:
        return [tok(o)], [tok(o_err)]
    do = dout.double().view(B, S, H, DV).transpose(1, 2).contiguous()
    dp = do @ v.transpose(-1, -2).contiguous()
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * grad
    size = do.abs() @ v.abs().transpose(-1, -2).contiguous()
    delta_err = (do.abs() * o_err).sum(-1, keepdim=True) \
        if S > 256 or rounded_ds else 0.0
    one = sees.sum(-1, keepdim=True) == 1
    ds_err = p * grad * (2.0 ** -12 * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))
                         + 2.0 ** -17 * (size + (p * size).sum(-1, keepdim=True)) + delta_err)
    ds_err = ds_err + U * ds.abs() if rounded_ds else torch.where(one, 0.0, ds_err)
    T = lambda t: t.transpose(-1, -2).contiguous()  # noqa: E731
    fold = lambda t: t.view(B, KV, G, S, -1).sum(2)  # noqa: E731
    dq, dk, dv = ds @ k * scale, fold(T(ds) @ q) * scale, fold(T(p) @ do)
    errs = [ds_err @ k.abs() * scale, fold(T(ds_err) @ q.abs()) * scale, fold(T(U * p) @ do.abs())]
    errs = [1.1 * (e + U * t.abs()) for e, t in zip(errs, (dq, dk, dv))]
    return [tok(o), dq, dk, dv], [tok(o_err), *errs]


def rope_ref(y, pos, inv, amplitude, heads, kv, D, rot, interleaved, norms=None, eps=1e-6):
    """q, k, v [B,h,S,D] float64 from float64 rows y [B*S, (heads+2kv)*D]."""
    B, S = pos.shape
    ang = pos.double()[:, None, :, None] * torch.tensor(inv, dtype=torch.float64, device=y.device)
    c, s = amplitude * ang.cos(), amplitude * ang.sin()
    q, k, v = y.view(B, S, heads + 2 * kv, D).transpose(1, 2).split([heads, kv, kv], 1)
    out = []
    for i, x in enumerate((q, k)):
        if norms is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * norms[i].double()
        r, rest = x[..., :rot], x[..., rot:]
        a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, -1)
        u, w = a * c - b * s, b * c + a * s
        t = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
        out.append(torch.cat((t, rest), -1))
    return out + [v]
