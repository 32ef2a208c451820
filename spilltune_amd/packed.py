"""Training on packed rows: several documents back to back in one sequence.

The reference trains one document a row (causal, right padding,
adapters/dense.py:232-248); these have no counterpart there.

* :func:`document_mask` -- the :class:`SpanMask` of a batch of packed rows: for
  every query the run of keys it sees (its document's, up to itself; with
  bidirectional runs and a window), each token's position in its document, and
  the kernels' tile plan.  Made once for a batch and read by every layer.
* :func:`span_attention` -- attention over those runs, optionally with scores
  capped by a tanh and a bias that falls with the distance, differentiable.
* :func:`positions_and_masks` and :func:`document_labels` -- what a model's
  blocks and its loss take for a batch of packed rows.
* :class:`Rotary` and :func:`rope_positions` -- rotation of query and key heads
  by per-token positions: whole heads or a part of them, half or interleaved
  pairs, the scalings for long contexts, optionally after Qwen3's per-head norms.

Ops run on the current stream of their operands' device and never fall back to
another implementation.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from .ops import _no_tangents, _once, _operand, _scratch

_BF16 = torch.bfloat16
_F32 = torch.float32


# ----------------------------------------------------------------- masks
@dataclass(frozen=True, eq=False)  # equal to itself alone: sizes do not make a mask
class SpanMask:
    """Query ``i`` of row ``b`` sees the keys ``[key_start[b, i], key_end[b, i])``
    (int32 [batch, length]); an empty run sees nothing.  ``positions`` (int32) is
    each token's place in its document, ``plan`` the kernels' tables of these
    runs: the tensors belong together and are not to be changed."""
    batch: int
    length: int
    key_start: torch.Tensor
    key_end: torch.Tensor
    positions: torch.Tensor
    plan: torch.Tensor


def span_mask(key_start: torch.Tensor, key_end: torch.Tensor, positions=None) -> SpanMask:
    """The mask of given runs (int32 [batch, length] on one device, bounds
    clamped to the row); ``positions`` default to 0..length-1."""
    for t, name in ((key_start, "key_start"), (key_end, "key_end"), (positions, "positions")):
        if t is None:
            continue
        if t.dtype != torch.int32 or t.dim() != 2 or t.shape != key_start.shape \
                or t.device != key_start.device:
            raise ValueError(f"unsupported_capability: {name} must be int32 [batch, length] on the "
                             "mask's device")
    B, S = key_start.shape
    if B < 1 or S < 1:
        raise ValueError("unsupported_capability: a mask needs at least one token")
    if not key_start.is_cuda:
        raise ValueError("unsupported_capability: a mask lives on the GPU")
    dev = key_start.device
    if positions is None:
        positions = torch.arange(S, dtype=torch.int32, device=dev).expand(B, S)
    # own copies: the plan below is of these values
    key_start, key_end, positions = (t.detach().clone(memory_format=torch.contiguous_format)
                                     for t in (key_start, key_end, positions))
    with _lib.on_device(dev):
        nbytes = _lib.query("st_span_plan_bytes", B, S)
        plan = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.call("st_span_plan", _lib.ptr(key_start), _lib.ptr(key_end), B, S, _lib.ptr(plan), nbytes,
                  _lib.stream_handle(dev))
    return SpanMask(B, S, key_start, key_end, positions, plan)


def document_runs(documents: torch.Tensor, *, bidirectional=None, window=None):
    """``(key_start, key_end, positions)`` (int32) of packed rows, in torch ops on
    the documents' device; see :func:`document_mask`."""
    if documents.dim() != 2 or documents.dtype not in (torch.int32, torch.int64):
        raise ValueError("unsupported_capability: documents must be int32/int64 [batch, length]")
    if bidirectional is not None and (bidirectional.dtype != torch.bool
                                      or bidirectional.shape != documents.shape
                                      or bidirectional.device != documents.device):
        raise ValueError("unsupported_capability: bidirectional must be bool [batch, length] on "
                         "the documents' device")
    if window is not None and (isinstance(window, bool) or not isinstance(window, int)
                               or window < 1):
        raise ValueError("unsupported_capability: window must be a positive integer")
    B, S = documents.shape
    at = torch.arange(S, device=documents.device).expand(B, S)
    real = documents >= 0
    fresh = torch.ones_like(real)
    fresh[:, 1:] = documents[:, 1:] != documents[:, :-1]
    start = torch.where(fresh, at, 0).cummax(1).values
    positions = torch.where(real, at - start, 0)
    end = at + 1
    if bidirectional is not None:
        # a run of marked tokens ends where the next token is unmarked or of another document
        last = torch.ones_like(real)
        last[:, :-1] = fresh[:, 1:] | ~bidirectional[:, 1:]
        stop = torch.where(last, end, S).flip(1).cummin(1).values.flip(1)
        end = torch.where(bidirectional, stop, end)
    if window is not None:
        start = torch.maximum(start, at - (window - 1))
    start, end = torch.where(real, start, 0), torch.where(real, end, 0)
    return start.to(torch.int32), end.to(torch.int32), positions.to(torch.int32)


def document_mask(documents: torch.Tensor, *, bidirectional=None, window=None) -> SpanMask:
    """Mask of packed rows.  ``documents`` (int [batch, length]) names each token's
    document: neighbours with one number belong together, a negative number is
    padding (sees nothing, seen by nothing).  A token sees its document up to
    itself; tokens marked in ``bidirectional`` (bool, e.g. a prompt) also see the
    rest of their unbroken run of marked tokens; with ``window`` only the last
    ``window`` keys before and with the token (and the run's later ones)."""
    if documents.device.type != "cuda":
        raise ValueError("unsupported_capability: documents must be on the GPU")
    return span_mask(*document_runs(documents, bidirectional=bidirectional, window=window))


# ----------------------------------------------------------------- attention
def _span_forward(q, k, v, scale, mask, cap, slopes):
    """(output, log-sum-exp)"""
    B, H, S, DQ = q.shape
    Hkv, DV = k.shape[1], v.shape[-1]
    dev = q.device
    out = torch.empty((B, S, H * DV), dtype=_BF16, device=dev)
    lse = torch.empty((B, H, S), dtype=_F32, device=dev)
    with _lib.on_device(dev):
        _lib.call("st_span_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), B, S, H, Hkv, DQ, DV,
                  scale, cap, _lib.ptr(slopes), mask.key_start.data_ptr(), mask.key_end.data_ptr(),
                  mask.plan.data_ptr(), out.data_ptr(), lse.data_ptr(), _lib.stream_handle(dev))
    return out, lse


class _SpanAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, mask, cap, slopes):
        out, lse = _span_forward(q, k, v, scale, mask, cap, slopes)
        ctx.save_for_backward(q, k, v, out, lse, slopes)
        ctx.meta = (scale, mask, cap)
        return out

    @staticmethod
    def backward(ctx, dout):
        _once()
        # addresses come from the saved tensors as they are now: a hook may have
        # moved them
        q, k, v, out, lse, slopes = ctx.saved_tensors
        scale, mask, cap = ctx.meta
        B, H, S, DQ = q.shape
        shape = (B, S, H, k.shape[1], DQ, v.shape[3])
        dev = dout.device
        dout = _operand(dout)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        with _lib.on_device(dev):
            nbytes = _lib.query("st_span_attn_workspace_bytes", *shape)
            ws = _scratch(dev, nbytes)
            _lib.call("st_span_attn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                      lse.data_ptr(), dout.data_ptr(), *shape, scale, cap, _lib.ptr(slopes),
                      mask.key_start.data_ptr(), mask.key_end.data_ptr(), mask.plan.data_ptr(),
                      dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(ws), nbytes,
                      _lib.stream_handle(dev))
        return dq, dk, dv, None, None, None, None


def span_attention(q, k, v, scale, mask: SpanMask, *, cap=None, slopes=None):
    """q [B,H,S,DQ], k [B,Hkv,S,DQ], v [B,Hkv,S,DV] (bf16, head dims 64/64,
    128/128 or 192/128) -> token-major [B,S,H*DV]: each query over its run of keys
    in ``mask``.  Scores are ``scale * q.k``, with ``cap`` ``cap * tanh(scale * q.k
    / cap)``; ``slopes`` (fp32 [H], constants) subtracts ``slopes[h] * |i - j|``.
    (``scale`` 1e-30 to 1e30, ``cap`` up to 1e30 and at least ``scale / 1e4``.)
    A query that sees nothing gets zeros and passes no gradient on.  Infinities and
    NaN reach what sees them and nothing else.  The gradients form the
    probabilities again from scores and their log-sum-exp in fp32: off by 2^-24 of
    the scores' size."""
    if not isinstance(mask, SpanMask):
        raise ValueError("unsupported_capability: span_attention needs a SpanMask")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or any(t.dtype != _BF16 for t in (q, k, v)):
        raise ValueError("unsupported_capability: span_attention expects 4-D bf16 q, k and v")
    B, H, S, DQ = q.shape
    Hkv, DV = k.shape[1], v.shape[-1]
    if k.shape != (B, Hkv, S, DQ) or v.shape != (B, Hkv, S, DV) or Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"unsupported_capability: q {tuple(q.shape)}, k {tuple(k.shape)} and v "
                         f"{tuple(v.shape)} do not fit")
    if (mask.batch, mask.length) != (B, S) or any(t.device != mask.plan.device for t in (q, k, v)):
        raise ValueError(f"unsupported_capability: a mask of {mask.batch} x {mask.length} tokens on "
                         f"{mask.plan.device} for {B} x {S} on {q.device}")
    scale, cap = float(scale), 0.0 if cap is None else float(cap)
    if cap < 0 or not math.isfinite(cap) or not math.isfinite(scale) or scale <= 0:
        raise ValueError("unsupported_capability: scale must be positive, cap None or positive")
    if slopes is not None:
        if slopes.dtype != _F32 or tuple(slopes.shape) != (H,) or slopes.device != q.device \
                or slopes.requires_grad:
            raise ValueError("unsupported_capability: slopes must be constant fp32 [heads] on the "
                             "attention's device")
        slopes = slopes.contiguous()
    _no_tangents(q, k, v, slopes)
    if not q.is_cuda:
        raise ValueError("unsupported_capability: span_attention runs on the GPU")
    args = (_operand(q), _operand(k), _operand(v), scale, mask, cap, slopes)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SpanAttention.apply(*args)
    return _span_forward(*args)[0]


# ----------------------------------------------------------------- rotation
_SCALING_KEYS = {
    "default": (), "linear": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
    "yarn": ("factor", "original_max_position_embeddings"),
}


def rotary_frequencies(dim: int, theta: float, scaling=None):
    """``(inverse frequencies [dim/2] as floats, amplitude)`` of a rotary
    embedding: ``scaling`` None or a ``rope_scaling`` table of type default,
    linear, llama3 or yarn.

    * linear: every frequency over ``factor``;
    * llama3: a pair that turns more than ``high_freq_factor`` times over the
      original context keeps its frequency, one below ``low_freq_factor`` turns is
      divided by ``factor``, between them they are mixed;
    * yarn: the same with the mix linear in the pair's index, between the pairs of
      ``beta_fast`` and ``beta_slow`` turns, and the amplitude 0.1 ln(factor) + 1
      (or ``attention_factor``, or the ratio of ``mscale`` and ``mscale_all_dim``)."""
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _SCALING_KEYS:
        raise ValueError(f"unsupported_capability: rotary scaling {kind!r}")
    missing = [n for n in _SCALING_KEYS[kind] if scaling.get(n) is None]
    if missing:
        raise ValueError(f"unsupported_capability: rotary scaling {kind!r} needs {missing}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError("unsupported_capability: theta must be positive")
    inv = [theta ** (-2.0 * i / dim) for i in range(dim // 2)]
    if kind == "default":
        return inv, 1.0
    factor = float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError("unsupported_capability: rotary scaling factor below 1")
    if kind == "linear":
        return [f / factor for f in inv], 1.0
    original = float(scaling["original_max_position_embeddings"])
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError("unsupported_capability: high_freq_factor must exceed low_freq_factor")
        keep = [min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low))) for f in inv]
        return [f * k + f / factor * (1.0 - k) for f, k in zip(inv, keep)], 1.0

    def index(turns):  # of the pair that turns so often over the original context
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = index(scaling.get("beta_fast") or 32), index(scaling.get("beta_slow") or 1)
    if scaling.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, dim - 1)
    if lo == hi:
        hi += 0.001
    slow = [min(1.0, max(0.0, (i - lo) / (hi - lo))) for i in range(dim // 2)]
    amplitude = scaling.get("attention_factor")
    if amplitude is None:
        def grown(s):
            return 1.0 if factor <= 1 else 0.1 * s * math.log(factor) + 1.0
        m, every = scaling.get("mscale"), scaling.get("mscale_all_dim")
        amplitude = grown(m) / grown(every) if m and every else grown(1.0)
    return [f / factor * s + f * (1.0 - s) for f, s in zip(inv, slow)], float(amplitude)


class Rotary:
    """A rotary embedding for :func:`rope_positions`: frequencies (fp64, on the
    device) and amplitude, made once for a model.  ``rotary_dim``: the first
    columns of each head that turn (default: all, even); ``interleaved``: pairs
    (2i, 2i+1) instead of (i, i + rotary_dim/2); ``scaling``: see
    :func:`rotary_frequencies`."""

    def __init__(self, head_dim: int, theta: float, *, rotary_dim=None, interleaved=False,
                 scaling=None, device):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 8 or head_dim % 8 or rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"unsupported_capability: rotary part {rotary_dim} of heads of {head_dim}")
        inv, self.amplitude = rotary_frequencies(rotary_dim, float(theta), scaling)
        self.head_dim, self.rotary_dim = int(head_dim), int(rotary_dim)
        self.interleaved = bool(interleaved)
        self.inv_freq = torch.tensor(inv, dtype=torch.float64, device=device)

    @property
    def device(self):
        return self.inv_freq.device


def _turn(positions, rotary, heads, kv_heads, wq, wk):
    """The arguments that both directions of the rotation share."""
    return (positions.data_ptr(), int(positions.dtype == torch.int64), rotary.inv_freq.data_ptr(),
            rotary.amplitude, *positions.shape, heads, kv_heads, rotary.head_dim, rotary.rotary_dim,
            int(rotary.interleaved), _lib.ptr(wq), _lib.ptr(wk))


def _rope_forward(y, positions, rotary, heads, kv_heads, wq, wk, eps):
    """(q, k, v, reciprocal norms or None)"""
    B, S = positions.shape
    D, dev = rotary.head_dim, y.device
    q = torch.empty((B, heads, S, D), dtype=_BF16, device=dev)
    k = torch.empty((B, kv_heads, S, D), dtype=_BF16, device=dev)
    v = torch.empty_like(k)
    rstd = None if wq is None else torch.empty((B * S, heads + kv_heads), dtype=_F32, device=dev)
    with _lib.on_device(dev):
        _lib.call("st_rope_pos_fwd", y.data_ptr(), y.stride(0),
                  *_turn(positions, rotary, heads, kv_heads, wq, wk), eps, q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), _lib.ptr(rstd), _lib.stream_handle(dev))
    return q, k, v, rstd


class _RopePositions(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, positions, rotary, heads, kv_heads, wq, wk, eps):
        q, k, v, rstd = _rope_forward(y, positions, rotary, heads, kv_heads, wq, wk, eps)
        if wq is None:  # the rotation's gradient does not read its input
            ctx.save_for_backward(positions)
        else:
            ctx.save_for_backward(positions, y, wq, wk, rstd)
        ctx.meta = (rotary, heads, kv_heads, tuple(y.shape))
        ctx.set_materialize_grads(False)
        return q, k, v

    @staticmethod
    def backward(ctx, dq, dk, dv):
        _once()
        # addresses come from the saved tensors as they are now: a hook may have
        # moved them
        positions, y, wq, wk, rstd = (*ctx.saved_tensors, None, None, None, None)[:5]
        rotary, heads, kv_heads, shape = ctx.meta
        (B, S), D, dev = positions.shape, rotary.head_dim, positions.device
        dy = torch.empty(shape, dtype=_BF16, device=dev)
        dq, dk, dv = (torch.zeros((B, n, S, D), dtype=_BF16, device=dev) if g is None else _operand(g)
                      for g, n in ((dq, heads), (dk, kv_heads), (dv, kv_heads)))
        with _lib.on_device(dev):
            _lib.call("st_rope_pos_bwd", dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(y),
                      shape[1] if y is None else y.stride(0),
                      *_turn(positions, rotary, heads, kv_heads, wq, wk), _lib.ptr(rstd),
                      dy.data_ptr(), shape[1], _lib.stream_handle(dev))
        return dy, None, None, None, None, None, None, None


def rope_positions(y, positions, rotary: Rotary, heads: int, kv_heads: int, *, norms=None, eps=1e-6):
    """q [B,heads,S,D], k and v [B,kv_heads,S,D] from a fused q|k|v output ``y``
    (bf16 [B*S, (heads + 2 kv_heads) * D], rows may be strided): query and key
    heads turned by ``positions`` (int32/int64 [B,S], e.g. ``SpanMask.positions``),
    with ``norms`` = (q weight, k weight) (bf16 [D], frozen) first RMS-normalised
    head by head; values copied.  fp32 arithmetic, one rounding; angles in fp64."""
    if not isinstance(rotary, Rotary):
        raise ValueError("unsupported_capability: rope_positions needs a Rotary")
    if positions.dim() != 2 or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("unsupported_capability: positions must be int32/int64 [batch, length]")
    B, S = positions.shape
    D = rotary.head_dim
    if heads < 1 or kv_heads < 1 or y.dim() != 2 or y.dtype != _BF16 \
            or tuple(y.shape) != (B * S, (heads + 2 * kv_heads) * D):
        raise ValueError(f"unsupported_capability: rope_positions expects bf16 "
                         f"[{B * S}, {(heads + 2 * kv_heads) * D}], got {y.dtype} {tuple(y.shape)}")
    if positions.device != y.device or rotary.device != y.device:
        raise ValueError("unsupported_capability: y, positions and the Rotary on one device")
    wq = wk = None
    if norms is not None:
        if any(w.requires_grad for w in norms):
            raise ValueError("unsupported_capability: norm weights are frozen")
        wq, wk = (_operand(w) for w in norms)
        if any(w.dtype != _BF16 or tuple(w.shape) != (D,) or w.device != y.device for w in (wq, wk)):
            raise ValueError("unsupported_capability: norm weights must be bf16 [head_dim]")
    _no_tangents(y, wq, wk)
    if not y.is_cuda:
        raise ValueError("unsupported_capability: rope_positions runs on the GPU")
    if y.stride(1) != 1 or y.stride(0) % 8 or y.stride(0) < y.shape[1] or y.data_ptr() % 16:
        y = y.clone(memory_format=torch.contiguous_format)
    args = (y, positions.contiguous(), rotary, int(heads), int(kv_heads), wq, wk, float(eps))
    if torch.is_grad_enabled() and y.requires_grad:
        return _RopePositions.apply(*args)
    return _rope_forward(*args)[:3]


# ----------------------------------------------------------------- a model's packed rows
@dataclass(frozen=True, eq=False)
class Positions:
    """Position embeddings of packed rows for a decoder block: per-token
    positions (int32 [batch, length]) and the rotary embedding they turn by, in
    the place of (cos, sin) tables."""
    positions: torch.Tensor
    rotary: Rotary


def positions_and_masks(documents: torch.Tensor, rotary: Rotary, *, bidirectional=None, window=None):
    """``(Positions, SpanMask)`` of packed rows, in the place of
    ``dense.positions_and_masks``; ``documents`` and ``bidirectional`` as for
    :func:`document_mask`, from the host or the device."""
    move = lambda t: None if t is None else t.to(rotary.device)  # noqa: E731
    mask = document_mask(move(documents), bidirectional=move(bidirectional), window=window)
    return Positions(mask.positions, rotary), mask


def document_labels(labels: torch.Tensor, documents: torch.Tensor) -> torch.Tensor:
    """``labels`` with -100 where no token of the same document comes before: a
    document's first token is not predicted from another document's last, and
    padding is not predicted at all."""
    if labels.shape != documents.shape or labels.dim() != 2:
        raise ValueError("unsupported_capability: labels and documents must be [batch, length]")
    documents = documents.to(labels.device)
    follows = torch.zeros(labels.shape, dtype=torch.bool, device=labels.device)
    follows[:, 1:] = (documents[:, 1:] == documents[:, :-1]) & (documents[:, 1:] >= 0)
    return torch.where(follows, labels, -100)


__all__ = ["SpanMask", "span_mask", "document_runs", "document_mask", "span_attention",
           "rotary_frequencies", "Rotary", "rope_positions", "Positions", "positions_and_masks",
           "document_labels"]
