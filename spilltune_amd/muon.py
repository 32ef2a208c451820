"""Orthogonalised updates of the adapters' factors (no counterpart in the reference,
whose optimizer is AdamW, finetune/optimizer.py:227-342).

* :func:`orthogonalize` -- every matrix of a list by a few Newton-Schulz steps, all
  of them in one call.
* :class:`Muon` -- the optimizer on it: momentum, orthogonalised, added to the
  factors; takes the place of ``engine.AdamW`` in ``engine.train``.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .ops import _no_tangents, _scratch

_DTYPES = {torch.bfloat16: _lib.ST_DTYPE_BF16, torch.float32: _lib.ST_DTYPE_F32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(matrices, *, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Each matrix of ``matrices`` (a tensor or a sequence of them, [..., rows,
    columns], bf16 or fp32, all of one type on one device) with its singular values
    pushed towards 1: ``X = U / (|U|_F + eps)`` and ``steps`` times ``X <- aX + (b XX'
    + c (XX')^2) X`` on the shorter side, which may have up to 1024 entries; the
    longer one is free.  Returns new tensors of the same shapes and type.

    The steps run in 64 bits, so the result is the formula's to the rounding of its
    type, also along directions whose singular value is far below the largest.
    ``|a|^(2 steps)`` may reach 1e13 (12 steps with the default coefficients).  A zero
    matrix stays zero; one with a value that is not finite turns into NaN."""
    single = isinstance(matrices, torch.Tensor)
    given = [matrices] if single else list(matrices)
    if not given:
        return []
    out = _run(_prepare(given, steps, coefficients, eps), given)
    return out[0] if single else out


def _rule(steps, coefficients, eps=1e-7):
    """``(steps, a, b, c, eps)``, checked."""
    a, b, c = (float(v) for v in coefficients)
    eps = float(eps)
    if isinstance(steps, bool) or not isinstance(steps, int):
        raise ValueError("unsupported_capability: steps must be an integer")
    if not (math.isfinite(a) and math.isfinite(b) and math.isfinite(c) and 0.0 <= eps < math.inf):
        raise ValueError("unsupported_capability: coefficients must be finite, eps not negative")
    if not 1 <= steps <= 64 or 2.0 * steps * math.log10(max(abs(a), 1.0)) > 13.0:
        raise ValueError("unsupported_capability: steps must be 1 to 64 with |a|^(2 steps) at most "
                         f"1e13, got {steps}")
    return steps, a, b, c, eps


def _prepare(given, steps, coefficients, eps):
    """Everything of a call that depends on sizes alone, checked."""
    if not all(isinstance(x, torch.Tensor) for x in given):
        raise ValueError("unsupported_capability: orthogonalize takes tensors")
    dtype, device = given[0].dtype, given[0].device
    if dtype not in _DTYPES or any(x.dtype != dtype or x.device != device or x.dim() < 2
                                   for x in given):
        raise ValueError("unsupported_capability: orthogonalize takes matrices of one type, bf16 or "
                         "fp32, on one device")
    if torch.is_grad_enabled() and any(x.requires_grad for x in given):
        raise ValueError("unsupported_capability: orthogonalize has no derivative")
    _no_tangents(*given)
    rule = _rule(steps, coefficients, eps)
    numbers = []  # st_matrix_batch: five 64-bit words each, addresses first
    for x in given:
        rows, cols = x.shape[-2:]
        numbers += (0, 0, x.numel() // (rows * cols) if rows and cols else 0, rows, cols)
    table = (ctypes.c_int64 * len(numbers))(*numbers)
    nbytes = _lib.query("st_orthogonalize_workspace_bytes", len(given), table)
    if nbytes < 0:
        _lib.check(_lib.ST_EUNSUPPORTED, "st_orthogonalize")
    if device.type != "cuda":
        raise ValueError("unsupported_capability: orthogonalize runs on the GPU")
    return table, nbytes, rule, dtype, device


def _run(plan, given):
    """The call on tensors of the sizes, type and device that ``plan`` was made for."""
    table, nbytes, rule, dtype, device = plan
    given = [x.contiguous() for x in given]
    out = [torch.empty_like(x) for x in given]
    at = 0
    for x, y in zip(given, out):
        table[at:at + 2] = x.data_ptr(), y.data_ptr()
        at += 5
    with _lib.on_device(device):
        ws = _scratch(device, nbytes)
        _lib.call("st_orthogonalize", len(given), table, _DTYPES[dtype], *rule, _lib.ptr(ws), nbytes,
                  _lib.stream_handle(device))
    return out


def _factors(proj):
    """``(parameter, gradient, momentum)`` of an adapter's two factors; of per-expert
    ones a view of the matrices, [matrices, rows, columns], whose fused gate and up are
    matrices of their own.  (For use without gradients.)"""
    n = getattr(proj, "segments", 1)
    for t in ((proj.A, proj.grad_A, proj.m_A), (proj.B, proj.grad_B, proj.m_B)):
        if t[0].dim() == 2:
            yield t
        else:
            shape = (t[0].shape[0] * n, t[0].shape[1] // n, t[0].shape[2])
            yield tuple(x.detach().view(shape) for x in t)


class Muon:
    """Momentum, orthogonalised, over LoRA projections (per-expert ones too)::

        m <- momentum m + (1 - momentum) g
        u  = momentum m + (1 - momentum) g   (nesterov; else m)
        p <- (1 - lr weight_decay) p - lr scale orthogonalize(u)

    ``scale`` is ``match_rms * sqrt(max(rows, columns))``, with which the entries of an
    update have a mean square of about ``match_rms`` squared whatever its shape; with
    ``match_rms=None`` it is ``sqrt(max(1, rows / columns))``.  ``m_A`` and ``m_B`` of a
    projection hold its momentum, ``v_A`` and ``v_B`` stay as they are.  A
    :class:`~spilltune_amd.embedding.TokenEmbedding` among the projections is updated
    by ``table`` (an ``engine.AdamW``)."""

    def __init__(self, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=COEFFICIENTS, match_rms=0.2, table=None):
        if not (math.isfinite(lr) and 0.0 <= momentum < 1.0 and weight_decay >= 0.0):
            raise ValueError("unsupported_capability: lr must be finite, momentum in [0, 1), "
                             "weight_decay not negative")
        self.lr, self.momentum, self.nesterov = lr, momentum, nesterov
        self.weight_decay, self.steps, self.coefficients = weight_decay, steps, tuple(coefficients)
        _rule(self.steps, self.coefficients)
        self.match_rms, self.table = match_rms, table
        self.step_count = 0

    def zero_grad(self, projections):
        for p in projections.values():
            p.zero_grad()

    def _scale(self, shape):
        rows, cols = shape[-2:]
        if self.match_rms is None:
            return math.sqrt(max(1.0, rows / cols))
        return self.match_rms * math.sqrt(max(rows, cols))

    def step(self, projections):
        tables = {k: p for k, p in projections.items() if not hasattr(p, "A")}
        if tables and self.table is None:
            raise ValueError(f"unsupported_capability: no optimizer for {sorted(tables)}")
        with torch.no_grad():
            factors = [f for k, p in projections.items() if k not in tables for f in _factors(p)]
            if factors:
                params, grads, moments = (list(t) for t in zip(*factors))
                # what the update refuses, it refuses before a momentum has moved
                plan = _prepare(moments, self.steps, self.coefficients, 1e-7)
                torch._foreach_lerp_(moments, grads, 1.0 - self.momentum)
                updates = torch._foreach_lerp(grads, moments, self.momentum) if self.nesterov \
                    else moments
                updates = _run(plan, updates)
                torch._foreach_mul_(updates, [-self.lr * self._scale(u.shape) for u in updates])
                if self.weight_decay:
                    torch._foreach_mul_(params, 1.0 - self.lr * self.weight_decay)
                torch._foreach_add_(params, updates)
        if tables:
            self.table.step(tables)
        self.step_count += 1


__all__ = ["orthogonalize", "Muon", "COEFFICIENTS"]
