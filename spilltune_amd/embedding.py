"""A token embedding that lives on the device and is trained (the reference looks
tokens up on the host and freezes the table; no counterpart there).

:class:`TokenEmbedding` takes the place of the host table in
``engine.DenseModel(embedding=...)``: the engine looks rows up through it, adds each
microbatch's gradient to its buffer and hands it to the optimizer with the adapters.
"""
from __future__ import annotations

import torch

from . import ops

_F32 = torch.float32


class TokenEmbedding:
    """``weight`` (fp32 [V, H], a copy on ``device``), its gradient buffer ``grad`` and
    the AdamW moments ``m`` and ``v``.  ``scale`` multiplies the rows that are looked
    up, as some models scale theirs by the root of the hidden size; tokens equal to
    ``padding_idx`` are looked up and not trained, nor does a weight decay reach their
    row.  A head that was tied to the table
    is a tensor of its own and stays frozen."""

    name = "embedding"

    def __init__(self, weight: torch.Tensor, *, device, scale=1.0, padding_idx=None):
        if weight.dim() != 2 or not weight.is_floating_point():
            raise ValueError("unsupported_capability: an embedding is a table [V, H]")
        self.weight = weight.detach().to(device, _F32, copy=True,
                                         memory_format=torch.contiguous_format)
        self.scale, self.padding_idx = scale, padding_idx
        ops._embedding_args(self.weight, torch.empty(0, dtype=torch.int64), scale, padding_idx)
        self.grad, self.m, self.v = (torch.zeros_like(self.weight) for _ in range(3))

    def __call__(self, ids: torch.Tensor) -> torch.Tensor:
        """bf16 rows [..., H] of ``ids``; no autograd node (see :meth:`add_grad`)."""
        return ops.embedding(self.weight, ids, scale=self.scale)

    def add_grad(self, ids: torch.Tensor, dout: torch.Tensor, accumulate: bool = True) -> None:
        """Adds the gradient that ``dout`` (bf16, of ``self(ids)``'s shape) means for the
        table to ``grad``, touching the rows that occur, or replaces ``grad``."""
        ids, scale = ops._embedding_args(self.weight, ids, self.scale, self.padding_idx)
        if dout.dtype != torch.bfloat16 or dout.shape != (*ids.shape, self.weight.shape[1]) \
                or dout.device != self.weight.device:
            raise ValueError("unsupported_capability: the gradient must be bf16 and shaped like the "
                             "rows that were looked up")
        ops._embedding_grad(self.grad, ids, ops._operand(dout.detach()), scale, self.padding_idx,
                            accumulate)

    def zero_grad(self) -> None:
        self.grad.zero_()


__all__ = ["TokenEmbedding"]
