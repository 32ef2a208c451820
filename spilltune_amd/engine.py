"""Causal-LM training step over 4-bit streamed blocks (mirror of
training/engine.py:21-195 and finetune/optimizer.py:227-342 in
/root/reference/src/ram_vram_finetune, without the config/dataset/checkpoint
I/O around it).

* :func:`forward` -- the per-layer loop through the streaming recompute driver
  (engine.py:36-45).
* :func:`microbatch` -- embedding, layers, full-sequence terminal norm,
  token-chunked head + summed cross-entropy / normaliser, norm VJP, one
  decoder backward (engine.py:48-79).  The terminal runs on the HIP path:
  RMSNorm kernels for the norm and its VJP, and ``ops.chunked_causal_loss``
  (native_terminal.py:11-47) -- per token chunk a bf16 head GEMM, one
  in-place cross-entropy/gradient pass over the bf16 logits and a bf16 GEMM
  back to the hidden size.
* :class:`AdamW` -- the fp32 update in torch.optim.AdamW's non-foreach order
  (optimizer.py:324-342), on the device.
* :func:`train` -- the optimizer-step loop with gradient accumulation over
  cyclic rows (engine.py:162-182), microbatch-major as the reference or
  layer-major (:func:`window_layer_major`: one layer load per phase per
  accumulation window instead of one per microbatch, same results).
* Packed rows (``documents``: several documents in a row, see
  :mod:`spilltune_amd.packed`) in all of the above, an ``objective`` on token log
  probabilities in the place of the cross-entropy, and :func:`score`, the log
  probabilities of given rows; these have no counterpart in the reference.
* A :class:`~spilltune_amd.embedding.TokenEmbedding` in the place of the host table:
  looked up on the device, scaled, trained with the adapters (no counterpart either).
* :class:`DenseModel` -- the adapter surface the engine uses
  (adapters/protocol.py:23-34) for a Llama-family model whose decoder
  matrices are stored 4-bit.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import ops, packed, slots
from .dense import positions_and_masks
from .embedding import TokenEmbedding
from .recompute import (_borrow_weights, _call_functional_block, block_adapter_backward,
                        streaming_block)


def flatten(model) -> dict:
    """``{"{layer}:{target}": projection}`` (engine.py:21-33)."""
    result, seen = {}, set()
    for block in model.blocks:
        for name, proj in block.adapters.items():
            key = f"{block.index}:{name}"
            if key in result or id(proj) in seen:
                raise ValueError("unsupported_capability: duplicate/shared trainable parameter")
            result[key] = proj
            seen.add(id(proj))
    if not result:
        raise ValueError("training plan has no trainable projections")
    return result


def forward(model, session, hidden, positions, masks, *, accumulate=False):
    for block in model.blocks:
        hidden = streaming_block(hidden, positions, masks[block.kind], block.functional, block.kwargs,
                                 session.reloader(block), block.adapters, block.index,
                                 accumulate_adapter_grads=accumulate)
    return hidden


def _trainables(model) -> dict:
    """What an optimizer steps: the projections, and ``"embedding"`` where the model's
    table is trained."""
    result = flatten(model)
    if isinstance(model.embedding, TokenEmbedding):
        result["embedding"] = model.embedding
    return result


def _embed(model, input_ids):
    """Rows of the model's table: a trained one's on the device, or the host's."""
    if isinstance(model.embedding, TokenEmbedding):
        return model.embedding(input_ids)
    return F.embedding(input_ids.cpu(), model.embedding).to(model.device)


def _embedding_grad(model, input_ids, gradient, accumulate):
    """Takes the embedded rows' gradient into a trained table's."""
    if isinstance(model.embedding, TokenEmbedding):
        model.embedding.add_grad(input_ids, gradient, accumulate)


def _row_inputs(model, input_ids, documents):
    """Positions and masks of a batch: all-valid rows, or packed documents."""
    if documents is None:
        return model.positions_and_masks(torch.ones_like(input_ids, dtype=torch.bool))
    if documents.shape != input_ids.shape:
        raise ValueError("unsupported_capability: documents must be shaped like the token rows")
    return model.packed_positions_and_masks(documents)


class LabelLogProbs(ops.TokenLogProbs):
    """What an objective is given: the :class:`~spilltune_amd.ops.TokenLogProbs`
    of a microbatch's labels, entry ``t`` of a row that of label ``t + 1``, with

    * ``labels`` (int64 [batch, length - 1], on the device): those labels, -100
      where none is to be learnt (dropped by the caller, a document's first token,
      padding).  Log probabilities are 0 there, entropies are real: a term on
      them is to be masked with ``labels != -100``;
    * ``normalization``: the labels of the whole accumulation window, so that the
      microbatches' terms, divided by it, add up to an average;
    * ``item``: which row this is -- its index in ``train``'s rows, or what the
      caller of ``microbatch`` names it."""
    labels: torch.Tensor
    normalization: int
    item: object


def _terminal(model, normalized, labels, *, normalization, token_chunk, objective, item=None):
    """The summed cross-entropy over ``normalization``, or the scalar that
    ``objective`` makes of the :class:`LabelLogProbs`."""
    if objective is not None:
        labels = labels[:, 1:].to(torch.int64)
        given = LabelLogProbs(*ops.token_logprobs(normalized[:, :-1], model.head, labels))
        given.labels = labels.to(normalized.device)
        given.normalization, given.item = normalization, item
        return objective(given)
    chunks = ops.supervised_chunk_intervals(labels, token_chunk)
    return ops.chunked_causal_loss(normalized, model.head, labels,
                                   normalization=normalization, token_chunk=token_chunk,
                                   supervised_chunks=chunks)


def microbatch(model, session, input_ids, labels, *, normalization, token_chunk, accumulate=False,
               documents=None, objective=None, item=None):
    """Exact shifted summed CE / window token count; one decoder backward.
    ``documents``: packed rows (labels across a document's start are dropped);
    ``objective``: a function of :class:`LabelLogProbs` (which tells it ``item``)
    to a scalar, in the place of the cross-entropy."""
    positions, masks = _row_inputs(model, input_ids, documents)
    if documents is not None:
        labels = packed.document_labels(labels, documents)
    embedded = _embed(model, input_ids).detach().requires_grad_(True)
    hidden = forward(model, session, embedded, positions, masks, accumulate=accumulate)
    terminal_input = hidden.detach().requires_grad_(True)
    normalized = model.terminal_norm(terminal_input)
    loss = _terminal(model, normalized, labels, normalization=normalization,
                     token_chunk=token_chunk, objective=objective, item=item)
    (gradient,) = torch.autograd.grad(loss, terminal_input)
    if not torch.isfinite(loss) or not torch.isfinite(gradient).all():
        raise FloatingPointError("non-finite causal loss/gradient")
    hidden.backward(gradient)
    _embedding_grad(model, input_ids, embedded.grad, accumulate)
    return float(loss.detach()), embedded.grad.detach().clone()


def score(model, session, input_ids, *, documents=None, top=0, temperature=1.0):
    """Log probabilities of given rows under the model, no gradients: a
    :class:`~spilltune_amd.ops.TokenLogProbs` of [batch, length - 1], whose entry
    ``t`` is token ``t + 1`` after the tokens up to ``t`` (0 where ``documents``
    starts another document or padding there), with the entropy and the ``top``
    alternatives of that place."""
    with torch.no_grad():
        positions, masks = _row_inputs(model, input_ids, documents)
        tokens = input_ids if documents is None else packed.document_labels(input_ids, documents)
        embedded = _embed(model, input_ids)
        normalized = model.terminal_norm(forward(model, session, embedded, positions, masks))
        return ops.token_logprobs(normalized[:, :-1], model.head, tokens[:, 1:].to(torch.int64),
                                  top=top, temperature=temperature)


def window_layer_major(model, session, items, *, normalization, token_chunk, objective=None,
                       names=None):
    """One gradient-accumulation window processed layer by layer, so each
    layer's 4-bit image crosses PCIe once per phase instead of once per
    microbatch (the reference streams every layer for every microbatch,
    engine.py:168-178):

    * forward: every microbatch through layer i (no grad) before layer i+1,
      keeping each microbatch's layer inputs (one bf16 [B,S,H] per layer and
      microbatch, as the recompute driver saves);
    * terminal per microbatch, in order (as ``microbatch``);
    * backward: per layer in reverse, the recompute + VJP of every microbatch
      in order, adding adapter gradients (the first microbatch replaces).

    For each layer the fp32 adapter-gradient sums take the microbatches in the
    same order as the microbatch-major loop, so the gradients and losses are
    the same bits.  ``objective`` as for :func:`microbatch`; ``names`` its ``item`` of
    each microbatch (default 0, 1, ...).  Returns the per-microbatch losses."""
    names = range(len(items)) if names is None else names
    if len(names) != len(items):
        raise ValueError(f"unsupported_capability: {len(names)} names for {len(items)} microbatches")
    mbs = []
    for ids, labels, *documents in items:
        positions, masks = _row_inputs(model, ids, *documents or [None])
        if documents and documents[0] is not None:
            labels = packed.document_labels(labels, documents[0])
        mbs.append({"ids": ids, "pos": positions, "masks": masks, "h": [_embed(model, ids)],
                    "labels": labels})
    for block in model.blocks:
        with _borrow_weights(session.reloader(block), "forward") as weights, torch.no_grad():
            for mb in mbs:
                mb["h"].append(_call_functional_block(block.functional, mb["h"][-1], mb["pos"],
                                                      mb["masks"][block.kind], weights,
                                                      block.kwargs))
    losses = []
    for mb, name in zip(mbs, names):
        terminal_input = mb["h"].pop().detach().requires_grad_(True)
        normalized = model.terminal_norm(terminal_input)
        loss = _terminal(model, normalized, mb["labels"], normalization=normalization,
                         token_chunk=token_chunk, objective=objective, item=name)
        (mb["g"],) = torch.autograd.grad(loss, terminal_input)
        if not torch.isfinite(loss) or not torch.isfinite(mb["g"]).all():
            raise FloatingPointError("non-finite causal loss/gradient")
        losses.append(float(loss.detach()))
    for block in reversed(model.blocks):
        ordered = sorted(block.adapters.values(), key=lambda p: p.name)
        with _borrow_weights(session.reloader(block), "backward") as weights:
            for k, mb in enumerate(mbs):
                hidden = mb["h"].pop().detach().requires_grad_(True)
                with torch.enable_grad():
                    out = _call_functional_block(block.functional, hidden, mb["pos"],
                                                 mb["masks"][block.kind], weights, block.kwargs)
                # the first microbatch replaces (zero + add), later ones accumulate
                mb["g"] = block_adapter_backward(out, hidden, ordered, mb["g"], k > 0, block.index)
    for k, mb in enumerate(mbs):
        _embedding_grad(model, mb["ids"], mb["g"], k > 0)
    return losses


def _tensors(projection):
    """``(parameter, gradient, m, v)`` of what a projection, or a trained embedding,
    holds."""
    p = projection
    if hasattr(p, "A"):
        return ((p.A, p.grad_A, p.m_A, p.v_A), (p.B, p.grad_B, p.m_B, p.v_B))
    return ((p.weight, p.grad, p.m, p.v),)


class AdamW:
    """Bias-corrected fp32 AdamW over LoRA projections (optimizer.py:227-342) and a
    trained embedding."""

    def __init__(self, lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0):
        self.lr, self.beta1, self.beta2, self.eps = lr, beta1, beta2, eps
        self.weight_decay = weight_decay
        self.step_count = 0

    def zero_grad(self, projections):
        for p in projections.values():
            for param, grad, _, _ in _tensors(p):
                grad.zero_()
                param.grad = None

    def step(self, projections):
        n = self.step_count + 1
        step_size = self.lr / (1.0 - self.beta1 ** n)
        bc2_sqrt = math.sqrt(1.0 - self.beta2 ** n)
        with torch.no_grad():
            for p in projections.values():
                for param, grad, m, v in _tensors(p):
                    if self.weight_decay != 0.0:
                        row = getattr(p, "padding_idx", None)  # of a table: not trained
                        kept = None if row is None else param[row].clone()
                        param.mul_(1.0 - self.lr * self.weight_decay)
                        if kept is not None:
                            param[row] = kept
                    m.lerp_(grad, 1.0 - self.beta1)
                    v.mul_(self.beta2).addcmul_(grad, grad, value=1.0 - self.beta2)
                    denom = (v.sqrt() / bc2_sqrt).add_(self.eps)
                    param.addcdiv_(m, denom, value=-step_size)
        self.step_count = n


def train(model, session, rows, *, steps, accumulation=1, lr=1e-4, weight_decay=0.0,
          token_chunk=64, layer_major=False, objective=None, optimizer=None):
    """Optimizer-step loop with cyclic rows (engine.py:162-182); returns losses.
    Rows are ``(ids, labels)`` or, packed, ``(ids, labels, documents)``.
    ``layer_major`` runs each accumulation window with ``window_layer_major``
    (same results, one layer load per phase per window).  ``objective``: in the
    place of the cross-entropy, see :func:`microbatch`.  ``optimizer`` (an
    :class:`AdamW` or :class:`~spilltune_amd.muon.Muon`, with its own rates) in the
    place of the AdamW of ``lr`` and ``weight_decay``."""
    projections = _trainables(model)
    if optimizer is None:
        optimizer = AdamW(lr=lr, weight_decay=weight_decay)
    cursor, losses = 0, []
    for _ in range(steps):
        names = [(cursor + i) % len(rows) for i in range(accumulation)]
        items = [rows[i] for i in names]
        normalization = sum(
            int(((labels if not docs or docs[0] is None else packed.document_labels(labels, docs[0]))
                 [:, 1:] != -100).sum()) for _, labels, *docs in items)
        optimizer.zero_grad(projections)
        loss = 0.0
        with session.run():
            if layer_major:
                for micro in window_layer_major(model, session, items,
                                                normalization=normalization,
                                                token_chunk=token_chunk, objective=objective,
                                                names=names):
                    loss += micro
            else:
                for i, (ids, labels, *docs) in enumerate(items):
                    micro, _ = microbatch(model, session, ids, labels,
                                          normalization=normalization, token_chunk=token_chunk,
                                          accumulate=i > 0, documents=docs[0] if docs else None,
                                          objective=objective, item=names[i])
                    loss += micro
            optimizer.step(projections)
        cursor += accumulation
        losses.append(loss)
    return losses


class DenseModel:
    """Llama-family model with 4-bit decoder matrices in slot images: the
    runtime surface of adapters/dense.py:178-263 the engine needs."""

    def __init__(self, *, embedding, norm, head, layers=None, heads, kv_heads, head_dim, eps,
                 theta, rank, alpha, targets, device, codec="nf4-g128", generator=None,
                 blocks=None, qk_norm=False, rotary=None, post_norms=False, residual_scale=1.0):
        """``embedding``: a host table, or a :class:`~spilltune_amd.embedding.TokenEmbedding`
        that is trained.  ``layers``: per-layer weight dicts, encoded here; or ``blocks``:
        prebuilt BlockPlans (e.g. ``slots.make_archive_block``).  ``rotary``: the
        model's :class:`~spilltune_amd.packed.Rotary`, of plain and of packed rows
        (default: whole heads, ``theta``, no scaling; plain rows then by bf16
        tables).  ``post_norms`` and ``residual_scale`` of ``layers``: see
        :func:`~spilltune_amd.dense.dense_block`."""
        self.device = torch.device(device)
        if isinstance(embedding, TokenEmbedding):
            if embedding.weight.device.type != self.device.type or (
                    self.device.index is not None
                    and embedding.weight.device.index != self.device.index):
                raise ValueError("unsupported_capability: a trained embedding lives on the model's "
                                 "device")
            self.embedding = embedding
        else:
            self.embedding = embedding.to(torch.bfloat16).contiguous()      # stays on the host
        self.norm = norm.to(torch.bfloat16).to(self.device)
        self.head = head.to(torch.bfloat16).to(self.device)
        self.eps, self.theta, self.head_dim = eps, theta, head_dim
        self.rotary = rotary
        self._plain = None  # of packed rows without one, made on their first use
        if (layers is None) == (blocks is None):
            raise ValueError("DenseModel needs exactly one of layers / blocks")
        self.blocks = list(blocks) if blocks is not None else [
            slots.make_dense_block(i, w, codec=codec, heads=heads, kv_heads=kv_heads,
                                   head_dim=head_dim, eps=eps, rank=rank, alpha=alpha,
                                   targets=targets, device=self.device, generator=generator,
                                   qk_norm=qk_norm, post_norms=post_norms,
                                   residual_scale=residual_scale)
            for i, w in enumerate(layers)]

    def positions_and_masks(self, valid):
        rot, mask = positions_and_masks(valid, head_dim=self.head_dim, theta=self.theta,
                                        device=self.device, rotary=self.rotary)
        return rot, {"full_attention": mask}

    def packed_positions_and_masks(self, documents, **kw):
        """Positions and masks of packed rows (packed.positions_and_masks)."""
        rotary = self.rotary
        if rotary is None:
            if self._plain is None:
                self._plain = packed.Rotary(self.head_dim, self.theta, device=self.device)
            rotary = self._plain
        positions, mask = packed.positions_and_masks(documents, rotary, **kw)
        return positions, {"full_attention": mask}

    def terminal_norm(self, hidden):
        B, S, H = hidden.shape
        return ops.rms_norm(hidden.reshape(B * S, H), self.norm, self.eps).view(B, S, H)

    def close(self):
        self.blocks.clear()
