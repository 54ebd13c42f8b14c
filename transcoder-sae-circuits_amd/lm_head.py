"""The end of a language model as differentiable operators: layer norm, and the cross entropy behind the unembedding without
the ``[rows, d_vocab]`` logits (``tsc_layer_norm*``, ``tsc_unembed_*`` through ``tsc_hip``).

    head = tsc_hip.UnembedHead(W_U, b_U)
    loss = unembed_loss(layer_norm(resid, w, b), targets, head)      # mean over the rows whose target counts
    loss.backward()                                                  # resid, w, b, W_U and b_U

Gradients are first-order (a second derivative raises) and the same call gives the same bits.  Both may be captured into a
HIP graph, the backward pass too.  A captured pass whose weights learn lays them out again on every replay (replays do not
tell torch that they changed the weights: ``head.refresh()`` before an eager call that follows them); a capture while an eager
pass over the same leaves is alive is refused (``_mark_leaves``), and so is one whose head is of a view (``W_E.t()``) that
learns.
"""
from __future__ import annotations

import weakref
from typing import Optional

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import get_gradient_edge

import tsc_hip

_MARK = "tsc_eager_stream"
_FINAL = "ln_final.hook_normalized"


def _mark_leaves(*tensors) -> list:
    """A leaf has one gradient accumulator for as long as any pass over it lives, and the accumulator belongs to the stream
    of the first.  A backward pass that is captured on another stream would wait for that stream inside the capture, which
    ends the process: so an eager pass leaves its stream at the accumulator (gone with the pass), and a capture that finds
    another stream's there refuses.  The caller holds what is returned until the pass itself holds the accumulators."""
    held = []
    for t in tensors:
        if t is None or not t.requires_grad or not t.is_leaf or not t.is_cuda:
            continue
        stream = torch.cuda.current_stream(t.device).cuda_stream
        held.append(get_gradient_edge(t).node)
        note = held[-1].metadata
        if not torch.cuda.is_current_stream_capturing():
            note.setdefault(_MARK, stream)
        elif note.get(_MARK, stream) != stream:
            raise tsc_hip.TscError(
                "an eager pass over the same leaf is alive (its loss or an output is still referenced) while this one is "
                "captured into a graph on another stream: delete its outputs first, or run it on the capture's stream")
    return held


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """A gradient may arrive broadcast or transposed: a copy where its rows are no ``tsc_rows_t``."""
    try:
        tsc_hip._rows(t, "t")
        return t
    except tsc_hip.TscError:
        return t.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, scale = tsc_hip.layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, scale)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, scale = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, db = tsc_hip.layer_norm_backward(_as_rows(dy), x, mean, scale, weight, bias if need_b else None, want_weight=need_w)
        return dx if need_x else None, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis (:func:`tsc_hip.layer_norm`: types, strides and
    refusals), differentiable in ``x``, ``weight`` and ``bias``."""
    held = _mark_leaves(x, weight, bias) if torch.is_grad_enabled() else None  # noqa: F841
    return _LayerNorm.apply(x, weight, bias, eps)


class _UnembedLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W_U, b_U, targets, head, ignore_index, laid_out):
        loss, lse = head._loss(x, targets, ignore_index, laid_out)
        # (the weights are saved for their version: a change in place between the two passes is an error, not a wrong gradient;
        # so the backward pass finds the forward pass' layout, which in a capture only the forward pass has captured)
        ctx.save_for_backward(x, W_U, b_U, targets, lse)
        ctx.head, ctx.ignore_index = head, ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, _, _, targets, lse = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, db = ctx.head._loss_backward(dloss.contiguous(), x, targets, lse, ctx.ignore_index, need_x, need_w, need_b,
                                             laid_out=True)
        return dx, dw, db, None, None, None, None


def _total(v: torch.Tensor) -> torch.Tensor:
    """Sum of all elements in rows of 1024: no reduction over several blocks, which clears its counters with a memset node
    in a captured graph."""
    v = v.reshape(-1)
    while v.numel() > 1024:
        n = -(-v.numel() // 1024)
        v = torch.nn.functional.pad(v, (0, n * 1024 - v.numel())).view(n, 1024).sum(1)
    return v.sum()


def unembed_loss(x: torch.Tensor, targets: torch.Tensor, head: "tsc_hip.UnembedHead", ignore_index: int = -100,
                 reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``x @ head.W_U + head.b_U`` with ``targets`` (:meth:`tsc_hip.UnembedHead.loss`), differentiable in
    ``x``, ``head.W_U`` and ``head.b_U``.  ``reduction``: ``"none"`` -- float32 of shape ``x.shape[:-1]``; ``"sum"``;
    ``"mean"`` -- over the rows whose target is not ``ignore_index`` (NaN where there are none)."""
    if reduction not in ("none", "sum", "mean"):
        raise tsc_hip.TscError(f"reduction must be 'none', 'sum' or 'mean' (got {reduction!r})")
    laid_out = False
    if torch.is_grad_enabled():
        held = _mark_leaves(x, head.W_U, head.b_U)  # noqa: F841
        learning = [p for p in (head.W_U, head.b_U) if p is not None and p.requires_grad]
        if learning and torch.cuda.is_current_stream_capturing():
            if not all(p.is_leaf for p in learning):
                raise tsc_hip.TscError("the head's W_U or b_U is a view of the leaf that learns, made before the capture: its "
                                       "accumulator may belong to another stream; make the head of leaves, or step eagerly")
            head.refresh()  # part of the graph: a replay finds the weights that the step before it left
            laid_out = True
    rows = _UnembedLoss.apply(x, head.W_U, head.b_U, targets, head, ignore_index, laid_out)
    if reduction == "none":
        return rows
    total = _total(rows)
    return total if reduction == "sum" else total / _total((targets != ignore_index).double()).float()


_heads: "weakref.WeakKeyDictionary" = weakref.WeakKeyDictionary()
_captured: "weakref.WeakKeyDictionary" = weakref.WeakKeyDictionary()  # model -> heads that a graph may hold


def model_head(model) -> "tsc_hip.UnembedHead":
    """The :class:`tsc_hip.UnembedHead` of ``model.W_U`` and ``model.b_U``, laid out once for as long as the model keeps these
    tensors (a change in place lays it out again; inference tensors do not tell of one, so a model of them lays out for every
    call).  A capture needs one that is there already; a head that was asked for inside
    a capture lives as long as the model, whatever tensors the model gets, because a graph may hold it.  A change that no loss
    has seen before the capture is laid out by every replay, which the caller then orders with losses on other streams."""
    key = tuple((t.data_ptr(), t.dtype, t.shape, t.stride()) for t in (model.W_U, model.b_U))
    entry = _heads.get(model)
    if entry is None or entry[0] != key:
        entry = _heads[model] = (key, tsc_hip.UnembedHead(model.W_U.detach(), model.b_U.detach()))
    elif model.W_U.is_inference() or model.b_U.is_inference():
        entry[1].refresh()
    if torch.cuda.is_current_stream_capturing():
        _captured.setdefault(model, set()).add(entry[1])
    return entry[1]


def next_token_loss(normalized: torch.Tensor, tokens: torch.Tensor, head: "tsc_hip.UnembedHead",
                    per_token: bool = False) -> torch.Tensor:
    """A model's training loss from its final normalised residual ``[batch, n, d_model]``: the cross entropy of token
    ``t + 1`` at position ``t``, as mean or ``[batch, n - 1]`` (padding counts like any token)."""
    return unembed_loss(normalized[:, :-1], tokens[:, 1:].contiguous(), head, reduction="none" if per_token else "mean")


def _plain_head(model) -> bool:
    """Are the model's logits ``hook_normalized @ W_U + b_U`` -- no weight of the final norm (not folded), no cap."""
    return (getattr(getattr(model, "ln_final", None), "w", None) is None
            and not (getattr(getattr(model, "cfg", None), "output_logits_soft_cap", None) or 0) > 0)


def hooked_loss(model, tokens: torch.Tensor, fwd_hooks) -> torch.Tensor:
    """Mean next-token loss of a hooked model under ``fwd_hooks``: ``model.run_with_hooks(tokens, return_type="loss", ...)``, on a
    GPU from the final normalised residual (``ln_final.hook_normalized``) and :func:`model_head`, so that the model makes no
    ``[batch, n, d_vocab]`` logits.  A model whose head is more than that -- a final norm with a weight of its own (not folded),
    capped logits, a loss that leaves out left padding, a type that the operator does not take -- computes its own loss."""

    def own():
        return model.run_with_hooks(tokens, return_type="loss", fwd_hooks=fwd_hooks)

    W, b = getattr(model, "W_U", None), getattr(model, "b_U", None)
    if not all(isinstance(t, torch.Tensor) for t in (W, b, tokens)) or not W.is_cuda or W.device != b.device or tokens.dim() > 2:
        return own()
    if W.dtype not in (torch.float32, torch.bfloat16, torch.float16) or b.dtype not in (W.dtype, torch.float32):
        return own()
    if (not _plain_head(model) or getattr(getattr(model, "tokenizer", None), "padding_side", None) == "left"
            or _FINAL not in getattr(model, "hook_dict", (_FINAL,))):
        return own()
    seen = []
    model.run_with_hooks(tokens, return_type=None, fwd_hooks=list(fwd_hooks) + [(_FINAL, lambda act, hook: seen.append(act))])
    if len(seen) != 1 or seen[0].dtype != W.dtype or seen[0].device != W.device:
        return own()
    return next_token_loss(seen[0], torch.atleast_2d(tokens).to(W.device, torch.int64), model_head(model))
