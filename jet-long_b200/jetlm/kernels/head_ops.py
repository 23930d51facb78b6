"""The vocabulary head without logits (see include/jetlong_b200_head.h): token scores and the cross-entropy loss with its
gradients, straight from the final hidden states and the lm_head weight.

A 131072-token prompt over a vocabulary of 151936 has 39.8 GB of bf16 logits; these operators hold a piece of the
vocabulary at a time.  The reference forms the logits of every position (modeling_qwen3_jetlong_fused.py:598-636) and
its perplexity driver reads them (jetlm/evaluation/ppl/growing_window.py:91-103).

Kernels run on the current torch CUDA stream; there is no PyTorch fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as N
from .draft_ops import _LAYOUTS, _keep_layout, _run, _sig
from .jetlong_ops import _SUPPORTED_DTYPES, _require_arch


class TokenScores(NamedTuple):
    """Per row: nll = lse - logit of the label (0 where ignored; None without labels), lse, and the most likely token
    (None unless asked for).  All have the shape of the rows."""
    nll: Optional[torch.Tensor]
    lse: torch.Tensor
    top: Optional[torch.Tensor]


def _rows(op: str, hidden: torch.Tensor, weight: torch.Tensor, labels: Optional[torch.Tensor]):
    """(hidden as (rows, H), labels as (rows,)) with the checks the kernels rely on; the layout checks are made once per layout."""
    key = (op, _sig(hidden), _sig(weight), None if labels is None else (labels.shape, labels.dtype, labels.get_device()))
    if key not in _LAYOUTS:
        _check_rows(op, hidden, weight, labels)
        _keep_layout(key, True)
    h = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])          # a copy only where the leading dimensions do not collapse
    if (h.data_ptr() | weight.data_ptr()) & 15:
        raise _bad_rows(op, "weight" if weight.data_ptr() & 15 else "hidden")
    if labels is not None and (labels.dim() != 1 or not labels.is_contiguous()):
        labels = labels.reshape(-1).contiguous()
    return h, labels


def _bad_rows(op, name):
    return ValueError(f"{op}: {name} rows must be contiguous, 16-byte aligned and a multiple of 8 elements apart; call {name}.contiguous()")


def _check_rows(op, hidden, weight, labels):
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{op}: expects hidden (..., H) and weight (V, H), got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype not in _SUPPORTED_DTYPES or weight.dtype != hidden.dtype:
        raise ValueError(f"{op}: hidden and weight must be torch.bfloat16, got {hidden.dtype} and {weight.dtype}")
    if not hidden.is_cuda or weight.device != hidden.device:
        raise ValueError(f"{op}: hidden and weight must be on one CUDA device")
    if weight.shape[0] < 1 or weight.shape[1] < 8 or weight.shape[1] % 8:
        raise ValueError(f"{op}: the hidden size must be a multiple of 8 and the vocabulary not empty, got {tuple(weight.shape)}")
    if labels is not None and (labels.shape != hidden.shape[:-1] or labels.dtype != torch.int64 or labels.device != hidden.device):
        raise ValueError(f"{op}: labels must be int64 with shape {tuple(hidden.shape[:-1])} on {hidden.device}")
    for name, t in (("hidden", hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])), ("weight", weight)):
        if t.shape[0] > 0 and (t.stride(1) != 1 or (t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < t.shape[1]))):
            raise _bad_rows(op, name)
    _require_arch(op, hidden.device)


def _row_stride(t: torch.Tensor) -> int:
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else cols


def _scores(h, w, labels, ignore_index, *, nll, top, reduction=None, skip_ignored=0):
    """One jl_head_scores call on (rows, H) operands; returns (nll, lse, top, loss, loss_count), None where not asked for."""
    n, dev, a = h.shape[0], h.device, N.HeadScoresArgs()
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    per_row = torch.empty_like(lse) if nll else None
    best = torch.empty_like(lse, dtype=torch.int64) if top else None
    loss = torch.empty((), dtype=torch.float32, device=dev) if reduction is not None else None
    count = torch.empty_like(loss) if reduction == "mean" else None
    lib = N.lib()
    ws = torch.empty(lib.jl_head_scores_workspace_bytes(n, w.shape[1], w.shape[0], skip_ignored), dtype=torch.uint8, device=dev)
    a.weight, a.hidden_stride, a.weight_stride, a.ignore_index = w.data_ptr(), _row_stride(h), _row_stride(w), int(ignore_index)
    a.hidden, a.rows, a.hidden_size, a.vocab = h.data_ptr() or a.weight, n, w.shape[1], w.shape[0]
    if labels is not None:
        a.labels = labels.data_ptr() or a.weight                # no rows: never read
    a.lse, a.skip_ignored = lse.data_ptr(), skip_ignored
    if nll:
        a.nll = per_row.data_ptr() or a.weight
    if top:
        a.top = best.data_ptr()
    if count is not None:
        a.loss_mean, a.loss_count = loss.data_ptr(), count.data_ptr()
    elif loss is not None:
        a.loss_sum = loss.data_ptr()
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _run("jl_head_scores", lib.jl_head_scores, a, dev.index)
    return per_row, lse, best, loss, count


def token_scores(hidden: torch.Tensor, weight: torch.Tensor, labels: Optional[torch.Tensor] = None, *, ignore_index: int = -100,
                 top: bool = False) -> TokenScores:
    """Negative log-likelihood of `labels` under softmax(hidden @ weight.T), the log of its normaliser and, with top=True,
    the most likely token of every row (the lowest index of equal ones) — in fp32, with no logits in memory.
    hidden (..., H) and weight (V, H) bf16, labels (...) int64.  A label that is neither ignore_index nor in [0, V) gives
    NaN.  Not differentiable: linear_cross_entropy is."""
    h, lab = _rows("token_scores", hidden.detach(), weight, labels)
    nll, lse, best, _, _ = _scores(h, weight, lab, ignore_index, nll=labels is not None, top=top)
    if hidden.dim() != 2:
        shape = hidden.shape[:-1]
        nll, lse, best = (t.view(shape) if t is not None else None for t in (nll, lse, best))
    return TokenScores(nll, lse, best)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        h, lab = _rows("linear_cross_entropy", hidden, weight, labels)
        per_row, grads = reduction == "none", any(ctx.needs_input_grad)
        nll, lse, _, loss, count = _scores(h, weight, lab, ignore_index, nll=per_row or grads, top=False, reduction=None if per_row else reduction,
                                           skip_ignored=1)
        if grads:
            ctx.save_for_backward(h, weight, lab, lse, nll, count if reduction == "mean" else None)
        ctx.ignore_index, ctx.per_row, ctx.shape = int(ignore_index), per_row, hidden.shape
        if not per_row:
            return loss
        # a copy of its own for the caller, who may write into it before the backward pass reads the losses
        return nll.view(labels.shape).clone() if grads else nll.view(labels.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        h, w, lab, lse, nll, count = ctx.saved_tensors
        n, dev, a, lib = h.shape[0], h.device, N.HeadGradsArgs(), N.lib()
        d_h = torch.empty(h.shape, dtype=h.dtype, device=dev) if ctx.needs_input_grad[0] else None
        d_w = torch.empty(w.shape, dtype=w.dtype, device=dev) if ctx.needs_input_grad[1] else None
        if grad.dtype != torch.float32 or (ctx.per_row and (grad.dim() != 1 or not grad.is_contiguous())):
            grad = grad.to(torch.float32).reshape(-1).contiguous()
        ws = torch.empty(lib.jl_head_grads_workspace_bytes(n, w.shape[1], w.shape[0]), dtype=torch.uint8, device=dev)
        a.weight, a.hidden_stride, a.weight_stride, a.ignore_index = w.data_ptr(), _row_stride(h), _row_stride(w), ctx.ignore_index
        a.hidden, a.labels, a.lse, a.nll, a.grad = (t.data_ptr() or a.weight for t in (h, lab, lse, nll, grad))      # no rows: never read
        a.rows, a.hidden_size, a.vocab, a.grad_stride = n, w.shape[1], w.shape[0], 1 if ctx.per_row else 0
        if count is not None:
            a.grad_count = count.data_ptr()
        if d_h is not None and n:
            a.d_hidden = d_h.data_ptr()
        if d_w is not None:
            a.d_weight = d_w.data_ptr()
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        _run("jl_head_grads", lib.jl_head_grads, a, dev.index)
        return d_h.view(ctx.shape) if d_h is not None else None, d_w, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of softmax(hidden @ weight.T) against `labels`, differentiable in hidden and weight, without the
    logits: torch.nn.functional.cross_entropy(hidden @ weight.T, labels) with fp32 logits.  hidden (..., H) and weight
    (V, H) bf16, labels (...) int64; reduction "mean" (over the labels that are not ignore_index; NaN if there is none, as
    in torch), "sum" or "none" (shape of labels).  The loss is fp32, the gradients are bf16.  The backward pass holds one
    piece of the vocabulary of d logits, in bf16; both gradients accumulate in fp32 and do not vary from run to run.
    Rows whose label is ignore_index take no part, whatever they hold: with more than 256 rows the others are packed and only
    they are multiplied.
    A label that is neither ignore_index nor in [0, V) makes the loss and the gradients NaN; nothing is read out of range.
    Both passes can be captured into a CUDA graph (with torch.autograd.grad, or .backward() while no eager graph of the
    same leaves is alive)."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"linear_cross_entropy: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    return _LinearCrossEntropy.apply(hidden, weight, labels, ignore_index, reduction)
