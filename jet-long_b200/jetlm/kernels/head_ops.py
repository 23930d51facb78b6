"""The vocabulary head without logits (see include/jetlong_b200_head.h): token scores and the cross-entropy loss with its
gradients, straight from the final hidden states and the lm_head weight.

A 131072-token prompt over a vocabulary of 151936 has 39.8 GB of bf16 logits; these operators hold a piece of the
vocabulary at a time.  The reference forms the logits of every position (modeling_qwen3_jetlong_fused.py:598-636) and
its perplexity driver reads them (jetlm/evaluation/ppl/growing_window.py:91-103).

Kernels run on the current torch CUDA stream; there is no PyTorch fallback.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .jetlong_ops import _SUPPORTED_DTYPES, _call, _require_arch, _stream


class TokenScores(NamedTuple):
    """Per row: nll = lse - logit of the label (0 where ignored; None without labels), lse, and the most likely token
    (None unless asked for).  All have the shape of the rows."""
    nll: Optional[torch.Tensor]
    lse: torch.Tensor
    top: Optional[torch.Tensor]


def _rows(op: str, hidden: torch.Tensor, weight: torch.Tensor, labels: Optional[torch.Tensor]):
    """(hidden as (rows, H), weight, labels as (rows,)) with the checks the kernels rely on."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{op}: expects hidden (..., H) and weight (V, H), got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype not in _SUPPORTED_DTYPES or weight.dtype != hidden.dtype:
        raise ValueError(f"{op}: hidden and weight must be torch.bfloat16, got {hidden.dtype} and {weight.dtype}")
    if not hidden.is_cuda or weight.device != hidden.device:
        raise ValueError(f"{op}: hidden and weight must be on one CUDA device")
    if weight.shape[0] < 1 or weight.shape[1] < 8 or weight.shape[1] % 8:
        raise ValueError(f"{op}: the hidden size must be a multiple of 8 and the vocabulary not empty, got {tuple(weight.shape)}")
    if labels is not None:
        if labels.shape != hidden.shape[:-1] or labels.dtype != torch.int64 or labels.device != hidden.device:
            raise ValueError(f"{op}: labels must be int64 with shape {tuple(hidden.shape[:-1])} on {hidden.device}")
        labels = labels.reshape(-1).contiguous()
    _require_arch(op, hidden.device)
    h = hidden.reshape(-1, hidden.shape[-1])          # a copy only where the leading dimensions do not collapse
    for name, t in (("hidden", h), ("weight", weight)):
        if t.shape[0] > 0 and (t.stride(1) != 1 or (t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < t.shape[1])) or t.data_ptr() % 16):
            raise ValueError(f"{op}: {name} rows must be contiguous, 16-byte aligned and a multiple of 8 elements apart; "
                             f"call {name}.contiguous()")
    return h, weight, labels


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _scores(op, h, w, labels, ignore_index, *, nll, lse, top, loss):
    """One jl_head_scores call on (rows, H) operands; returns (nll, lse, top, loss_sum, loss_count), None where not asked for."""
    n, dev = h.shape[0], h.device
    f32 = lambda *s: torch.empty(*s, dtype=torch.float32, device=dev)      # noqa: E731
    out = (f32(n) if nll else None, f32(n) if lse else None, torch.empty(n, dtype=torch.int64, device=dev) if top else None,
           f32(()) if loss else None, f32(()) if loss else None)
    lib = N.lib()
    ws = torch.empty(lib.jl_head_scores_workspace_bytes(n, w.shape[1], w.shape[0]), dtype=torch.uint8, device=dev)
    ptr = lambda t: t.data_ptr() if t is not None else None                # noqa: E731
    a = N.HeadScoresArgs(h.data_ptr() if n else w.data_ptr(), w.data_ptr(), _row_stride(h), _row_stride(w),
                         ptr(labels) if n or labels is None else w.data_ptr(), int(ignore_index),
                         n, w.shape[1], w.shape[0], *(ptr(t) for t in out), ws.data_ptr(), ws.numel())
    with torch.cuda.device(dev):
        _call("jl_head_scores", lambda: lib.jl_head_scores(C.byref(a), _stream()))
    return out


def token_scores(hidden: torch.Tensor, weight: torch.Tensor, labels: Optional[torch.Tensor] = None, *, ignore_index: int = -100,
                 top: bool = False) -> TokenScores:
    """Negative log-likelihood of `labels` under softmax(hidden @ weight.T), the log of its normaliser and, with top=True,
    the most likely token of every row (the lowest index of equal ones) — in fp32, with no logits in memory.
    hidden (..., H) and weight (V, H) bf16, labels (...) int64.  A label that is neither ignore_index nor in [0, V) gives
    NaN.  Not differentiable: linear_cross_entropy is."""
    op = "token_scores"
    with torch.no_grad():
        h, w, lab = _rows(op, hidden.detach(), weight.detach(), labels)
        nll, lse, best, _, _ = _scores(op, h, w, lab, ignore_index, nll=labels is not None, lse=True, top=top, loss=False)
    shape = hidden.shape[:-1]
    return TokenScores(nll.view(shape) if nll is not None else None, lse.view(shape), best.view(shape) if best is not None else None)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        h, w, lab = _rows("linear_cross_entropy", hidden, weight, labels)
        nll, lse, _, total, count = _scores("linear_cross_entropy", h, w, lab, ignore_index, nll=reduction == "none", lse=True,
                                            top=False, loss=reduction != "none")
        ctx.save_for_backward(hidden, weight, lab, lse, count if reduction == "mean" else None)
        ctx.ignore_index, ctx.per_row = int(ignore_index), reduction == "none"
        return nll.view(labels.shape) if ctx.per_row else total / count if reduction == "mean" else total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, lab, lse, count = ctx.saved_tensors
        h, w, _ = _rows("linear_cross_entropy", hidden, weight, None)
        n, dev = h.shape[0], h.device
        d_h = torch.empty(h.shape, dtype=h.dtype, device=dev) if ctx.needs_input_grad[0] else None
        d_w = torch.empty(w.shape, dtype=w.dtype, device=dev) if ctx.needs_input_grad[1] else None
        grad = grad.to(torch.float32).reshape(-1).contiguous()
        lib = N.lib()
        ws = torch.empty(lib.jl_head_grads_workspace_bytes(n, w.shape[1], w.shape[0]), dtype=torch.uint8, device=dev)
        some = lambda t: t.data_ptr() if t.numel() else w.data_ptr()       # noqa: E731  (no rows: never read)
        a = N.HeadGradsArgs(some(h), w.data_ptr(), _row_stride(h), _row_stride(w), some(lab), ctx.ignore_index, n, w.shape[1], w.shape[0],
                            some(lse), some(grad), 1 if ctx.per_row else 0, count.data_ptr() if count is not None else None,
                            d_h.data_ptr() if d_h is not None and n else None, d_w.data_ptr() if d_w is not None else None,
                            ws.data_ptr(), ws.numel())
        with torch.cuda.device(dev):
            _call("jl_head_grads", lambda: lib.jl_head_grads(C.byref(a), _stream()))
        return d_h.view(hidden.shape) if d_h is not None else None, d_w, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of softmax(hidden @ weight.T) against `labels`, differentiable in hidden and weight, without the
    logits: torch.nn.functional.cross_entropy(hidden @ weight.T, labels) with fp32 logits.  hidden (..., H) and weight
    (V, H) bf16, labels (...) int64; reduction "mean" (over the labels that are not ignore_index; NaN if there is none, as
    in torch), "sum" or "none" (shape of labels).  The loss is fp32, the gradients are bf16.  The backward pass holds one
    piece of the vocabulary of d logits, in bf16; both gradients accumulate in fp32 and do not vary from run to run.
    A label that is neither ignore_index nor in [0, V) makes the loss and the gradients NaN; nothing is read out of range.
    Both passes can be captured into a CUDA graph (with torch.autograd.grad, or .backward() while no eager graph of the
    same leaves is alive)."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"linear_cross_entropy: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    return _LinearCrossEntropy.apply(hidden, weight, labels, ignore_index, reduction)
