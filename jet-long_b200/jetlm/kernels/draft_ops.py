"""Drafted tokens on the bifocal cache: verify a TREE of them in one pass (see include/jetlong_b200_tree.h).

A step takes T drafted tokens per sample.  `parents[b, t]` is -1 for a child of the last committed token, the index of
an earlier node, or -2 for a place that sample b does not use.  Node t is stored in cache row lens[b] + t and sits at
position lens[b] + depth; it attends the committed rows [0, lens[b]) and the nodes on its own path.

    tree = draft_tree(parents)                                                       # once per step
    q_base, q_group = tree_append(q, k, v, ..., key_rows, value_rows, tree, lens)    # per layer
    out, lse = tree_attention(q_base, q_group, key_rows, value_rows, tree, lens, w_0=..., key_group_rows=...)
    keep_path(buffer, path, start)                                                   # after the path has been chosen

The reference decodes one token per call (jetlm/kernels/cute_decode_sm90.py:2748-2799); these operators have no
counterpart there.  Kernels run on the current torch CUDA stream; nothing here computes attention in PyTorch.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .jetlong_ops import _SUPPORTED_DTYPES, _call, _check_view, _require_arch, _require_contiguous, _st, _stream


class DraftTree(NamedTuple):
    """What the kernels need of a draft's parent links: `depth` (B, T) int32, -1 for an absent node, and `mask`
    (B, T, (T + 63) // 64) int64 words whose bit u says that the node attends node u (itself and its ancestors)."""
    depth: torch.Tensor
    mask: torch.Tensor


def _require_cuda(op: str, *tensors) -> torch.device:
    if not all(t.is_cuda for t in tensors if t is not None):
        raise ValueError(f"{op} requires CUDA tensors")
    dev = tensors[0].device
    if not all(t.device == dev for t in tensors if t is not None):
        raise ValueError(f"{op}: all tensors must be on the same CUDA device")
    return dev


def _require_ints(op: str, name: str, t: torch.Tensor, shape: tuple, dtype) -> None:
    if tuple(t.shape) != shape or t.dtype != dtype:
        raise ValueError(f"{op}: {name} must be {dtype} with shape {shape}, got {t.dtype} {tuple(t.shape)}")
    _require_contiguous(op, name, t)


def _require_tree(op: str, tree: DraftTree, lens: torch.Tensor, B: int, T: int) -> None:
    if not 1 <= T <= N.JL_TREE_MAX_NODES:
        raise ValueError(f"{op}: between 1 and {N.JL_TREE_MAX_NODES} nodes, got {T}")
    _require_ints(op, "tree.depth", tree.depth, (B, T), torch.int32)
    _require_ints(op, "tree.mask", tree.mask, (B, T, (T + 63) // 64), torch.int64)
    _require_ints(op, "lens", lens, (B,), torch.int32)


def draft_tree(parents: torch.Tensor) -> DraftTree:
    """Depths and ancestor masks of parent links (B, T) or (T,), int32 or int64 on the device (see jl_tree_plan).
    A link that is neither -1 nor an earlier node makes the node, and every node below it, an absent one."""
    op = "draft_tree"
    if parents.dim() == 1:
        parents = parents.unsqueeze(0)
    if parents.dim() != 2 or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{op}: parents must be int32 or int64 with shape (B, T)")
    B, T = parents.shape
    if not 1 <= T <= N.JL_TREE_MAX_NODES:
        raise ValueError(f"{op}: between 1 and {N.JL_TREE_MAX_NODES} nodes, got {T}")
    dev = _require_cuda(op, parents)
    _require_arch(op, dev)
    parents = parents.clamp(-2, T).to(torch.int32) if parents.dtype == torch.int64 else parents
    parents = parents.contiguous()
    depth = torch.empty(B, T, dtype=torch.int32, device=dev)
    mask = torch.empty(B, T, (T + 63) // 64, dtype=torch.int64, device=dev)
    a = N.TreePlanArgs(parents.data_ptr(), depth.data_ptr(), mask.data_ptr(), B, T)
    if B > 0:
        with torch.cuda.device(dev):
            _call("jl_tree_plan", lambda: N.lib().jl_tree_plan(C.byref(a), _stream()))
    return DraftTree(depth, mask)


def tree_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                inv_freq: torch.Tensor, key_rows: torch.Tensor, value_rows: torch.Tensor, tree: DraftTree, lens: torch.Tensor, *,
                q_eps: float, k_eps: float, group_size: int = 1, key_group_rows: Optional[torch.Tensor] = None):
    """One launch between the projections and the attention of a tree step (see jl_tree_append): per-head RMSNorm + RoPE
    of q (B,T,H,D) and k (B,T,Hk,D) at the nodes' positions, the regrouped query when group_size > 1, and the write of
    keys and values into rows lens[b] + t of key_rows / value_rows (B,rows,Hk,D views of the cache buffers).
    key_group_rows (shape and strides of key_rows) receives the regrouped keys.  Absent nodes get zero queries and write
    nothing.  Returns (q_base, q_group), each (B,T,H,D); q_group is q_base when group_size == 1."""
    op = "tree_append"
    for name, t in (("q", q), ("k", k), ("v", v), ("key_rows", key_rows), ("value_rows", value_rows)):
        _check_view(op, name, t)
        if t.dtype not in _SUPPORTED_DTYPES:
            raise ValueError(f"{op}: {name} must be torch.bfloat16, got {t.dtype}")
    B, T, H, D = q.shape
    Hk = k.shape[2]
    if k.shape != (B, T, Hk, D) or v.shape != k.shape:
        raise ValueError(f"{op}: expects q (B,T,H,D) and k, v (B,T,Hk,D)")
    if key_rows.shape[0] != B or key_rows.shape[2:] != (Hk, D) or value_rows.shape != key_rows.shape:
        raise ValueError(f"{op}: key_rows and value_rows must be (B, rows, Hk, D)")
    _require_tree(op, tree, lens, B, T)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.numel() != D or not w.is_contiguous() or w.dtype != q.dtype:
            raise ValueError(f"{op}: {name} must be a contiguous ({D},) tensor of the query dtype")
    if inv_freq.numel() < D // 2:
        raise ValueError(f"{op}: inv_freq must have shape ({D // 2},) or larger")
    if int(group_size) < 1:
        raise ValueError(f"{op}: group_size must be >= 1")
    if key_group_rows is not None and (key_group_rows.shape != key_rows.shape or key_group_rows.dtype != key_rows.dtype
                                       or [_st(key_group_rows, i) for i in range(3)] != [_st(key_rows, i) for i in range(3)]):
        raise ValueError(f"{op}: key_group_rows must match key_rows in shape, strides and dtype")
    dev = _require_cuda(op, q, k, v, q_weight, k_weight, key_rows, value_rows, key_group_rows, tree.depth, tree.mask, lens)
    _require_arch(op, dev)
    inv_freq = inv_freq.to(device=dev, dtype=torch.float32).contiguous()
    q_base = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    q_group = torch.empty(B, T, H, D, dtype=q.dtype, device=dev) if group_size > 1 else None
    a = N.TreeAppendArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         *(_st(t, i) for t in (q, k, v) for i in range(3)),
                         q_weight.data_ptr(), k_weight.data_ptr(), float(q_eps), float(k_eps),
                         q_base.data_ptr(), q_group.data_ptr() if q_group is not None else None,
                         key_rows.data_ptr(), value_rows.data_ptr(),
                         key_group_rows.data_ptr() if key_group_rows is not None else None,
                         *(_st(t, i) for t in (key_rows, value_rows) for i in range(3)), int(key_rows.shape[1]),
                         B, T, H, Hk, D, int(group_size), inv_freq.data_ptr(), lens.data_ptr(), tree.depth.data_ptr())
    with torch.cuda.device(dev):
        _call("jl_tree_append", lambda: N.lib().jl_tree_append(C.byref(a), _stream()))
    return q_base, (q_group if q_group is not None else q_base)


def tree_attention(q_base: torch.Tensor, q_group: torch.Tensor, key_rows: torch.Tensor, value_rows: torch.Tensor,
                   tree: DraftTree, lens: torch.Tensor, *, w_0: int, key_group_rows: Optional[torch.Tensor] = None,
                   softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = True):
    """Bifocal attention of a drafted tree over the cache (see jl_tree_attention).  q_base / q_group (B,T,H,D) views
    sharing strides; key_rows / key_group_rows / value_rows (B,rows,Hk,D) views of this layer's whole cache buffers, the
    nodes' rows included; lens (B,) int32 committed tokens per sample, on the device, lens[b] + T <= rows.  Pairs more
    than w_0 positions apart are scored q_group . key_group_rows, the others q_base . key_rows; without key_group_rows
    (group size 1) every pair is scored q_base . key_rows.  Nothing depends on lens on the host, so the launches can sit
    in a CUDA graph.  Returns (out (B,T,H,D), lse (B,H,T) fp32) or out; a row that sees no key is zero with lse -inf."""
    op = "tree_attention"
    tensors = [("q_base", q_base), ("q_group", q_group), ("key_rows", key_rows), ("value_rows", value_rows)]
    if key_group_rows is not None:
        tensors.append(("key_group_rows", key_group_rows))
    for name, t in tensors:
        _check_view(op, name, t)
        if t.dtype not in _SUPPORTED_DTYPES:
            raise ValueError(f"{op}: {name} must be torch.bfloat16, got {t.dtype}")
    B, T, H, D = q_base.shape
    rows, Hk = key_rows.shape[1], key_rows.shape[2]
    if q_group.shape != q_base.shape or [_st(q_group, i) for i in range(3)] != [_st(q_base, i) for i in range(3)]:
        raise ValueError(f"{op}: q_base and q_group must share shape and strides")
    if key_rows.shape != (B, rows, Hk, D) or value_rows.shape != key_rows.shape:
        raise ValueError(f"{op}: key_rows and value_rows must be (B, rows, Hk, D)")
    if key_group_rows is not None and (key_group_rows.shape != key_rows.shape
                                       or [_st(key_group_rows, i) for i in range(3)] != [_st(key_rows, i) for i in range(3)]):
        raise ValueError(f"{op}: key_group_rows must match key_rows in shape and strides")
    for name, t in tensors:
        if any(t.shape[i] > 1 and t.stride(i) <= 0 for i in range(3)):
            raise ValueError(f"{op}: {name} must not be a broadcast view; call {name}.contiguous()")
    if Hk < 1 or H % Hk != 0:
        raise ValueError(f"{op}: query heads must be divisible by kv heads")
    if int(w_0) < 0:
        raise ValueError(f"{op}: w_0 must be >= 0")
    _require_tree(op, tree, lens, B, T)
    if rows < T:
        raise ValueError(f"{op}: the cache ({rows} rows) does not hold the {T} nodes")
    dev = _require_cuda(op, *(t for _, t in tensors), tree.depth, tree.mask, lens, out)
    _require_arch(op, dev)
    if out is None:
        out = torch.empty(B, T, H, D, dtype=q_base.dtype, device=dev)
    else:
        if tuple(out.shape) != (B, T, H, D) or out.dtype != q_base.dtype:
            raise ValueError(f"{op}: out must be {q_base.dtype} with shape {(B, T, H, D)}")
        _check_view(op, "out", out)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=dev) if return_lse else None
    lib = N.lib()
    # split partials: this call's own memory from the stream-ordered allocator, so concurrent calls and captured graphs
    # never share it
    ws = torch.empty(max(16, lib.jl_tree_attention_workspace_bytes(B, T, H, Hk, rows)), dtype=torch.uint8, device=dev)
    two = key_group_rows is not None
    a = N.TreeAttentionArgs(q_base.data_ptr(), q_group.data_ptr() if two else None, key_rows.data_ptr(),
                            key_group_rows.data_ptr() if two else None, value_rows.data_ptr(),
                            *(_st(t, i) for t in (q_base, key_rows, value_rows) for i in range(3)),
                            lens.data_ptr(), tree.depth.data_ptr(), tree.mask.data_ptr(), out.data_ptr(),
                            lse.data_ptr() if lse is not None else None, *(_st(out, i) for i in range(3)),
                            B, T, H, Hk, D, rows, int(w_0),
                            float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D), 0,
                            ws.data_ptr(), ws.numel())
    with torch.cuda.device(dev):
        _call("jl_tree_attention", lambda: lib.jl_tree_attention(C.byref(a), _stream()))
    return (out, lse) if return_lse else out


def keep_path(buffer: torch.Tensor, path: torch.Tensor, start: int) -> None:
    """Move the rows of the accepted nodes together: buffer (B, rows, ...) gets rows start + path[i] in rows
    start + i.  `path` (n,) int64 node indices on the device, root first.  Positions do not change (node path[i] has
    depth i), so base-rotated and regrouped keys stay valid where they land."""
    if path.dim() != 1 or path.dtype != torch.int64:
        raise ValueError("keep_path: path must be int64 with shape (n,)")
    buffer[:, start: start + path.numel()] = buffer.index_select(1, path + start)
