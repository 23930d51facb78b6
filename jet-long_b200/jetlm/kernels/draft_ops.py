"""Drafted tokens on the bifocal cache: verify a TREE of them in one pass (see include/jetlong_b200_tree.h).

A step takes T drafted tokens per sample.  `parents[b, t]` is -1 for a child of the last committed token, the index of
an earlier node, or -2 for a place that sample b does not use.  Node t is stored in cache row lens[b] + t and sits at
position lens[b] + depth; it attends the committed rows [0, lens[b]) and the nodes on its own path.

    tree = draft_tree(parents)                                                       # once per step
    q_base, q_group = tree_append(q, k, v, ..., key_rows, value_rows, tree, lens)    # per layer
    out, lse = tree_attention(q_base, q_group, key_rows, value_rows, tree, lens, w_0=..., key_group_rows=...)
    tree_keep(key_rows, value_rows, path, lens, key_group_rows=...)                  # per layer, after a path has been chosen

The reference decodes one token per call (jetlm/kernels/cute_decode_sm90.py:2748-2799); these operators have no
counterpart there.  Kernels run on the current torch CUDA stream; nothing here computes attention in PyTorch.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .jetlong_ops import _SUPPORTED_DTYPES, _check_view, _require_arch, _require_contiguous, _st

# Checked call layouts: what a call's shapes, strides, types and devices were found to allow, with the argument structure
# filled in except for its pointers.  A decode loop makes the same call for every layer and step, and the checks took longer
# than the kernels (host time of an attention call: 78 us with them, 20 with the layouts kept).
_LAYOUTS: dict = {}


def _keep_layout(key, value):
    if len(_LAYOUTS) >= 1024:
        _LAYOUTS.clear()
    _LAYOUTS[key] = value
    return value


def _sig(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _misaligned(op: str, **tensors) -> ValueError:
    return ValueError(f"{op}: {next(n for n, t in tensors.items() if t is not None and t.data_ptr() % 16)} must be 16-byte aligned")


def _current_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the handle alone, without the Python object around it (0.2 us against 5), and the current device without the wrapper's checks
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _run(op: str, fn, args, index: int) -> None:
    """One C call on the current stream of the tensors' device."""
    if _current_device() == index:
        status = fn(C.byref(args), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(C.byref(args), _raw_stream(index))
    if status != N.JL_OK:
        N.check(op, status)


def _no_broadcast(op: str, name: str, t: torch.Tensor) -> None:
    if any(t.shape[i] > 1 and t.stride(i) <= 0 for i in range(3)):
        raise ValueError(f"{op}: {name} must not be a broadcast view; call {name}.contiguous()")


class DraftTree(NamedTuple):
    """What the kernels need of a draft's parent links: `depth` (B, T) int32, -1 for an absent node and below T otherwise,
    and `mask` (B, T, (T + 63) // 64) int64 words whose bit u says that the node attends node u (itself and its ancestors)."""
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
    key = (op, parents.shape, parents.dtype, parents.get_device())
    if key not in _LAYOUTS:
        if parents.dim() != 2 or parents.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{op}: parents must be int32 or int64 with shape (B, T)")
        if not 1 <= parents.shape[1] <= N.JL_TREE_MAX_NODES:
            raise ValueError(f"{op}: between 1 and {N.JL_TREE_MAX_NODES} nodes, got {parents.shape[1]}")
        _require_arch(op, _require_cuda(op, parents))
        _keep_layout(key, True)
    B, T = parents.shape
    dev = parents.device
    parents = parents.clamp(-2, T).to(torch.int32) if parents.dtype == torch.int64 else parents
    parents = parents.contiguous()
    depth = torch.empty_like(parents)
    mask = torch.empty(B, T, (T + 63) // 64, dtype=torch.int64, device=dev)
    if B > 0:
        _run("jl_tree_plan", N.lib().jl_tree_plan, N.TreePlanArgs(parents.data_ptr(), depth.data_ptr(), mask.data_ptr(), B, T), dev.index)
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
    q_eps, k_eps, group_size = float(q_eps), float(k_eps), int(group_size)
    key = (op, _sig(q), _sig(k), _sig(v), _sig(q_weight), _sig(k_weight), _sig(inv_freq), _sig(key_rows), _sig(value_rows),
           _sig(key_group_rows), _sig(tree.depth), _sig(tree.mask), _sig(lens), q_eps, k_eps, group_size)
    template = _LAYOUTS.get(key)
    if template is None:
        template = _keep_layout(key, _append_layout(op, q, k, v, q_weight, k_weight, inv_freq, key_rows, value_rows, tree, lens,
                                                    q_eps, k_eps, group_size, key_group_rows))
    if inv_freq.device != q.device or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(device=q.device, dtype=torch.float32).contiguous()
    q_base = torch.empty_like(q, memory_format=torch.contiguous_format)
    q_group = torch.empty_like(q_base) if group_size > 1 else None
    a = N.TreeAppendArgs.from_buffer_copy(template)
    a.q, a.k, a.v, a.q_weight, a.k_weight = ptrs = (q.data_ptr(), k.data_ptr(), v.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr())
    a.k_cache, a.v_cache = kc, vc = key_rows.data_ptr(), value_rows.data_ptr()
    a.q_base = q_base.data_ptr()
    if q_group is not None:
        a.q_group = q_group.data_ptr()
    kg = 0
    if key_group_rows is not None:
        a.k_group_cache = kg = key_group_rows.data_ptr()
    a.inv_freq, a.lens, a.depth = inv_freq.data_ptr(), lens.data_ptr(), tree.depth.data_ptr()
    if (ptrs[0] | ptrs[1] | ptrs[2] | ptrs[3] | ptrs[4] | kc | vc | kg) & 15:
        raise _misaligned(op, q=q, k=k, v=v, q_weight=q_weight, k_weight=k_weight, key_rows=key_rows, value_rows=value_rows,
                          key_group_rows=key_group_rows)
    _run("jl_tree_append", N.lib().jl_tree_append, a, q.device.index)
    return q_base, (q_group if q_group is not None else q_base)


def _append_layout(op, q, k, v, q_weight, k_weight, inv_freq, key_rows, value_rows, tree, lens, q_eps, k_eps, group_size, key_group_rows):
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
    for name, t in (("key_rows", key_rows), ("value_rows", value_rows)):
        _no_broadcast(op, name, t)                    # two samples or heads would write the same rows
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
    _require_arch(op, _require_cuda(op, q, k, v, q_weight, k_weight, key_rows, value_rows, key_group_rows, tree.depth, tree.mask, lens))
    a = N.TreeAppendArgs()
    for name, t in (("q", q), ("k", k), ("v", v), ("kc", key_rows), ("vc", value_rows)):
        for i, axis in enumerate("bsh"):
            setattr(a, f"{name}_stride_{axis}", _st(t, i))
    a.q_eps, a.k_eps, a.cache_rows, a.group_size = float(q_eps), float(k_eps), int(key_rows.shape[1]), int(group_size)
    a.batch, a.nodes, a.heads, a.kv_heads, a.head_dim = B, T, H, Hk, D
    return a


def tree_attention(q_base: torch.Tensor, q_group: torch.Tensor, key_rows: torch.Tensor, value_rows: torch.Tensor,
                   tree: DraftTree, lens: torch.Tensor, *, w_0: int, key_group_rows: Optional[torch.Tensor] = None,
                   softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = True):
    """Bifocal attention of a drafted tree over the cache (see jl_tree_attention).  q_base / q_group (B,T,H,D) views
    sharing strides; key_rows / key_group_rows / value_rows (B,rows,Hk,D) views of this layer's whole cache buffers, the
    nodes' rows included; lens (B,) int32 committed tokens per sample, on the device.  A node whose row lens[b] + t is past
    the cache is an absent one (places of a padded batch may reach there, nodes should not).  Pairs more than w_0 positions apart are scored q_group . key_group_rows, the others q_base . key_rows; without key_group_rows
    (group size 1) every pair is scored q_base . key_rows.  Nothing depends on lens on the host, so the launches can sit
    in a CUDA graph.  Returns (out (B,T,H,D), lse (B,H,T) fp32) or out; a row that sees no key is zero with lse -inf."""
    op = "tree_attention"
    w_0, softmax_scale = int(w_0), None if softmax_scale is None else float(softmax_scale)
    key = (op, _sig(q_base), _sig(q_group), _sig(key_rows), _sig(value_rows), _sig(key_group_rows), _sig(tree.depth), _sig(tree.mask),
           _sig(lens), _sig(out), w_0, softmax_scale)
    plan = _LAYOUTS.get(key)
    if plan is None:
        plan = _keep_layout(key, _attention_layout(op, q_base, q_group, key_rows, value_rows, tree, lens, w_0, key_group_rows,
                                                   softmax_scale, out))
    template, ws_bytes = plan
    dev = q_base.device
    if out is None:
        out = torch.empty_like(q_base, memory_format=torch.contiguous_format)
    # split partials: this call's own memory from the stream-ordered allocator, so concurrent calls and captured graphs
    # never share it
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    a = N.TreeAttentionArgs.from_buffer_copy(template)
    a.q_base, a.k_base, a.v, a.out = ptrs = (q_base.data_ptr(), key_rows.data_ptr(), value_rows.data_ptr(), out.data_ptr())
    qg = kg = 0
    if key_group_rows is not None:
        a.q_group, a.k_group = qg, kg = q_group.data_ptr(), key_group_rows.data_ptr()
    if (ptrs[0] | ptrs[1] | ptrs[2] | ptrs[3] | qg | kg) & 15:
        raise _misaligned(op, q_base=q_base, key_rows=key_rows, value_rows=value_rows, out=out, q_group=q_group, key_group_rows=key_group_rows)
    a.lens, a.depth, a.mask, a.workspace = lens.data_ptr(), tree.depth.data_ptr(), tree.mask.data_ptr(), ws.data_ptr()
    lse = None
    if return_lse:
        lse = torch.empty(a.batch, a.heads, a.nodes, dtype=torch.float32, device=dev)
        a.lse = lse.data_ptr()
    _run("jl_tree_attention", N.lib().jl_tree_attention, a, dev.index)
    return (out, lse) if return_lse else out


def _attention_layout(op, q_base, q_group, key_rows, value_rows, tree, lens, w_0, key_group_rows, softmax_scale, out):
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
        _no_broadcast(op, name, t)
    if Hk < 1 or H % Hk != 0:
        raise ValueError(f"{op}: query heads must be divisible by kv heads")
    if int(w_0) < 0:
        raise ValueError(f"{op}: w_0 must be >= 0")
    if softmax_scale is not None and not 0.0 < softmax_scale < math.inf:
        raise ValueError(f"{op}: softmax_scale must be positive and finite, got {softmax_scale}")
    _require_tree(op, tree, lens, B, T)
    if rows < T:
        raise ValueError(f"{op}: the cache ({rows} rows) does not hold the {T} nodes")
    if out is not None:
        if tuple(out.shape) != (B, T, H, D) or out.dtype != q_base.dtype:
            raise ValueError(f"{op}: out must be {q_base.dtype} with shape {(B, T, H, D)}")
        _check_view(op, "out", out)
        _no_broadcast(op, "out", out)
    _require_arch(op, _require_cuda(op, *(t for _, t in tensors), tree.depth, tree.mask, lens, out))
    o_st = [_st(out, i) for i in range(3)] if out is not None else [T * H * D, H * D, D]
    ws_bytes = max(16, N.lib().jl_tree_attention_workspace_bytes(B, T, H, Hk, rows))
    a = N.TreeAttentionArgs()
    for name, st in (("q", [_st(q_base, i) for i in range(3)]), ("k", [_st(key_rows, i) for i in range(3)]),
                     ("v", [_st(value_rows, i) for i in range(3)]), ("o", o_st)):
        for axis, x in zip("bsh", st):
            setattr(a, f"{name}_stride_{axis}", x)
    a.batch, a.nodes, a.heads, a.kv_heads, a.head_dim, a.rows, a.w_0 = B, T, H, Hk, D, rows, int(w_0)
    a.softmax_scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(D)
    a.workspace_bytes = ws_bytes
    return a, ws_bytes


def tree_keep(key_rows: torch.Tensor, value_rows: torch.Tensor, path: torch.Tensor, lens: torch.Tensor, *,
              key_group_rows: Optional[torch.Tensor] = None) -> None:
    """Moves the rows of the accepted nodes together, in place (see jl_tree_keep): row lens[b] + i of key_rows, value_rows and
    key_group_rows (B,rows,Hk,D views) becomes what row lens[b] + path[b, i] was.  path (B, n) int32 node indices on the
    device, root first; a path ends at its first entry that is not larger than the one before (-1 pads).  Positions do not
    change (node path[b, i] has depth i), so base-rotated and regrouped keys stay valid where they land."""
    op = "tree_keep"
    key = (op, _sig(key_rows), _sig(value_rows), _sig(path), _sig(lens), _sig(key_group_rows))
    template = _LAYOUTS.get(key)
    if template is None:
        template = _keep_layout(key, _tree_keep_layout(op, key_rows, value_rows, path, lens, key_group_rows))
    a = N.TreeKeepArgs.from_buffer_copy(template)
    a.k_cache, a.v_cache = kc, vc = key_rows.data_ptr(), value_rows.data_ptr()
    kg = 0
    if key_group_rows is not None:
        a.k_group_cache = kg = key_group_rows.data_ptr()
    if (kc | vc | kg) & 15:
        raise _misaligned(op, key_rows=key_rows, value_rows=value_rows, key_group_rows=key_group_rows)
    a.path, a.lens = path.data_ptr(), lens.data_ptr()
    _run("jl_tree_keep", N.lib().jl_tree_keep, a, key_rows.device.index)


def _tree_keep_layout(op, key_rows, value_rows, path, lens, key_group_rows):
    caches = [("key_rows", key_rows), ("value_rows", value_rows)] + ([("key_group_rows", key_group_rows)] if key_group_rows is not None else [])
    for name, t in caches:
        _check_view(op, name, t)
        _no_broadcast(op, name, t)
        if t.dtype not in _SUPPORTED_DTYPES:
            raise ValueError(f"{op}: {name} must be torch.bfloat16, got {t.dtype}")
        if t.shape != key_rows.shape:
            raise ValueError(f"{op}: key_rows, value_rows and key_group_rows must share their shape")
    if key_group_rows is not None and [_st(key_group_rows, i) for i in range(3)] != [_st(key_rows, i) for i in range(3)]:
        raise ValueError(f"{op}: key_group_rows must match key_rows in shape and strides")
    B, rows, Hk, D = key_rows.shape
    if path.dim() != 2 or path.shape[1] > N.JL_TREE_MAX_NODES:
        raise ValueError(f"{op}: path must be (B, n) with at most {N.JL_TREE_MAX_NODES} nodes, got {tuple(path.shape)}")
    _require_ints(op, "path", path, (B, path.shape[1]), torch.int32)
    _require_ints(op, "lens", lens, (B,), torch.int32)
    _require_arch(op, _require_cuda(op, *(t for _, t in caches), path, lens))
    a = N.TreeKeepArgs()
    for name, t in (("kc", key_rows), ("vc", value_rows)):
        for i, axis in enumerate("bsh"):
            setattr(a, f"{name}_stride_{axis}", _st(t, i))
    a.cache_rows, a.batch, a.kept, a.kv_heads, a.head_dim = rows, B, path.shape[1], Hk, D
    return a
