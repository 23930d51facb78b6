"""CPU checks of the drafted-token and vocabulary-head operators: symbols, structure layout, and every refusal that is made
before a device is touched."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT


def _n():
    from jetlm.kernels import _native
    return _native


@pytest.mark.parametrize("header, exports, structs", [
    ("jetlong_b200_tree.h", "TREE_EXPORTS", {"jl_tree_plan_args": "TreePlanArgs", "jl_tree_append_args": "TreeAppendArgs",
                                             "jl_tree_attention_args": "TreeAttentionArgs", "jl_tree_keep_args": "TreeKeepArgs"}),
    ("jetlong_b200_head.h", "HEAD_EXPORTS", {"jl_head_scores_args": "HeadScoresArgs", "jl_head_grads_args": "HeadGradsArgs"}),
])
def test_header_matches_the_binding(tmp_path, header, exports, structs):
    n = _n()
    text = open(os.path.join(ROOT, "include", header)).read()
    declared = set(re.findall(r"^(?:int|size_t) (jl_[a-z0-9_]+)\(", text, re.M))
    assert declared == {name for name, _, _ in getattr(n, exports)}
    for name in declared:
        assert getattr(n.lib(), name) is not None
    assert set(re.findall(r"}\s*(jl_[a-z0-9_]+)\s*;", text)) == set(structs)
    lines = []
    for c, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in getattr(n, py)._fields_]
    src = tmp_path / "sz.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(){{{"".join(lines)}return 0;}}\n')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "sz"), str(src)])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "sz")]).split()]
    want = []
    for py in structs.values():
        t = getattr(n, py)
        want += [C.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]
    assert got == want


def test_c_entries_refuse_before_they_touch_a_device():
    n = _n()
    lib = n.lib()
    for fn in ("jl_tree_plan", "jl_tree_append", "jl_tree_attention", "jl_tree_keep", "jl_head_scores", "jl_head_grads"):
        assert getattr(lib, fn)(None, None) == n.JL_ERR_BAD_ARG
        assert b"NULL" in lib.jl_last_error()
    p = n.TreePlanArgs(1024, 1024, 1024, 1, 0)
    assert lib.jl_tree_plan(C.byref(p), None) == n.JL_ERR_BAD_ARG
    p.nodes = n.JL_TREE_MAX_NODES + 1
    assert lib.jl_tree_plan(C.byref(p), None) == n.JL_ERR_BAD_ARG

    def attention(**kw):
        a = n.TreeAttentionArgs()
        a.q_base = a.k_base = a.v = a.out = a.lens = a.depth = a.mask = 1024
        a.batch, a.nodes, a.heads, a.kv_heads, a.head_dim, a.rows, a.w_0, a.softmax_scale = 1, 4, 4, 2, 128, 64, 16, 0.125
        for t in "qkvo":
            setattr(a, f"{t}_stride_s", 512)
            setattr(a, f"{t}_stride_h", 128)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jl_tree_attention(C.byref(a), None)

    bad, no = n.JL_ERR_BAD_ARG, n.JL_ERR_UNSUPPORTED
    for want, kw in [(no, dict(head_dim=64)), (bad, dict(kv_heads=3)), (bad, dict(nodes=0)), (bad, dict(nodes=257)), (bad, dict(rows=3)),
                     (bad, dict(w_0=-1)), (bad, dict(q_group=1024)), (bad, dict(k_group=1024)), (bad, dict(v=None)), (bad, dict(mask=None)),
                     (bad, dict(q_base=1032)), (bad, dict(k_stride_s=129)), (bad, dict(o_stride_h=4)), (bad, dict(batch=-1)),
                     (no, dict(heads=258, kv_heads=2)), (no, dict(k_stride_s=0)), (no, dict(q_stride_h=-128)), (no, dict(batch=2)),
                     (bad, dict(softmax_scale=0.0)), (bad, dict(softmax_scale=-0.1)), (bad, dict(softmax_scale=float("nan"))),
                     (bad, dict(softmax_scale=float("inf")))]:
        assert attention(**kw) == want, kw
    assert attention(batch=0) == n.JL_OK

    def append(**kw):
        a = n.TreeAppendArgs()
        for f in ("q", "k", "v", "q_weight", "k_weight", "q_base", "k_cache", "v_cache", "inv_freq", "lens", "depth"):
            setattr(a, f, 1024)
        a.batch, a.nodes, a.heads, a.kv_heads, a.head_dim, a.cache_rows, a.group_size = 1, 4, 4, 2, 128, 64, 1
        a.kc_stride_s = a.vc_stride_s = 256
        a.kc_stride_h = a.vc_stride_h = 128
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jl_tree_append(C.byref(a), None)

    for want, kw in [(no, dict(head_dim=96)), (bad, dict(depth=None)), (bad, dict(nodes=0)), (bad, dict(q_group=1024, group_size=0)),
                     (bad, dict(q=1028)), (bad, dict(kc_stride_s=2)), (bad, dict(cache_rows=-1)),
                     (no, dict(vc_stride_h=0)), (no, dict(batch=2))]:
        assert append(**kw) == want, kw
    assert append(batch=0) == n.JL_OK

    def keep(**kw):
        a = n.TreeKeepArgs()
        a.k_cache = a.v_cache = a.path = a.lens = 1024
        a.batch, a.kept, a.kv_heads, a.head_dim, a.cache_rows = 1, 4, 2, 128, 64
        a.kc_stride_s = a.vc_stride_s = 256
        a.kc_stride_h = a.vc_stride_h = 128
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jl_tree_keep(C.byref(a), None)

    for want, kw in [(no, dict(head_dim=64)), (bad, dict(kept=257)), (bad, dict(kept=-1)), (bad, dict(path=None)), (bad, dict(lens=1026)),
                     (bad, dict(v_cache=1032)), (bad, dict(kc_stride_s=132)), (no, dict(vc_stride_h=0)), (no, dict(batch=2)), (bad, dict(batch=65536))]:
        assert keep(**kw) == want, kw
    assert keep(batch=0) == keep(kept=0) == n.JL_OK

    def scores(**kw):
        a = n.HeadScoresArgs()
        a.hidden = a.weight = a.labels = a.nll = a.workspace = 1024
        a.hidden_stride = a.weight_stride = a.hidden_size = 64
        a.rows, a.vocab = 3, 100
        a.workspace_bytes = lib.jl_head_scores_workspace_bytes(3, 64, 100, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jl_head_scores(C.byref(a), None)

    for want, kw in [(bad, dict(rows=-1)), (bad, dict(vocab=0)), (no, dict(hidden_size=60)), (bad, dict(hidden_stride=68)), (bad, dict(weight_stride=56)),
                     (bad, dict(labels=None)), (bad, dict(hidden=1032)), (n.JL_ERR_WORKSPACE, dict(workspace_bytes=16)),
                     (n.JL_ERR_WORKSPACE, dict(workspace=None)), (no, dict(rows=(1 << 22) + 1)),
                     (bad, dict(skip_ignored=1, top=1024)), (bad, dict(skip_ignored=1, labels=None, nll=None))]:
        assert scores(**kw) == want, kw

    def grads(**kw):
        a = n.HeadGradsArgs()
        a.hidden = a.weight = a.labels = a.lse = a.grad = a.d_hidden = a.workspace = 1024
        a.hidden_stride = a.weight_stride = a.hidden_size = 64
        a.rows, a.vocab = 3, 100
        a.workspace_bytes = lib.jl_head_grads_workspace_bytes(3, 64, 100)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jl_head_grads(C.byref(a), None)

    for want, kw in [(bad, dict(lse=None)), (bad, dict(grad_stride=2)), (bad, dict(d_weight=1028)), (n.JL_ERR_WORKSPACE, dict(workspace_bytes=16)),
                     (no, dict(hidden_size=60))]:
        assert grads(**kw) == want, kw


def test_draft_ops_refuse():
    from jetlm.kernels import draft_ops as d
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)      # noqa: E731
    with pytest.raises(ValueError, match="int32 or int64"):
        d.draft_tree(torch.zeros(1, 4))
    with pytest.raises(ValueError, match="between 1 and 256"):
        d.draft_tree(torch.zeros(1, 257, dtype=torch.int32))
    with pytest.raises(ValueError, match="between 1 and 256"):
        d.draft_tree(torch.zeros(1, 0, dtype=torch.int32))
    with pytest.raises(ValueError, match="requires CUDA"):
        d.draft_tree(torch.zeros(1, 4, dtype=torch.int32))
    B, T, H, Hk, R = 2, 3, 4, 2, 16
    tree = d.DraftTree(torch.zeros(B, T, dtype=torch.int32), torch.zeros(B, T, 1, dtype=torch.int64))
    lens = torch.zeros(B, dtype=torch.int32)
    ok = dict(q_base=bf(B, T, H, 128), q_group=bf(B, T, H, 128), key_rows=bf(B, R, Hk, 128), value_rows=bf(B, R, Hk, 128),
              tree=tree, lens=lens, w_0=4)
    for match, kw in [("requires CUDA", {}), ("rank-4", dict(q_base=bf(T, H, 128))), ("bfloat16", dict(value_rows=torch.zeros(B, R, Hk, 128))),
                      ("share shape and strides", dict(q_group=bf(B, T, H + 1, 128))), ("key_rows and value_rows", dict(value_rows=bf(B, R + 1, Hk, 128))),
                      ("match key_rows", dict(key_group_rows=bf(B, R + 1, Hk, 128))), ("divisible", dict(key_rows=bf(B, R, 3, 128), value_rows=bf(B, R, 3, 128))),
                      ("w_0", dict(w_0=-1)), ("tree.depth", dict(tree=tree._replace(depth=tree.depth.long()))),
                      ("tree.mask", dict(tree=tree._replace(mask=torch.zeros(B, T, 2, dtype=torch.int64)))),
                      ("lens", dict(lens=torch.zeros(B, dtype=torch.int64))), ("does not hold", dict(key_rows=bf(B, 2, Hk, 128), value_rows=bf(B, 2, Hk, 128))),
                      ("multiples of 8", dict(key_rows=torch.zeros(B, R, Hk, 132, dtype=torch.bfloat16)[..., :128])),
                      ("softmax_scale", dict(softmax_scale=0.0)), ("softmax_scale", dict(softmax_scale=float("nan"))),
                      ("broadcast", dict(value_rows=bf(1, R, Hk, 128).expand(B, -1, -1, -1))), ("broadcast", dict(out=bf(B, 1, H, 128).expand(-1, T, -1, -1)))]:
        with pytest.raises(ValueError, match=match):
            d.tree_attention(**{**ok, **kw})
    w = bf(128)
    ok = dict(q=bf(B, T, H, 128), k=bf(B, T, Hk, 128), v=bf(B, T, Hk, 128), q_weight=w, k_weight=w, inv_freq=torch.ones(64),
              key_rows=bf(B, R, Hk, 128), value_rows=bf(B, R, Hk, 128), tree=tree, lens=lens, q_eps=1e-6, k_eps=1e-6)
    for match, kw in [("requires CUDA", {}), ("expects q", dict(v=bf(B, T, Hk + 1, 128))), ("key_rows and value_rows", dict(key_rows=bf(B, R, H, 128))),
                      ("q_weight", dict(q_weight=bf(64))), ("inv_freq", dict(inv_freq=torch.ones(8))), ("group_size", dict(group_size=0)),
                      ("key_group_rows", dict(key_group_rows=bf(B, R, H, 128))), ("broadcast", dict(key_rows=bf(1, R, Hk, 128).expand(B, -1, -1, -1))),
                      ("broadcast", dict(value_rows=bf(B, R, 1, 128).expand(-1, -1, Hk, -1)))]:
        with pytest.raises(ValueError, match=match):
            d.tree_append(**{**ok, **kw})
    path = torch.zeros(B, T, dtype=torch.int32)
    ok = dict(key_rows=bf(B, R, Hk, 128), value_rows=bf(B, R, Hk, 128), path=path, lens=lens)
    for match, kw in [("requires CUDA", {}), ("path", dict(path=path.long())), ("path", dict(path=path[0])), ("path", dict(path=path[:1])),
                      ("at most 256", dict(path=torch.zeros(B, 257, dtype=torch.int32))), ("lens", dict(lens=lens.long())),
                      ("share their shape", dict(value_rows=bf(B, R, 1, 128))), ("match key_rows", dict(key_group_rows=bf(B, Hk, R, 128).transpose(1, 2))),
                      ("bfloat16", dict(value_rows=torch.zeros(B, R, Hk, 128))), ("broadcast", dict(value_rows=bf(1, R, Hk, 128).expand(B, -1, -1, -1)))]:
        with pytest.raises(ValueError, match=match):
            d.tree_keep(**{**ok, **kw})


def test_head_ops_refuse():
    from jetlm.kernels import head_ops as hd
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)      # noqa: E731
    lab = torch.zeros(3, dtype=torch.int64)
    for match, a in [("expects hidden", (bf(3, 64), bf(10, 72), lab)), ("bfloat16", (torch.zeros(3, 64), torch.zeros(10, 64), lab)),
                     ("CUDA", (bf(3, 64), bf(10, 64), lab))]:
        with pytest.raises(ValueError, match=match):
            hd.token_scores(*a)
        with pytest.raises(ValueError, match=match):
            hd.linear_cross_entropy(*a)
    with pytest.raises(ValueError, match="reduction"):
        hd.linear_cross_entropy(bf(3, 64), bf(10, 64), lab, reduction="max")
