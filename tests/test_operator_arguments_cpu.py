"""Arguments of the drafted-token and vocabulary-head C entries that are refused, or need nothing, before a device is touched."""
import ctypes as C

import pytest


def _n():
    from jetlm.kernels import _native
    return _native


def grads(**kw):
    n = _n()
    a = n.HeadGradsArgs()
    a.hidden = a.weight = a.labels = a.lse = a.nll = a.grad = a.d_hidden = a.workspace = 1024
    a.hidden_stride = a.weight_stride = a.hidden_size = 64
    a.rows, a.vocab = 3, 100
    a.workspace_bytes = n.lib().jl_head_grads_workspace_bytes(3, 64, 100)
    for k, v in kw.items():
        setattr(a, k, v)
    return n.lib().jl_head_grads(C.byref(a), None)


def test_gradients_need_the_losses_of_the_forward_pass():
    n = _n()
    assert grads(nll=None) == n.JL_ERR_BAD_ARG and b"nll" in n.lib().jl_last_error()


def plan(**kw):
    n = _n()
    a = n.TreePlanArgs(1024, 1024, 1024, 1, 4)
    for k, v in kw.items():
        setattr(a, k, v)
    return n.lib().jl_tree_plan(C.byref(a), None)


def append(**kw):
    n = _n()
    a = n.TreeAppendArgs()
    for f in ("q", "k", "v", "q_weight", "k_weight", "q_base", "k_cache", "v_cache", "inv_freq", "lens", "depth"):
        setattr(a, f, 1024)
    a.batch, a.nodes, a.heads, a.kv_heads, a.head_dim, a.cache_rows, a.group_size = 1, 4, 4, 2, 128, 64, 1
    a.kc_stride_s = a.vc_stride_s = 256
    a.kc_stride_h = a.vc_stride_h = 128
    for k, v in kw.items():
        setattr(a, k, v)
    return n.lib().jl_tree_append(C.byref(a), None)


def attention(**kw):
    n = _n()
    a = n.TreeAttentionArgs()
    a.q_base = a.k_base = a.v = a.out = a.lens = a.depth = a.mask = 1024
    a.batch, a.nodes, a.heads, a.kv_heads, a.head_dim, a.rows, a.w_0, a.softmax_scale = 1, 4, 4, 2, 128, 64, 16, 0.125
    for t in "qkvo":
        setattr(a, f"{t}_stride_s", 512)
        setattr(a, f"{t}_stride_h", 128)
    for k, v in kw.items():
        setattr(a, k, v)
    return n.lib().jl_tree_attention(C.byref(a), None)


def test_no_samples_need_no_arrays():
    n = _n()
    assert plan(batch=0, parents=None, depth=None, mask=None) == n.JL_OK
    assert append(batch=0, q=None, k=None, v=None, q_base=None, k_cache=None, v_cache=None, lens=None, depth=None) == n.JL_OK
    assert attention(batch=0, q_base=None, k_base=None, v=None, out=None, lens=None, depth=None, mask=None) == n.JL_OK
    # sizes that are out of range stay so
    assert plan(batch=0, nodes=0) == append(batch=0, nodes=300) == attention(batch=0, kv_heads=3) == n.JL_ERR_BAD_ARG
    assert append(batch=0, head_dim=64) == n.JL_ERR_UNSUPPORTED


def scores(**kw):
    n = _n()
    a = n.HeadScoresArgs()
    a.hidden = a.weight = a.labels = a.nll = a.workspace = 1024
    a.hidden_stride = a.weight_stride = a.hidden_size = 64
    a.rows, a.vocab = 3, 100
    a.workspace_bytes = n.lib().jl_head_scores_workspace_bytes(3, 64, 100, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return n.lib().jl_head_scores(C.byref(a), None)


@pytest.mark.parametrize("call, field, address", [
    *[(append, f, 1026) for f in ("inv_freq", "lens", "depth")], *[(attention, f, 1026) for f in ("lens", "depth", "lse")], (attention, "mask", 1028),
    (scores, "labels", 1028), (scores, "top", 1028), *[(scores, f, 1026) for f in ("nll", "lse", "loss_sum", "loss_count", "loss_mean")],
    (grads, "labels", 1028), *[(grads, f, 1026) for f in ("lse", "nll", "grad", "grad_count")]])
def test_misaligned_arrays_are_refused(call, field, address):
    """The kernels load whole words; nothing of such a call may reach the device (there is none here, and one is asked for last)."""
    n = _n()
    assert call(**{field: address}) == n.JL_ERR_BAD_ARG and b"aligned" in n.lib().jl_last_error()


def test_the_attention_workspace_does_not_grow_with_the_batch():
    """A part of the line of visits leaves two partial results at most: 148 parts, two row tiles of 128 rows, 512 bytes of O and 4 of lse."""
    n = _n()
    size = n.lib().jl_tree_attention_workspace_bytes
    for nodes, heads, kv in [(1, 8, 8), (16, 32, 8), (64, 32, 8), (80, 32, 8), (256, 8, 1), (256, 128, 1), (255, 64, 1)]:
        one = size(1, nodes, heads, kv, 4096)
        assert 0 < one <= 2 * (148 * 2 + 1) * 128 * 516
        assert size(65535 // kv, nodes, heads, kv, 4096) == one
