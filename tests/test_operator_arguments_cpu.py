"""Arguments of the drafted-token and vocabulary-head C entries that are refused, or need nothing, before a device is touched."""
import ctypes as C


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
