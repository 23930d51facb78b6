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
