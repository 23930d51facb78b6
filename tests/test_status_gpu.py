"""The status words of the kernels' bounded waits: read after the work of every stream, and read by the drafted and scoring paths of a
model that asks for it."""
import pytest
import torch

from test_model_gpu import _tiny_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["jl_prefill_status", "jl_tree_status", "jl_head_status"])
def test_status_waits_for_other_streams(name):
    from jetlm.kernels import _native
    assert getattr(_native.lib(), name)() == 0        # (the first call may allocate, which waits for everything)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                # some 50 ms
    assert not side.query()
    assert getattr(_native.lib(), name)() == 0
    assert side.query()


def _raise_after(monkeypatch, module, name, word):
    """kernel_status as if a wait had given up in the last call of module.name; a read clears it."""
    from jetlm.kernels import jetlong_ops as ops
    word_up, real_fn, real_status = [], getattr(module, name), ops.kernel_status

    def fn(*a, **k):
        word_up.append(1)
        return real_fn(*a, **k)

    def status():
        st = real_status()
        if word_up:
            word_up.clear()
            st[word] = 1
        return st

    monkeypatch.setattr(module, name, fn)
    monkeypatch.setattr(ops, "kernel_status", status)


@torch.inference_mode()
@pytest.mark.parametrize("where, name, word", [("draft", "tree_attention", "tree_wait_timeouts"), ("head", "token_scores", "head_wait_timeouts")])
def test_drafted_generation_reads_the_status(golden, monkeypatch, where, name, word):
    from jetlm.kernels import draft_ops, head_ops
    from jetlm.kernels import jetlong_ops as ops
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    ids = g["input_ids"].cuda()[:, :100]
    model.generate_drafted(ids, 3, lambda i: ([1], [-1]))
    _raise_after(monkeypatch, dict(draft=draft_ops, head=head_ops)[where], name, word)
    model.generate_drafted(ids, 3, lambda i: ([1], [-1]))                  # off by default
    with pytest.raises(RuntimeError, match="gave up"):                     # what that call left
        ops.check_status()
    model.model.check_kernel_status = True
    with pytest.raises(RuntimeError, match="gave up"):
        model.generate_drafted(ids, 2, lambda i: ([1], [-1]))              # one step behind the prompt


@torch.inference_mode()
def test_the_last_step_of_a_drafted_generation_is_checked_too(golden, monkeypatch):
    from jetlm.kernels import jetlong_ops as ops
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    model.model.check_kernel_status = True
    ids = g["input_ids"].cuda()[:, :100]
    order, real = [], ops.check_status
    from jetlm.kernels import draft_ops, head_ops
    scores, attend = head_ops.token_scores, draft_ops.tree_attention
    monkeypatch.setattr(ops, "check_status", lambda: (order.append("check"), real())[1])
    monkeypatch.setattr(head_ops, "token_scores", lambda *a, **k: (order.append("head"), scores(*a, **k))[1])
    monkeypatch.setattr(draft_ops, "tree_attention", lambda *a, **k: (order.append("tree"), attend(*a, **k))[1])
    model.generate_drafted(ids, 4, lambda i: ([], []))
    assert order.count("head") == 4 and order[-1] == "check"
    assert all(b == "check" for a, b in zip(order, order[1:]) if a == "head")


@torch.inference_mode()
def test_scores_and_losses_read_the_status(golden, monkeypatch):
    from jetlm.kernels import head_ops
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    ids = g["input_ids"].cuda()[:, :100]
    model.fused_loss = True
    _raise_after(monkeypatch, head_ops, "token_scores", "head_wait_timeouts")
    _raise_after(monkeypatch, head_ops, "linear_cross_entropy", "head_wait_timeouts")
    model.score_tokens(ids)
    model(input_ids=ids, labels=ids)
    from jetlm.kernels import jetlong_ops as ops
    with pytest.raises(RuntimeError, match="gave up"):                     # what the calls above left
        ops.check_status()
    model.model.check_kernel_status = True
    with pytest.raises(RuntimeError, match="gave up"):
        model.score_tokens(ids)
    with pytest.raises(RuntimeError, match="gave up"):
        model(input_ids=ids, labels=ids)
