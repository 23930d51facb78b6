"""The drafted-token and vocabulary-head operators together, as the model runs them."""
import math

import pytest
import torch

from test_model_gpu import _tiny_model

pytestmark = pytest.mark.gpu

HALF = torch.finfo(torch.bfloat16).eps / 2


def _greedy(model, ids, n, chunk):
    """One token per call through the decode path, the choice made by the fp32 head."""
    from jetlm.kernels import head_ops
    from jetlm.kernels.kv_cache import BifocalKVCache
    cache = BifocalKVCache(model.config, ids.shape[1] + n, device="cuda", dtype=torch.bfloat16)
    for lo in range(0, ids.shape[1], chunk):
        hidden = model.model(input_ids=ids[:, lo: lo + chunk], past_key_values=cache, use_cache=True).last_hidden_state
    toks = []
    for _ in range(n):
        tok = head_ops.token_scores(hidden[:, -1], model.lm_head.weight, top=True).top
        toks.append(int(tok))
        hidden = model.model(input_ids=tok.view(1, 1), past_key_values=cache, use_cache=True).last_hidden_state
    return toks


def _tree_draft(truth, n_prompt, wrong):
    """Drafts of depth 3: the true continuation (if `wrong` is not hit) among false branches, in a mixed order."""
    def draft(ids):
        done = len(ids) - n_prompt
        nxt = truth[done: done + 3]
        tokens, parents = [(ids[-1] + 1) % 128, 5], [-1, 0]
        up = -1
        for i, t in enumerate(nxt):
            t = (t + 1) % 128 if (done + i) % wrong == wrong - 1 else t
            tokens += [t, (t + 3) % 128]
            parents += [up, up]
            up = len(tokens) - 2
        return tokens, parents
    return draft


@torch.inference_mode()
@pytest.mark.parametrize("regrouped", [True, False])
@pytest.mark.parametrize("prompt, chunk, new", [(186, 64, 14), (150, 150, 9)])
def test_drafted_generation_equals_greedy(golden, prompt, chunk, new, regrouped):
    """The tokens do not depend on the drafts — none, right ones, partly wrong ones — across a change of the group size
    (w = 64: G goes 3 -> 4 at 193 tokens), with and without regrouped copies in the cache; right drafts take fewer steps."""
    from jetlm.kernels.kv_cache import BifocalKVCache
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    ids = g["input_ids"].cuda()[:, :prompt]
    want = _greedy(model, ids, new, chunk)
    steps = []
    for draft in (lambda i: ([], []), _tree_draft(want, prompt, 1 << 30), _tree_draft(want, prompt, 3)):
        cache = BifocalKVCache(model.config, 512, device="cuda", dtype=torch.bfloat16, regrouped_far_keys=regrouped)
        got = model.generate_drafted(ids, new, draft, chunk_tokens=chunk, past_key_values=cache)
        assert got.tolist() == [want]
        steps.append(model.drafted_steps)
    assert steps[0] == new - 1 and steps[1] < steps[2] < steps[0], steps
    # the kept rows are those that one-token decoding writes: the caches agree on keys to the rounding of the projections
    n = cache.get_seq_length()
    ref = BifocalKVCache(model.config, 512, device="cuda", dtype=torch.bfloat16)
    for lo in range(0, prompt, chunk):
        model.model(input_ids=ids[:, lo: lo + chunk], past_key_values=ref, use_cache=True)
    for t in want[: n - prompt]:
        model.model(input_ids=torch.tensor([[t]], device="cuda"), past_key_values=ref, use_cache=True)
    for a, b in zip(cache.layers, ref.layers):
        scale = b.keys[:, :n].float().abs().max()
        assert (a.keys[:, :n].float() - b.keys[:, :n].float()).abs().max() <= 16 * HALF * scale
        assert (a.values[:, :n].float() - b.values[:, :n].float()).abs().max() <= 16 * HALF * b.values[:, :n].float().abs().max()


@torch.inference_mode()
def test_drafted_generation_inside_the_window_and_refusals(golden):
    from jetlm.kernels.kv_cache import BifocalKVCache
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    ids = g["input_ids"].cuda()[:, :30]
    model.model.kernels_within_window = True
    want = _greedy(model, ids, 8, 30)
    assert model.generate_drafted(ids, 8, _tree_draft(want, 30, 1 << 30)).tolist() == [want]
    with pytest.raises(ValueError, match="one prompt"):
        model.generate_drafted(ids.repeat(2, 1), 4, lambda i: ([], []))
    with pytest.raises(ValueError, match="parent"):
        model.generate_drafted(ids, 4, lambda i: ([1, 2], [1, -1]))
    with pytest.raises(ValueError, match="token 1 must be in"):
        model.generate_drafted(ids, 4, lambda i: ([1, 128], [-1, 0]))
    small = BifocalKVCache(model.config, 32, device="cuda", dtype=torch.bfloat16)          # whole blocks of 128 rows
    with pytest.raises(RuntimeError, match="capacity"):
        model.generate_drafted(ids, 120, lambda i: ([], []), past_key_values=small)


@torch.inference_mode()
@pytest.mark.parametrize("batch", [1, 2])
def test_score_tokens_equals_the_logits(golden, batch):
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    ids = g["input_ids"].cuda()
    ids = torch.cat([ids[:, i * 7: i * 7 + 150] for i in range(batch)])
    got = model.score_tokens(ids, chunk_tokens=64)
    from jetlm.kernels.kv_cache import BifocalKVCache
    cache = BifocalKVCache(model.config, 256, batch=batch, device="cuda", dtype=torch.bfloat16)
    z = torch.cat([model(input_ids=ids[:, lo: min(lo + 64, 149)], past_key_values=cache, use_cache=True).logits.float()
                   for lo in range(0, 149, 64)], 1)
    want = torch.logsumexp(z, -1) - z.gather(-1, ids[:, 1:, None])[..., 0]
    # the logits were rounded to bf16 once: half a step in the label's and in the largest ones
    assert got.shape == (batch, 149) and (got - want).abs().max() <= 2 * HALF * z.abs().max() + 1e-5
    assert model.score_tokens(ids[:, :1]).shape == (batch, 0)


def test_fused_loss_trains_inside_the_window(golden):
    """fused_loss gives the loss of the logits path to the rounding of its logits, and the same gradients as the same head in
    fp32 torch on the same hidden states; num_items_in_batch and ignored labels follow transformers."""
    g = golden("model_tiny.npz")
    model = _tiny_model(g).train()
    ids = g["input_ids"].cuda()[:, :50]
    labels = ids.clone()
    labels[:, :10] = -100
    out = model(input_ids=ids, labels=labels)
    model.fused_loss = True
    fused = model(input_ids=ids, labels=labels)
    assert fused.logits is None
    assert abs(float(fused.loss.detach() - out.loss.detach())) <= 2 * HALF * float(out.logits.abs().max()) + 1e-5
    summed = model(input_ids=ids, labels=labels, num_items_in_batch=80)
    assert math.isclose(float(summed.loss.detach()), float(fused.loss.detach()) * 40 / 80, rel_tol=1e-5)      # positions 10 .. 49 are counted
    hidden = model.model(input_ids=ids).last_hidden_state
    h = hidden.detach().requires_grad_(True)
    w = model.lm_head.weight.detach().clone().requires_grad_(True)
    shifted = torch.cat([labels[:, 1:], torch.full((1, 1), -100, device="cuda")], 1)
    torch.nn.functional.cross_entropy((h.float() @ w.float().T)[0], shifted[0]).backward()
    fh, = torch.autograd.grad(model._fused_loss(hidden, labels), hidden, retain_graph=True)
    # d logits rounded to bf16, results rounded to bf16: two half-steps of terms that do not cancel to less than 1/16 of their sum
    assert (fh.float() - h.grad.float()).abs().max() <= 32 * HALF * h.grad.float().abs().max()
    model.zero_grad()
    fused.loss.backward()
    grads = {n: p.grad for n, p in model.named_parameters()}
    assert all(x is not None and torch.isfinite(x).all() for x in grads.values())
    model.zero_grad()
    model.fused_loss = False
    model(input_ids=ids, labels=labels).loss.backward()
    for n, p in model.named_parameters():
        a, b = grads[n].double().flatten(), p.grad.double().flatten()
        assert float((a @ b) / (a.norm() * b.norm())) > 0.99, n      # the logits path rounds logits and their gradient
