"""Drafted generation with drafts deeper than the near window, and behind a cache that holds tokens already."""
import pytest
import torch

from test_drafted_model_gpu import _greedy
from test_model_gpu import _tiny_model

pytestmark = pytest.mark.gpu


def _chain(truth, n_prompt, depth, branch):
    """The true continuation `depth` tokens deep, with a false token beside every one that a child hangs on."""
    def draft(ids):
        nxt = truth[len(ids) - n_prompt:][:depth]
        tokens, parents, up = [], [], -1
        for t in nxt:
            if branch:
                tokens.append((t + 5) % 128)
                parents.append(up)
            tokens.append(t)
            parents.append(up)
            up = len(tokens) - 1
        return tokens, parents
    return draft


@torch.inference_mode()
@pytest.mark.parametrize("regrouped", [True, False])
@pytest.mark.parametrize("branch", [True, False])
def test_drafts_deeper_than_the_near_window(golden, regrouped, branch):
    """w_0 = 16 and chains of 40: drafted keys are in the far class of the nodes at their end."""
    from jetlm.kernels.kv_cache import BifocalKVCache
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    w_0 = model.model.rotary_emb.jetlong_w_0
    depth = w_0 + 24
    ids = g["input_ids"].cuda()[:, :130]
    want = _greedy(model, ids, depth + 6, 130)
    cache = BifocalKVCache(model.config, 512, device="cuda", dtype=torch.bfloat16, regrouped_far_keys=regrouped)
    got = model.generate_drafted(ids, depth + 6, _chain(want, 130, depth, branch), past_key_values=cache)
    assert got.tolist() == [want] and model.drafted_steps <= 3


@torch.inference_mode()
def test_a_cache_that_holds_tokens_and_one_that_ends_with_the_last_token(golden):
    from jetlm.kernels.kv_cache import BifocalKVCache
    g = golden("model_tiny.npz")
    model = _tiny_model(g)
    ids = g["input_ids"].cuda()[:, :120]
    want = _greedy(model, ids, 9, 60)
    # 120 prompt tokens and 8 of the 9 new ones are the 128 rows of the smallest cache: the last step's places end at its last row
    cache = BifocalKVCache(model.config, 128, device="cuda", dtype=torch.bfloat16)
    model.model(input_ids=ids[:, :60], past_key_values=cache, use_cache=True)
    got = model.generate_drafted(ids[:, 60:], 9, _chain(want, 60, 3, True), past_key_values=cache)
    assert got.tolist() == [want] and cache.get_seq_length() == 128
