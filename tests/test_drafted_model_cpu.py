"""Refusals of the model's drafted generation that are made before a kernel runs."""
import pytest
import torch

from test_model_surface_cpu import _make_model_dir


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    from transformers import AutoConfig
    from jetlm.modeling.jetlong_fused import Qwen3JetLongFusedForCausalLM
    d = _make_model_dir(tmp_path_factory.mktemp("model"))
    return Qwen3JetLongFusedForCausalLM(AutoConfig.from_pretrained(str(d), trust_remote_code=True)).eval()


def _draft(ids):
    raise AssertionError("no draft is asked for")


@pytest.mark.parametrize("rank", [0, 1])
def test_sharded_caches_are_refused(model, rank):
    from jetlm.kernels.kv_cache import BifocalKVCache
    from jetlm.kernels.sequence_parallel import SequenceShard
    cache = BifocalKVCache(model.config, 64, dtype=torch.float32, shard=SequenceShard(rank, 2, 16))
    with pytest.raises(ValueError, match="must not be sharded"):
        model.generate_drafted(torch.zeros(1, 8, dtype=torch.long), 4, _draft, past_key_values=cache)
    assert cache.get_seq_length() == 0


def test_other_caches_are_refused(model):
    from transformers import DynamicCache
    with pytest.raises(TypeError, match="BifocalKVCache"):
        model.generate_drafted(torch.zeros(1, 8, dtype=torch.long), 4, _draft, past_key_values=DynamicCache(config=model.config))
