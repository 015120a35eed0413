"""Rope scaling of checkpoints' configurations, from the file to the tables."""
import logging

import pytest
import torch

from mini_vllm_b200.config.config import _flatten_hf
from mini_vllm_b200.models.layers.rotary import build_cos_sin_cache

LINEAR = {"rope_type": "linear", "factor": 8.0}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 256}


def ours(caplog):
    return [r for r in caplog.records if r.name.startswith("mini_vllm_b200")]


def gemma3(**kw):
    from transformers import Gemma3TextConfig
    return Gemma3TextConfig(hidden_size=64, num_attention_heads=4, num_key_value_heads=1, head_dim=16, num_hidden_layers=6, vocab_size=64, **kw)


def qwen3(**kw):
    from transformers import Qwen3Config
    return Qwen3Config(hidden_size=64, num_attention_heads=4, head_dim=16, num_hidden_layers=1, vocab_size=64, **kw)


@pytest.mark.parametrize("make,scaling", [(gemma3, LINEAR), (qwen3, LINEAR), (qwen3, YARN)])
@pytest.mark.parametrize("through_a_file", [False, True])
def test_scaling_of_both_families(make, scaling, through_a_file, tmp_path, caplog):
    cfg = make(rope_scaling=dict(scaling), rope_theta=1e6, max_position_embeddings=2048)
    if through_a_file:
        from transformers import AutoConfig
        cfg.save_pretrained(tmp_path)
        cfg = AutoConfig.from_pretrained(tmp_path)
    with caplog.at_level(logging.WARNING):
        flat = _flatten_hf(cfg)
    assert not ours(caplog)
    assert flat.rope_scaling["rope_type"] == scaling["rope_type"] and flat.rope_scaling["factor"] == scaling["factor"] and flat.rope_theta == 1e6
    assert flat.rope_scaling["original_max_position_embeddings"] == scaling.get("original_max_position_embeddings", 2048)


def test_only_gemmas_layers_without_a_window_are_scaled():
    from mini_vllm_b200.models.models.gemma3 import Gemma3ForCausalLM
    flat = _flatten_hf(gemma3(rope_scaling=dict(LINEAR), rope_theta=1e6, max_position_embeddings=512))
    model = Gemma3ForCausalLM(flat)
    assert torch.equal(model.rotary.cos_sin_cache, build_cos_sin_cache(16, 512, 1e6, scaling=LINEAR))
    assert torch.equal(model.rotary_local.cos_sin_cache, build_cos_sin_cache(16, 512, flat.rope_local_base_freq))
    assert not torch.equal(model.rotary.cos_sin_cache, build_cos_sin_cache(16, 512, 1e6))


def test_what_is_left_out_is_said(caplog):
    plain = _flatten_hf(gemma3())
    assert not hasattr(plain, "rope_scaling") and not hasattr(_flatten_hf(qwen3()), "rope_scaling")
    cfg = gemma3()
    cfg.rope_parameters = {"full_attention": {"rope_type": "dynamic", "factor": 2.0, "rope_theta": 1e6},
                           "sliding_attention": {"rope_type": "linear", "factor": 2.0, "rope_theta": 1e4}}
    with caplog.at_level(logging.WARNING):
        assert not hasattr(_flatten_hf(cfg), "rope_scaling")
    assert len(ours(caplog)) == 2
    cfg.rope_parameters = {"full_attention": {**YARN, "rope_theta": 1e6}, "sliding_attention": {"rope_type": "default", "rope_theta": 1e4}}
    flat = _flatten_hf(cfg)
    assert flat.rope_scaling["factor"] == 4.0 and flat.rope_theta == 1e6 and flat.rope_local_base_freq == 1e4 and len(ours(caplog)) == 2


def test_a_configuration_with_the_older_names():
    from types import SimpleNamespace
    cfg = SimpleNamespace(hidden_size=64, num_attention_heads=4, head_dim=16, rope_theta=1e6, max_position_embeddings=2048,
                          rope_scaling={"type": "linear", "factor": 2.0})
    assert _flatten_hf(cfg).rope_scaling == {"type": "linear", "factor": 2.0, "original_max_position_embeddings": 2048}
