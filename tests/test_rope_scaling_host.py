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


@pytest.mark.parametrize("scaling,most,model_len,want", [(YARN, 256, 4096, 1024), (YARN, 2048, 4096, 2048), ({**YARN, "factor": 2.5}, 100, 64, 640),
                                                         ({"rope_type": "linear", "factor": 4.0}, 512, 4096, 2048),
                                                         ({"rope_type": "linear", "factor": 4.0}, 512, 1500, 1500),
                                                         ({"type": "linear", "factor": 4.0}, 512, 100, 512), (None, 512, 4096, 512),
                                                         ({"rope_type": "default"}, 512, 4096, 512)])
def test_tables_reach_as_far_as_the_scaling(scaling, most, model_len, want):
    from mini_vllm_b200.config import Config, qwen3_shape
    shape = qwen3_shape(num_hidden_layers=1, hidden_size=64, intermediate_size=64, num_attention_heads=4, num_key_value_heads=2, head_dim=16, vocab_size=64,
                        max_position_embeddings=most, **({} if scaling is None else {"rope_scaling": dict(scaling)}))
    for _ in range(2):                                              # the same description twice: the same tables
        cfg = Config(hf_config=shape, max_model_len=model_len).hf_config
        assert cfg.max_position_embeddings == want
    from mini_vllm_b200.models.models.qwen3 import Qwen3ForCausalLM
    table = Qwen3ForCausalLM(cfg).rotary.cos_sin_cache
    assert table.shape == (want, 16)
    assert torch.equal(table[:most], build_cos_sin_cache(16, most, 1e6, scaling=scaling))


def test_a_scaling_that_is_not_known_is_the_models_matter():
    from mini_vllm_b200.config import Config, qwen3_shape
    from mini_vllm_b200.models.models.qwen3 import Qwen3ForCausalLM
    cfg = Config(hf_config=qwen3_shape(rope_scaling={"rope_type": "longrope", "short_factor": [1.0]})).hf_config
    assert cfg.max_position_embeddings == 40960
    with pytest.raises(ValueError, match="not supported"):
        Qwen3ForCausalLM(cfg)


def test_requests_past_the_tables_are_refused():
    from types import SimpleNamespace
    from mini_vllm_b200.config import SamplingParams
    from mini_vllm_b200.engine.engine import Engine

    def engine(limit, eos=()):
        e, taken = Engine.__new__(Engine), []
        e.config = SimpleNamespace(hf_config=None, eos_token_ids=set(eos))
        e.executor, e.scheduler = SimpleNamespace(max_positions=limit), SimpleNamespace(submit=taken.append)
        return e, taken

    e, taken = engine(100)
    e.submit([1] * 91, SamplingParams(max_tokens=10))               # (the last token has no position)
    for prompt, new in ((92, 10), (101, 1), (5, 97)):
        with pytest.raises(ValueError, match="100 positions"):
            e.submit([1] * prompt, SamplingParams(max_tokens=new))
    assert len(taken) == 1
    e, taken = engine(100, eos=[2])
    e.submit([1] * 100, SamplingParams(max_tokens=500))             # may stop in front of it
    for prompt, params in ((101, SamplingParams(max_tokens=1)), (92, SamplingParams(max_tokens=10, ignore_eos=True))):
        with pytest.raises(ValueError, match="100 positions"):
            e.submit([1] * prompt, params)
    assert len(taken) == 1
    e, taken = engine(None)
    e.submit([1] * 1000, SamplingParams(max_tokens=1000))
    assert len(taken) == 1
    with pytest.raises(ValueError, match="100 positions"):          # none of a job's requests is taken then
        e, taken = engine(100)
        e.generate([[1] * 5, [1] * 200], SamplingParams(max_tokens=3))
    assert not taken
