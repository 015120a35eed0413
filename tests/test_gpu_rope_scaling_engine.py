"""The engine on positions that only a scaled rotation reaches."""
import pytest

from mini_vllm_b200.config import Config, SamplingParams
from mini_vllm_b200.engine.engine import Engine
from tests.test_gpu_engine import small_qwen3
from tests.test_gpu_kv4_engine import Twin

pytestmark = pytest.mark.gpu
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 256}


def trained_on_256(scaling=None):
    shape = small_qwen3(**({} if scaling is None else {"rope_scaling": dict(scaling)}))
    shape.max_position_embeddings = 256
    return shape


@pytest.mark.parametrize("extra", [{}, {"decode_spans": 12}])
def test_contexts_past_the_trained_length(cuda, monkeypatch, extra):
    """Up to 600 tokens beside the oracle model, all of a context's spans chosen among the rest."""
    Twin(monkeypatch, "qwen3", trained_on_256(YARN), scaling=YARN, **extra).run(singles=3)


@pytest.mark.parametrize("bits", [16, 4])
def test_generation_past_the_trained_length_and_past_the_tables(cuda, bits):
    engine = Engine(Config(hf_config=trained_on_256(YARN), kv_cache_num_blocks=16, max_num_batched_seqs=2, max_num_batched_tokens=2048, gpu_memory_utilization=0.2,
                           kv_cache_bits=bits))
    out = engine.generate([[7] * 500, [9] * 1000], SamplingParams(max_tokens=25, ignore_eos=True), use_tqdm=False)
    assert [len(o["tokens"]) for o in out] == [25, 25]
    with pytest.raises(ValueError, match="1024 positions"):
        engine.generate([[7] * 1000], SamplingParams(max_tokens=26, ignore_eos=True), use_tqdm=False)
    with pytest.raises(ValueError, match="4096 positions"):
        Engine(Config(hf_config=small_qwen3(), kv_cache_num_blocks=20, max_num_batched_seqs=2, gpu_memory_utilization=0.2, use_cuda_graph=False,
                      kv_cache_bits=bits)).submit([7] * 4097, SamplingParams(max_tokens=1))
