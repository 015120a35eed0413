"""A step's prompts unpack no more context than the executor has kept memory for."""
import pytest
import torch

from mini_vllm_b200 import ops
from mini_vllm_b200.config import Config, SamplingParams
from mini_vllm_b200.engine.engine import Engine
from mini_vllm_b200.workloads import generator
from tests.test_gpu_engine import small_gemma3, small_qwen3

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [small_qwen3, small_gemma3])
def test_portions_behind_long_contexts(cuda, monkeypatch, shape):
    g = generator(11)
    prompts = [torch.randint(0, 2048, (n,), generator=g).tolist() for n in (1500, 1400, 1300, 40, 900, 1200)]
    cfg = Config(hf_config=shape(), kv_cache_num_blocks=64, max_num_batched_seqs=8, max_num_batched_tokens=400, gpu_memory_utilization=0.3, seed=4, kv_cache_bits=4,
                 enable_chunked_prefill=True)
    engine = Engine(cfg)
    assert cfg.max_prompt_keys == 4096 and engine.scheduler.max_prompt_keys == 4096      # the longest context that the tables allow
    engine.scheduler.max_prompt_keys = 1600
    rows, gather = [], ops.kv4_gather
    monkeypatch.setattr(ops, "kv4_gather", lambda cache, cu, table, n, *a, **kw: rows.append(n) or gather(cache, cu, table, n, *a, **kw))
    out = engine.generate(prompts, SamplingParams(max_tokens=5, ignore_eos=True), use_tqdm=False)
    assert all(len(o["tokens"]) == 5 for o in out) and max(rows) <= 1600 and max(rows) > 1400
    heads = max(4 * m.num_kv_heads * m.head_dim for m in engine.executor.attention_layers)
    assert engine.executor._kv4_blocks_and_keys(10 ** 9, engine.executor._kv4_block_bytes()) == (64, 4096)
    tight = 20 * engine.executor._kv4_block_bytes() + 4096 * heads
    blocks, keys = engine.executor._kv4_blocks_and_keys(tight, engine.executor._kv4_block_bytes())
    assert (blocks, keys) == (20, 4096)
