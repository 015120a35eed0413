"""Which layers a cache in 4 bits stands in for, and how much of the pool's memory goes to unpacked contexts (no GPU)."""
from types import SimpleNamespace

import pytest
import torch

from mini_vllm_b200.config import SamplingParams
from mini_vllm_b200.engine.request import Request
from mini_vllm_b200.executor.executor import Executor
from mini_vllm_b200.models.layers.branches import AttentionBranch, alibi_slopes
from mini_vllm_b200.scheduler.batch import Batch
from mini_vllm_b200.scheduler.scheduler import Scheduler

BF = torch.bfloat16


def branch(**kw) -> AttentionBranch:
    return AttentionBranch(4, 2, 128, 128, 128 ** -0.5, None, 0, 128, **kw)


@pytest.mark.parametrize("options", [{"gate": "head"}, {"gate": "head", "norm_eps": 1e-6}, {"norm_eps": 1e-6}, {"row_norm_eps": 1e-6}, {"value_norm_eps": 1e-6},
                                     {"sink": "zero"}, {"slopes": alibi_slopes(4)}, {"window": 64, "keep_first": 4}])
def test_branches_that_are_refused(options):
    """What ``forward_fused`` would refuse at the first prompt is refused when the engine is made."""
    assert not branch(**options).attn.takes_kv4(BF)


@pytest.mark.parametrize("options", [{}, {"gate": "value"}, {"window": 64}, {"softcap": 30.0}, {"in_bias": True, "out_bias": True}, {"keys_are_values": True}])
def test_branches_that_are_taken(options):
    assert branch(**options).attn.takes_kv4(BF) and not branch(**options).attn.takes_kv4(torch.float32)


def test_branches_that_share_keys_are_refused():
    lender = branch()
    assert lender.attn.takes_kv4(BF)
    borrower = branch(source=lender)
    assert not lender.attn.takes_kv4(BF) and not borrower.attn.takes_kv4(BF)


# ---- memory for unpacked contexts ---------------------------------------------------------------------------------------------------------
def pool(room, block_bytes, blocks, batched=64, positions=4096, heads=((2, 128), (1, 256))):
    ex = object.__new__(Executor)
    ex.config = SimpleNamespace(kv_cache_num_blocks=blocks, max_num_batched_tokens=batched)
    ex.block_size, ex.max_positions = 256, positions
    ex.attention_layers = [SimpleNamespace(num_kv_heads=h, head_dim=d) for h, d in heads]
    return ex._kv4_blocks_and_keys(room, block_bytes)


@pytest.mark.parametrize("room", [0, 10 ** 6, 5 * 10 ** 6, 10 ** 7, 10 ** 9])
@pytest.mark.parametrize("positions", [None, 300, 4096])
@pytest.mark.parametrize("batched", [64, 2048])
def test_the_pool_leaves_room_to_unpack(room, positions, batched):
    """As many blocks as fit beside the rows of the longest context, and not one fewer."""
    row, block_bytes, most = 4 * 256, 256 * 300, 500
    blocks, keys = pool(room, block_bytes, most, batched, positions)
    need = lambda n: n * block_bytes + row * max(batched, min(positions or most * 256, n * 256))
    assert blocks == max((n for n in range(most + 1) if need(n) <= room), default=0)
    assert keys == max(batched, min(positions or most * 256, blocks * 256))


def scheduler(keys, prefix=False, batched=64):
    return Scheduler(SimpleNamespace(max_num_batched_seqs=8, max_num_batched_tokens=batched, eos_token_ids=set(), enable_chunked_prefill=True, enable_prefix_cache=prefix,
                                     kv_cache_num_blocks=200, kv_cache_block_size=16, max_prompt_keys=keys))


def drive(sch, prompts):
    """Steps until every prompt has its first token: (context tokens of the step's prompts, their number) of each."""
    reqs = [Request(p, SamplingParams(max_tokens=1, ignore_eos=True)) for p in prompts]
    for r in reqs:
        sch.submit(r)
    steps = []
    while not sch.finished:
        batch = sch.schedule()
        assert batch.type == Batch.PREFILL
        steps.append((sum(r.step_len for r in batch.requests), len(batch.requests)))
        assert sum(r.step_len - r.num_cached_tokens for r in batch.requests) <= sch.max_num_batched_tokens
        sch.update(batch, [1] * len(batch.requests))
    assert all(len(r.tokens) == len(p) + 1 for r, p in zip(reqs, prompts))
    return steps


@pytest.mark.parametrize("prefix", [False, True])
def test_portions_keep_to_the_context_that_can_be_unpacked(prefix):
    shared = list(range(160))
    prompts = [shared + [1000 + i, i] for i in range(7)] + [list(range(5)), list(range(300))]
    free, bound = drive(scheduler(None, prefix), prompts), drive(scheduler(330, prefix), prompts)
    assert all(keys <= 330 for keys, _ in bound)
    if prefix:
        assert max(keys for keys, _ in free) > 700                  # what had to be unpacked at once: the same prefix seven times
    assert any(n > 1 for _, n in bound)
    assert drive(scheduler(10 ** 6, prefix), prompts) == free


def test_one_context_may_always_come():
    steps = drive(scheduler(50), [list(range(200)), list(range(10))])
    assert steps[0] == (64, 1) and max(keys for keys, _ in steps) == 200
