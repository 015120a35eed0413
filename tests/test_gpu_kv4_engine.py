"""The engine over a cache in 4 bits beside the oracle model that reads the same 4-bit rows."""
import copy

import pytest
import torch

from mini_vllm_b200.config import Config, SamplingParams
from mini_vllm_b200.engine.engine import Engine
from mini_vllm_b200.executor.context import Context
from mini_vllm_b200 import ops
from mini_vllm_b200.engine.request import Request
from mini_vllm_b200.models.layers.attention import FlashAttention
from mini_vllm_b200.models.layers.rotary import build_cos_sin_cache
from mini_vllm_b200.workloads import generator, randint
from oracle import rope_kv
from oracle import attention as oattn
from oracle.model import OracleModel, reference_names
from tests import kv4_helpers as kh
from tests.helpers import assert_close_attn
from tests.test_gpu_engine import small_gemma3, small_qwen3

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rows_of(cache: ops.KV4Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    at = (slots.long() // cache.block_size, slice(None), slots.long() % cache.block_size)
    return (kh.values(cache.k_codes[at], cache.k_affine[at], True, torch.float32), kh.values(cache.v_codes[at], cache.v_affine[at], False, torch.float32))


class Twin:
    """An engine over given tokens beside the oracle model.  Quantising is a step function, so that two bf16 neighbours may get codes one
    apart: the oracle's cache takes the engine's own rows, which have to be within half a code (and the scale's rounding over 15 of
    them) of the oracle's, plus what bf16 arithmetic of the layers below may differ by, and all attention reads the same values."""

    def __init__(self, monkeypatch, family, shape, scaling=None, **extra):
        self.cfg = Config(hf_config=shape, kv_cache_num_blocks=40, max_num_batched_seqs=8, max_num_batched_tokens=2048, gpu_memory_utilization=0.3, seed=3,
                          kv_cache_bits=4, **extra)
        self.engine = Engine(self.cfg)
        self.layers = self.engine.executor.attention_layers
        weights = reference_names({k: v.detach() for k, v in self.engine.executor.model.state_dict().items()}, family, self.cfg.hf_config)
        if scaling is not None:
            monkeypatch.setattr(rope_kv, "cos_sin_table", lambda d, n, theta: build_cos_sin_cache(d, n, theta, scaling=scaling))
        self.model = OracleModel(weights, self.cfg.hf_config, family, self.cfg.kv_cache_num_blocks, 256, device=self.engine.executor.device)
        for name in ("k_cache", "v_cache"):
            setattr(self.model, name, [c.float() for c in getattr(self.model, name)])
        plain = oattn.prefill

        def store(k, v, k_cache, v_cache, slots):
            layer = next(i for i, c in enumerate(self.model.k_cache) if c is k_cache)
            for x, cache, rows in zip((k, v), (k_cache, v_cache), rows_of(self.layers[layer].kv4, slots)):
                g, y = x.float().unflatten(-1, (-1, 64)), rows.unflatten(-1, (-1, 64))
                spread, size = g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True), g.abs().amax(-1, keepdim=True)
                assert ((g - y).abs() <= spread / 15 * (0.5 + 16 * 2.0 ** -8) + size * 2.0 ** -5).all()
                cache.view(-1, *cache.shape[2:])[slots.long()] = rows

        def prefill(q, k, v, cu_q, cu_k, table, scale, window):
            return plain(q, k.to(BF), v.to(BF), cu_q, cu_k, table, scale, window)     # prompts read rows unpacked to bf16, single tokens the values

        monkeypatch.setattr(rope_kv, "store_kvcache", store)
        monkeypatch.setattr(oattn, "prefill", prefill)
        self.requests, self.steps, self.exact = {}, 0, 0

    def step(self, entries, g):
        """entries: (name, number of new tokens)."""
        new = {name: torch.randint(0, 2048, (n,), generator=g).tolist() for name, n in entries}
        got = self.engine.replay_step([(self.requests.setdefault(name, Request([])), new[name], [n - 1]) for name, n in entries])
        self.engine.executor.check_device_status()
        dev = self.engine.executor.device
        for row, (name, n) in enumerate(entries):
            r = self.requests[name]
            total = len(r.tokens)
            p = torch.arange(total - n, total, device=dev)
            table = torch.tensor([r.blocks], dtype=torch.int32, device=dev)
            ctx = {"prefill": n > 1, "slot_mapping": (table[0, p // 256] * 256 + p % 256).int(), "block_table": table,
                   "cu_seqlens_q": torch.tensor([0, n], dtype=torch.int32, device=dev), "cu_seqlens_k": torch.tensor([0, total], dtype=torch.int32, device=dev),
                   "cache_seqlens": torch.tensor([total], dtype=torch.int32, device=dev)}
            want = self.model.forward(ctx, torch.tensor(new[name], device=dev), p)[0].float()
            chosen = int(got[row].argmax())
            worst = (want.max() - want[chosen]) / want.max().abs().clamp_min(1.0)
            assert worst <= 4 * 2 ** -8, f"{name} after {total} tokens: {float(worst):.4f}"          # as for the 16-bit cache
            self.steps += 1
            self.exact += chosen == int(want.argmax())

    def run(self, seed=5, singles=12):
        g = generator(seed)
        self.step([("a", 300), ("b", 40), ("c", 257)], g)           # prompts
        self.step([("a", 90), ("d", 600)], g)                       # a portion behind cached tokens, and a prompt
        self.step([("b", 1), ("e", 70), ("c", 1)], g)               # a mixed step
        for _ in range(singles):
            self.step([(name, 1) for name in "abcde"], g)
        assert self.exact >= 0.95 * self.steps


@pytest.mark.parametrize("family,shape,graphs", [("qwen3", small_qwen3, True), ("qwen3", small_qwen3, False), ("gemma3", small_gemma3, True)])
def test_engine_beside_the_oracle(cuda, monkeypatch, family, shape, graphs):
    Twin(monkeypatch, family, shape(), use_cuda_graph=graphs).run()


def test_stand_alone_norms(cuda, monkeypatch):
    Twin(monkeypatch, "qwen3", small_qwen3(), fuse_qk_norm=False).run(singles=3)


def test_spans_that_cover_everything(cuda, monkeypatch):
    """Contexts of at most 12 spans: a selection of 12 of them reads all."""
    twin = Twin(monkeypatch, "qwen3", small_qwen3(), decode_spans=12)
    assert all(m.summaries is not None for m in twin.layers)
    twin.run()


def test_long_contexts_scaled(cuda, monkeypatch):
    """A checkpoint's rope scaling reaches the tables."""
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 256}
    Twin(monkeypatch, "qwen3", small_qwen3(rope_scaling=scaling), scaling=scaling).run(singles=3)


@pytest.mark.parametrize("extra", [{"enable_prefix_cache": True, "kv_cache_num_blocks": 14}, {"enable_mixed_steps": True}, {"enable_chunked_prefill": True, "max_num_batched_tokens": 300},
                                   {"decode_spans": 3}, {"decode_spans": 2, "use_cuda_graph": False}])
def test_generation_under_every_scheduler_option(cuda, extra):
    """Shared prefixes under preemption, mixed steps, prompts in portions, few spans: whole answers, no bad index anywhere, twice the same."""
    g = generator(6)
    shared = torch.randint(0, 2048, (512,), generator=g).tolist()
    prompts = [(shared if i % 2 else []) + torch.randint(0, 2048, (int(n),), generator=g).tolist() for i, n in enumerate(randint(g, 10, 300, 8))]
    params = [SamplingParams(max_tokens=30, ignore_eos=True) for _ in prompts]
    shape = small_gemma3() if extra.get("decode_spans") == 3 else small_qwen3()
    answers = []
    for _ in range(2):
        engine = Engine(Config(hf_config=shape, max_num_batched_seqs=6, gpu_memory_utilization=0.3, seed=4, kv_cache_bits=4,
                               **{"max_num_batched_tokens": 2048, "kv_cache_num_blocks": 40, **extra}))
        out = engine.generate(prompts, copy.deepcopy(params), use_tqdm=False)
        engine.executor.check_device_status()
        answers.append([o["tokens"] for o in out])
    assert all(len(t) == 30 and min(t) >= 0 for t in answers[0]) and answers[0] == answers[1]


def test_four_bits_make_room_for_more_blocks(cuda):
    blocks = lambda bits: Engine(Config(hf_config=small_qwen3(), kv_cache_num_blocks=10 ** 8, gpu_memory_utilization=0.05, use_cuda_graph=False, kv_cache_bits=bits,
                                        max_num_batched_seqs=2)).config.kv_cache_num_blocks
    few, many = blocks(16), blocks(4)
    assert 3.3 < many / few < 3.7                                   # 16 bits against 4.5


def test_models_that_are_refused(cuda):
    with pytest.raises(ValueError, match="kv_cache_bits=4"):
        Engine(Config(hf_config=_odd_heads(), kv_cache_num_blocks=8, gpu_memory_utilization=0.2, kv_cache_bits=4, use_cuda_graph=False))


def _odd_heads():
    cfg = small_qwen3()
    cfg.num_attention_heads, cfg.num_key_value_heads = 10, 1        # ten query heads to a KV head
    return cfg


def test_layer_mixed_step(cuda):
    """One layer: prompts behind cached tokens and single tokens in one step, and the reference's unrotated entry."""
    g, hq, hkv, d, size = generator(9), 4, 2, 128, 256
    lens, cached = [300, 40, 257, 90], [256, 0, 256, 89]            # the last two decode
    table, blocks = kh.block_lists(g, lens, size)
    layer = FlashAttention(hq, d, d ** -0.5, hkv)
    layer.kv4 = ops.KV4Cache.empty(blocks, size, hkv, d, cuda)
    k, v = ([torch.randn(n, hkv, d, generator=g).to(BF) for n in lens] for _ in range(2))
    slot = lambda b, a, n: table[b, torch.arange(a, n) // size] * size + torch.arange(a, n) % size
    for b, n in enumerate(cached):
        if n:
            ops.rotary_kv4_write(None, k[b][:n].to(cuda), v[b][:n].to(cuda), None, None, slot(b, 0, n).int().to(cuda), layer.kv4)
    q = torch.randn(sum(n - c for n, c in zip(lens, cached)), hq, d, generator=g).to(BF)
    cu = lambda xs: torch.tensor([0] + list(torch.tensor(xs).cumsum(0)), dtype=torch.int32, device=cuda)
    new = [n - c for n, c in zip(lens, cached)]
    ctx = Context(prefill=True, num_decode=2, cu_seqlens_q=cu(new), cu_seqlens_k=cu(lens), max_seqlen_q=max(new[:2]), block_table=table.to(cuda),
                  slot_mapping=torch.cat([slot(b, c, n) for b, (c, n) in enumerate(zip(cached, lens))]).int().to(cuda),
                  cache_seqlens=torch.tensor(lens[2:], dtype=torch.int32, device=cuda), prompt_keys=sum(lens[:2]), status=ops.new_status(cuda))
    cut = lambda xs: torch.cat([x[c:] for x, c in zip(xs, cached)]).to(cuda)
    out = layer(ctx, q.to(cuda), cut(k), cut(v))
    ops.check_status(ctx.status)
    at = 0
    for b, n in enumerate(lens):
        ks, vs = (kh.stored(x[b], keys, torch.float32) for x, keys in ((k, True), (v, False)))
        want = oattn.prefill(q[at:at + new[b]], ks, vs, torch.tensor([0, new[b]]), torch.tensor([0, n]))
        assert_close_attn(out[at:at + new[b]], want, f"sequence {b}")
        at += new[b]
