"""Rotation tables for long contexts, the 4-bit cache's handle, and every refusal that needs no GPU."""
import ctypes

import pytest
import torch

from mini_vllm_b200 import _cabi, ops
from mini_vllm_b200.config import Config, qwen3_shape
from mini_vllm_b200.config.config import _flatten_hf
from mini_vllm_b200.models.layers.rotary import build_cos_sin_cache, scaled_frequencies
from tests import kv4_helpers as kh

A = 1 << 20                                          # an address that no call below follows


def cache_struct(blocks=8, size=256, hkv=2, d=128, **other):
    s = _cabi.KV4Cache(A, A, A, A, blocks, size, hkv, d)
    for name, v in other.items():
        setattr(s, name, v)
    return ctypes.byref(s)


# ---- tables ---------------------------------------------------------------------------------------------------------------------------
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 8192}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}


@pytest.mark.parametrize("scaling,head_dim,partial", [(YARN, 128, 1.0), ({**YARN, "beta_fast": 16, "beta_slow": 2}, 64, 1.0), (LLAMA3, 128, 1.0),
                                                      ({"rope_type": "linear", "factor": 4.0}, 128, 0.5), ({**YARN, "truncate": False}, 128, 1.0),
                                                      ({**YARN, "mscale": 1.0, "mscale_all_dim": 0.707}, 64, 1.0), ({**YARN, "attention_factor": 1.5}, 64, 1.0)])
def test_frequencies_are_those_of_hugging_face(scaling, head_dim, partial):
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=4 * head_dim, num_attention_heads=4, head_dim=head_dim, max_position_embeddings=32768)
    cfg.rope_parameters = {**scaling, "rope_theta": 1e6, "partial_rotary_factor": partial}
    want, grow = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    got, factor = scaled_frequencies(int(head_dim * partial), 1e6, scaling)
    assert got.dtype == torch.float64 and abs(factor - grow) < 1e-6
    # theirs is fp32 throughout: the power and two products, each good to a few 2^-24
    assert torch.allclose(got, want.double(), rtol=2 ** -20, atol=0)


def test_frequencies_default_and_unknown():
    freq, grow = scaled_frequencies(64, 1e4, {"type": "default"})
    assert grow == 1.0 and torch.equal(freq, 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.double) / 64))
    with pytest.raises(ValueError, match="not supported"):
        scaled_frequencies(64, 1e4, {"rope_type": "dynamic", "factor": 2.0})


def test_table_far_positions_and_growth():
    table = build_cos_sin_cache(128, 40000, 1e6, scaling=YARN)
    freq, grow = scaled_frequencies(128, 1e6, YARN)
    assert table.shape == (40000, 128) and table.dtype == torch.float32 and grow > 1
    angle = 39999 * freq
    assert torch.equal(table[39999], (torch.cat([angle.cos(), angle.sin()]) * grow).float())
    assert torch.allclose(table[:, :64] ** 2 + table[:, 64:] ** 2, torch.full((40000, 64), grow ** 2), rtol=1e-6)
    # without a scaling the table is what it was
    plain = build_cos_sin_cache(128, 64, 1e6)
    inv = 1.0 / (1e6 ** (torch.arange(0, 128, 2, dtype=torch.float) / 128))
    f = torch.einsum("i,j -> ij", torch.arange(64, dtype=torch.float), inv)
    assert torch.equal(plain, torch.cat((f.cos(), f.sin()), -1))


def test_scaling_comes_out_of_a_hugging_face_config():
    from transformers import Qwen3Config
    cfg = Qwen3Config(hidden_size=64, num_attention_heads=4, head_dim=16, num_hidden_layers=1)
    assert not hasattr(_flatten_hf(cfg), "rope_scaling")
    cfg.rope_parameters = {**YARN, "rope_theta": 1e6}
    flat = _flatten_hf(cfg)
    assert flat.rope_scaling["factor"] == 4.0 and flat.rope_theta == 1e6 and flat.rope_scaling["original_max_position_embeddings"] == 8192
    cfg.rope_parameters = {"rope_type": "yarn", "factor": 2.0, "rope_theta": 1e6}
    assert _flatten_hf(cfg).rope_scaling["original_max_position_embeddings"] == cfg.max_position_embeddings
    cfg.rope_parameters = {"rope_type": "dynamic", "factor": 2.0, "rope_theta": 1e6}
    assert not hasattr(_flatten_hf(cfg), "rope_scaling")            # (left out, as it always was)


# ---- configuration and handle ---------------------------------------------------------------------------------------------------------
def test_config_values():
    assert Config(hf_config=qwen3_shape()).kv_cache_bits == 16
    Config(hf_config=qwen3_shape(), kv_cache_bits=4, decode_spans=2)
    for bad in ({"kv_cache_bits": 8}, {"decode_spans": 4}, {"kv_cache_bits": 4, "decode_spans": 1}):
        with pytest.raises(ValueError):
            Config(hf_config=qwen3_shape(), **bad)


def test_cache_handle():
    c = ops.KV4Cache.empty(3, 128, 2, 256, "cpu")
    assert (c.num_blocks, c.block_size, c.num_kv_heads, c.head_dim) == (3, 128, 2, 256)
    size = sum(t.numel() * t.element_size() for t in (c.k_codes, c.k_affine, c.v_codes, c.v_affine))
    assert size == 3 * 128 * ops.KV4Cache.token_bytes(2, 256)
    with pytest.raises(TypeError):
        ops.KV4Cache(c.k_codes, c.k_affine.float(), c.v_codes, c.v_affine)
    with pytest.raises(ValueError):
        ops.KV4Cache(c.k_codes, c.k_affine[:, :, :64], c.v_codes, c.v_affine)
    with pytest.raises(ValueError):
        ops.KV4Cache(c.k_codes[:, :, ::2], c.k_affine[:, :, ::2], c.v_codes[:, :, ::2], c.v_affine[:, :, ::2])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("keys", [True, False])
def test_layout_is_a_permutation_and_values_come_back(d, keys):
    assert sorted(kh.places(d, keys).tolist()) == list(range(d))
    x = torch.randn(5, d, generator=torch.Generator().manual_seed(d)).to(torch.bfloat16)
    y = kh.stored(x, keys)
    g, z = x.double().unflatten(-1, (-1, 64)), y.unflatten(-1, (-1, 64))
    spread = g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)
    # half a code, and the scale's own rounding over 15 codes
    assert ((g - z).abs() <= spread / 15 * (0.5 + 16 * 2.0 ** -8)).all()


def test_layer_refuses_what_four_bits_do_not_serve():
    from mini_vllm_b200.executor.context import Context
    from mini_vllm_b200.models.layers.attention import FlashAttention
    layer = FlashAttention(4, 128, 1.0, 2)
    assert layer.takes_kv4(torch.bfloat16) and not layer.takes_kv4(torch.float32)
    assert not FlashAttention(4, 64, 1.0, 2).takes_kv4(torch.bfloat16) and not FlashAttention(18, 128, 1.0, 2).takes_kv4(torch.bfloat16)
    layer.kv4 = ops.KV4Cache.empty(1, 128, 2, 128, "cpu")
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="block table"):
        layer(Context(prefill=True), x, x, x)
    with pytest.raises(ValueError, match="no norms"):
        layer.forward_fused(Context(prefill=True), x, x, x, torch.zeros(3, dtype=torch.int64), None, norm=(128, 1e-6))
    layer.sinks = torch.zeros(4)
    assert not layer.takes_kv4(torch.bfloat16)
    with pytest.raises(ValueError, match="no sinks"):
        layer(Context(prefill=False), x, x, x)


# ---- refusals at the C entries (nothing is launched: no address is followed) ---------------------------------------------------------------
def test_rotary_refusals():
    f = _cabi.load().mvb_rotary
    call = lambda tokens=4, hq=2, hkv=1, d=64, rot=64, dtype=0, q=A, out=A, pos=A, cs=A, mp=10: f(
        q, 128, A, 64, out, 128, A, 64, pos, cs, mp, tokens, hq, hkv, d, rot, 0, dtype, None, None)
    assert call(tokens=-1) == -1 and call(hq=0, hkv=0) == -1 and call(rot=0) == -1 and call(mp=0) == -1
    assert call(rot=7) == -2 and call(rot=66) == -2 and call(dtype=2) == -2
    assert call(q=None) == -1 and call(out=None) == -1 and call(pos=None) == -1 and call(cs=None) == -1
    assert call(q=A + 1) == -5 and call(dtype=1, q=A + 2) == -5 and call(pos=A + 4) == -5
    assert call(tokens=0) == 0
    assert call(tokens=1 << 30, hq=64) == -2                        # more units than a launch numbers


def test_cache_refusals():
    f = _cabi.load().mvb_kv4_gather
    call = lambda c, n=1, rows=4, width=2, k=A: f(c, A, A, 2, width, n, rows, k, A, None, None)
    assert call(None) == -1 and call(cache_struct(k_codes=None)) == -1 and call(cache_struct(num_blocks=0)) == -1
    assert call(cache_struct(head_dim=96)) == -2 and call(cache_struct(block_size=96)) == -2
    assert call(cache_struct(blocks=1 << 24, size=256)) == -2       # slots past 2^31
    assert call(cache_struct(v_affine=A + 8)) == -5
    assert call(cache_struct(), n=-1) == -1 and call(cache_struct(), width=0) == -1 and call(cache_struct(), k=A + 2) == -5
    assert call(cache_struct(), n=0) == 0 and call(cache_struct(), rows=0) == 0


def test_write_refusals():
    f = _cabi.load().mvb_rotary_kv4_write
    call = lambda c, tokens=4, hq=2, rot=128, cs=A, pos=A, slots=A, k=A, stride=256, mp=9: f(
        A, stride, A, 256, k, 256, A, 256, pos, cs, mp, rot, 0, slots, c, tokens, hq, 0, None, None)
    assert call(cache_struct(), tokens=-1) == -1 and call(cache_struct(), slots=None) == -1 and call(cache_struct(), k=None) == -1
    assert call(cache_struct(), pos=None) == -1 and call(cache_struct(), mp=0) == -1
    assert call(cache_struct(), rot=24) == -2 and call(cache_struct(), rot=144) == -2
    assert call(cache_struct(), stride=252) == -5 and call(cache_struct(), k=A + 8) == -5
    assert call(cache_struct(), tokens=0) == 0


def test_decode_refusals():
    lib = _cabi.load()
    need = lib.mvb_decode_attn4_workspace_bytes(4, 8, 2, 128)
    assert need > 0 and lib.mvb_decode_attn4_workspace_bytes(0, 8, 2, 128) == 0 and lib.mvb_decode_attn4_workspace_bytes(4, 7, 2, 128) == 0
    call = lambda c, n=4, hq=8, window=-1, cap=0.0, spans=None, budget=0, ws=A, size=need, q=A, stride=1024, width=4, tstride=4: lib.mvb_decode_attn4(
        q, stride, c, A, A, tstride, width, spans, budget, n, hq, 1.0, window, cap, 1.0, A, 1024, ws, size, None, None)
    c = cache_struct()
    assert call(c, n=-1) == -1 and call(c, cap=-1.0) == -1 and call(c, cap=float("nan")) == -1 and call(c, tstride=3) == -1
    assert call(c, spans=A) == -1 and call(c, spans=A, budget=4, window=3) == -1 and call(c, ws=None) == -1 and call(c, q=None) == -1
    assert call(c, hq=7) == -2 and call(c, hq=18) == -2 and call(c, n=70000, size=1 << 40) == -2
    assert call(c, stride=1020) == -5 and call(c, q=A + 8) == -5 and call(c, ws=A + 128) == -5
    assert call(c, size=need - 1) == -7
    assert call(c, n=0) == 0


def test_span_refusals():
    lib = _cabi.load()
    assert lib.mvb_kv4_summarise(cache_struct(), A, -1, A, None, None) == -1
    assert lib.mvb_kv4_summarise(cache_struct(), None, 4, A, None, None) == -1
    assert lib.mvb_kv4_summarise(cache_struct(), A, 4, A + 8, None, None) == -5
    assert lib.mvb_kv4_summarise(cache_struct(), A, 0, A, None, None) == 0
    call = lambda n=2, hq=8, hkv=2, d=128, most=4096, budget=4, width=16, bs=256, q=A, tstride=None: lib.mvb_kv4_select(
        q, 1024, A, 8, bs, A, A, width if tstride is None else tstride, width, n, hq, hkv, d, most, budget, A, None, None)
    assert call(budget=1) == -1 and call(n=-1) == -1 and call(most=0) == -1 and call(q=None) == -1 and call(tstride=8) == -1
    assert call(d=96) == -2 and call(hq=9) == -2 and call(hq=18) == -2 and call(bs=96) == -2 and call(n=70000) == -2
    assert call(most=1 << 30, width=1 << 14) == -2                  # more keys than shared memory holds
    assert call(n=0) == 0


def test_wrappers_refuse_cpu_tensors():
    c = ops.KV4Cache.empty(2, 64, 1, 64, "cpu")
    q, k = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    i32, pos = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    table, ws = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(64, dtype=torch.uint8)
    for call in (lambda: ops.rotary(q, k, pos, torch.zeros(4, 64)), lambda: ops.rotary_kv4_write(q, k, k, pos, torch.zeros(4, 64), i32, c),
                 lambda: ops.kv4_gather(c, i32, table, 4), lambda: ops.decode_attn4(q, c, i32, table, 1.0, -1, ws),
                 lambda: ops.kv4_summarise(c, i32, ops.kv4_summaries(c)), lambda: ops.kv4_select(q, ops.kv4_summaries(c), i32, table, 64, 2)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError):
        ops.rotary(None, None, pos, torch.zeros(4, 64))
    with pytest.raises(TypeError):
        ops.rotary(q.half(), None, pos, torch.zeros(4, 64))
