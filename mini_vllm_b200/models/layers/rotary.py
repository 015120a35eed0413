"""Rotary position embedding table (the rotation itself is fused into the KV-write kernel).

The table is built exactly as ``minivllm/models/layers/rotary.py:32-47`` builds it — fp32,
``[max_position_embeddings, rotary_dim] = cat(cos, sin)`` — but always on the CPU, then moved:
``cos``/``sin`` can differ by an ulp between devices, and bit-exact KV contents need the one
table everywhere.  ``forward`` keeps the reference signature and runs the CUDA kernel with the
cache write disabled.
"""
from __future__ import annotations

import math

import torch
from torch import nn

from ... import ops


def scaled_frequencies(rotary_dim: int, rope_theta: float, scaling: dict) -> tuple[torch.Tensor, float]:
    """(radians per position of every pair, fp64 on the CPU; the factor of the rotated vectors' length) for contexts beyond the trained one.

    ``scaling`` as Hugging Face configurations have it, ``rope_type`` (or ``type``) being

    * ``default``: as trained;
    * ``linear``: every position counts as ``1 / factor``;
    * ``yarn``: pairs that turn less than ``beta_slow`` times over ``original_max_position_embeddings`` are slowed by ``factor``, those that turn
      more than ``beta_fast`` times stay, a ramp over the pairs' numbers between; vectors grow by ``attention_factor``, or by ``g(1)`` with
      ``g(m) = 0.1 m ln(factor) + 1``, or by ``g(mscale) / g(mscale_all_dim)`` where both are given; ``truncate`` False: the ramp's ends are not rounded;
    * ``llama3``: pairs with wavelengths above ``original / low_freq_factor`` are slowed by ``factor``, those below ``original /
      high_freq_factor`` stay, blended by the wavelength between.
    """
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    freq = rope_theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.double, device="cpu") / max(rotary_dim, 1))
    if kind == "default":
        return freq, 1.0
    if kind not in ("linear", "yarn", "llama3"):
        raise ValueError(f"rope scaling of type {kind!r} is not supported (default, linear, yarn, llama3)")
    factor = float(scaling["factor"])
    if kind == "linear":
        return freq / factor, 1.0
    trained = float(scaling["original_max_position_embeddings"])
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = trained * freq / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return freq / factor * (1 - keep) + freq * keep, 1.0
    pair = lambda turns: rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(rope_theta))   # the pair that turns so often
    whole = scaling.get("truncate", True)                    # the ramp goes from pair to pair
    low, high = pair(float(scaling.get("beta_fast") or 32)), pair(float(scaling.get("beta_slow") or 1))
    low, high = max(math.floor(low) if whole else low, 0), min(math.ceil(high) if whole else high, rotary_dim - 1)
    slowed = ((torch.arange(rotary_dim // 2, dtype=torch.double, device="cpu") - low) / max(high - low, 0.001)).clamp(0, 1)
    grow = scaling.get("attention_factor")
    if grow is None:
        growth = lambda m: 0.1 * m * math.log(factor) + 1 if factor > 1 else 1.0
        m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        grow = growth(float(m)) / growth(float(m_all)) if m and m_all else growth(1.0)
    return freq / factor * slowed + freq * (1 - slowed), float(grow)


def build_cos_sin_cache(rotary_dim: int, max_position_embeddings: int, rope_theta: float,
                        head_dim: int | None = None, scaling: dict | None = None) -> torch.Tensor:
    """``scaling``: frequencies for long contexts (``scaled_frequencies``); the angles are then exact to fp32 rounding at any position, and
    the vectors' growth is in the table.  ``head_dim`` larger than ``rotary_dim``: the pairs past the rotated ones keep angle 0 (cos 1, sin 0), for heads
    whose rotated coordinates ``i`` and ``i + rotary_dim/2`` have been laid out at ``i`` and ``i + head_dim/2``."""
    # the plain table is built in fp32 as the reference builds it; a table with a layout of its own has nothing to match
    # and is exact to fp32 rounding at any position
    work = torch.float if head_dim is None and scaling is None else torch.double
    grow = 1.0
    if scaling is None:
        exponent = torch.arange(0, rotary_dim, 2, dtype=work, device="cpu") / max(rotary_dim, 1)
        inv_freq = 1.0 / (rope_theta ** exponent)
    else:
        inv_freq, grow = scaled_frequencies(rotary_dim, rope_theta, scaling)
    t = torch.arange(max_position_embeddings, dtype=work, device="cpu")
    freqs = torch.einsum("i,j -> ij", t, inv_freq)
    rest = 0 if head_dim is None else head_dim // 2 - rotary_dim // 2
    freqs = torch.cat((freqs, freqs.new_zeros(freqs.shape[0], rest)), dim=-1)
    table = torch.cat((freqs.cos(), freqs.sin()), dim=-1)
    return (table if grow == 1.0 else table * grow).float()


class RotaryEmbedding(nn.Module):
    def __init__(self, rotary_dim: int, max_position_embeddings: int, rope_theta: float, device=None,
                 head_dim: int | None = None, scaling: dict | None = None, interleaved: bool = False) -> None:
        super().__init__()
        self.interleaved = interleaved          # pairs (2i, 2i + 1) instead of halves
        self.rotary_dim = rotary_dim
        self.max_position_embeddings = max_position_embeddings
        self.rope_theta = rope_theta
        cache = build_cos_sin_cache(rotary_dim, max_position_embeddings, rope_theta, head_dim, scaling)
        self.register_buffer("cos_sin_cache", cache.to(device) if device is not None else cache, persistent=False)

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor):
        """Rotate ``query [T,Hq,D]`` and ``key [T,Hkv,D]`` in place and return them."""
        if self.interleaved or query.dtype != torch.bfloat16 or self.cos_sin_cache.shape[1] != query.shape[2]:
            return ops.rotary(query, key, positions, self.cos_sin_cache, interleaved=self.interleaved)
        ops.rope_kv_write(query, key, key, positions, self.cos_sin_cache, None, None, None, k_in_place=True)
        return query, key
