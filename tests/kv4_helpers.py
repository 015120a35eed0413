"""The 4-bit cache and what reads it, in plain torch: from the definitions, value by value, without the package's kernels."""
from __future__ import annotations

import torch

BF, F64 = torch.bfloat16, torch.float64
GROUP, SPAN = 64, 64


def word_of(channel: int, d: int, keys: bool) -> tuple[int, int]:
    """(32-bit word of a row, shift inside it) of a channel."""
    level, e = channel // 8, channel % 8
    word = (d // 32) * (level % 4) + level // 4 if keys else (d // 64) * (level % 8) + level // 8
    return word, 4 * (e // 2) + 16 * (e % 2)


def places(d: int, keys: bool) -> torch.Tensor:
    """For every channel its 4-bit place (byte * 2 + half) in a row."""
    return torch.tensor([w * 8 + s // 4 for w, s in (word_of(c, d, keys) for c in range(d))])


def quantise(x: torch.Tensor, keys: bool):
    """x [..., d] bf16 -> codes [..., d / 2] uint8, affine [..., d / 64, 2] bf16; fp32 steps, each rounded by itself."""
    d = x.shape[-1]
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).to(BF).float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    code = torch.where(scale > 0, torch.round((g - lo) / safe).clamp(max=15.0), torch.zeros_like(g)).flatten(-2).to(torch.int64)
    flat = torch.zeros_like(code)
    flat[..., places(d, keys).to(x.device)] = code
    return (flat[..., 0::2] + 16 * flat[..., 1::2]).to(torch.uint8), torch.cat([scale, lo], -1).to(BF)


def values(codes: torch.Tensor, affine: torch.Tensor, keys: bool, dtype=F64) -> torch.Tensor:
    """What rows stand for."""
    d = codes.shape[-1] * 2
    flat = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    code = flat[..., places(d, keys).to(codes.device)].to(dtype).unflatten(-1, (-1, GROUP))
    return (affine[..., 1:].to(dtype) + affine[..., :1].to(dtype) * code).flatten(-2)


def stored(x: torch.Tensor, keys: bool, dtype=F64) -> torch.Tensor:
    return values(*quantise(x, keys), keys, dtype)


def turn(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, inter: bool, dtype=F64) -> torch.Tensor:
    """Rotated by the table's angles, in the given type; not rounded to x's."""
    rot = table.shape[1]
    y = x.to(dtype).clone()
    c, s = (t[:, None].to(dtype) for t in table[positions].split(rot // 2, -1))
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = y[..., one].clone(), y[..., two].clone()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    return y


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, seen: torch.Tensor, cap: float = 0.0):
    """q [heads, d] of one KV head, k and v [n, d], seen [n] -> ([heads, d] in fp64, the largest |v| seen)."""
    if not bool(seen.any()):
        return torch.zeros_like(q, dtype=F64), 0.0
    z = q.to(F64) @ k[seen].to(F64).T * scale
    if cap > 0:
        z = cap * torch.tanh(z / cap)
    return torch.softmax(z, -1) @ v[seen].to(F64), float(v[seen].abs().max())


def make_cache(g: torch.Generator, blocks: int, hkv: int, size: int, d: int, v_size: float = 1.0):
    """Codes and affines of random rows in every slot (CPU), in the order of ``ops.KV4Cache``."""
    rows = lambda f: (torch.randn(blocks, hkv, size, d, generator=g) * f).to(BF)
    k = rows(1.0)
    k[..., d // 3] *= 5
    return (*quantise(k, True), *quantise(rows(v_size), False))


def poison(cache, table: torch.Tensor, lens, size: int) -> None:
    """Rows that no sequence has written hold NaN scales and minima and full codes."""
    used = torch.zeros(cache[0].shape[0], size, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(-(-n // size)):
            used[table[b, i], :min(size, n - i * size)] = True
    for t in cache:
        t.transpose(1, 2)[~used] = 255 if t.dtype == torch.uint8 else float("nan")


def block_lists(g: torch.Generator, lens, size: int, width: int | None = None, spare: int = 2):
    need = [-(-n // size) for n in lens]
    pool = torch.randperm(sum(need) + spare, generator=g).tolist()
    table, at = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(pool[at:at + n], dtype=torch.int32)
        at += n
    return table, sum(need) + spare


def context(cache, table: torch.Tensor, b: int, n: int, dtype=F64):
    """Keys and values of a sequence's n tokens, [kv heads, n, d] each."""
    size = cache[0].shape[2]
    blocks = table[b, :-(-n // size)].long()
    k = values(cache[0][blocks], cache[1][blocks], True, dtype).transpose(0, 1).flatten(1, 2)[:, :n]
    return k, values(cache[2][blocks], cache[3][blocks], False, dtype).transpose(0, 1).flatten(1, 2)[:, :n]


def decode(q: torch.Tensor, cache, table: torch.Tensor, lens, scale: float, window: int = -1, cap: float = 0.0, spans=None):
    """([B, heads, d] in fp64, [B, heads] largest |v| that a head reads)."""
    hkv = cache[0].shape[1]
    group = q.shape[1] // hkv
    out, big = torch.zeros(q.shape, dtype=F64), torch.zeros(q.shape[:2], dtype=F64)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        k, v = context(cache, table, b, n)
        t = torch.arange(n)
        for h in range(hkv):
            seen = t >= n - 1 - window if window >= 0 else torch.ones(n, dtype=torch.bool)
            if spans is not None:
                chosen = torch.zeros(-(-n // SPAN), dtype=torch.bool)
                chosen[[s for s in spans[b, h].tolist() if 0 <= s < chosen.numel()]] = True
                seen = chosen[t // SPAN]
            heads = slice(h * group, (h + 1) * group)
            out[b, heads], big[b, heads] = attend(q[b, heads], k[h], v[h], scale, seen, cap)
    return out, big


def assert_decode(got: torch.Tensor, want: torch.Tensor, big: torch.Tensor, what: str = "") -> None:
    """Rounding of the output: half a step of bf16, 2^-8 of the value.  Of a weight p s to fp16: 2^-11 of it, and sum p (s c) <= sum p times the
    spread of a group <= 2 max |v|: 2^-10 max |v|.  Scores: fp32 sums of 256 products at most, good to 2^-14 and with them each weight, twice
    (numerator and sum): 2^-13 max |v|; weights below fp16's normal numbers: 2^-25 each of the greatest's 15 codes, 40000 times at most."""
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bound = want.abs() * 2.0 ** -8 + big[..., None] * (2.0 ** -10 + 2.0 ** -13 + 40000 * 2.0 ** -25)
    worst = ((got - want).abs() / bound.clamp(min=1e-300)).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


def bounds(cache, rows: int = SPAN):
    """bf16 [blocks, kv heads, spans, 2, d] over all rows of every span."""
    k = values(cache[0], cache[1], True, torch.float32).unflatten(2, (-1, SPAN))
    return torch.stack([k.amin(3), k.amax(3)], 3).to(BF)


def select(q: torch.Tensor, summaries: torch.Tensor, table: torch.Tensor, lens, budget: int) -> torch.Tensor:
    hkv = summaries.shape[1]
    group = q.shape[1] // hkv
    per_block = summaries.shape[2]
    out = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        count = -(-n // SPAN) if n > 0 else 0
        for h in range(hkv):
            if count <= budget:
                chosen = list(range(count))
            else:
                s = summaries[table[b, :-(-count // per_block)].long(), h].flatten(0, 1)[:count].to(F64)
                qs = q[b, h * group:(h + 1) * group].to(F64)
                score = torch.maximum(qs[:, None] * s[:, 0], qs[:, None] * s[:, 1]).sum((0, 2)).tolist()
                rest = sorted(range(1, count - 1), key=lambda i: (-score[i], i))
                chosen = sorted([0, count - 1] + rest[:budget - 2])
            out[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out
