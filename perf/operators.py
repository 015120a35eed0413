"""Operators around a paged cache of keys and values held in 4 bits, as this package's users call them, with their plain forms.

A case is a dict of plain values; ``op`` names the operator:

  rotary   rotation of queries and keys by position, in either pairing and for part of the head (``ops.rotary``)
  write    a step's queries rotated, its keys rotated and quantised with the values into the cache, and the sequences' whole contexts
           unpacked as the prompt kernel reads them (``ops.rotary_kv4_write``, ``ops.kv4_gather``)
  decode   attention of one new token per sequence over the cache (``ops.decode_attn4``)
  sparse   the same over a few spans of 64 tokens: the bounds of the spans just written renewed, the spans chosen for every sequence and
           KV head, attention over them (``ops.kv4_summarise``, ``ops.kv4_select``, ``ops.decode_attn4``)

Cache, per layer, for keys and for values: 4-bit codes ``[blocks, kv heads, 256, dim / 2]`` (uint8) and, for each group of 64 channels of
a row, a bf16 (scale, minimum) ``[blocks, kv heads, 256, dim / 64, 2]``; a code c stands for ``minimum + scale * c``.  With m and M a
group's least and greatest value: minimum m, scale bf16((M - m) * fp32(1/15)), code round((x - m) / scale) held to 0..15.

Sizes are those of the repository's shapes: 16 query heads of 128 with 8 KV heads, 32 with 8, or 4 of 256 with one; blocks of 256.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK, SPAN, GROUP = 256, 64, 64
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF, "fp32": F32}


def listed() -> list[dict]:
    return [
        # the smallest call: one conversation's new token of a small model with an odd head size, a quarter of it rotated, in fp32
        {"name": "rotary_token", "op": "rotary", "tokens": 1, "hq": 12, "hkv": 4, "dim": 80, "rot": 20, "inter": True, "type": "fp32", "scaling": "none"},
        # a decode step of many conversations, positions far beyond the trained length
        {"name": "rotary_step", "op": "rotary", "tokens": 256, "hq": 16, "hkv": 8, "dim": 128, "rot": 128, "inter": False, "type": "bf16", "scaling": "yarn"},
        # the prompts of one step, half of the head rotated by neighbouring pairs
        {"name": "rotary_prompts", "op": "rotary", "tokens": 16384, "hq": 32, "hkv": 8, "dim": 128, "rot": 64, "inter": True, "type": "bf16", "scaling": "linear"},
        # a few short requests that join
        {"name": "write_short", "op": "write", "seqs": 5, "low": 1, "high": 9, "prefix": 0, "hq": 8, "hkv": 2, "dim": 64, "rot": 32, "inter": True, "scaling": "none"},
        # the prompts of one step, ragged, behind an instruction that the cache holds already
        {"name": "write_prompts", "op": "write", "seqs": 16, "low": 100, "high": 2048, "prefix": 500, "hq": 16, "hkv": 8, "dim": 128, "rot": 128, "inter": False, "scaling": "yarn"},
        # the next portion of long documents, heads of 256
        {"name": "write_portions", "op": "write", "seqs": 4, "low": 1024, "high": 1024, "prefix": 6000, "hq": 4, "hkv": 1, "dim": 256, "rot": 256, "inter": False, "scaling": "linear"},
        # one conversation's next token: latency
        {"name": "decode_one", "op": "decode", "seqs": 1, "low": 700, "high": 700, "hq": 16, "hkv": 8, "dim": 128, "window": -1, "cap": 0.0},
        # one long document
        {"name": "decode_document", "op": "decode", "seqs": 1, "low": 40951, "high": 40951, "hq": 32, "hkv": 8, "dim": 128, "window": -1, "cap": 0.0},
        # a step of many conversations, ragged: the largest call
        {"name": "decode_batch", "op": "decode", "seqs": 240, "low": 128, "high": 8192, "hq": 16, "hkv": 8, "dim": 128, "window": -1, "cap": 0.0},
        # the layers with a window of the 256-wide heads, scores capped
        {"name": "decode_window", "op": "decode", "seqs": 128, "low": 200, "high": 4096, "hq": 4, "hkv": 1, "dim": 256, "window": 512, "cap": 30.0},
        # a few long documents, 32 spans of each
        {"name": "sparse_documents", "op": "sparse", "seqs": 4, "low": 9000, "high": 40000, "hq": 32, "hkv": 8, "dim": 128, "budget": 32},
        # a step of many long conversations
        {"name": "sparse_batch", "op": "sparse", "seqs": 96, "low": 1000, "high": 16000, "hq": 16, "hkv": 8, "dim": 128, "budget": 16},
    ]


def _log(rng, low, high) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["rotary", "write", "decode", "decode", "sparse"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _log(rng, 1, 4096), "hq": hkv * rng.choice([1, 2, 3, 4]), "hkv": hkv, "dim": dim,
                "rot": 2 * rng.randint(1, dim // 2) if rng.random() < 0.4 else rng.choice([dim, dim // 2]), "inter": rng.random() < 0.5,
                "type": rng.choice(["bf16", "bf16", "fp32"]), "scaling": rng.choice(["none", "linear", "yarn"])}
    hq, hkv, dim = rng.choice([(16, 8, 128), (16, 8, 128), (32, 8, 128), (4, 1, 256), (8, 2, 64), (6, 2, 128), (5, 5, 128), (7, 1, 64)])
    if op == "write":
        seqs = _log(rng, 1, 32)
        high = _log(rng, 1, 12288 // seqs)
        return {"op": op, "seqs": seqs, "low": _log(rng, 1, high), "high": high, "prefix": rng.choice([0, 0, 1, 255, 512, 700]), "hq": hq, "hkv": hkv,
                "dim": dim, "rot": 16 * rng.randint(1, dim // 16) if rng.random() < 0.5 else dim, "inter": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "yarn"])}
    seqs = _log(rng, 1, 200)
    if op == "decode":
        high = _log(rng, 1, min(40000, 400000 // seqs))
        window, cap = rng.choice([(-1, 0.0), (-1, 0.0), (-1, 50.0), (0, 0.0), (100, 0.0), (1024, 30.0)])
        return {"op": op, "seqs": seqs, "low": _log(rng, 1, high), "high": high, "hq": hq, "hkv": hkv, "dim": dim, "window": window, "cap": cap}
    high = _log(rng, 1, min(40000, 400000 // seqs))
    return {"op": op, "seqs": seqs, "low": _log(rng, 1, high), "high": high, "hq": hq, "hkv": hkv, "dim": dim, "budget": rng.choice([2, 5, 16, 33, 64])}


def _lens(case) -> list[int]:
    """A case's lengths follow from its own numbers; the shortest and the longest are among them."""
    rng = random.Random("%d/%d/%d" % (case["seqs"], case["low"], case["high"]))
    lens = [_log(rng, case["low"], case["high"]) for _ in range(case["seqs"])]
    lens[0] = case["high"]
    if len(lens) > 1:
        lens[-1] = case["low"]
    return lens


def _visible(case) -> list[int]:
    """Tokens that each sequence's query reads."""
    if case["op"] == "sparse":
        return [min(n, case["budget"] * SPAN) for n in _lens(case)]
    return [n if case["window"] < 0 else min(n, case["window"] + 1) for n in _lens(case)]


def work(case) -> dict:
    """Inputs read once and outputs written once; multiplications and additions apart."""
    d, hq, hkv = case["dim"], case["hq"], case["hkv"]
    if case["op"] == "rotary":
        t, size = case["tokens"], TYPES[case["type"]].itemsize
        return {"bytes": t * (2 * (hq + hkv) * d * size + case["rot"] * 4 + 8), "flops": t * (hq + hkv) * case["rot"] * 3}
    row = 2 * (d // 2 + d // GROUP * 4)                     # a token's key and value of one head in the cache
    if case["op"] == "write":
        new, all_ = sum(_lens(case)), sum(n + case["prefix"] for n in _lens(case))
        step = new * ((2 * hq + 2 * hkv) * d * 2 + hkv * row + case["rot"] * 4 + 12)
        return {"bytes": step + all_ * hkv * (row + 4 * d), "flops": new * ((hq + hkv) * case["rot"] * 3 + hkv * d * 8) + all_ * hkv * d * 4}
    seen = sum(_visible(case))
    total = {"bytes": seen * hkv * row + 2 * case["seqs"] * hq * d * 2, "flops": 4 * seen * hq * d}
    if case["op"] == "sparse":
        spans = sum(-(-n // SPAN) for n in _lens(case) if -(-n // SPAN) > case["budget"])     # bounds that have to be looked at
        total["bytes"] += spans * hkv * 4 * d + case["seqs"] * hkv * (SPAN // 2 * row // 2 + 4 * d + 4 * case["budget"])
        total["flops"] += spans * hq * d * 3
    return total


# ---- layout -------------------------------------------------------------------------------------------------------------------------
def _order(dim: int, keys: bool, device) -> torch.Tensor:
    """The channel that each 4-bit place of a row holds.  A 32-bit word holds channels 8L .. 8L + 7, the even ones in its low half; word
    (dim / 32) c + j is L = 4 j + c for keys (c < 4), word (dim / 64) g + j is L = 8 j + g for values (g < 8)."""
    words, inside = dim // 8, [0, 2, 4, 6, 1, 3, 5, 7]
    order = []
    for p in range(words):
        per = words // 4 if keys else words // 8
        first, j = divmod(p, per)
        order += [8 * ((4 if keys else 8) * j + first) + e for e in inside]
    return torch.tensor(order, device=device)


def _quantise(x: torch.Tensor, keys: bool):
    """x [..., dim] bf16 -> (codes [..., dim / 2] uint8, affine [..., dim / 64, 2] bf16)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    least, most = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((most - least) * (1.0 / 15.0)).to(BF).float()
    code = torch.where(scale > 0, torch.round((g - least) / scale).clamp(0, 15), torch.zeros_like(g))
    code = code.flatten(-2).to(torch.uint8)[..., _order(x.shape[-1], keys, x.device)]
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([scale, least], -1).to(BF)


def _values(codes: torch.Tensor, affine: torch.Tensor, keys: bool, dtype=F32) -> torch.Tensor:
    """What the cache's rows stand for."""
    dim = codes.shape[-1] * 2
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    back = torch.argsort(_order(dim, keys, codes.device))
    code = code[..., back].to(dtype).unflatten(-1, (-1, GROUP))
    return (code * affine[..., 0:1].to(dtype) + affine[..., 1:2].to(dtype)).flatten(-2)


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _table(rot: int, rows: int, scaling: str, device) -> torch.Tensor:
    """fp32 [rows, rot]: cosines, then sines.  linear: positions four times as dense; yarn: slow pairs four times as dense, fast ones as
    they were, a ramp between, and the rotation longer by 1 + 0.1 ln 4."""
    half, theta = rot // 2, 1e6
    freq = theta ** (-torch.arange(half, dtype=F64, device=device) / half)
    grow = 1.0
    if scaling == "linear":
        freq = freq / 4
    elif scaling == "yarn":
        turns = 8192 * freq / (2 * math.pi)                 # over the trained length
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        freq, grow = freq / 4 * (1 - keep) + freq * keep, 1 + 0.1 * math.log(4)
    angle = torch.arange(rows, dtype=F64, device=device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], -1) * grow).float()


def _keys(g, *shape) -> torch.Tensor:
    """Keys as layers make them: a few channels much larger than the others."""
    d = shape[-1]
    size = torch.ones(d, device="cuda")
    size[d // 5] = size[d // 2 + 1] = 6.0
    return (torch.randn(*shape, device="cuda", generator=g) * size).to(BF)


def _cache(g, blocks: int, hkv: int, dim: int) -> dict:
    """A layer's cache, every row of it filled."""
    k, v = [], []
    for first in range(0, blocks, 512):
        n = min(512, blocks - first)
        k.append(_quantise(_keys(g, n, hkv, BLOCK, dim), True))
        v.append(_quantise(torch.randn(n, hkv, BLOCK, dim, device="cuda", generator=g).to(BF), False))
    (kc, ka), (vc, va) = (tuple(torch.cat(part) for part in zip(*rows)) for rows in (k, v))
    return {"k_codes": kc, "k_affine": ka, "v_codes": vc, "v_affine": va}


def _blocks(lens: list[int], seed: int):
    """Block lists over a shuffled pool, as a table padded with -1; the pool has three blocks more than are used."""
    need = [-(-n // BLOCK) for n in lens]
    pool = list(range(sum(need) + 3))
    random.Random(seed).shuffle(pool)
    table, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(pool[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda(), len(pool)


def _summaries(cache: dict) -> torch.Tensor:
    """bf16 [blocks, kv heads, 4, 2, dim]: least and greatest key of every span of 64 rows, channel by channel."""
    out = []
    for c, a in zip(cache["k_codes"].split(256), cache["k_affine"].split(256)):
        k = _values(c, a, True).unflatten(2, (-1, SPAN))
        out.append(torch.stack([k.amin(3), k.amax(3)], 3).to(BF))
    return torch.cat(out)


def _inputs(case, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["op"] == "rotary":
        t, dtype = case["tokens"], TYPES[case["type"]]
        rows = 40960
        first = torch.randint(0, rows - t, (1,), device="cuda", generator=g)
        pos = first + torch.arange(t, device="cuda") if t > 512 else torch.randint(0, rows, (t,), device="cuda", generator=g)
        q, k = (torch.randn(t, h, dim, device="cuda", generator=g).to(dtype) for h in (hq, hkv))
        return {"q": q, "k": k, "positions": pos, "table": _table(case["rot"], rows, case["scaling"], "cuda")}
    lens = _lens(case)
    if case["op"] == "write":
        whole = [n + case["prefix"] for n in lens]
        table, pool = _blocks(whole, seed)
        slots, pos = [], []
        for b, n in enumerate(whole):
            p = torch.arange(case["prefix"], n, device="cuda")
            slots.append(table[b, p // BLOCK] * BLOCK + p % BLOCK)
            pos.append(p)
        packed = _keys(g, sum(lens), hq + 2 * hkv, dim)         # the projection's output: q, k and v are views of it
        cu = [0]
        for n in whole:
            cu.append(cu[-1] + n)
        return {"q": packed[:, :hq], "k": packed[:, hq:hq + hkv], "v": packed[:, hq + hkv:], "positions": torch.cat(pos),
                "slots": torch.cat(slots).int(), "table": _table(case["rot"], max(whole), case["scaling"], "cuda"),
                "cache": _cache(g, pool, hkv, dim), "block_table": table, "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"), "whole": whole}
    table, pool = _blocks(lens, seed)
    s = {"q": torch.randn(len(lens), hq, dim, device="cuda", generator=g).to(BF), "cache": _cache(g, pool, hkv, dim),
         "block_table": table, "seqlens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "lens": lens}
    if case["op"] == "sparse":
        last = torch.tensor([n - 1 for n in lens], device="cuda")
        s["slots"] = (table[torch.arange(len(lens), device="cuda"), last // BLOCK] * BLOCK + last % BLOCK).int()
        s["summaries"] = _summaries(s["cache"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _handles(s)
    return s


def _handles(s) -> None:
    """What a user's program keeps for the framework's calls: the cache's handle, the workspace."""
    from mini_vllm_b200 import ops
    if "cache" in s:
        s["kv4"] = ops.KV4Cache(**s["cache"])
    if s["case"]["op"] in ("decode", "sparse"):
        c = s["case"]
        s["workspace"] = ops.decode4_workspace(c["seqs"], c["hq"], c["hkv"], c["dim"], "cuda")


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "rotary":
        return [_rotate(x, s["positions"], s["table"], case["inter"]) for x in (s["q"], s["k"])]
    if case["op"] == "write":
        return _write(s)
    spans = None
    if case["op"] == "sparse":
        _renew(s)
        spans = _select(s, case["budget"])
    out = _attend(s, case["dim"] ** -0.5, case.get("window", -1), case.get("cap", 0.0), spans)
    return out if spans is None else {"out": out, "spans": spans, "summaries": s["summaries"]}


def _run_own(s):
    from mini_vllm_b200 import ops
    case = s["case"]
    if "kv4" not in s and "cache" in s:
        _handles(s)
    if case["op"] == "rotary":
        return list(ops.rotary(s["q"], s["k"], s["positions"], s["table"], interleaved=case["inter"], q_out=torch.empty_like(s["q"]),
                               k_out=torch.empty_like(s["k"])))
    if case["op"] == "write":
        q = torch.empty(s["q"].shape, dtype=BF, device="cuda")
        ops.rotary_kv4_write(s["q"], s["k"], s["v"], s["positions"], s["table"], s["slots"], s["kv4"], interleaved=case["inter"], q_out=q)
        k, v = ops.kv4_gather(s["kv4"], s["cu"], s["block_table"], sum(s["whole"]))
        return {"q": q, "k": k, "v": v}
    scale = case["dim"] ** -0.5
    if case["op"] == "decode":
        return ops.decode_attn4(s["q"], s["kv4"], s["seqlens"], s["block_table"], scale, case["window"], s["workspace"], softcap=case["cap"])
    ops.kv4_summarise(s["kv4"], s["slots"], s["summaries"])
    spans = ops.kv4_select(s["q"], s["summaries"], s["seqlens"], s["block_table"], BLOCK, case["budget"])
    out = ops.decode_attn4(s["q"], s["kv4"], s["seqlens"], s["block_table"], scale, -1, s["workspace"], spans=spans)
    return {"out": out, "spans": spans, "summaries": s["summaries"]}


# ---- plain forms --------------------------------------------------------------------------------------------------------------------
def _rotate(x, positions, table, inter: bool) -> torch.Tensor:
    """Pairs (2i, 2i + 1), or (i, i + rot / 2), of the first rot channels; products and sums in fp32, one rounding."""
    rot = table.shape[1]
    row = table[positions][:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:]
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if inter else (y[..., :rot // 2], y[..., rot // 2:rot])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if inter else torch.cat(turned, -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _write(s) -> dict:
    inter, cache = s["case"]["inter"], s["cache"]
    q, k = (_rotate(s[n], s["positions"], s["table"], inter) for n in ("q", "k"))
    block, row = s["slots"].long() // BLOCK, s["slots"].long() % BLOCK
    for name, x, keys in (("k", k, True), ("v", s["v"], False)):
        codes, affine = _quantise(x, keys)
        cache[name + "_codes"][block, :, row] = codes
        cache[name + "_affine"][block, :, row] = affine
    back = {"q": q}
    for name in "kv":
        rows = []
        for b, n in enumerate(s["whole"]):
            blocks = s["block_table"][b, :-(-n // BLOCK)].long()
            x = _values(cache[name + "_codes"][blocks], cache[name + "_affine"][blocks], name == "k")
            rows.append(x.transpose(1, 2).flatten(0, 1)[:n].to(BF))
        back[name] = torch.cat(rows)
    return back


def _context(s, b: int, dtype):
    """Keys and values of a sequence, [kv heads, blocks * 256, dim] each."""
    blocks = s["block_table"][b, :-(-s["lens"][b] // BLOCK)].long()
    return (_values(s["cache"][n + "_codes"][blocks], s["cache"][n + "_affine"][blocks], n == "k", dtype).transpose(0, 1).flatten(1, 2) for n in "kv")


def _attend(s, scale: float, window: int, cap: float, spans) -> torch.Tensor:
    out = torch.empty_like(s["q"])
    for b, n in enumerate(s["lens"]):
        k, v = _context(s, b, F32)
        hkv = k.shape[0]
        if spans is not None:
            at = (spans[b].long()[..., None] * SPAN + torch.arange(SPAN, device="cuda")).flatten(1)   # [kv heads, tokens]; < 0: no span
            seen = (at >= 0) & (at < n)
            at = at.clamp(0, k.shape[1] - 1)[..., None].expand(-1, -1, k.shape[2])
            k, v = k.gather(1, at), v.gather(1, at)
        else:
            first = max(0, n - 1 - window) if window >= 0 else 0
            k, v, seen = k[:, first:n], v[:, first:n], None
        score = (s["q"][b].float().unflatten(0, (hkv, -1)) @ k.transpose(1, 2)) * scale
        if cap > 0:
            score = cap * torch.tanh(score / cap)
        if seen is not None:
            score = score.masked_fill(~seen[:, None], -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        out[b] = ((p @ v) / p.sum(-1, keepdim=True)).flatten(0, 1).to(BF)
    return out


def _renew(s) -> None:
    """The bounds of the spans that the step's tokens lie in, over their rows up to the new one."""
    slot = s["slots"].long()
    block, span, end = slot // BLOCK, slot % BLOCK // SPAN, slot % SPAN
    c, a = (s["cache"][n].unflatten(2, (-1, SPAN))[block, :, span] for n in ("k_codes", "k_affine"))
    k = _values(c, a, True)                                                                            # [seqs, kv heads, 64, dim]
    seen = (torch.arange(SPAN, device="cuda") <= end[:, None])[:, None, :, None]
    least, most = k.masked_fill(~seen, math.inf).amin(2), k.masked_fill(~seen, -math.inf).amax(2)
    s["summaries"][block, :, span] = torch.stack([least, most], 2).to(BF)


def _select(s, budget: int) -> torch.Tensor:
    """int32 [seqs, kv heads, budget], ascending, -1 behind them: the first and the last span and the ones whose bound
    sum over the group's heads and channels of max(q least, q greatest) is greatest, the lower index first among equals.
    The sums run in 64 bits, where they are exact."""
    lens, hkv = s["lens"], s["summaries"].shape[1]
    out = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        count = -(-n // SPAN)
        if count <= budget:
            out[b, :, :count] = torch.arange(count, dtype=torch.int32, device="cuda")
            continue
        bounds = s["summaries"][s["block_table"][b, :-(-n // BLOCK)].long()].transpose(0, 1).flatten(1, 2)[:, :count].to(F64)
        q = s["q"][b].to(F64).unflatten(0, (hkv, -1))
        score = torch.zeros(hkv, count, dtype=F64, device="cuda")
        for i in range(q.shape[1]):
            score += (bounds * q[:, i, None, None]).amax(2).sum(-1)
        score[:, 0] = score[:, -1] = math.inf
        best = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :budget]
        out[b] = best.sort(-1).values.int()
    return out


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------------------
def _unpack64(codes, affine, keys: bool):
    """Word by word: channel 8 L + e of a row lies in a word's bits 4 (e / 2), + 16 where e is odd."""
    dim = codes.shape[-1] * 2
    word = codes.to(torch.int64).unflatten(-1, (-1, 4))
    word = word[..., 0] + (word[..., 1] << 8) + (word[..., 2] << 16) + (word[..., 3] << 24)
    value = torch.empty(*codes.shape[:-1], dim, dtype=F64, device=codes.device)
    for p in range(dim // 8):
        level = 4 * (p % (dim // 32)) + p // (dim // 32) if keys else 8 * (p % (dim // 64)) + p // (dim // 64)
        for e in range(8):
            code = (word[..., p] >> (4 * (e // 2) + 16 * (e % 2))) & 15
            pair = affine[..., level // 8, :].to(F64)
            value[..., 8 * level + e] = pair[..., 1] + pair[..., 0] * code
    return value


def _turn64(x, positions, table, inter: bool):
    y, rot = x.to(F64).clone(), table.shape[1]
    for i in range(rot // 2):
        c, w = table[positions, i].to(F64)[:, None], table[positions, rot // 2 + i].to(F64)[:, None]
        one, two = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        u, v = y[..., one].clone(), y[..., two].clone()
        y[..., one], y[..., two] = u * c - v * w, v * c + u * w
    return y


def _stored64(x):
    """What rows x [..., dim] of 64-bit values stand for once they are in the cache."""
    y = torch.empty_like(x)
    for g in range(x.shape[-1] // GROUP):
        part = x[..., g * GROUP:(g + 1) * GROUP]
        low = part.min(-1, keepdim=True).values
        step = ((part.max(-1, keepdim=True).values - low) / 15).to(BF).to(F64)
        code = torch.minimum(torch.round((part - low) / torch.where(step > 0, step, torch.ones_like(step))), torch.full_like(step, 15.0))
        y[..., g * GROUP:(g + 1) * GROUP] = low + step * torch.where(step > 0, code, torch.zeros_like(code))
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":
        return [_turn64(s[n], s["positions"], s["table"], case["inter"]) for n in ("q", "k")]
    if case["op"] == "write":
        if sum(s["whole"]) * case["hkv"] * case["dim"] > 1 << 27:
            return None
        res = {"q": _turn64(s["q"], s["positions"], s["table"], case["inter"])}
        new = {"k": _turn64(s["k"], s["positions"], s["table"], case["inter"]).to(BF).to(F64), "v": s["v"].to(F64)}
        for n in "kv":
            fresh, at, rows = _stored64(new[n]), 0, []
            for b, total in enumerate(s["whole"]):
                blocks = s["block_table"][b, :-(-total // BLOCK)].long()
                old = _unpack64(s["cache"][n + "_codes"][blocks], s["cache"][n + "_affine"][blocks], n == "k")
                old = old.permute(0, 2, 1, 3).reshape(-1, *new[n].shape[1:])[:case["prefix"]]
                rows += [old, fresh[at:at + total - case["prefix"]]]
                at += total - case["prefix"]
            res[n] = torch.cat(rows)
        return res
    sparse = case["op"] == "sparse"
    res = torch.empty(s["q"].shape, dtype=F64, device="cuda")
    if sparse:
        bounds = s["summaries"].to(F64)
        for b, slot in enumerate(s["slots"].tolist()):
            i, r = divmod(slot, BLOCK)
            first = r // SPAN * SPAN
            k = _unpack64(s["cache"]["k_codes"][i, :, first:r + 1], s["cache"]["k_affine"][i, :, first:r + 1], True)
            bounds[i, :, r // SPAN, 0], bounds[i, :, r // SPAN, 1] = k.min(1).values, k.max(1).values
        stored = bounds.to(BF).to(F64)
    group = case["hq"] // case["hkv"]
    for b, n in enumerate(s["lens"]):
        blocks = s["block_table"][b, :-(-n // BLOCK)].long()
        k, v = (_unpack64(s["cache"][m + "_codes"][blocks], s["cache"][m + "_affine"][blocks], m == "k").permute(1, 0, 2, 3).flatten(1, 2)[:, :n]
                for m in "kv")
        for h in range(case["hkv"]):
            q = s["q"][b, h * group:(h + 1) * group].to(F64)
            seen = torch.ones(n, dtype=torch.bool, device="cuda")
            if sparse:
                count = (n + SPAN - 1) // SPAN
                low, high = (stored[blocks, h].flatten(0, 1)[:count, m] for m in (0, 1))
                bound = torch.maximum(q[:, None] * low, q[:, None] * high).sum((0, 2))
                bound[0] = bound[count - 1] = math.inf
                rank = torch.sort(bound, descending=True, stable=True).indices[:case["budget"]]
                chosen = torch.zeros(count, dtype=torch.bool, device="cuda")
                chosen[rank] = True
                seen = chosen.repeat_interleave(SPAN)[:n]
            elif case["window"] >= 0:
                seen[:max(0, n - 1 - case["window"])] = False
            z = (k[h] @ q.T) / math.sqrt(case["dim"])                       # [tokens, heads of the group]
            if case.get("cap", 0.0) > 0:
                z = case["cap"] * torch.tanh(z / case["cap"])
            w = torch.softmax(z.masked_fill(~seen[:, None], -math.inf), 0)
            res[b, h * group:(h + 1) * group] = w.T @ v[h]
    return {"out": res, "spans": None, "summaries": bounds} if sparse else res
