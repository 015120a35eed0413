"""The 4-bit cache (CUDA) where its users rarely go."""
import pytest
import torch

from mini_vllm_b200 import ops
from tests import kv4_helpers as kh

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def on(cuda, cache) -> ops.KV4Cache:
    return ops.KV4Cache(*(t.to(cuda) for t in cache))


def call(cuda, q, cache, table, lens, window=-1, spans=None, room=None, status=None):
    """``room``: blocks in the pool and columns in the table, more than anyone holds."""
    dev, (blocks, hkv, size), d = on(cuda, cache), cache[0].shape[:3], q.shape[2]
    if room is not None:
        wide = torch.full((table.shape[0], room), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        big, table = ops.KV4Cache.empty(room, size, hkv, d, cuda), wide
        for to, rows in zip((big.k_codes, big.k_affine, big.v_codes, big.v_affine), (dev.k_codes, dev.k_affine, dev.v_codes, dev.v_affine)):
            to[:blocks] = rows
        dev = big
    ws = ops.decode4_workspace(len(lens), q.shape[1], hkv, d, cuda)
    return ops.decode_attn4(q.to(cuda), dev, torch.tensor(lens, dtype=torch.int32, device=cuda), table.to(cuda), d ** -0.5, window, ws,
                            spans=None if spans is None else spans.to(cuda), status=status).double().cpu()


# ---- groups of unequal size ---------------------------------------------------------------------------------------------------------------
def group_bound(q, cache, table, lens):
    """Per sequence, head and group of 64 channels, the bound that goes with that group alone.  With p the softmax: a weight p s to fp16 is off
    by 2^-11 of itself and meets codes of at most 15: 2^-11 sum p (15 s).  Scores are fp32 sums, good to 2^-14, and with them each weight, twice
    (numerator and sum): 2^-13 sum p |v|.  Weights below fp16's normal numbers are off by 2^-25, the group's greatest being 2^8 at least:
    2^-33 of the greatest p (15 s) for each token.  Sums run in fp32, a step for 16 tokens, each good to 2^-23: n 2^-27 of what is added up."""
    hkv, d = cache[0].shape[1], q.shape[2]
    group, out = q.shape[1] // hkv, torch.zeros(*q.shape[:2], d // 64, dtype=kh.F64)
    for b, n in enumerate(lens):
        k, v = kh.context(cache, table, b, n)
        size = cache[0].shape[2]
        s = cache[3][table[b, :-(-n // size)].long()].transpose(0, 1).flatten(1, 2)[:, :n, :, 0].to(kh.F64) * 15
        for h in range(hkv):
            p = torch.softmax(q[b, h * group:(h + 1) * group].to(kh.F64) @ k[h].T * d ** -0.5, -1)
            v_size = v[h].abs().unflatten(-1, (-1, 64)).amax(-1)
            sums = p @ s[h], p @ v_size
            out[b, h * group:(h + 1) * group] = ((2.0 ** -11 + n * 2.0 ** -27) * sums[0] + (2.0 ** -13 + n * 2.0 ** -27) * sums[1] +
                                                 n * 2.0 ** -33 * (p[..., None] * s[h]).amax(1))
    return out


def check_groups(cuda, change, hq, hkv, d, lens, seed, **kw):
    g = gen(seed)
    table, blocks = kh.block_lists(g, lens, 256)
    cache = kh.make_cache(g, blocks, hkv, 256, d)
    change(cache, table)
    kh.poison(cache, table, lens, 256)
    q = torch.randn(len(lens), hq, d, generator=g).to(BF)
    got, (want, _) = call(cuda, q, cache, table, lens, **kw), kh.decode(q, cache, table, lens, d ** -0.5)
    assert torch.isfinite(got).all()
    bound = want.abs() * 2.0 ** -8 + group_bound(q, cache, table, lens).repeat_interleave(64, -1)
    worst = ((got - want).abs() / bound.clamp(min=1e-300)).unflatten(-1, (-1, 64)).amax((0, 1, 3))
    assert (worst <= 1.0).all(), f"of the bound, per group: {worst.tolist()}"


@pytest.mark.parametrize("r", [0, 12, 16, 20, 26, 60, 100])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (4, 1, 256)])
def test_a_small_group_beside_a_large_one(cuda, hq, hkv, d, r):
    def change(cache, table):
        cache[3][..., 1, :] *= 2.0 ** -r
    check_groups(cuda, change, hq, hkv, d, [650, 33, 1], seed=r)
    check_groups(cuda, change, hq, hkv, d, [3000, 700], seed=r, room=2000)


@pytest.mark.parametrize("r", [18, 40, 110])
def test_one_token_with_a_large_group(cuda, r):
    """Its other group and all other tokens' are what they were."""
    def change(cache, table):
        cache[3][table[0, 0], :, 70, 0] *= 2.0 ** r
        cache[3][table[1, 0], :, 5, 0] *= 2.0 ** r
    check_groups(cuda, change, 8, 2, 128, [700, 40, 9], seed=r)


@pytest.mark.parametrize("up", [True, False])
def test_groups_that_grow_and_shrink_along_a_row(cuda, up):
    """Every tile's first group 2^4 larger, its second 2^4 smaller than the tile's before."""
    def change(cache, table):
        size, n = 256, 640
        step = (torch.arange(3 * size) // 32 - 10).clamp(-10, 10) * (4 if up else -4)
        for i in range(3):
            f = torch.exp2(step[i * size:(i + 1) * size].float())[None, :, None]
            cache[3][table[0, i], :, :, 0] = (cache[3][table[0, i], :, :, 0].float() * f).to(BF)
            cache[3][table[0, i], :, :, 1] = (cache[3][table[0, i], :, :, 1].float() / f).to(BF)
    check_groups(cuda, change, 4, 2, 128, [640], seed=3)
    check_groups(cuda, change, 1, 1, 128, [640], seed=4)


@pytest.mark.parametrize("first", [32, 64, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_head_whose_first_scores_pass_below_all_numbers(cuda, d, first):
    """Keys of 2^126 that one head meets with zeros and the other with negative numbers: for that one they weigh nothing, and the rest is what it was."""
    g, lens = gen(first), [700]
    table, blocks = kh.block_lists(g, lens, 256)
    cache = kh.make_cache(g, blocks, 1, 256, d)
    for t in range(first):
        cache[1][table[0, t // 256], 0, t % 256, :, 0], cache[1][table[0, t // 256], 0, t % 256, :, 1] = 0, 2.0 ** 126
    q = torch.zeros(1, 2, d, dtype=BF)
    q[0, 1] = -8.0
    got, (want, _) = call(cuda, q, cache, table, lens), kh.decode(q, cache, table, lens, d ** -0.5)
    bound = want.abs() * 2.0 ** -8 + group_bound(q, cache, table, lens).repeat_interleave(64, -1)
    # (the second head's scores are sums of numbers of one sign, up to 2^7: good to 2^-14 as a difference, too)
    assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all()


# ---- what is not a number -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [NAN, -NAN, INF, -INF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_are_not_numbers_stay_visible(cuda, d, bad):
    """A NaN makes its whole group of 64 one; an infinity leaves no channel of its group finite.  Every other group is what it was."""
    g, n, hkv = gen(d), 90, 2
    x = torch.randn(n, 2 * hkv, d, generator=g).to(BF)
    hit = torch.zeros(n, 2 * hkv, d // 64, dtype=torch.bool)
    for t, h, c in ((0, 0, 0), (5, 1, d - 1), (6, 2, 17), (40, 3, d // 2), (89, 0, d - 7), (88, 2, 63)):
        x[t, h, c] = bad
        hit[t, h, c // 64] = True
    cache = ops.KV4Cache.empty(2, 64, hkv, d, cuda)
    slots, dev = torch.arange(n, dtype=torch.int32, device=cuda), x.to(cuda)
    ops.rotary_kv4_write(None, dev[:, :hkv], dev[:, hkv:], None, None, slots, cache)
    k, v = ops.kv4_gather(cache, torch.tensor([0, n], dtype=torch.int32, device=cuda), torch.tensor([[0, 1]], dtype=torch.int32, device=cuda), n)
    got = torch.cat([k, v], 1).cpu().unflatten(-1, (-1, 64))
    if bad != bad:
        assert torch.isnan(got[hit]).all()
    else:
        assert not torch.isfinite(got[hit]).any()
    clean = x.clone()
    clean[~torch.isfinite(clean)] = 0
    want = torch.cat([kh.stored(clean[:, :hkv], True, torch.float32), kh.stored(clean[:, hkv:], False, torch.float32)], 1).to(BF).unflatten(-1, (-1, 64))
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("n", [20, 700, 9000])
def test_a_value_that_is_not_a_number_is_its_groups_matter(cuda, n, bad):
    g, hq, hkv, d = gen(n), 4, 2, 128
    table, blocks = kh.block_lists(g, [n, n], 256)
    cache = kh.make_cache(g, blocks, hkv, 256, d)
    q = torch.randn(2, hq, d, generator=g).to(BF)
    want, big = kh.decode(q, cache, table, [n, n], d ** -0.5)
    t = n // 2
    cache[3][table[1, t // 256], 1, t % 256, 0] = torch.tensor([abs(bad), 0.5 if bad == INF else bad]).to(BF)     # what a write makes of it
    got = call(cuda, q, cache, table, [n, n])
    assert not torch.isfinite(got[1, 2:, :64]).any()
    others = torch.ones(2, hq, 2, dtype=torch.bool)
    others[1, 2:, 0] = False
    kh.assert_decode(got.unflatten(-1, (2, 64))[others], want.unflatten(-1, (2, 64))[others], big[..., None].expand(2, hq, 2)[others], "the other groups")


def test_a_key_that_is_not_a_number_reaches_its_queries_and_is_chosen(cuda):
    g, hq, hkv, d, n = gen(3), 4, 2, 128, 64 * 40
    x = torch.randn(n, 2 * hkv, d, generator=g).to(BF)
    x[64 * 17 + 3, 1, 100] = NAN                                    # a key of the second head
    dev, slots = x.to(cuda), torch.arange(n, dtype=torch.int32, device=cuda)
    cache = ops.KV4Cache.empty(n // 256, 256, hkv, d, cuda)
    ops.rotary_kv4_write(None, dev[:, :hkv], dev[:, hkv:], None, None, slots, cache)
    summaries = ops.kv4_summarise(cache, slots, ops.kv4_summaries(cache))
    q = torch.randn(3, hq, d, generator=g).to(BF).to(cuda)
    lens = torch.tensor([n, 64 * 17 + 3, n], dtype=torch.int32, device=cuda)             # (the second sequence ends in front of it)
    table = torch.arange(n // 256, dtype=torch.int32, device=cuda).repeat(3, 1)
    ws = ops.decode4_workspace(3, hq, hkv, d, cuda)
    out = ops.decode_attn4(q, cache, lens, table, d ** -0.5, -1, ws)
    nan = torch.isnan(out).all(-1).cpu()
    assert nan.tolist() == [[False, False, True, True], [False] * 4, [False, False, True, True]] and not torch.isnan(out[nan.logical_not().to(cuda)]).any()
    spans = ops.kv4_select(q[:1], summaries, lens[:1], table[:1], 256, 4).cpu()
    assert 17 in spans[0, 1].tolist()
    few = ops.kv4_summarise(cache, slots[64 * 17:64 * 17 + 64], ops.kv4_summaries(cache))    # by eight warps a span, as by one
    assert torch.equal(few[4, :, 1].view(torch.int16), summaries[4, :, 1].view(torch.int16))
    assert torch.isnan(summaries[4, 1, 1, :, 64:]).all() and not torch.isnan(summaries[4, 1, 1, :, :64]).any()


# ---- lists of spans with gaps -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("budget", [5, 31, 40, 100])
@pytest.mark.parametrize("hq,hkv,d,size", [(8, 2, 128, 256), (2, 1, 256, 64), (8, 2, 64, 64)])
def test_spans_behind_gaps(cuda, hq, hkv, d, size, budget):
    """Entries below 0 anywhere in a list, more of them than the sequence has spans."""
    g, lens = gen(budget), [1, 64, 100, 700, 0, 5000, 130, 1300]
    spans = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        count = -(-n // 64)
        for h in range(hkv):
            m = int(torch.randint(0, min(count, budget) + 1, (1,), generator=g))
            at = torch.randperm(budget, generator=g)[:m]
            spans[b, h, at] = torch.randperm(count, generator=g)[:m].int() if m else spans[b, h, at]
    if budget == 5:
        spans[2] = torch.tensor([-1, -1, 0, 1, -1])
        spans[0] = torch.tensor([-1, -1, -1, -1, 0])
    table, blocks = kh.block_lists(g, lens, size)
    cache = kh.make_cache(g, blocks, hkv, size, d)
    kh.poison(cache, table, lens, size)
    q = torch.randn(len(lens), hq, d, generator=g).to(BF)
    want, big = kh.decode(q, cache, table, lens, d ** -0.5, spans=spans)
    for room in (None, 2000):
        status = ops.new_status(cuda)
        got = call(cuda, q, cache, table, lens, spans=spans, room=room, status=status)
        ops.check_status(status)
        kh.assert_decode(got, want, big, f"budget {budget}")


def test_spans_outside_the_sequence_in_front_of_others(cuda):
    g = gen(2)
    table, blocks = kh.block_lists(g, [100], 64)
    cache = kh.make_cache(g, blocks, 1, 64, 128)
    q, spans = torch.randn(1, 2, 128, generator=g).to(BF), torch.tensor([[[9, 2, 1, 1 << 20, 0]]], dtype=torch.int32)
    status = ops.new_status(cuda)
    got = call(cuda, q, cache, table, [100], spans=spans, status=status)
    assert status[0].item() == 5 and status[1].item() == 0
    kh.assert_decode(got, *kh.decode(q, cache, table, [100], 128 ** -0.5), "both spans")


# ---- single rows ----------------------------------------------------------------------------------------------------------------------
def test_a_single_row_of_any_stride(cuda):
    """One token cut out of rows whose length is no multiple of eight: its own stride leads nowhere."""
    g, hq, hkv, d = gen(1), 4, 2, 128
    odd = torch.zeros(3, (hq + 2 * hkv) * d + 3, dtype=BF, device=cuda)
    odd[0, :-3] = torch.randn((hq + 2 * hkv) * d, generator=g).to(BF)
    q, k, v = (odd.as_strided((1, h, d), (odd.stride(0), d, 1), at * d) for h, at in ((hq, 0), (hkv, hq), (hkv, hq + hkv)))
    assert q.stride(0) % 8 and q.shape == (1, hq, d)
    slots, table, lens = torch.zeros(1, dtype=torch.int32, device=cuda), torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda)
    pos, cos, ws = torch.ones(1, dtype=torch.int64, device=cuda), torch.randn(2, d, generator=g).to(cuda), ops.decode4_workspace(1, hq, hkv, d, cuda)
    got = []
    for rows in ((q, k, v), (q.contiguous().clone(), k.contiguous(), v.contiguous())):
        cache = ops.KV4Cache.empty(1, 256, hkv, d, cuda)
        out = ops.rotary_kv4_write(*rows, pos, cos, slots, cache, q_out=torch.empty_strided((1, hq, d), (hq * d + 1, d, 1), dtype=BF, device=cuda))
        summaries = ops.kv4_summarise(cache, slots, ops.kv4_summaries(cache))
        spans = ops.kv4_select(out, summaries, lens, table, 256, 2)
        got.append((out, spans, ops.decode_attn4(out, cache, lens, table, 1.0, -1, ws, spans=spans), ops.rotary(rows[0], None, pos, cos)[0]))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 32 + 64, 2 ** 63 - 1])
def test_windows_and_contexts_beyond_32_bits(cuda, far):
    """As long as can be, not what is left of them in 32 bits."""
    g, lens, hq, hkv, d = gen(5), [3000, 64, 2600], 4, 2, 128
    table, blocks = kh.block_lists(g, lens, 256)
    cache = kh.make_cache(g, blocks, hkv, 256, d)
    q = torch.randn(3, hq, d, generator=g).to(BF)
    assert torch.equal(call(cuda, q, cache, table, lens, window=far), call(cuda, q, cache, table, lens))
    status, summaries = ops.new_status(cuda), torch.randn(blocks, hkv, 4, 2, d, generator=g).to(BF).sort(3).values
    got = ops.kv4_select(q.to(cuda), summaries.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), table.to(cuda), 256, 5, status=status, max_context=far)
    ops.check_status(status)
    assert torch.equal(got.cpu(), kh.select(q, summaries, table, lens, 5))


# ---- every tile counts ------------------------------------------------------------------------------------------------------------------
def tile_marks(cache, table, lens, size, d):
    """Values that say where they come from: channel c is 1 in the tiles of 32 tokens whose number leaves c when divided by d, else 0."""
    t = torch.arange(table.shape[1] * size)
    one = torch.nn.functional.one_hot(t // 32 % d, d).to(BF)
    codes, affine = kh.quantise(one, False)
    for b, n in enumerate(lens):
        for i in range(-(-n // size)):
            cache[2][table[b, i]], cache[3][table[b, i]] = codes[i * size:(i + 1) * size], affine[i * size:(i + 1) * size]


@pytest.mark.parametrize("lens,room", [([9000], None), ([9000], 2000), ([40000], None), ([40000], 2000), ([9000, 3, 700, 0, 4000, 31], None),
                                       ([9000, 3, 700, 0, 4000, 31], 2000), ([2500 + 33 * i for i in range(12)], 2000)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (16, 8, 128), (2, 1, 256), (2, 2, 64)])
def test_every_tile_counts_once(cuda, hq, hkv, d, lens, room):
    """A channel's output is the weight of its few tiles, and has to be right as a number of that size.  All values are 0 or 1, so each error is
    relative: a weight's rounding 2^-11, scores good to 2^-14 twice (numerator and sum), the rounding of the output 2^-8."""
    g, size = gen(len(lens)), 256
    table, blocks = kh.block_lists(g, lens, size)
    cache = kh.make_cache(g, blocks, hkv, size, d)
    tile_marks(cache, table, lens, size, d)
    kh.poison(cache, table, lens, size)
    q = (torch.randn(len(lens), hq, d, generator=g) * 0.25).to(BF)
    q[:, 0] = 0                                                     # a head whose weights are all alike
    for window in (-1, 2600):
        got, (want, _) = call(cuda, q, cache, table, lens, window=window, room=room), kh.decode(q, cache, table, lens, d ** -0.5, window)
        worst = ((got - want).abs() / want.clamp(min=1e-300))[want > 0].max() / (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -12)
        assert worst <= 1.0 and (got[want == 0] == 0).all(), f"window {window}: {worst:.3f}"


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (2, 1, 256), (2, 2, 64)])
def test_every_tile_of_a_list_counts_once(cuda, hq, hkv, d):
    g, lens, size, budget = gen(d), [9000, 64, 3000, 12000], 256, 70
    table, blocks = kh.block_lists(g, lens, size)
    cache = kh.make_cache(g, blocks, hkv, size, d)
    tile_marks(cache, table, lens, size, d)
    kh.poison(cache, table, lens, size)
    spans = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            chosen = torch.randperm(-(-n // 64), generator=g)[:budget - 9 * h % 20]
            spans[b, h, torch.randperm(budget, generator=g)[:len(chosen)]] = chosen.int()
    q = (torch.randn(len(lens), hq, d, generator=g) * 0.25).to(BF)
    want, _ = kh.decode(q, cache, table, lens, d ** -0.5, spans=spans)
    for room in (None, 2000):
        got = call(cuda, q, cache, table, lens, spans=spans, room=room)
        worst = ((got - want).abs() / want.clamp(min=1e-300))[want > 0].max() / (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -12)
        assert worst <= 1.0 and (got[want == 0] == 0).all(), f"{worst:.3f}"
