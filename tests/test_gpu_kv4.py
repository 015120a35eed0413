"""The 4-bit cache (CUDA): written, unpacked, attended, its spans bounded and chosen, against plain forms in 64 bits."""
import pytest
import torch

from mini_vllm_b200 import ops
from mini_vllm_b200.models.layers.rotary import build_cos_sin_cache
from tests import kv4_helpers as kh

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def on(cuda, cache) -> ops.KV4Cache:
    return ops.KV4Cache(*(t.to(cuda) for t in cache))


# ---- writing and unpacking ------------------------------------------------------------------------------------------------------------
WRITES = [(1, 1, 1, 64, 64, 64), (9, 8, 2, 64, 32, 128), (33, 16, 8, 128, 128, 256), (300, 4, 1, 256, 256, 256), (41, 7, 1, 128, 16, 64),
          (700, 6, 3, 128, 96, 128), (257, 5, 5, 64, 48, 64), (130, 0, 2, 256, 32, 64)]


@pytest.mark.parametrize("tokens,hq,hkv,d,rot,size", WRITES)
@pytest.mark.parametrize("inter", [False, True])
def test_write_is_exact(cuda, tokens, hq, hkv, d, rot, size, inter):
    """Codes, scales and minima bit by bit; slots that got no row and the input's other columns stay as they were."""
    g = gen(tokens + d)
    blocks = -(-tokens // size) + 2
    packed = torch.randn(tokens, hq + 2 * hkv, d, generator=g).to(BF)
    packed[0, -1] = 0.25                                            # a row of one value: scale 0
    if tokens > 2:
        packed[1, hq:] *= 2.0 ** -60
        packed[2, hq:] *= 2.0 ** 60
    q, k, v = packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:]
    pos = torch.randint(0, 3000, (tokens,), generator=g)
    slots = torch.randperm(blocks * size, generator=g)[:tokens].to(torch.int32)
    slots[3::7] = -1
    table = build_cos_sin_cache(rot, 3000, 1e4, scaling={"rope_type": "default"})
    turned = [kh.turn(x, pos, table, inter, torch.float32).to(BF) for x in (q, k)]
    cache = ops.KV4Cache.empty(blocks, size, hkv, d, cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0xA5)
    for t in (cache.k_affine, cache.v_affine):
        t.fill_(3.0)
    want = [t.cpu().clone() for t in (cache.k_codes, cache.k_affine, cache.v_codes, cache.v_affine)]
    ok = slots >= 0
    at = (slots[ok].long() // size, slice(None), slots[ok].long() % size)
    for i, x, keys in ((0, turned[1], True), (2, v, False)):
        want[i][at], want[i + 1][at] = (t[ok] for t in kh.quantise(x, keys))
    dev = packed.to(cuda)
    status = ops.new_status(cuda)
    q_out = torch.empty(tokens, hq, d, dtype=BF, device=cuda) if hq else None
    got = ops.rotary_kv4_write(dev[:, :hq] if hq else None, dev[:, hq:hq + hkv], dev[:, hq + hkv:], pos.to(cuda), table.to(cuda), slots.to(cuda), cache,
                               interleaved=inter, q_out=q_out, status=status)
    ops.check_status(status)
    for a, b in zip((cache.k_codes, cache.k_affine, cache.v_codes, cache.v_affine), want):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(dev.cpu(), packed)
    if hq:
        assert got is q_out and torch.equal(q_out.cpu(), turned[0])
        # in place, k too; the cache gets the same
        again = ops.KV4Cache.empty(blocks, size, hkv, d, cuda)
        ops.rotary_kv4_write(dev[:, :hq], dev[:, hq:hq + hkv], dev[:, hq + hkv:], pos.to(cuda), table.to(cuda), slots.to(cuda), again, interleaved=inter,
                             k_in_place=True)
        assert torch.equal(dev[:, :hq].cpu(), turned[0]) and torch.equal(dev[:, hq:hq + hkv].cpu(), turned[1])
        assert torch.equal(again.k_codes.cpu()[at], want[0][at])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_write_of_every_kind_of_group(cuda, d):
    """Halves between two codes, tiny and huge spreads, zeros of both signs, without rotation."""
    g = gen(d)
    rows = [torch.randint(-60, 60, (400, 1, d), generator=g).float() / 8,               # many exact halves
            torch.randn(200, 1, d, generator=g) * 2.0 ** torch.randint(-126, 100, (200, 1, 1), generator=g),
            torch.randn(50, 1, d, generator=g) * 2.0 ** -132, torch.zeros(3, 1, d) * -1.0,
            torch.randint(0, 3, (50, 1, d), generator=g).float() * 2.0 ** -133]
    x = torch.cat(rows).to(BF)
    n = x.shape[0]
    cache = ops.KV4Cache.empty(-(-n // 64), 64, 1, d, cuda)
    slots = torch.arange(n, dtype=torch.int32, device=cuda)
    assert ops.rotary_kv4_write(None, x.to(cuda), x.flip(0).to(cuda), None, None, slots, cache) is None
    for codes, affine, y, keys in ((cache.k_codes, cache.k_affine, x, True), (cache.v_codes, cache.v_affine, x.flip(0), False)):
        c, a = kh.quantise(y, keys)
        assert torch.equal(codes.cpu().flatten(0, 2)[:n], c[:, 0])
        assert (affine.cpu().flatten(0, 2)[:n] == a[:, 0]).all()                        # (as values: a zero minimum may have either sign)


def test_write_reports_bad_slots_and_positions(cuda):
    cache = ops.KV4Cache.empty(2, 64, 1, 64, cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.zero_()
    table = build_cos_sin_cache(64, 8, 1e4).to(cuda)
    x = torch.randn(3, 1, 64, device=cuda, dtype=BF)
    for slots, pos, code in (([0, 128, 1], [0, 1, 2], 1), ([0, -2, 1], [0, 1, 2], 1), ([0, 1, 2], [0, 8, 2], 3)):
        status = ops.new_status(cuda)
        ops.rotary_kv4_write(None, x, x, torch.tensor(pos, device=cuda), table, torch.tensor(slots, dtype=torch.int32, device=cuda), cache, status=status)
        assert status[0].item() == code and status[1].item() == 1


@pytest.mark.parametrize("d,hkv,size", [(64, 3, 64), (128, 8, 256), (256, 1, 128)])
def test_gather(cuda, d, hkv, size):
    g, lens = gen(d), [1, 0, size, size + 1, 3 * size - 1, 70]
    table, blocks = kh.block_lists(g, lens, size, width=5)
    cache = kh.make_cache(g, blocks, hkv, size, d)
    kh.poison(cache, table, lens, size)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    total, status = sum(lens), ops.new_status(cuda)
    out = [torch.full((total + 5, hkv, d), 7.0, dtype=BF, device=cuda) for _ in range(2)]
    ops.kv4_gather(on(cuda, cache), cu.to(cuda), table.to(cuda), total + 5, *out, status=status)
    ops.check_status(status)
    for i, o in enumerate(out):
        want = torch.cat([kh.context(cache, table, b, n, torch.float32)[i].transpose(0, 1) for b, n in enumerate(lens) if n]).to(BF)
        assert torch.equal(o[:total].cpu(), want)
        assert (o[total:] == 7.0).all()                             # rows behind the last sequence
    bad = table.clone()
    bad[4, 1] = blocks
    k, v = ops.kv4_gather(on(cuda, cache), cu.to(cuda), bad.to(cuda), total, status=status)
    assert status[0].item() == 2 and status[1].item() == 4
    first = int(cu[4]) + size
    assert (k[first:first + size] == 0).all() and (v[first:first + size] == 0).all()
    late, status = (cu + 3).to(torch.int32), ops.new_status(cuda)   # lists that do not begin at 0: the rows before them read as zeros
    k, v = ops.kv4_gather(on(cuda, cache), late.to(cuda), table.to(cuda), total + 3, status=status)
    assert status[0].item() == 2 and status[1].item() == 0 and (k[:3] == 0).all() and (v[:3] == 0).all()
    assert torch.equal(k[3:].cpu(), out[0][:total].cpu()) and torch.equal(v[3:].cpu(), out[1][:total].cpu())


# ---- attention of single tokens ---------------------------------------------------------------------------------------------------------
def run_decode(cuda, lens, hq, hkv, d, size=256, window=-1, cap=0.0, spans=None, seed=0, v_size=1.0, width=None, workspace=None, change=None, q_scale=1.0, pool=0):
    g = gen(seed)
    table, blocks = kh.block_lists(g, lens, size, width)
    cache = kh.make_cache(g, blocks, hkv, size, d, v_size)
    if change is not None:
        change(cache, table)
    kh.poison(cache, table, lens, size)
    q = (torch.randn(len(lens), hq, d, generator=g) * q_scale).to(BF)
    want, big = kh.decode(q, cache, table, lens, d ** -0.5, window, cap, spans)
    status = ops.new_status(cuda)
    ws = ops.decode4_workspace(len(lens), hq, hkv, d, cuda) if workspace is None else workspace
    out = torch.full((len(lens), hq, d), float("nan"), dtype=BF, device=cuda)
    packed = torch.zeros(len(lens), hq * d + 16, dtype=BF, device=cuda)                 # rows further apart than they are long
    qd = packed[:, 8:8 + hq * d].view(len(lens), hq, d)
    qd.copy_(q)
    dev = on(cuda, cache)
    if pool > blocks:                                               # more blocks than anyone holds
        big_one = ops.KV4Cache.empty(pool, size, hkv, d, cuda)
        for to, rows in ((big_one.k_codes, dev.k_codes), (big_one.k_affine, dev.k_affine), (big_one.v_codes, dev.v_codes), (big_one.v_affine, dev.v_affine)):
            to[:blocks] = rows
        dev = big_one
    got = ops.decode_attn4(qd, dev, torch.tensor(lens, dtype=torch.int32, device=cuda), table.to(cuda), d ** -0.5, window, ws,
                           spans=None if spans is None else spans.to(cuda), out=out, status=status, softcap=cap)
    ops.check_status(status)
    assert got is out
    kh.assert_decode(out, want, big, f"{lens[:8]} {hq}/{hkv} x {d} window {window}")
    for b, n in enumerate(lens):
        if n <= 0:
            assert (out[b] == 0).all()
    return out


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (32, 8, 128), (4, 1, 256), (8, 1, 256), (8, 2, 64), (7, 1, 64), (6, 2, 128), (5, 5, 128), (3, 1, 256),
                                      (24, 3, 128), (1, 1, 64)])
def test_decode_head_shapes(cuda, hq, hkv, d):
    run_decode(cuda, [5, 129, 640, 2049, 77, 1], hq, hkv, d, seed=hq * 10 + hkv)


@pytest.mark.parametrize("size", [64, 128, 256])
def test_decode_lengths_around_tiles_and_blocks(cuda, size):
    run_decode(cuda, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 0, 1000], 4, 2, 128, size=size, seed=size)


@pytest.mark.parametrize("lens", [[1], [32], [700], [9000], [9000] + [3] * 40 + [0, 700], [0, 0, 5, 0], [40] * 300, [1] * 1100, [300, 0, 280, 310, 0] * 20])
def test_decode_splits(cuda, lens):
    """One row over many CTAs, many rows in one, more sequences than threads, empty ones between."""
    run_decode(cuda, lens, 4, 2, 128, seed=len(lens))
    run_decode(cuda, lens[:64], 2, 1, 256, seed=len(lens), width=40)


def test_decode_nothing_to_read(cuda):
    assert (run_decode(cuda, [0, 0, -3], 2, 1, 128, width=2) == 0).all()
    c = ops.KV4Cache.empty(1, 64, 1, 64, cuda)
    empty = torch.zeros(0, dtype=torch.int32, device=cuda)
    out = ops.decode_attn4(torch.zeros(0, 2, 64, dtype=BF, device=cuda), c, empty, torch.zeros(1, 1, dtype=torch.int32, device=cuda), 1.0, -1,
                           ops.decode4_workspace(1, 2, 1, 64, cuda))
    assert out.shape == (0, 2, 64)


@pytest.mark.parametrize("window", [0, 1, 31, 32, 100, 512, 5000])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_decode_windows_and_caps(cuda, window, cap):
    run_decode(cuda, [1, 40, 512, 513, 514, 1500, 3000], 4, 1, 256, window=window, cap=cap, seed=window)
    run_decode(cuda, [1, 33, 700], 4, 2, 64, window=window, cap=cap, seed=window, q_scale=20.0)


@pytest.mark.parametrize("v_size", [2.0 ** -90, 2.0 ** -20, 2.0 ** 15, 2.0 ** 60])
def test_decode_sizes_of_values(cuda, v_size):
    """The weights p s are scaled by the values' own sizes: nothing overflows, nothing is lost."""
    run_decode(cuda, [700, 33], 4, 2, 128, v_size=v_size, seed=3)


def test_decode_values_of_very_different_sizes(cuda):
    def change(cache, table):
        cache[3][:, :, ::5] *= 2.0 ** 20                            # every fifth row of every block: a million times larger
        cache[3][:, :, 1::7] = 0                                    # constant rows of zeros
    run_decode(cuda, [900, 64, 1], 4, 2, 128, seed=4, change=change)

    def constant(cache, table):
        cache[3][..., 0] = 0                                        # scales of zero: a row is its minimum
    run_decode(cuda, [300, 7], 2, 1, 64, seed=5, change=constant)


@pytest.mark.parametrize("q_scale", [0.0, 2.0 ** -100, 2.0 ** 30])
def test_decode_sizes_of_queries(cuda, q_scale):
    """All weights alike; and scores so far apart that one key takes all."""
    run_decode(cuda, [600, 31], 4, 1, 128, seed=6, q_scale=q_scale)


def test_decode_one_workspace_for_every_shape(cuda):
    """The counters in a workspace are zero between calls, whatever shape used it last, and whatever it held of parts."""
    ws = ops.decode4_workspace(64, 16, 8, 256, cuda)
    for hq, hkv, d in ((16, 8, 128), (8, 1, 256), (2, 2, 64), (32, 8, 256), (16, 8, 128)):
        run_decode(cuda, [3000, 40, 900], hq, hkv, d, workspace=ws, seed=d)


WIDE = dict(width=2000, pool=2000)                                  # room for contexts of half a million tokens: sixteen warps a block


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (16, 8, 128), (8, 2, 64), (14, 2, 64)])
@pytest.mark.parametrize("lens", [[1], [700], [9000], [9000] + [3] * 40 + [0, 700], [40] * 150, [300, 0, 280, 310, 0] * 20, [31, 32, 33, 63, 64, 65, 255, 256, 257, 0]])
def test_decode_with_room_for_long_contexts(cuda, lens, hq, hkv, d):
    run_decode(cuda, lens, hq, hkv, d, seed=len(lens), **WIDE)


def test_decode_both_kinds_of_blocks_on_one_workspace(cuda):
    ws = ops.decode4_workspace(64, 16, 8, 256, cuda)
    for more in ({}, WIDE, {}, dict(WIDE, cap=30.0), dict(cap=30.0), WIDE):
        run_decode(cuda, [3000, 40, 900, 0], 16, 8, 128, workspace=ws, seed=9, **more)


def test_decode_windows_and_spans_of_many_sequences(cuda):
    g, lens = gen(6), [(i * 37) % 400 + 1 for i in range(240)]
    run_decode(cuda, lens, 16, 8, 128, window=600, width=40, pool=600, seed=5)
    spans = torch.stack([torch.stack([torch.cat([torch.randperm(-(-n // 64), generator=g)[:4].int(), torch.full((60,), -1, dtype=torch.int32)])[:12] for _ in range(8)])
                         if n > 192 else torch.cat([torch.arange(-(-n // 64)), torch.full((12,), -1)])[:12].int().repeat(8, 1) for n in lens]).contiguous()
    run_decode(cuda, lens, 16, 8, 128, spans=spans, seed=5)


def test_decode_same_bits_every_time(cuda):
    first = run_decode(cuda, [9000, 500, 33], 16, 8, 128, seed=8)
    assert all(torch.equal(first, run_decode(cuda, [9000, 500, 33], 16, 8, 128, seed=8)) for _ in range(3))


def test_decode_reports_bad_blocks_and_lengths(cuda):
    g = gen(1)
    table, blocks = kh.block_lists(g, [300, 300], 64)
    cache = kh.make_cache(g, blocks, 1, 64, 128)
    q = torch.randn(2, 2, 128, generator=g).to(BF)
    ws = ops.decode4_workspace(2, 2, 1, 128, cuda)
    lens = torch.tensor([300, 300], dtype=torch.int32, device=cuda)
    bad = table.clone()
    bad[1, 2] = blocks
    status = ops.new_status(cuda)
    out = ops.decode_attn4(q.to(cuda), on(cuda, cache), lens, bad.to(cuda), 1.0, -1, ws, status=status)
    assert status[0].item() == 2 and status[1].item() == 1 and torch.isfinite(out).all()
    status.zero_()
    lens[0] = 5 * 64 + 1                                            # one token more than its five columns hold
    ops.decode_attn4(q.to(cuda), on(cuda, cache), lens, table.to(cuda), 1.0, -1, ws, status=status)
    assert status[0].item() == 5 and status[1].item() == 0


@pytest.mark.parametrize("n", [20, 700, 9000])
def test_decode_a_query_that_is_not_a_number_stays_one_heads_matter(cuda, n):
    """Within one warp, over the warps of a CTA and over CTAs."""
    g, hq, hkv, d = gen(n), 4, 2, 128
    table, blocks = kh.block_lists(g, [n, n], 256)
    cache = kh.make_cache(g, blocks, hkv, 256, d)
    q = torch.randn(2, hq, d, generator=g).to(BF)
    want, big = kh.decode(q, cache, table, [n, n], d ** -0.5)
    q[1, 2, 77] = float("nan")
    got = ops.decode_attn4(q.to(cuda), on(cuda, cache), torch.tensor([n, n], dtype=torch.int32, device=cuda), table.to(cuda), d ** -0.5, -1,
                           ops.decode4_workspace(2, hq, hkv, d, cuda))
    assert torch.isnan(got[1, 2]).all()
    others = torch.ones(2, hq, dtype=torch.bool)
    others[1, 2] = False
    kh.assert_decode(got.cpu()[others], want[others], big[others], "the other heads")


def test_decode_capture_replay_and_two_graphs_of_one_workspace(cuda):
    """Lengths change between replays of a captured step; two graphs take turns on one workspace and another stream."""
    g, hq, hkv, d, most = gen(12), 8, 2, 128, [2000, 700, 90, 300]
    table, blocks = kh.block_lists(g, most, 256)
    cache = kh.make_cache(g, blocks, hkv, 256, d)
    dev, ws, stream = on(cuda, cache), ops.decode4_workspace(4, hq, hkv, d, cuda), torch.cuda.Stream()
    steps = []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for batch in (4, 2):
            q, lens = torch.randn(batch, hq, d, generator=g).to(BF), torch.zeros(batch, dtype=torch.int32, device=cuda)
            qd, td, out = q.to(cuda), table[:batch].to(cuda), torch.empty(batch, hq, d, dtype=BF, device=cuda)
            call = lambda: ops.decode_attn4(qd, dev, lens, td, d ** -0.5, -1, ws, out=out)
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                call()
            steps.append((graph, q, lens, out, (qd, td)))
        for now in ([2000, 0, 90, 1], [31, 700, 0, 300], [0, 0, 0, 0]):
            for graph, q, lens, out, _ in steps:
                n = now[:len(q)]
                lens.copy_(torch.tensor(n, dtype=torch.int32))
                out.fill_(float("nan"))
                graph.replay()
                stream.synchronize()
                kh.assert_decode(out, *kh.decode(q, cache, table, n, d ** -0.5), f"replay {n}")


def test_wrappers_refuse(cuda):
    c = ops.KV4Cache.empty(4, 64, 2, 128, cuda)
    q, i32 = torch.zeros(2, 4, 128, dtype=BF, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    k = q[:, :2].contiguous()
    table, ws = torch.zeros(2, 2, dtype=torch.int32, device=cuda), ops.decode4_workspace(2, 4, 2, 128, cuda)
    cs, pos = torch.zeros(4, 128, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    spans, s = torch.zeros(2, 2, 3, dtype=torch.int32, device=cuda), ops.kv4_summaries(c)
    dec = lambda **kw: ops.decode_attn4(**{**dict(q=q, cache=c, cache_seqlens=i32, block_table=table, scale=1.0, window_left=-1, workspace=ws), **kw})
    wr = lambda **kw: ops.rotary_kv4_write(**{**dict(q=q, k=k, v=k, positions=pos, cos_sin=cs, slot_mapping=i32, cache=c), **kw})
    sel = lambda **kw: ops.kv4_select(**{**dict(q=q, summaries=s, cache_seqlens=i32, block_table=table, block_size=64, budget=2), **kw})
    dec(), wr(), sel(), dec(spans=spans)
    for bad in (lambda: dec(q=q.float()), lambda: dec(cache_seqlens=i32.long()), lambda: dec(workspace=ws.view(torch.int32)), lambda: dec(spans=spans.long()),
                lambda: wr(k=k.float()), lambda: wr(positions=i32), lambda: wr(slot_mapping=pos), lambda: sel(summaries=s.float()),
                lambda: ops.kv4_summarise(c, pos, s), lambda: ops.kv4_gather(c, pos, table, 4)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: dec(q=q[..., :64]), lambda: dec(cache_seqlens=i32[:1]), lambda: dec(block_table=table[:1]), lambda: dec(block_table=table.t()[::2]),
                lambda: dec(spans=spans[:1]), lambda: dec(out=q[:1]), lambda: dec(out=q), lambda: wr(k=q), lambda: wr(v=k[:1]), lambda: wr(slot_mapping=i32[:1]),
                lambda: wr(cos_sin=cs[:, ::2]), lambda: wr(positions=None), lambda: wr(q=None, q_out=q), lambda: sel(block_size=128), lambda: sel(summaries=s[:, :, :, :1]),
                lambda: sel(out=spans), lambda: ops.kv4_summarise(c, i32, s[:2]), lambda: ops.kv4_gather(c, i32, table, 4, k_out=k),
                lambda: dec(q=q[0]), lambda: dec(q=torch.zeros(2, 128, 4, dtype=BF, device=cuda).transpose(1, 2))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: dec(softcap=-1.0), lambda: dec(window_left=4, spans=spans), lambda: dec(workspace=ws[:256]), lambda: sel(budget=1),
                lambda: wr(cos_sin=torch.zeros(4, 24, device=cuda)), lambda: dec(q=torch.zeros(2, 18, 128, dtype=BF, device=cuda))):
        with pytest.raises(ops._cabi.KernelError):
            bad()


# ---- spans ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,hkv,size", [(64, 3, 64), (128, 8, 256), (256, 1, 128)])
@pytest.mark.parametrize("many", [False, True])
def test_bounds_of_written_spans(cuda, d, hkv, size, many):
    """A step of prompts (some behind cached tokens), of single tokens, and of both, over rows poisoned behind each sequence."""
    g = gen(d)
    lens = [1, 64, 65, 3 * size - 1, 200, size] + ([700] * 8 if many else [])            # many: more than 4096 (token, head) pairs with 8 heads
    start = [0, 0, 60, 0, 199, size - 64] + ([0] * 8 if many else [])
    table, blocks = kh.block_lists(g, lens, size)
    cache = kh.make_cache(g, blocks, hkv, size, d)
    kh.poison(cache, table, lens, size)
    slots = []
    for b, n in enumerate(lens):
        p = torch.arange(start[b], n)
        slots.append(table[b, p // size] * size + p % size)
    slots.insert(2, torch.tensor([-1, -1]))
    slots = torch.cat(slots).to(torch.int32)
    want = torch.full((blocks, hkv, size // 64, 2, d), 9.0, dtype=BF)
    for b, n in enumerate(lens):
        k = kh.context(cache, table, b, n, torch.float32)[0]
        for s in range(start[b] // 64, -(-n // 64)):
            part = k[:, 64 * s:min(n, 64 * s + 64)]
            want[table[b, 64 * s // size], :, 64 * s % size // 64] = torch.stack([part.amin(1), part.amax(1)], 1).to(BF)
    got = torch.full_like(want, 9.0, device=cuda)
    status = ops.new_status(cuda)
    ops.kv4_summarise(on(cuda, cache), slots.to(cuda), got, status=status)
    ops.check_status(status)
    assert torch.equal(got.cpu(), want)
    ops.kv4_summarise(on(cuda, cache), torch.tensor([blocks * size, 0], dtype=torch.int32, device=cuda), got, status=status)
    assert status[0].item() == 1 and status[1].item() == 0


@pytest.mark.parametrize("hq,hkv,d,size", [(16, 8, 128, 256), (4, 1, 256, 128), (7, 1, 64, 64), (6, 2, 128, 256)])
@pytest.mark.parametrize("budget", [2, 5, 16, 33, 200])
def test_selection(cuda, hq, hkv, d, size, budget):
    """Exactly the spans that the sums in 64 bits choose, on both sides of the 256 spans that a block ranks at once."""
    g, lens = gen(budget), [1, 64, 65, 0, 128, 64 * budget, 64 * budget + 1, 5000, 64 * 256, 64 * 256 + 1, 21000]
    table, blocks = kh.block_lists(g, lens, size)
    summaries = torch.randn(blocks, hkv, size // 64, 2, d, generator=g).to(BF).sort(3).values
    q = torch.randn(len(lens), hq, d, generator=g).to(BF)
    want = kh.select(q, summaries, table, lens, budget)
    status = ops.new_status(cuda)
    args = (q.to(cuda), summaries.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), table.to(cuda), size, budget)
    got = ops.kv4_select(*args, status=status)
    ops.check_status(status)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(ops.kv4_select(*args, max_context=21000).cpu(), want)
    one = [a[7:8].contiguous() if i in (0, 2, 3) else a for i, a in enumerate(args)]      # few rows: clusters of blocks
    assert torch.equal(ops.kv4_select(*one).cpu(), want[7:8])
    ops.kv4_select(*args, max_context=20000, status=status)
    assert status[0].item() == 5 and status[1].item() == 10
    longest = args[2].clone()
    longest[10] = 2 ** 31 - 1                                       # longer than its list of blocks holds: cut there
    status = ops.new_status(cuda)
    cut = ops.kv4_select(*args[:2], longest, *args[3:], status=status)[10]
    assert status[0].item() == 5 and status[1].item() == 10 and (cut[:, -1] == table.shape[1] * (size // 64) - 1).all()


def test_selection_for_many_sequences(cuda):
    """More rows than SMs, on both sides of the 128 spans that such rows are ranked up to."""
    g, hkv, d, size, budget = gen(77), 8, 64, 256, 20
    lens = [64 * n + i % 3 for i, n in enumerate([1, 20, 21, 126, 127, 128, 129, 200, 255, 256, 257] * 3)]
    table, blocks = kh.block_lists(g, lens, size)
    summaries = torch.randn(blocks, hkv, size // 64, 2, d, generator=g).to(BF).sort(3).values
    q = torch.randn(len(lens), 16, d, generator=g).to(BF)
    got = ops.kv4_select(q.to(cuda), summaries.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), table.to(cuda), size, budget)
    assert torch.equal(got.cpu(), kh.select(q, summaries, table, lens, budget))


@pytest.mark.parametrize("count", [40, 500])
def test_selection_among_equals_takes_the_lower_index(cuda, count):
    """Equal sums (all, or from some span on), negative ones, and an infinity in a query."""
    hkv, d, budget, size = 2, 64, 9, 256
    table = torch.arange(-(-count // 4), dtype=torch.int32)[None]
    summaries = torch.zeros(table.shape[1], hkv, 4, 2, d, dtype=BF)
    flat = summaries.transpose(1, 2).flatten(0, 1)
    flat[:, 0] = -1.0
    flat[:, 1, 0], flat[:, 1, 1] = -3.0, -2.0
    flat[7::11, 1, 1] = -1.0
    summaries = flat.view(table.shape[1], 4, hkv, 2, d).transpose(1, 2).contiguous()
    q = torch.ones(1, 4, d, dtype=BF)
    got = ops.kv4_select(q.to(cuda), summaries.to(cuda), torch.tensor([64 * count], dtype=torch.int32, device=cuda), table.to(cuda), size, budget).cpu()
    assert torch.equal(got, kh.select(q, summaries, table, [64 * count], budget))
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, count - 1]
    q[0, 2, 5] = float("inf")
    got = ops.kv4_select(q.to(cuda), summaries.to(cuda), torch.tensor([64 * count], dtype=torch.int32, device=cuda), table.to(cuda), size, budget).cpu()
    assert ((got >= 0) & (got < count)).all() and (got[..., 1:] > got[..., :-1]).all()
    bad, status = table.clone(), ops.new_status(cuda)
    bad[0, 3] = 1 << 20
    ops.kv4_select(q.to(cuda), summaries.to(cuda), torch.tensor([64 * count], dtype=torch.int32, device=cuda), bad.to(cuda), size, budget, status=status)
    assert status[0].item() == 2


@pytest.mark.parametrize("hq,hkv,d,size", [(16, 8, 128, 256), (4, 1, 256, 128), (8, 2, 64, 64)])
def test_decode_over_spans(cuda, hq, hkv, d, size):
    lens, g = [5000, 64, 65, 1, 0, 700, 127], gen(21)
    spans = torch.full((len(lens), hkv, 6), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        count = -(-n // 64)
        for h in range(hkv):
            chosen = torch.randperm(count, generator=g)[:6].tolist() if count else []
            spans[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)          # in no order
    spans[5, 0] = torch.tensor([-1, 3, -1, -1, 10, -7])             # gaps, and the last span, which ends early
    run_decode(cuda, lens, hq, hkv, d, size=size, spans=spans, seed=22)
    spans[0, 0] = -1                                                # a head that reads nothing
    out = run_decode(cuda, lens, hq, hkv, d, size=size, spans=spans, seed=22)
    assert (out[0, :hq // hkv] == 0).all()
    long = torch.arange(100, dtype=torch.int32).repeat(1, hkv, 1)
    run_decode(cuda, [64 * 100 - 5], hq, hkv, d, size=size, spans=long, seed=23)         # a list of more than 32 entries: all tokens


def test_decode_reports_spans_outside_the_sequence(cuda):
    g = gen(2)
    table, blocks = kh.block_lists(g, [300, 300], 64)
    cache = kh.make_cache(g, blocks, 1, 64, 128)
    spans = torch.tensor([[[0, 4]], [[0, 5]]], dtype=torch.int32, device=cuda)           # spans 0 .. 4
    status = ops.new_status(cuda)
    out = ops.decode_attn4(torch.randn(2, 2, 128, generator=g).to(BF).to(cuda), on(cuda, cache), torch.tensor([300, 300], dtype=torch.int32, device=cuda),
                           table.to(cuda), 1.0, -1, ops.decode4_workspace(2, 2, 1, 128, cuda), spans=spans, status=status)
    assert status[0].item() == 5 and status[1].item() == 1 and torch.isfinite(out).all()


def test_a_step_of_all_of_them(cuda):
    """Prompts written, then single tokens: written, bounded, chosen and attended, as a decoding engine runs them; captured and replayed."""
    g, hq, hkv, d, size, budget = gen(31), 8, 2, 128, 128, 4
    lens = [500, 90, 1]
    table, blocks = kh.block_lists(g, [n + 2 for n in lens], size)
    cos = build_cos_sin_cache(d, 1024, 1e4, scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 256})
    cache = ops.KV4Cache.empty(blocks, size, hkv, d, cuda)
    for t in (cache.k_affine, cache.v_affine):
        t.fill_(float("nan"))
    summaries, ws = ops.kv4_summaries(cache), ops.decode4_workspace(3, hq, hkv, d, cuda)
    slot = lambda b, p: table[b, p // size] * size + p % size
    pos = torch.cat([torch.arange(n) for n in lens])
    slots = torch.cat([slot(b, torch.arange(n)) for b, n in enumerate(lens)]).to(torch.int32)
    x = torch.randn(len(pos), hq + 2 * hkv, d, generator=g).to(BF)
    dev = x.to(cuda)
    ops.rotary_kv4_write(dev[:, :hq], dev[:, hq:hq + hkv], dev[:, hq + hkv:], pos.to(cuda), cos.to(cuda), slots.to(cuda), cache)
    ops.kv4_summarise(cache, slots.to(cuda), summaries)
    plain = [t.cpu().clone() for t in (cache.k_codes, cache.k_affine, cache.v_codes, cache.v_affine)]
    step, pos_d, slot_d = torch.zeros(3, hq + 2 * hkv, d, dtype=BF, device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    lens_d, out, td, cd = torch.zeros(3, dtype=torch.int32, device=cuda), torch.zeros(3, hq, d, dtype=BF, device=cuda), table.to(cuda), cos.to(cuda)
    spans = torch.zeros(3, hkv, budget, dtype=torch.int32, device=cuda)
    q_d = torch.zeros(3, hq, d, dtype=BF, device=cuda)

    def run():
        ops.rotary_kv4_write(step[:, :hq], step[:, hq:hq + hkv], step[:, hq + hkv:], pos_d, cd, slot_d, cache, q_out=q_d)
        ops.kv4_summarise(cache, slot_d, summaries)
        ops.kv4_select(q_d, summaries, lens_d, td, size, budget, out=spans)
        ops.decode_attn4(q_d, cache, lens_d, td, d ** -0.5, -1, ws, spans=spans, out=out)

    slot_d.fill_(-1)
    run()                                                           # nothing cached, nothing read
    assert (out == 0).all() and (spans == -1).all()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for k in range(2):
        now = [n + k for n in lens]
        y = torch.randn(3, hq + 2 * hkv, d, generator=g).to(BF)
        p = torch.tensor(now)
        step.copy_(y); pos_d.copy_(p); lens_d.copy_((p + 1).int())
        s = torch.stack([slot(b, p[b]) for b in range(3)])
        slot_d.copy_(s.int())
        graph.replay()
        torch.cuda.synchronize()
        q, key = (kh.turn(t, p, cos, False, torch.float32).to(BF) for t in (y[:, :hq], y[:, hq:hq + hkv]))
        assert torch.equal(q_d.cpu(), q)
        at = (s.long() // size, slice(None), s.long() % size)
        for i, rows, keys in ((0, key, True), (2, y[:, hq + hkv:], False)):
            plain[i][at], plain[i + 1][at] = kh.quantise(rows, keys)
        seen = [n + 1 for n in now]
        assert torch.equal(cache.k_codes.cpu()[at], plain[0][at])
        tight = torch.zeros_like(summaries.cpu())
        for b, n in enumerate(seen):
            kk = kh.context(plain, table, b, n, torch.float32)[0]
            for j in range(-(-n // 64)):
                part = kk[:, 64 * j:min(n, 64 * j + 64)]
                tight[table[b, 64 * j // size], :, 64 * j % size // 64] = torch.stack([part.amin(1), part.amax(1)], 1).to(BF)
        want = kh.select(q, tight, table, seen, budget)
        assert torch.equal(spans.cpu(), want)
        kh.assert_decode(out, *kh.decode(q, plain, table, seen, d ** -0.5, spans=want), f"step {k}")


def test_a_cache_whose_offsets_pass_32_bits(cuda):
    """The last blocks of 18 M slots (2.3 GB of codes a side) hold and give what the first ones do, bit for bit."""
    g, hq, hkv, d, size, blocks, n = gen(40), 8, 1, 256, 256, 70000, 1500
    cache = ops.KV4Cache.empty(blocks, size, hkv, d, cuda)
    summaries, ws = ops.kv4_summaries(cache), ops.decode4_workspace(2, hq, hkv, d, cuda)
    x = torch.randn(n, hq + 2 * hkv, d, generator=g).to(BF).to(cuda)
    pos = torch.arange(n, device=cuda)
    cos = build_cos_sin_cache(d, n, 1e4).to(cuda)
    used = -(-n // size)
    near = torch.arange(used, dtype=torch.int32, device=cuda)[None]
    far = blocks - 1 - near
    assert blocks * size * (d // 2) > 2 ** 31
    got = []
    for table in (near, far):
        slots = (table[0].repeat_interleave(size) * size + torch.arange(size, dtype=torch.int32, device=cuda).repeat(used))[:n].contiguous()
        q = ops.rotary_kv4_write(x[:, :hq], x[:, hq:hq + 1], x[:, hq + 1:], pos, cos, slots, cache, q_out=torch.empty(n, hq, d, dtype=BF, device=cuda))
        ops.kv4_summarise(cache, slots, summaries)
        lens, last, status = torch.tensor([n], dtype=torch.int32, device=cuda), q[-1:], ops.new_status(cuda)
        spans = ops.kv4_select(last, summaries, lens, table, size, 6, status=status)
        rows = ops.kv4_gather(cache, torch.tensor([0, n], dtype=torch.int32, device=cuda), table, n, status=status)
        got.append((spans, *rows, ops.decode_attn4(last, cache, lens, table, d ** -0.5, -1, ws, status=status),
                    ops.decode_attn4(last, cache, lens, table, d ** -0.5, -1, ws, spans=spans, status=status)))
        ops.check_status(status)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.equal(got[1][2].cpu(), kh.stored(x[:, hq + 1:].cpu(), False, torch.float32).to(BF))
