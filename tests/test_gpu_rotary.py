"""Rotation in either pairing and for part of the head (CUDA) against the formula in 64 bits."""
import pytest
import torch

from mini_vllm_b200 import ops
from mini_vllm_b200.models.layers.rotary import RotaryEmbedding, build_cos_sin_cache
from tests.kv4_helpers import turn

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def check(got, x, pos, table, inter):
    """Two products and a sum in fp32, each off by half a step of what it is (the products' sizes bound all three): 3 * 2^-24 (|a c| + |b s|);
    then half a step of the type."""
    want = turn(x, pos, table, inter)
    rot = table.shape[1]
    c, s = (t[:, None].double() for t in table[pos].split(rot // 2, -1))
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    size = torch.zeros_like(want)
    a, b = x[..., one].double().abs(), x[..., two].double().abs()
    size[..., one], size[..., two] = a * c.abs() + b * s.abs(), b * c.abs() + a * s.abs()
    bound = size * 3 * 2.0 ** -24 + want.abs() * torch.finfo(x.dtype).eps / 2 * (1 + 2.0 ** -20)
    assert ((got.double().cpu() - want).abs() <= bound).all()
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])          # the others: carried along, bit by bit


SHAPES = [(1, 1, 1, 128, 128), (7, 16, 8, 128, 64), (64, 12, 4, 80, 20), (301, 3, 1, 96, 96), (33, 2, 2, 64, 2), (5, 4, 1, 256, 130),
          (3000, 16, 8, 128, 128), (2500, 5, 3, 64, 32)]


@pytest.mark.parametrize("tokens,hq,hkv,d,rot", SHAPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_against_the_formula(cuda, tokens, hq, hkv, d, rot, inter, dtype):
    g = torch.Generator().manual_seed(tokens + rot)
    table = build_cos_sin_cache(rot, 5000, 1e4, scaling={"rope_type": "linear", "factor": 2.0})
    packed = torch.randn(tokens, (hq + hkv) * d + 8, generator=g).to(dtype)
    q, k = packed[:, :hq * d].view(tokens, hq, d), packed[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    pos = torch.randint(0, 5000, (tokens,), generator=g)
    dev = packed.to(cuda)
    qd, kd = dev[:, :hq * d].view(tokens, hq, d), dev[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    status = ops.new_status(cuda)
    q_out, k_out = ops.rotary(qd, kd, pos.to(cuda), table.to(cuda), interleaved=inter, q_out=torch.full((tokens, hq, d), float("nan"), dtype=dtype, device=cuda),
                              k_out=torch.full((tokens, hkv, d), float("nan"), dtype=dtype, device=cuda), status=status)
    check(q_out, q, pos, table, inter)
    check(k_out, k, pos, table, inter)
    assert torch.equal(dev.cpu(), packed)                           # the inputs are as they were
    ops.rotary(qd, kd, pos.to(cuda), table.to(cuda), interleaved=inter, status=status)           # in place: the same bits
    assert torch.equal(qd, q_out) and torch.equal(kd, k_out) and torch.equal(dev[:, (hq + hkv) * d:].cpu(), packed[:, (hq + hkv) * d:])
    ops.check_status(status)


@pytest.mark.parametrize("inter", [False, True])
def test_one_side_only_and_unaligned_rows(cuda, inter):
    g = torch.Generator().manual_seed(2)
    table = build_cos_sin_cache(64, 100, 1e4)
    flat = torch.randn(40 * 131 + 3, generator=g).to(BF)
    x = flat.as_strided((40, 1, 128), (131, 128, 1), 3)             # rows that no vector load reaches
    pos = torch.arange(40)
    dev = flat.to(cuda)
    xd = dev.as_strided((40, 1, 128), (131, 128, 1), 3)
    out, none = ops.rotary(xd, None, pos.to(cuda), table.to(cuda), interleaved=inter, q_out=torch.empty(40, 1, 128, dtype=BF, device=cuda))
    assert none is None
    check(out, x, pos, table, inter)
    none, out = ops.rotary(None, xd, pos.to(cuda), table.to(cuda), interleaved=inter)
    assert none is None and out is xd
    check(out, x, pos, table, inter)


def test_no_tokens_and_positions_outside_the_table(cuda):
    table = build_cos_sin_cache(64, 16, 1e4).to(cuda)
    q = torch.randn(3, 2, 64, device=cuda)
    assert ops.rotary(q[:0], None, torch.zeros(0, dtype=torch.int64, device=cuda), table)[0].shape == (0, 2, 64)
    status, was = ops.new_status(cuda), q.clone()
    ops.rotary(q, None, torch.tensor([1, 16, -1], device=cuda), table, status=status)
    assert status[0].item() == 3 and torch.equal(q[1:], was[1:]) and not torch.equal(q[0], was[0])


def test_refusals(cuda):
    table, pos = torch.zeros(8, 64, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    q = torch.zeros(2, 2, 64, device=cuda, dtype=BF)
    for bad in (lambda: ops.rotary(q, q.float(), pos, table), lambda: ops.rotary(q, None, pos.int(), table), lambda: ops.rotary(q, None, pos, table.double()),
                lambda: ops.rotary(q, None, pos, table, q_out=q.float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.rotary(q, None, pos[:1], table), lambda: ops.rotary(q.transpose(1, 2), None, pos, table),
                lambda: ops.rotary(q, None, pos, table[:, ::2]), lambda: ops.rotary(q, None, pos, table, q_out=q[:1]),
                lambda: ops.rotary(q, q[:, :, :32], pos, table), lambda: ops.rotary(q, None, pos, table, k_out=q), lambda: ops.rotary(q[0], None, pos, table)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ops._cabi.KernelError):
        ops.rotary(q[..., :32].contiguous(), None, pos, table)       # more rotated channels than the head has


def test_capture_and_another_stream(cuda):
    table = build_cos_sin_cache(128, 64, 1e4).to(cuda)
    x = torch.randn(9, 2, 128, device=cuda, dtype=BF)
    pos, out = torch.zeros(9, dtype=torch.int64, device=cuda), torch.empty_like(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.rotary(x, None, pos, table, q_out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.rotary(x, None, pos, table, q_out=out)
    torch.cuda.current_stream().wait_stream(stream)
    pos.copy_(torch.arange(9))
    graph.replay()
    torch.cuda.synchronize()
    check(out, x.cpu(), torch.arange(9), table.cpu(), False)


@pytest.mark.parametrize("inter,rot,dtype", [(True, 64, BF), (False, 32, BF), (False, 64, F32)])
def test_embedding_module_takes_every_form(cuda, inter, rot, dtype):
    emb = RotaryEmbedding(rot, 512, 1e4, device=cuda, scaling={"rope_type": "linear", "factor": 2.0}, interleaved=inter)
    q, k = torch.randn(17, 4, 64).to(dtype), torch.randn(17, 2, 64).to(dtype)
    pos = torch.arange(100, 117)
    qd, kd = q.to(cuda), k.to(cuda)
    got = emb(pos.to(cuda), qd, kd)
    assert got[0] is qd and got[1] is kd
    for a, x in ((qd, q), (kd, k)):
        check(a, x, pos, emb.cos_sin_cache.cpu(), inter)
