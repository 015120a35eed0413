"""Which layers a cache in 4 bits stands in for, and how much of the pool's memory goes to unpacked contexts (no GPU)."""
import pytest
import torch

from mini_vllm_b200.models.layers.branches import AttentionBranch, alibi_slopes

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
