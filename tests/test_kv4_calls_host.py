"""Calls around the 4-bit cache that are refused, and what the wrappers hand to the C entries (nothing is launched: no address is followed)."""
import ctypes

import pytest

from mini_vllm_b200 import _cabi

A, B = 1 << 20, 1 << 21


def cache_struct():
    return ctypes.byref(_cabi.KV4Cache(A, A, A, A, 8, 256, 2, 128))


@pytest.mark.parametrize("k,v,in_place,cs,tokens,want", [(A, A, 1, A, 0, 0), (A, A, 1, A, 4, -1)])
def test_values_apart_from_keys_that_are_turned_in_place(k, v, in_place, cs, tokens, want):
    """The values are read while the keys are written: one tensor cannot be both."""
    assert _cabi.load().mvb_rotary_kv4_write(None, 0, None, 0, k, 256, v, 256, A, cs, 9, 128, 0, A, cache_struct(), tokens, 0, in_place, None, None) == want
