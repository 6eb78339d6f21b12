"""Heads so many that the drafted-token kernels' 32-bit numbers would not hold a slot's bytes: refused before anything
is launched (no GPU is touched)."""
import pytest

from tests.test_abi import call, desc
from tests.test_tree_host import ECAP, EUNSUPPORTED, EWORKSPACE, Z, tree


def wide(nkv, fmt):
    return desc(nkv=nkv, nh=nkv, cap=64, n_layers=1, k_fmt=fmt, v_fmt=fmt)


@pytest.mark.parametrize("fmt,row", [(0, 512), (1, 256)])
def test_attn_tree_refuses_steps_of_more_than_32_bits(fmt, row):
    """31 slots' bytes, the last key of a step, are counted in 32 bits."""
    most = (2**32 - 1 - row) // (31 * row)         # heads
    assert tree(wide(most, fmt), pos0=10, n=1, ws=None) == EWORKSPACE    # (as far as the next check)
    assert tree(wide(most + 1, fmt), pos0=10, n=1, ws=None) == EUNSUPPORTED
    one = desc(nkv=most + 1, nh=most + 1, cap=64, n_layers=1, k_fmt=fmt, v_fmt=1 - fmt)   # (either tensor's)
    assert tree(one, pos0=10, n=1, ws=None) == EUNSUPPORTED
    assert tree(wide(most + 1, fmt), pos0=64, n=1, ws=None) == ECAP


@pytest.mark.parametrize("fmt,row", [(0, 512), (1, 256)])
def test_commit_refuses_slots_of_more_than_31_bits(fmt, row):
    heads = 2**31 // row
    assert call("bkv_kv_commit", wide(heads, fmt), 0, 8, 4, None, None) == EUNSUPPORTED
    assert call("bkv_kv_commit", wide(heads - 1, fmt), 0, 8, 4, Z + 2, None) == -4          # (as far as the next check)
