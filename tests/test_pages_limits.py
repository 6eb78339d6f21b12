"""Pages and pools that are too large for the page calls' counts. (No counterpart in the reference. No GPU: every call is refused, the
ones within the limits for their missing workspace.)"""
import pytest

from bonsai_vk_amd._lib import BKV_F16, BKV_Q4_0, BKV_Q8_0, BkvCacheDesc, lib

EWORKSPACE, EUNSUPPORTED = -5, -7
PTR = 0x7F0000000000                               # (an address that is never followed)


def answers(hd, nkv, k_fmt, v_fmt, page, pages=1):
    """What extend and compact say to a pool of `pages` pages of `page` positions, without a workspace."""
    d = BkvCacheDesc()
    d.n_layers, d.nh, d.nkv, d.hd, d.cap, d.k_fmt, d.v_fmt, d.scale = 1, nkv, nkv, hd, page * pages, k_fmt, v_fmt, 0.0625
    d.k_data = d.k_scales = d.v_data = d.v_scales = d.block_table = PTR
    for i in range(4):
        d.layer_stride_bytes[i] = 1 << 50
    d.page_tokens, d.max_pages = page, 1
    return {lib().bkv_pages_extend(d, 1, PTR, PTR, PTR, PTR, PTR, None, 0, None), lib().bkv_pages_compact(d, 1, PTR, PTR, PTR, PTR, None, 0, None)}


# (chunks of 16 bytes, or of 4 where a position's scales are fewer: 2^31 of them a page)
@pytest.mark.parametrize("hd, nkv, k_fmt, v_fmt, chunks", [(256, 4, BKV_Q4_0, BKV_Q4_0, 72), (256, 1, BKV_Q8_0, BKV_F16, 49), (64, 1, BKV_Q8_0, BKV_Q4_0, 26),
                                                           (128, 1, BKV_F16, BKV_Q4_0, 82)])
def test_a_page_of_more_chunks_than_are_counted(hd, nkv, k_fmt, v_fmt, chunks):
    most = (1 << 31) // chunks
    assert answers(hd, nkv, k_fmt, v_fmt, most) == {EWORKSPACE}
    assert answers(hd, nkv, k_fmt, v_fmt, most + 1) == {EUNSUPPORTED}
    assert answers(hd, nkv, k_fmt, v_fmt, min(2 * most, 2**31 - 1)) == {EUNSUPPORTED}
    assert answers(hd, nkv, k_fmt, v_fmt, 64) == {EWORKSPACE}


def test_a_page_whose_bytes_pass_64_bits():
    assert answers(1 << 30, 1 << 30, BKV_F16, BKV_F16, 1 << 30) == {EUNSUPPORTED}


def test_a_pool_of_more_pages_than_are_counted():
    assert answers(64, 1, BKV_Q8_0, BKV_Q4_0, 1, 1 << 30) == {EWORKSPACE}
    for pages in ((1 << 30) + 1, 2**31 - 1):
        assert answers(64, 1, BKV_Q8_0, BKV_Q4_0, 1, pages) == {EUNSUPPORTED}
    d = BkvCacheDesc()
    d.n_layers, d.nh, d.nkv, d.hd, d.cap, d.scale, d.page_tokens, d.max_pages = 1, 1, 1, 64, 2**31 - 1, 0.0625, 1, 1
    d.k_data = d.v_data = d.block_table = PTR
    assert lib().bkv_pages_workspace_bytes(d) == 0
    assert lib().bkv_pages_fork(d, 1, PTR, PTR, None, PTR, None) == EUNSUPPORTED
