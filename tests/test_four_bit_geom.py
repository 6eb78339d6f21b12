"""The geometry of a 4-bit cache on the Python side: words and bytes of a slot as the library has them, and the block policy that
counts by them."""
import ctypes

import pytest

from bonsai_vk_amd import BKV_F16, BKV_Q4_0, BKV_Q8_0, BkvCacheDesc, KvCache, lib
from bonsai_vk_amd.cache import KvGeom
from bonsai_vk_amd.guard import KvGuard

FORMATS = [BKV_F16, BKV_Q8_0, BKV_Q4_0]


def slot_bytes(nkv, hd, k_fmt, v_fmt):
    d = BkvCacheDesc()
    d.n_layers, d.nh, d.nkv, d.hd, d.cap, d.k_fmt, d.v_fmt = 1, nkv, nkv, hd, 1, k_fmt, v_fmt
    return [lib().bkv_slot_bytes(ctypes.byref(d), i) for i in range(4)]


@pytest.mark.parametrize("nkv, hd", [(4, 256), (1, 64), (3, 128), (8, 512)])
@pytest.mark.parametrize("k_fmt", FORMATS)
@pytest.mark.parametrize("v_fmt", FORMATS)
def test_words_of_every_format(nkv, hd, k_fmt, v_fmt):
    g = KvGeom(nkv=nkv, hd=hd, n_attn=5, v_q8=int(v_fmt == BKV_Q8_0), k_q8=int(k_fmt == BKV_Q8_0), v_q4=int(v_fmt == BKV_Q4_0), k_q4=int(k_fmt == BKV_Q4_0))
    kd, ks, vd, vs = slot_bytes(nkv, hd, k_fmt, v_fmt)
    assert (4 * g.w_k, 4 * g.w_vd, 4 * g.w_vs) == (kd + ks, vd, vs)
    assert g.bytes_slot == 5 * (kd + ks + vd + vs) and g.check() == ""


def test_a_cache_and_its_blocks():
    cache = KvCache(n_layers=8, nh=16, nkv=4, cap=64, k_fmt=BKV_Q4_0, v_fmt=BKV_Q4_0, device="cpu")
    assert cache.geom.bytes_slot == 9216 == sum(x.shape[2] for x in (cache.k_data, cache.k_scales, cache.v_data, cache.v_scales)) * 8
    assert KvGuard(blk_slots=16).init(cache.geom, cache.cap, 1 << 30, evict=False).bytes_per_blk == 16 * 9216
    for k, v, size in ((BKV_Q8_0, BKV_Q4_0, 1024 + 64 + 512 + 64), (BKV_Q4_0, BKV_F16, 512 + 64 + 2048)):
        g = KvCache(n_layers=1, nh=16, nkv=4, cap=8, k_fmt=k, v_fmt=v, device="cpu").geom
        assert g.bytes_slot == size
