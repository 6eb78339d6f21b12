"""The TSV dump refuses formats that it has no lines for, before it reads or writes anything."""
import pytest

from bonsai_vk_amd import BKV_F16, BKV_Q4_0, BKV_Q8_0, KvCache, kvdump


@pytest.mark.parametrize("k_fmt, v_fmt", [(BKV_Q4_0, BKV_Q4_0), (BKV_Q8_0, BKV_Q4_0), (BKV_Q4_0, BKV_F16)])
def test_four_bits_are_refused(k_fmt, v_fmt, tmp_path):
    cache = KvCache(n_layers=1, nh=4, nkv=1, cap=8, k_fmt=k_fmt, v_fmt=v_fmt, device="cpu")
    for n in (0, 3):
        with pytest.raises(ValueError, match="fp16 and q8_0"):
            kvdump.dump_cache(cache, 0, n, tmp_path / "dump.tsv")
        with pytest.raises(ValueError, match="fp16 and q8_0"):
            list(kvdump.dump_lines(cache.host_arrays(), 0, n, 8, 1, 256, k_fmt, v_fmt))
    assert not (tmp_path / "dump.tsv").exists()
