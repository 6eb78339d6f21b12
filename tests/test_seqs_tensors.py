"""What may be put in the place of KvSeqs' tables and counts. (No counterpart in the reference.)"""
import pytest
import torch

from bonsai_vk_amd import BKV_Q4_0, KvCache, KvSeqs

from seqs_util import Pages, device_ints, make


def paged():
    cache = KvCache(n_layers=2, nh=4, nkv=1, cap=64, k_fmt=BKV_Q4_0, v_fmt=BKV_Q4_0, page_tokens=16, max_pages=3,
                    block_table=torch.full((2, 3), -1), device="cpu")
    return KvSeqs(cache, 5)


@pytest.mark.parametrize("name, shape", [("tables", (5, 2, 3)), ("refs", (2, 4))])
def test_tensors_of_another_kind_are_refused(name, shape):
    seqs = paged()
    old = getattr(seqs, name)
    assert tuple(old.shape) == shape
    larger = tuple(2 * n for n in shape)
    for bad in (torch.zeros(shape, dtype=torch.int64), torch.zeros(shape[:-1], dtype=torch.int32), torch.zeros((shape[0] - 1, *shape[1:]), dtype=torch.int32),
                torch.zeros(larger, dtype=torch.int32)[tuple(slice(0, None, 2) for _ in shape)]):
        with pytest.raises(ValueError):
            setattr(seqs, name, bad)
        assert getattr(seqs, name) is old
    new = torch.ones(shape, dtype=torch.int32)
    setattr(seqs, name, new)
    assert getattr(seqs, name) is new and seqs.desc.block_table == seqs.tables.data_ptr()


def test_a_contiguous_cache_has_none():
    seqs = KvSeqs(KvCache(n_layers=1, nh=4, nkv=1, cap=64, k_fmt=BKV_Q4_0, v_fmt=BKV_Q4_0, device="cpu"), 1)
    assert seqs.tables is None and seqs.refs is None
    for name in ("tables", "refs"):
        with pytest.raises(ValueError, match="no pages"):
            setattr(seqs, name, torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
def test_host_tensors_are_refused_and_compacted_ones_taken():
    cache, seqs = make([40, 20, 0], 16, layers=2, spare=9, room=80)
    for name in ("tables", "refs"):
        with pytest.raises(ValueError):
            setattr(seqs, name, getattr(seqs, name).cpu())
    want = Pages(seqs)
    want.compact()
    seqs.tables, seqs.refs = seqs.compact(torch.empty_like(seqs.tables), torch.empty_like(seqs.refs))
    assert (seqs.tables.cpu().numpy() == want.tables).all() and (seqs.refs.cpu().numpy() == want.refs).all()
    assert seqs.extend(device_ints([1, 20, 3])).tolist() == want.extend([1, 20, 3])[0] == [0, 0]
    assert (seqs.tables.cpu().numpy() == want.tables).all() and (seqs.refs.cpu().numpy() == want.refs).all()
    seqs.fork(device_ints([1, 1, -1]))
    want.fork([1, 1, -1])
    assert (seqs.tables.cpu().numpy() == want.tables).all() and (seqs.refs.cpu().numpy() == want.refs).all()
