"""Pages of several sequences: fork, extend and compact (bkv_pages_*) against one page after another in Python. (No
counterpart in the reference.)"""
import numpy as np
import pytest
import torch

from seqs_util import Pages, arrays, copied, device_ints, make, random_bytes

pytestmark = pytest.mark.gpu


def same(seqs, want, before=None, copies=None):
    torch.cuda.synchronize()
    assert np.array_equal(seqs.tables.cpu().numpy(), want.tables)
    assert np.array_equal(seqs.refs.cpu().numpy(), want.refs)
    assert np.array_equal(seqs.len.cpu().numpy(), want.len)
    if before is not None:
        for a, b in zip(arrays(seqs.cache), copied(before, copies, want.page)):
            assert torch.equal(a, b)


def count(seqs):
    """refs as the tables say."""
    t, n = seqs.tables.cpu().numpy(), seqs.refs.shape[1]
    return np.stack([np.bincount(t[:, layer].reshape(-1)[(t[:, layer].reshape(-1) >= 0) & (t[:, layer].reshape(-1) < n)], minlength=n)
                     for layer in range(t.shape[1])])


def extend(seqs, n_new, want):
    before = [a.clone() for a in arrays(seqs.cache)]
    lack = seqs.extend(device_ints(n_new))
    said, copies = want.extend(n_new)
    assert lack.tolist() == said
    same(seqs, want, before, copies)
    return said


@pytest.mark.parametrize("k, v", [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("f16", "f16"), ("f16", "q8_0")])
@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("nkv", [1, 4])
def test_a_life_of_sequences(k, v, page, nkv):
    """Prompts, forks, copies on write, ends and compactions in any order: counts, tables and every byte of the pool."""
    r = np.random.default_rng(page * 7 + nkv)
    cache, seqs = make([0] * 9, page, nkv, 2, k, v, layers=3, cap=page * 60, room=40 * page)
    random_bytes(cache, page)
    want = Pages(seqs)
    for step in range(25):
        what = r.integers(0, 6)
        if what <= 2:
            n = [int(x) for x in r.integers(0, 2 * page + 2, 9)]
            if not any(extend(seqs, n, want)):
                want.len += np.array(n, np.int32)
                seqs.len += device_ints(n)
        elif what <= 4:
            parent = [int(x) for x in r.integers(-1 if what == 4 else 0, 9, 9)]
            seqs.fork(device_ints(parent))
            want.fork(parent)
            same(seqs, want)
        else:
            before = [a.clone() for a in arrays(cache)]
            seqs.compact()
            same(seqs, want, before, want.compact())
        assert np.array_equal(count(seqs), want.refs)


@pytest.mark.parametrize("hd, nkv", [(64, 1), (64, 3), (128, 1), (192, 2)])
@pytest.mark.parametrize("page", [3, 16])
def test_rows_of_few_scales(hd, nkv, page):
    """4, 12, 8 and 24 bytes of scales a position: what is held of a page ends inside 16 bytes, and so may a page begin."""
    cache, seqs = make([0] * 4, page, nkv, 2, "q8_0", "q4_0", layers=2, cap=page * 40, room=10 * page, hd=hd)
    random_bytes(cache, hd + page)
    want = Pages(seqs)
    for n in ([page - 1, 1, 2 * page + 2, 5], [1, 2, 3, 1]):
        extend(seqs, n, want)
        want.len += np.array(n, np.int32)
        seqs.len += device_ints(n)
        parent = [0, 0, 2, 2] if page == 3 else [3, 1, 3, 2]
        seqs.fork(device_ints(parent))
        want.fork(parent)
        extend(seqs, [1, 1, 1, 1], want)
        before = [a.clone() for a in arrays(cache)]
        seqs.compact()
        same(seqs, want, before, want.compact())


def test_the_last_keeps_a_page_that_nobody_else_would():
    cache, seqs = make([0] * 4, 16, layers=2, cap=16 * 20, room=64)
    random_bytes(cache)
    want = Pages(seqs)
    extend(seqs, [20, 0, 0, 0], want)
    for p in (want.len, seqs.len):
        p[0] = 20
    for parent, n in (([0, 0, 0, 0], [1, 1, 1, 1]), ([0, 0, 0, 0], [1, 0, 1, 0]), ([2, 2, 2, -1], [0, 1, 1, 0]), ([3, 0, 0, 0], [5, 5, 5, 40])):
        seqs.fork(device_ints(parent))
        want.fork(parent)
        extend(seqs, n, want)


def test_nothing_changes_where_pages_lack():
    """One layer is short of one page: no layer is touched. Rows that are too short, lengths past them."""
    cache, seqs = make([0] * 3, 16, layers=3, cap=16 * 6, room=64)
    random_bytes(cache)
    seqs.refs[1, 2] = 1                            # (in use by something else)
    want = Pages(seqs)
    assert extend(seqs, [32, 32, 32], want) == [0, 1, 0]
    assert extend(seqs, [16, 65, 0], want) == [1, 1, 1]
    assert extend(seqs, [32, 32, 16], want) == [0, 0, 0]
    seqs.len.copy_(device_ints([64, 70, 1000]))
    want.len = np.array([64, 70, 1000], np.int32)
    assert extend(seqs, [1, 0, 0], want) == [1, 1, 1]
    assert extend(seqs, [0, 3, 40], want) == [4, 4, 4]
    assert extend(seqs, [0, 0, 0], want) == [0, 0, 0]
    assert extend(seqs, [-5, 0, -1], want) == [0, 0, 0]


def test_very_many_new_positions_are_a_lack():
    cache, seqs = make([0] * 2, 1, nkv=1, grp=1, cap=50, room=40)
    seqs.len.copy_(device_ints([7, -3]))
    lack = seqs.extend(device_ints([2**31 - 1, 2**31 - 1]))
    assert lack.tolist()[0] > 50 and int((seqs.tables >= 0).sum()) == 0 and int(seqs.refs.sum()) == 0


def test_entries_outside_the_pool():
    """They name nothing: no count, no copy; a fork carries them along, an extend replaces them, a compaction leaves them."""
    cache, seqs = make([40, 40], 16, layers=2, room=80)
    random_bytes(cache)
    seqs.tables[0, 0, 4], seqs.tables[1, 1, 4], seqs.tables[1, 0, 3] = 2**31 - 1, cache.cap // 16, -2**31
    want = Pages(seqs)
    seqs.fork(device_ints([1, 0]))
    want.fork([1, 0])
    same(seqs, want)
    before = [a.clone() for a in arrays(cache)]
    seqs.compact()
    same(seqs, want, before, want.compact())
    extend(seqs, [40, 0], want)


def test_parents_outside_the_sequences_empty_a_row():
    cache, seqs = make([40, 16, 1, 30], 16, layers=2)
    want = Pages(seqs)
    parent = [-1, 4, 2, 2**31 - 1]
    seqs.fork(device_ints(parent))
    want.fork(parent)
    same(seqs, want)
    assert seqs.len.tolist() == [0, 0, 1, 0] and int(seqs.refs.sum()) == 2


@pytest.mark.parametrize("n", [1, 15, 16, 17, 255, 1024])
def test_many_sequences_and_long_tables(n):
    r = np.random.default_rng(n)
    cache, seqs = make([int(x) for x in r.integers(1, 30, n)], 2, 1, 1, layers=1, room=70, spare=n + 7)
    random_bytes(cache)
    want = Pages(seqs)
    parent = [int(x) for x in r.integers(0, n, n)]
    seqs.fork(device_ints(parent))
    want.fork(parent)
    same(seqs, want)
    extend(seqs, [1] * n, want)
    for parent in ([n - 1] * n, [n - 1] * n, [-1] * (n - 1) + [0]):   # (all from one; nothing new; one is left)
        seqs.fork(device_ints(parent))
        want.fork(parent)
        same(seqs, want)
        extend(seqs, [2] * n, want)
    before = [a.clone() for a in arrays(cache)]
    seqs.compact()
    same(seqs, want, before, want.compact())


def test_large_pools():
    """More pages than a workgroup looks at at once, few of them used, and a long first prompt."""
    cache, seqs = make([0, 0], 4, 1, 1, cap=4 * 20011, room=4 * 15000)
    r = np.random.default_rng(5)
    taken = r.random(20011) < 0.1
    seqs.refs[0] = torch.from_numpy(taken.astype(np.int32)).cuda()
    want = Pages(seqs)
    random_bytes(cache)
    assert extend(seqs, [4 * 14000 + 1, 4 * 3000], want) == [0]
    parent = [-1, 1]
    seqs.fork(device_ints(parent))
    want.fork(parent)
    before = [a.clone() for a in arrays(cache)]
    seqs.compact()
    same(seqs, want, before, want.compact())


def test_compact_beside_the_old_tables():
    """The new tables elsewhere: the old ones and the bytes that they name stay."""
    cache, seqs = make([0] * 5, 16, layers=2, cap=16 * 40, room=160)
    random_bytes(cache)
    want = Pages(seqs)
    extend(seqs, [33, 100, 17, 64, 90], want)
    seqs.fork(device_ints([0, -1, 2, 2, 4]))
    want.fork([0, -1, 2, 2, 4])
    tables, refs = torch.empty_like(seqs.tables), torch.empty_like(seqs.refs)
    old = seqs.tables.clone(), seqs.refs.clone()
    before = [a.clone() for a in arrays(cache)]
    got = seqs.compact(tables, refs)
    assert got[0] is tables and got[1] is refs
    assert torch.equal(old[0], seqs.tables) and torch.equal(old[1], seqs.refs)
    copies = want.compact()
    assert np.array_equal(tables.cpu().numpy(), want.tables) and np.array_equal(refs.cpu().numpy(), want.refs)
    for a, b in zip(arrays(cache), copied(before, copies, 16)):
        assert torch.equal(a, b)
    assert copies and all(refs[layer, b] > 0 and old[1][layer, a] > 0 for layer, a, b, _ in copies)


def test_an_empty_and_a_full_pool():
    cache, seqs = make([0, 0], 16, layers=2, cap=16 * 8, room=128)
    want = Pages(seqs)
    random_bytes(cache)
    before = [a.clone() for a in arrays(cache)]
    seqs.compact()
    same(seqs, want, before, want.compact())
    extend(seqs, [64, 64], want)
    seqs.compact()
    same(seqs, want, None, want.compact())


def test_replays_of_a_captured_step():
    """fork, extend and compact in one graph, from different tables at every replay."""
    cache, seqs = make([0] * 6, 16, layers=2, cap=16 * 60, room=160)
    random_bytes(cache)
    want = Pages(seqs)
    n0 = [40, 25, 60, 3, 0, 16]
    extend(seqs, n0, want)
    seqs.len += device_ints(n0)
    want.len += np.array(n0, np.int32)
    parent, n_new, lack = device_ints([0] * 6), device_ints([1] * 6), device_ints([0, 0])
    graph = torch.cuda.CUDAGraph()
    start = [x.clone() for x in (seqs.tables, seqs.refs, seqs.len)]
    with torch.cuda.graph(graph):
        seqs.fork(parent)
        seqs.extend(n_new, lack)
        seqs.compact()
    for x, y in zip((seqs.tables, seqs.refs, seqs.len), start):
        assert torch.equal(x, y)
    for p, n in (([0, 0, 1, 1, 2, 2], [1, 1, 1, 1, 1, 1]), ([5, 4, 3, 2, 1, 0], [0, 20, 3, 0, 7, 1]), ([1, 1, 1, 1, 1, 1], [16, 1, 2, 0, 0, 5]),
                 ([-1, 0, -1, 0, 0, 9], [5, 0, 0, 1, 0, 0])):
        parent.copy_(device_ints(p))
        n_new.copy_(device_ints(n))
        before = [a.clone() for a in arrays(cache)]
        graph.replay()
        torch.cuda.synchronize()
        want.fork(p)
        said, first = want.extend(n)
        then = want.compact()
        mid = copied(before, first, 16)
        assert lack.tolist() == said
        same(seqs, want, mid, then)


def test_bytes_past_4_gib():
    cache, seqs = make([0, 0], 64, cap=64 * 147500, room=640)
    assert cache.k_data.numel() > 1 << 32
    n = seqs.refs.shape[1]
    seqs.refs[0, :n - 3] = 1
    seqs.refs[0, 5] = 0
    part = [a[0, (n - 3) * 64:] for a in arrays(cache)]
    for i, a in enumerate(part):
        a.copy_(torch.randint(0, 256, a.shape, dtype=torch.uint8, device="cuda"))
    seqs.tables[0, 0, 0] = seqs.tables[1, 0, 0] = n - 1
    seqs.refs[0, n - 1] = 2
    seqs.len.copy_(device_ints([50, 50]))
    seqs.refs[0, 5] = 1
    last = [a[0, (n - 1) * 64:(n - 1) * 64 + 50].clone() for a in arrays(cache)]
    assert seqs.extend(device_ints([1, 1])).tolist() == [0]
    assert seqs.tables[0, 0, 0] == n - 3 and seqs.tables[1, 0, 0] == n - 1
    for a, b in zip(arrays(cache), last):
        assert torch.equal(a[0, (n - 3) * 64:(n - 3) * 64 + 50], b)
    seqs.refs[0, 7] = 0
    seqs.compact()
    assert seqs.tables[0, 0, 0] == n - 3 and seqs.tables[1, 0, 0] == 7
    for a, b in zip(arrays(cache), last):
        assert torch.equal(a[0, 7 * 64:7 * 64 + 50], b)
