"""Attention of several sequences over a 4-bit cache (bkv_seqs_attn) against its formula in 64 bits. (No counterpart in the
reference.)"""
import numpy as np
import pytest
import torch

from bonsai_vk_amd import KvSeqs

from seqs_util import arrays, attention, device_ints, fill, make, slots, starts_of

pytestmark = pytest.mark.gpu
SCALE = 1.0 / 16.0


def queries(n, nh, seed, mul=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(n, nh, 256, generator=g, device="cuda") * mul


def check(seqs, q, n, lens, out, layer=0, norm=2e-6):
    """Every output within its bound (seqs_util.attention), and the whole within `norm`: the roundings of the bound are
    independent, so that their sum's 2-norm is that of the square root of their number: of a score 16 eps of its partial sums
    (about 20 / 16 here) and eps * 16 of its distance to the reference, 1e-6 together, each output a mean of such p's."""
    want, bound = attention(seqs, layer, q, starts_of(n), lens, SCALE)
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"{float((off - bound).max()):.3e} over the bound"
    if float(want.norm()) > 0:
        assert float(off.norm() / want.norm()) < norm, float(off.norm() / want.norm())


def run(lens, n, page, nkv=4, grp=4, seed=1, gate=False, max_q=0, q_mul=1.0, **more):
    cache, seqs = make(lens, page, nkv, grp, seed=seed, **more)
    fill(cache, seed)
    q = queries(sum(n), nkv * grp, seed, q_mul)
    g = queries(sum(n), nkv * grp, seed + 1) if gate else None
    out, gated = seqs.attn(0, q, device_ints(starts_of(n)), gate=g, max_q=max_q)
    check(seqs, q, n, lens, out)
    if gate:
        want = out.double() * torch.sigmoid(g.double())
        assert float((gated.double() - want).abs().max()) <= 2.0 ** -21 * float(want.abs().max()) + 1e-30
    return cache, seqs, q, out


@pytest.mark.parametrize("page", [0, 16, 32, 48, 64, 100, 1])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 127, 128, 129, 300, 1000])
def test_one_token(page, length):
    run([length], [1], page, gate=length == 300)


@pytest.mark.parametrize("grp", [1, 2, 3, 4, 5, 8, 16, 17, 40])
@pytest.mark.parametrize("nkv", [1, 3, 4])
def test_head_layouts(nkv, grp):
    run([70, 200], [1, 3], 32, nkv, grp)


def test_many_kv_heads():
    run([40, 33], [1, 2], 16, 40, 2)


@pytest.mark.parametrize("page", [16, 64, 100])
def test_ragged_batch(page):
    lens = [1, 500, 33, 32, 31, 2, 900, 64, 65, 1300, 7, 128]
    run(lens, [1] * len(lens), page, gate=True)


def test_as_many_sequences_as_there_may_be():
    r = np.random.default_rng(3)
    lens = [int(x) for x in r.integers(1, 40, 1024)]
    run(lens, [1] * 1024, 16, nkv=1, grp=2)


@pytest.mark.parametrize("page", [0, 16, 48, 256])
@pytest.mark.parametrize("n, length", [(2, 2), (5, 40), (17, 17), (33, 500), (64, 64), (100, 700), (300, 301)])
def test_chunk(page, n, length):
    run([length], [n], page, gate=n == 33)


def test_many_tiles():
    """More tiles than pieces of a KV head, and pieces that have the ends of two tiles and whole ones between."""
    run([1600], [1500], 64, nkv=1, grp=8)
    run([700, 900, 650, 30], [640, 700, 650, 30], 48, nkv=2, grp=16)
    run([40] * 90 + [3000], [33] * 90 + [40], 16, nkv=1, grp=4)
    run([40] * 90 + [3000], [33] * 90 + [40], 16, nkv=4, grp=4)


def test_tiles_that_equal_pieces_would_share_out_badly():
    """5 x 8 tiles of a KV head for 64 pieces: whole ones would be twice as long as an equal share; 33 of which one is long."""
    run([4000] * 5, [256] * 5, 64)
    run([150] * 32 + [6000], [33] * 33, 48)


def test_blocks_of_several_rows_and_tiles_of_more_than_64_sequences():
    run([300] * 40 + [90] * 40, [1] * 20 + [9, 20, 24, 25] * 10 + [3] * 20, 32, nkv=2, grp=4)


def test_one_workspace_for_calls_of_all_sizes():
    """It is as large as the largest call wants, and the calls before leave nothing in it that one after them would take."""
    cache, seqs = make([2000, 600, 90], 32)
    fill(cache)
    seqs.workspace(700)
    outs = []
    for n in ([300, 1, 90], [1, 1, 1], [2, 300, 4], [1, 1, 1], [300, 1, 90], [0, 0, 1], [2, 300, 4]):
        q = queries(sum(n), 16, sum(n))
        out, _ = seqs.attn(0, q, device_ints(starts_of(n)))
        check(seqs, q, n, [2000, 600, 90], out)
        outs.append(out)
    assert torch.equal(outs[0], outs[4]) and torch.equal(outs[1], outs[3]) and torch.equal(outs[2], outs[6])


def test_chunks_and_tokens_together():
    run([700, 3, 1200, 90, 400, 64], [90, 1, 1, 64, 200, 1], 48, gate=True)


def test_sequences_without_tokens():
    run([50, 300, 20, 60, 70], [0, 3, 0, 0, 1], 32)
    run([50] * 70 + [33], [0] * 70 + [2], 16)


def test_queries_before_the_first_position_see_nothing():
    """More tokens than positions: the first of them get 0, as do all of a sequence without positions."""
    for n, length in ((5, 3), (40, 7), (3, 0), (150, 20)):
        cache, seqs = make([max(length, 1), 64], 32)
        fill(cache)
        seqs.len[0] = length
        q = queries(n + 1, 16, 2)
        out, _ = seqs.attn(0, q, device_ints([0, n, n + 1]), out=torch.full((n + 1, 16, 256), 7.0, device="cuda"))
        check(seqs, q, [n, 1], [length, 64], out)
        assert float(out[:n - length].abs().max()) == 0.0


def test_pages_outside_the_pool_are_not_seen():
    for page in (32, 48):
        lens = [300, 200, 100]
        cache, seqs = make(lens, page)
        fill(cache)
        seqs.tables[0, 0, 1] = -1
        seqs.tables[1, 0, 0] = cache.cap // page
        seqs.tables[1, 0, 2] = 2**31 - 1
        seqs.tables[2] = -1
        n = [3, 1, 2]
        q = queries(6, 16, 3)
        out, _ = seqs.attn(0, q, device_ints(starts_of(n)))
        check(seqs, q, n, lens, out)
        assert float(out[4:].abs().max()) == 0.0


@pytest.mark.parametrize("byte", [0xFF, 0x7C])
def test_bytes_of_unseen_positions_have_no_effect(byte):
    """Infs, NaNs and scales past the largest in every slot that is no sequence's, behind a sequence's end and later in a
    chunk than the query."""
    lens, n, page = [70, 33, 140], [20, 1, 130], 32
    cache, seqs = make(lens, page)
    fill(cache)
    q = queries(sum(n), 16, 4)
    clean, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    used = np.concatenate([slots(seqs, 0, s, x) for s, x in enumerate(lens)])
    others = np.setdiff1d(np.arange(cache.cap), used)
    for a in arrays(cache):
        a[0, torch.from_numpy(others).cuda()] = byte
    dirty, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    assert torch.equal(clean, dirty)
    # the last position, seen by the last query of each sequence only
    for s, x in enumerate(lens):
        for a in arrays(cache):
            a[0, int(slots(seqs, 0, s, x)[-1])] = byte
    dirty, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    check(seqs, q, n, lens, dirty)
    rows = [i for s in range(3) for i in range(sum(n[:s]), sum(n[:s + 1]) - 1)]
    assert torch.equal(clean[rows], dirty[rows])


def test_rows_of_no_sequence_are_left_as_they_were():
    cache, seqs = make([40, 70], 16)
    fill(cache)
    q, g = queries(9, 16, 5), queries(9, 16, 6)
    out, gated = torch.full((9, 16, 256), 3.5, device="cuda"), torch.full((9, 16, 256), -2.5, device="cuda")
    got = seqs.attn(0, q, device_ints([2, 3, 6]), g, out, gated)
    assert got[0] is out and got[1] is gated
    for t, x in ((out, 3.5), (gated, -2.5)):
        assert bool((t[:2] == x).all()) and bool((t[6:] == x).all())
    want, bound = attention(seqs, 0, q, [2, 3, 6], [40, 70], SCALE)
    assert bool(((out.double() - want).abs() <= bound)[2:6].all())


def test_strided_rows():
    """q and the gate in the engine's interleaved rows, and a fused buffer's."""
    cache, seqs = make([300], 0)
    fill(cache)
    qg = queries(3, 32, 7).view(3, 16, 512)
    q, g = qg[:, :, :256], qg[:, :, 256:]
    a = seqs.attn(0, q, device_ints([0, 3]), g)
    b = seqs.attn(0, q.contiguous(), device_ints([0, 3]), g.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = queries(3, 17, 8)[:, 1:]
    assert torch.equal(seqs.attn(0, odd, device_ints([0, 3]))[0], seqs.attn(0, odd.contiguous(), device_ints([0, 3]))[0])


@pytest.mark.parametrize("mul", [0.0, 30.0])
def test_flat_and_sharp_rows(mul):
    """Every key alike, and one key that takes it all (scores of hundreds)."""
    lens, n = [600, 77], [2, 1]
    cache, seqs = make(lens, 32)
    fill(cache)
    q = queries(3, 16, 9, mul)
    out, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    # (scores of 30 times the size: their roundings too)
    check(seqs, q, n, lens, out, norm=2e-6 if mul == 0.0 else 6e-5)


@pytest.mark.parametrize("v_mul", [1e-3, 3e-6, 5000.0])
def test_small_and_large_values(v_mul):
    """Scales below fp16's normal numbers (values a coarse multiple of 2^-21 then), and near the largest."""
    lens = [200, 50]
    cache, seqs = make(lens, 32)
    fill(cache, v_mul=v_mul)
    q = queries(2, 16, 10)
    out, _ = seqs.attn(0, q, device_ints([0, 1, 2]))
    want, bound = attention(seqs, 0, q, [0, 1, 2], lens, SCALE)
    assert bool(((out.double() - want).abs() <= bound).all())


def test_infinite_and_nan_queries_stay_in_their_row():
    cache, seqs = make([200, 100], 32)
    fill(cache)
    q = queries(4, 16, 11)
    want, _ = seqs.attn(0, q, device_ints([0, 3, 4]))
    q[1, 5, 7], q[3, 2, 200] = float("nan"), float("inf")
    out, _ = seqs.attn(0, q, device_ints([0, 3, 4]))
    other = torch.ones(4, 16, dtype=torch.bool, device="cuda")
    other[1, 5] = other[3, 2] = False
    assert torch.equal(out[other], want[other])
    assert not bool(torch.isfinite(out[1, 5]).any())


def test_the_same_from_call_to_call():
    lens, n = [3000, 100, 700], [40, 1, 3]
    cache, seqs = make(lens, 64)
    fill(cache)
    q = queries(44, 16, 12)
    first, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    for _ in range(5):
        assert torch.equal(seqs.attn(0, q, device_ints(starts_of(n)))[0], first)


def test_layers_are_apart():
    lens = [90, 40]
    cache, seqs = make(lens, 16, layers=3)
    fill(cache)
    q = queries(2, 16, 13)
    for layer in range(3):
        out, _ = seqs.attn(layer, q)
        check(seqs, q, [1, 1], lens, out, layer)


def test_max_q_is_only_a_hint():
    lens, n = [400, 300, 20], [200, 1, 9]
    cache, seqs = make(lens, 32)
    fill(cache)
    q = queries(210, 16, 14)
    for max_q in (0, 1, 8, 200, 100000):
        out, _ = seqs.attn(0, q, device_ints(starts_of(n)), max_q=max_q)
        check(seqs, q, n, lens, out)


def test_inconsistent_starts_and_lengths_stay_in_bounds():
    """Starts that go back, past the rows or below 0, lengths past the table and below 0: nothing but the results is lost."""
    cache, seqs = make([100, 90, 80], 16)
    fill(cache)
    q = queries(50, 16, 15)
    want, _ = seqs.attn(0, q[:3])
    for starts in ([0, 50, 0, 50], [40, 10, 45, 2], [-5, 70, 2**31 - 1, -2**31], [0, 2**30, 2**30, 2**30]):
        for lens in ([100, 90, 80], [2**31 - 1, -7, 5], [-2**31, 10**6, 96]):
            seqs.len.copy_(device_ints(lens))
            seqs.attn(0, q, device_ints(starts))
            seqs.attn(0, q, device_ints(starts), max_q=3)
            seqs.read(0, device_ints(starts), 50)
    seqs.len.copy_(device_ints([100, 90, 80]))
    assert torch.equal(seqs.attn(0, q[:3])[0], want)


def test_no_rows():
    cache, seqs = make([10], 16)
    out, _ = seqs.attn(0, torch.empty(0, 16, 256, device="cuda"), device_ints([0, 0]))
    assert out.shape == (0, 16, 256)


def test_graph_replays_with_other_lengths():
    """One captured call serves a sequence as it grows, and other sequences' starts."""
    cache, seqs = make([600, 500], 16, room=700)
    fill(cache)
    q = queries(40, 16, 16)
    starts = device_ints([0, 1, 40])
    seqs.workspace(40)
    out = torch.zeros(40, 16, 256, device="cuda")
    seqs.attn(0, q, starts, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seqs.attn(0, q, starts, out=out)
    for lens, st in (([600, 500], [0, 1, 40]), ([17, 300], [0, 20, 40]), ([1, 499], [0, 1, 40]), ([600, 39], [0, 39, 40])):
        seqs.len.copy_(device_ints(lens))
        starts.copy_(device_ints(st))
        q.normal_()
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager, _ = seqs.attn(0, q, starts)
        assert torch.equal(got, eager)
        check(seqs, q, [st[1], st[2] - st[1]], lens, got)


def test_workspace_asked_for_inside_a_capture_is_refused():
    cache, seqs = make([60], 16)
    fill(cache)
    q, starts = queries(1, 16, 17), device_ints([0, 1])
    out = torch.empty(1, 16, 256, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            seqs.attn(0, q, starts, out=out)
    seqs.workspace(1)
    seqs.attn(0, q, starts, out=out)
    torch.cuda.synchronize()


def test_another_stream():
    cache, seqs = make([900], 0)
    fill(cache)
    q = queries(1, 16, 18)
    want, _ = seqs.attn(0, q)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got, _ = seqs.attn(0, q)
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("page", [64, 80])
def test_bytes_past_4_gib(page):
    """Pages at the end of a pool whose K and V are past 2^32 bytes each."""
    pool = (9 << 20) // page
    cache, seqs = make([130, 70], page, cap=pool * page)
    assert cache.k_data.numel() > 1 << 32
    top = torch.arange(pool - 5, pool, dtype=torch.int32, device="cuda")
    seqs.tables[0, 0, :3], seqs.tables[1, 0, :2] = top[[4, 0, 2]][:seqs.tables.shape[2]], top[[1, 3]]
    part = slice((pool - 5) * page, pool * page)
    small, _ = make([130, 70], page, cap=5 * page)
    fill(small)
    for a, b in zip(arrays(cache), arrays(small)):
        a[0, part] = b[0]
    view = KvSeqs(small, 2)
    view.tables.copy_(seqs.tables - (pool - 5))
    view.len.copy_(seqs.len)
    n = [20, 1]
    q = queries(21, 16, 19)
    out, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    assert torch.equal(out, view.attn(0, q, device_ints(starts_of(n)))[0])
    check(view, q, n, [130, 70], out)
    for a, b in zip(seqs.read(0, device_ints([0, 130, 200]), 200), view.read(0, device_ints([0, 130, 200]), 200)):
        assert torch.equal(a, b)


def test_a_longer_context():
    run([20000, 5], [1, 1], 64)
    run([9000], [40], 256)
