"""The 4-bit format as it is written and read, rotary positions of several axes, ragged appends and reads
(bkv_seqs_rope_append, bkv_seqs_read), and all calls for several sequences together. (No counterpart in the reference.)"""
import ctypes

import numpy as np
import pytest
import torch

from bonsai_vk_amd import BkvError, KvCache, KvSeqs, Rope, RopeAxes
from bonsai_vk_amd._lib import lib

from seqs_util import FMT, HD, arrays, attention, device_ints, make, q4_pack, q4_quantise, q4_values, random_bytes, slots, starts_of

pytestmark = pytest.mark.gpu
NONE = Rope(0)


def special_rows():
    """Head rows with blocks that can go wrong: ties of size, borders of two codes, values that saturate, vanish or are not
    finite, and ordinary ones of all sizes."""
    r = np.random.default_rng(1)
    rows = [np.zeros(256), np.arange(256) - 128.0, np.tile([3.0, -3.0], 128), np.tile([-5.0, 5.0, 4.0, -4.0], 64)]
    rows += [r.standard_normal(256) * 10.0 ** e for e in (-9, -8, -7, -6, -5, -4, -3, 0, 2, 3, 4, 5, 8, 30)]
    rows += [r.uniform(0, 1, 256), -r.uniform(0, 1, 256), r.integers(-16, 17, 256) / 2.0, r.integers(-8, 8, 256) * 0.37]
    rows += [np.full(256, 16384.0), np.full(256, -16384.0), np.full(256, 16385.0), np.full(256, 65000.0), np.full(256, 3.4e38)]
    # scales on the border of 8 significant bits, both ways, and of a step of the exponent
    rows += [np.where(np.arange(256) % 32 == 5, -8.0 * x, 0.3 * x) for x in (1 + 1 / 256, 1 + 3 / 256, 2 - 1 / 256, 2 - 1 / 1024, 2.0 ** -14, 2.0 ** -14 - 2.0 ** -24)]
    for bad in (np.nan, np.inf, -np.inf):
        x = r.standard_normal(256)
        x[[3, 70, 71]] = bad
        rows.append(x)
    x = np.full(256, np.nan)
    x[40] = 2.0
    rows.append(x)
    x = np.tile([np.inf, -np.inf], 128)
    rows.append(x)
    return np.stack(rows).astype(np.float32)


def cache_rows(cache, name):
    """(bytes [cap][nkv][128], scale words [cap][nkv][8]) of layer 0."""
    d = getattr(cache, name + "_data")[0].cpu().numpy().reshape(cache.cap, cache.nkv, 128)
    s = getattr(cache, name + "_scales")[0].cpu().numpy().reshape(cache.cap, cache.nkv, 16)
    return d, np.ascontiguousarray(s).view(np.uint16).reshape(cache.cap, cache.nkv, 8)


def scales_without_nan(x, d):
    """A block whose values are all NaN has a scale that means nothing (every value of it is 0)."""
    b = np.isnan(x.reshape(*x.shape[:-1], 8, 32)).all(-1)
    return np.where(b, 0, d)


@pytest.mark.parametrize("how", ["append", "rope_append", "seqs"])
def test_the_format_bit_for_bit(how):
    x = special_rows()
    n = len(x)
    k = torch.from_numpy(x).cuda().view(n, 1, 256)
    v = k.flip(0).contiguous()
    if how == "seqs":
        cache, seqs = make([n], 16, 1, 2)
        q = seqs.rope_append(0, None, k, v, NONE, device_ints([0, n]))
        assert q is None
        at = slots(seqs, 0, 0, n)
    else:
        cache = KvCache(n_layers=1, nh=2, nkv=1, cap=n, k_fmt=FMT["q4_0"], v_fmt=FMT["q4_0"])
        if how == "append":
            cache.append(0, 0, k, v)
        else:
            cache.rope_append(0, 0, None, k, v, NONE)
        at = np.arange(n)
    for name, y in (("k", x), ("v", x[::-1])):
        c, d = q4_quantise(y)
        got_d, got_s = cache_rows(cache, name)
        assert np.array_equal(got_d[at, 0], q4_pack(c))
        assert np.array_equal(scales_without_nan(y, got_s[at, 0]), scales_without_nan(y, d))
        fine = np.isfinite(y).reshape(n, 8, 32).all(-1)
        assert np.isfinite(q4_values(got_d[at, 0], got_s[at, 0])).all()
        # half a step off at most (and the last step's half on the other side), where the block does not saturate or vanish
        top = np.abs(np.where(np.isfinite(y), y, 0)).reshape(n, 8, 32).max(-1)
        mid = fine & (top <= 16384) & (top >= 2.0 ** -11)
        off = np.abs(q4_values(got_d[at, 0], got_s[at, 0]) - y.astype(np.float64)).reshape(n, 8, 32).max(-1)
        # a scale of 8 bits is 2^-9 off (and 2^-12 from fp16), so x / d is past 7.5 or 8 by 8 (2^-9 + 2^-12) at most, or in
        # the other direction: where the largest of the other sign is as far as x_m, 8 is cut to 7
        assert (off[mid] <= top[mid] / 8 * (1.0 + 2.0 ** -8) * (1.0 + 8 * (2.0 ** -9 + 2.0 ** -12))).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_reading_any_bytes(dtype):
    """Every scale word, Infs and NaNs among them, is the value that the format says."""
    cache = KvCache(n_layers=1, nh=4, nkv=2, cap=600, k_fmt=FMT["q4_0"], v_fmt=FMT["q4_0"])
    random_bytes(cache, 3)
    cache.k_scales[0, :8] = 0xFF
    cache.v_scales[0, :8] = 0x7C
    want = [q4_values(*cache_rows(cache, name)) for name in "kv"]
    for got, w in zip(cache.read(0, 0, 600, dtype=dtype), want):
        w = torch.from_numpy(w)
        assert torch.equal(got.cpu(), w.to(dtype))
        if dtype != torch.bfloat16:
            assert torch.equal(got.cpu().double(), w)          # (exact in fp16)
    part = torch.empty(2, 7, HD, device="cuda").transpose(0, 1)
    cache.read(0, 593, 7, v_out=part)
    assert torch.equal(part.cpu().double(), torch.from_numpy(want[1][593:]))
    paged, seqs = make([600], 48, 2, 2)
    for a, b in zip(arrays(paged), arrays(cache)):
        a[0, torch.from_numpy(slots(seqs, 0, 0, 600)).cuda()] = b[0]
    for got, w in zip(seqs.read(0, device_ints([0, 600]), 600, dtype=dtype), want):
        assert torch.equal(got.cpu(), torch.from_numpy(w).to(dtype))


@pytest.mark.parametrize("k, v", [("q4_0", "q4_0"), ("q4_0", "f16"), ("q8_0", "q4_0"), ("f16", "q8_0"), ("q8_0", "q8_0")])
def test_a_ragged_append_is_the_single_ones(k, v):
    """Every sequence's tokens as bkv_rope_append writes them: the same bytes (without a norm, whose sum is formed otherwise
    there), and the same queries."""
    lens, n = [70, 5, 33, 64, 1], [20, 5, 0, 1, 1]
    cache, seqs = make(lens, 16, 2, 3, k, v)
    random_bytes(cache)
    before = [a.clone() for a in arrays(cache)]
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    t = sum(n)
    rows = torch.randn(t, 10, 256, device="cuda", generator=g)
    q, kk, vv = rows[:, :6], rows[:, 6:8], rows[:, 8:]
    rope = Rope(128, "interleaved")
    got = seqs.rope_append(0, q, kk, vv, rope, device_ints(starts_of(n)))
    mine = [a.clone() for a in arrays(cache)]
    for a, b in zip(arrays(cache), before):
        a.copy_(b)
    ref = KvCache(n_layers=1, nh=6, nkv=2, cap=cache.cap, k_fmt=cache.k_fmt, v_fmt=cache.v_fmt, page_tokens=16,
                  max_pages=cache.max_pages, block_table=seqs.tables[0])
    for a, b in zip(arrays(ref), before):
        a.copy_(b)
    for s, (x, m) in enumerate(zip(lens, n)):
        if m:
            ref.block_table.copy_(seqs.tables[s])
            a = starts_of(n)[s]
            want = ref.rope_append(0, x - m, q[a:a + m], kk[a:a + m], vv[a:a + m], rope)
            assert torch.equal(got[a:a + m], want)
    for a, b in zip(mine, arrays(ref)):
        assert torch.equal(a, b)


def plain_rope(x, rope, axis, at, w, eps=1e-6):
    """Rows [n][heads][256] in 64 bits; at [axes][n]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    nrot, half = rope.params.nrot, rope.params.nrot // 2
    turns = torch.tensor(list(rope.params.turns[:half]), dtype=torch.float64, device="cuda")
    a = (at.double()[axis].t() * turns)
    a = ((a - a.round()) * (2 * np.pi))[:, None]
    i = torch.arange(half, device="cuda")
    one, two = (i, i + half) if rope.params.layout == 0 else (2 * i, 2 * i + 1)
    y, m = x.clone(), float(rope.params.mscale)
    y[..., one] = (x[..., one] * torch.cos(a) - x[..., two] * torch.sin(a)) * m
    y[..., two] = (x[..., two] * torch.cos(a) + x[..., one] * torch.sin(a)) * m
    return y


@pytest.mark.parametrize("pairs, order", [((32,), "blocks"), ((11, 11, 10), "dealt"), ((8, 12, 12), "blocks"), ((24, 20, 20), "dealt"),
                                          ((0, 5, 5), "blocks"), ((1, 0, 9), "dealt"), ((16,) * 8, "dealt"), ((16,) * 8, "blocks"), ((0, 0), "dealt")])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
def test_axes(pairs, order, layout, norm):
    """Queries against the formula: the norm's factor is rounded 3 times, the value 2, cosine and sine once each, both
    products and their sum: 8 roundings of values that are no larger than the pair's |x1| + |x2| times mscale."""
    nrot, t = 2 * sum(pairs), 37
    rope = Rope(nrot, layout, scaling="yarn", factor=4.0, trained_ctx=32768) if nrot else NONE
    axes = RopeAxes(list(pairs), order)
    left, axis = list(pairs), []
    while sum(left):
        for a in range(len(left)):
            for _ in range(left[a] if order == "blocks" else min(left[a], 1)):
                axis.append(a)
                left[a] -= 1
    assert axes.axis == axis
    cache, seqs = make([37, 60], 16, 1, 2)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    q, k, v = (torch.randn(t, h, 256, device="cuda", generator=g) for h in (2, 1, 1))
    at = torch.randint(-50, 300000, (len(pairs), t), device="cuda", generator=g, dtype=torch.int32)
    at[:, 0] = 0
    qw, kw = (torch.rand(256, device="cuda", generator=g) + 0.5 for _ in range(2)) if norm else (None, None)
    got = seqs.rope_append(0, q, k, v, rope, device_ints([0, 20, t]), positions=at, axes=axes, qn_w=qw, kn_w=kw)
    ax = torch.tensor(axis, dtype=torch.long, device="cuda")
    want = plain_rope(q, rope, ax, at, qw)
    size = float(want.abs().max()) * 2
    assert float((got.double() - want).abs().max()) <= 8 * 2.0 ** -24 * size
    # K: within its 64-bit value's step, half of it but next to a border of two codes (and a scale's)
    kd, vd = seqs.read(0, device_ints([0, 20, t]), t)
    for x, y in ((kd, plain_rope(k, rope, ax, at, kw)), (vd, v.double())):
        top = y.reshape(t, 1, 8, 32).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(y.shape)
        assert bool(((x.double() - y).abs() <= top / 8 * 1.05).all())


@pytest.mark.parametrize("n_seq", [63, 64, 65, 200])
def test_appends_of_many_sequences(n_seq):
    """Some without tokens, some rows before the first and behind the last sequence: every token's codes and scales are its
    row's, at its own position, and it reads back as them."""
    r = np.random.default_rng(n_seq)
    n = [int(x) for x in r.integers(0, 4, n_seq)]
    lens = [m + int(x) for m, x in zip(n, r.integers(0, 40, n_seq))]
    cache, seqs = make(lens, 16, 1, 2, room=64)
    random_bytes(cache)
    before = [a.clone() for a in arrays(cache)]
    t, starts = sum(n) + 5, [x + 2 for x in starts_of(n)]
    g = torch.Generator(device="cuda")
    g.manual_seed(n_seq)
    q, k, v = (torch.randn(t, h, 256, device="cuda", generator=g) for h in (2, 1, 1))
    out = torch.full((t, 2, 256), 4.0, device="cuda")
    seqs.rope_append(0, q, k, v, NONE, device_ints(starts), q_out=out)
    end = starts[-1]
    assert torch.equal(out[2:end], q[2:end]) and bool((out[:2] == 4.0).all()) and bool((out[end:] == 4.0).all())
    got = seqs.read(0, device_ints(starts), t)
    want = [a.cpu().numpy().reshape(cache.cap, -1).copy() for a in before]
    for i, x in enumerate((k, v)):
        c, d = q4_quantise(x.cpu().numpy()[:, 0])
        values = q4_values(q4_pack(c), d)
        assert np.array_equal(got[i][2:end, 0].cpu().numpy(), values[2:end].astype(np.float32))
        for s in range(n_seq):
            for j, slot in enumerate(slots(seqs, 0, s, lens[s])[lens[s] - n[s]:]):
                want[2 * i][slot] = q4_pack(c[starts[s] + j])
                want[2 * i + 1][slot] = d[starts[s] + j].view(np.uint8)
    for a, b in zip(arrays(cache), want):
        assert np.array_equal(a.cpu().numpy().reshape(cache.cap, -1), b)


@pytest.mark.parametrize("nkv, grp", [(1, 1), (3, 1), (1, 9), (8, 8), (5, 3)])
@pytest.mark.parametrize("t", [1, 300])
def test_any_number_of_rows(nkv, grp, t):
    """Row counts that do not divide into a workgroup's, with and without norms and queries: Q against the formula, K and V the
    same bytes with Q beside them or not."""
    cache, seqs = make([t], 64, nkv, grp)
    g = torch.Generator(device="cuda")
    g.manual_seed(nkv)
    q, k, v = (torch.randn(t, h, 256, device="cuda", generator=g) for h in (nkv * grp, nkv, nkv))
    qw, kw = (torch.rand(256, device="cuda", generator=g) + 0.5 for _ in range(2))
    rope, start = Rope(64), device_ints([0, t])
    for a, b in ((None, None), (qw, kw)):
        got = seqs.rope_append(0, q, k, v, rope, start, qn_w=a, kn_w=b)
        want = plain_rope(q, rope, torch.zeros(32, dtype=torch.long, device="cuda"), torch.arange(t, device="cuda")[None], a)
        assert float((got.double() - want).abs().max()) <= 8 * 2.0 ** -24 * 2 * float(want.abs().max())
        with_q = seqs.read(0, start, t)
        bytes_with_q = [x.clone() for x in arrays(cache)]
        random_bytes(cache)
        assert seqs.rope_append(0, None, k, v, rope, start, qn_w=a, kn_w=b) is None
        for x, y in zip(with_q, seqs.read(0, start, t)):
            assert torch.equal(x, y)
        for x, y in zip(arrays(cache), bytes_with_q):
            at = torch.from_numpy(slots(seqs, 0, 0, t)).cuda()
            assert torch.equal(x[0].view(cache.cap, -1)[at], y[0].view(cache.cap, -1)[at])


def test_tokens_without_a_place():
    """Rows of no sequence are left as they are; tokens of negative positions or of missing pages are rotated and not
    written; nothing else in the cache changes."""
    lens = [4, 40]
    cache, seqs = make([20, 40], 16, 1, 2)
    seqs.len.copy_(device_ints(lens))
    random_bytes(cache)
    seqs.tables[1, 0, 1] = -1
    before = [a.clone() for a in arrays(cache)]
    q, k, v = (torch.randn(40, h, 256, device="cuda") for h in (2, 1, 1))
    out = torch.full((40, 2, 256), 4.0, device="cuda")
    starts = [2, 9, 38]                            # 7 tokens of 4 positions, 29 of 40: 11 .. 39, of which 16 .. 31 have no page
    got = seqs.rope_append(0, q, k, v, NONE, device_ints(starts), q_out=out)
    assert got is out and torch.equal(out[2:38], q[2:38])
    assert bool((out[:2] == 4.0).all()) and bool((out[38:] == 4.0).all())
    where = {5 + i: (0, i) for i in range(4)} | {9 + i: (1, 11 + i) for i in range(29)}
    table = seqs.tables.cpu().numpy()
    changed = {}
    for t, (s, p) in where.items():
        if not 16 <= p < 32 or s == 0:
            changed[int(table[s, 0, p // 16]) * 16 + p % 16] = t
    assert len(changed) == 4 + 29 - 16
    for name, x in (("k", k), ("v", v)):
        c, d = q4_quantise(x.cpu().numpy()[:, 0])
        want_d = dict(zip(range(40), q4_pack(c)))
        got_d, got_s = cache_rows(cache, name)
        old_d = before[0 if name == "k" else 2][0].cpu().numpy().reshape(-1, 1, 128)
        for slot in range(cache.cap):
            assert np.array_equal(got_d[slot, 0], want_d[changed[slot]] if slot in changed else old_d[slot, 0])
            if slot in changed:
                assert np.array_equal(got_s[slot, 0], d[changed[slot]])
    kd, vd = seqs.read(0, device_ints(starts), 40)
    for t, (s, p) in where.items():
        if s == 1 and 16 <= p < 32:
            assert float(kd[t].abs().max()) == 0.0 == float(vd[t].abs().max())
    assert float(kd[2:5].abs().max()) == 0.0


def test_appends_without_room_are_dropped():
    cache, seqs = make([30], 16, 1, 2)
    random_bytes(cache)
    before = [a.clone() for a in arrays(cache)]
    k = torch.randn(3, 1, 256, device="cuda")
    for n in (1000, 2**31 - 1, -4):
        seqs.len.fill_(n)
        seqs.rope_append(0, None, k, k, NONE, device_ints([0, 3]))
    for a, b in zip(arrays(cache), before):
        assert torch.equal(a, b)
    one = KvCache(n_layers=1, nh=2, nkv=1, cap=8, k_fmt=FMT["q4_0"], v_fmt=FMT["q4_0"])
    for call in (lambda: one.append(0, 6, k, k), lambda: one.rope_append(0, 6, None, k, k, NONE), lambda: one.read(0, 6, 3)):
        with pytest.raises(BkvError, match="ECAP"):
            call()


def test_commit_moves_4_bit_rows():
    cache = KvCache(n_layers=2, nh=4, nkv=2, cap=64, k_fmt=FMT["q4_0"], v_fmt=FMT["q4_0"])
    random_bytes(cache)
    before = [a.clone() for a in arrays(cache)]
    cache.commit(20, 30, device_ints([0, 3, 1, 29, 8]))
    for a, b in zip(arrays(cache), before):
        b[:, 20:25] = b[:, [20, 23, 21, 49, 28]]
        assert torch.equal(a, b)


def test_synthetic_fill():
    cache = KvCache(n_layers=2, nh=4, nkv=1, cap=10, k_fmt=FMT["q4_0"], v_fmt=FMT["q8_0"])
    cache.fill_synthetic()
    for a in arrays(cache):
        assert bool((a.view(torch.int32) == 0x3C003C00).all())


def test_calls_that_do_not_take_4_bits():
    cache = KvCache(n_layers=1, nh=4, nkv=1, cap=64, k_fmt=FMT["q4_0"], v_fmt=FMT["q8_0"])
    cache.workspace = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    q, k = torch.randn(4, 256, device="cuda"), torch.randn(1, 1, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    for call in (lambda: cache.decode(0, 3, q), lambda: cache.decode_step(0, 3, k, k, q), lambda: cache.decode_window(0, 1, 3, q),
                 lambda: cache.norm_rope_append(0, 0, q[None], k, k, w, w), cache.check_workspace):
        with pytest.raises(BkvError, match="EUNSUPPORTED"):
            call()
    with pytest.raises(BkvError, match="EUNSUPPORTED"):    # (one format of 4 bits is not enough)
        KvSeqs(cache, 1).attn(0, q[None])
    assert cache.decode_path(3) == -1
    assert lib().bkv_decode_step_static(ctypes.byref(cache.desc), 0, 3, k.data_ptr(), k.data_ptr(), q.data_ptr(), None, q.data_ptr(), None, 0) == -7
    assert lib().bkv_workspace_bytes(ctypes.byref(cache.desc), 0, 64) == 0 == lib().bkv_workspace_bytes(ctypes.byref(cache.desc), 2, 64)


def test_append_and_read_in_a_graph():
    """One captured step at other positions, lengths and tables of each replay."""
    cache, seqs = make([30, 50, 20], 16, 1, 2, room=64, spare=6)
    random_bytes(cache)
    q, k, v = (torch.randn(12, h, 256, device="cuda") for h in (2, 1, 1))
    axes, rope = RopeAxes([8, 8], "dealt"), Rope(32)
    at, starts = torch.zeros(2, 12, dtype=torch.int32, device="cuda"), device_ints([0, 4, 8, 12])
    out = torch.zeros(12, 2, 256, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seqs.rope_append(0, q, k, v, rope, starts, at, axes, q_out=out)
        got = seqs.read(0, starts, 12)
    for lens, st in (([30, 50, 20], [0, 4, 8, 12]), ([12, 1, 7], [0, 11, 12, 12]), ([1, 2, 20], [0, 0, 0, 12])):
        seqs.len.copy_(device_ints(lens))
        starts.copy_(device_ints(st))
        at.random_(0, 5000)
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        a, b = out.clone(), [x.clone() for x in got]
        data = [x.clone() for x in arrays(cache)]
        assert torch.equal(a, seqs.rope_append(0, q, k, v, rope, starts, at, axes))
        for x, y in zip(b, seqs.read(0, starts, 12)):
            rows = [i for s in range(3) for i in range(st[s], st[s + 1])]
            assert torch.equal(x[rows], y[rows])
        for x, y in zip(data, arrays(cache)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("page", [16, 48])
def test_a_server_step_by_step(page):
    """Two prompts, one with a picture; samples of both; a beam step; a conversation that ends; a compaction: every step's
    attention against the formula, over what the sequence's own history is."""
    layers, nkv, grp, n_seq = 2, 2, 4, 6
    nh = nkv * grp
    cache, seqs = make([0] * n_seq, page, nkv, grp, layers=layers, cap=page * 60, room=10 * page)
    rope, axes = Rope(64), RopeAxes([12, 10, 10], "dealt")
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    history = [[torch.empty(0, nkv, 256, device="cuda") for _ in range(2 * layers)] for _ in range(n_seq)]

    def step(n):
        t, starts = sum(n), device_ints(starts_of(n))
        assert seqs.extend(device_ints(n)).tolist() == [0] * layers
        seqs.len += device_ints(n)
        at = torch.randint(0, 500, (3, t), device="cuda", generator=g, dtype=torch.int32)
        for layer in range(layers):
            q, k, v = (torch.randn(t, h, 256, device="cuda", generator=g) for h in (nh, nkv, nkv))
            q = seqs.rope_append(layer, q, k, v, rope, starts, at, axes)
            out, _ = seqs.attn(layer, q, starts)
            new = seqs.read(layer, starts, t)
            for s in range(n_seq):
                a, b = starts_of(n)[s], starts_of(n)[s + 1]
                for i in range(2):
                    history[s][2 * layer + i] = torch.cat([history[s][2 * layer + i], new[i][a:b]])
            lens = seqs.len.tolist()
            want, bound = attention(seqs, layer, q, starts_of(n), lens, cache.scale)
            assert bool(((out.double() - want).abs() <= bound).all())
        same()

    def same():
        """The cache holds each sequence's history, in its own order."""
        lens = seqs.len.tolist()
        for layer in range(layers):
            got = seqs.read(layer, device_ints(starts_of(lens)), sum(lens))
            for s in range(n_seq):
                a, b = starts_of(lens)[s], starts_of(lens)[s + 1]
                for i in range(2):
                    assert torch.equal(got[i][a:b], history[s][2 * layer + i])

    def fork(parent):
        seqs.fork(device_ints(parent))
        old = [list(h) for h in history]
        for s, p in enumerate(parent):
            history[s] = list(old[p]) if 0 <= p < n_seq else [x[:0] for x in old[s]]
        same()

    step([page + 5, 0, 0, 3 * page, 0, 0])
    fork([0, 0, 0, 3, 3, 3])
    step([1, 1, 1, 1, 1, 1])
    step([1, 2, 1, 1, 5, 1])
    fork([1, 1, 2, 4, 4, 4])
    step([1, 1, 1, 1, 1, page])
    fork([0, -1, 2, 3, -1, 5])
    seqs.compact()
    same()
    used = (seqs.refs > 0).sum(1)
    assert bool(((seqs.refs > 0) == (torch.arange(seqs.refs.shape[1], device="cuda") < used[:, None])).all())
    step([2, 7, 0, 1, 30, 1])
    fork([-1] * 6)
    assert int(seqs.refs.abs().sum()) == 0 and int((seqs.tables >= 0).sum()) == 0
