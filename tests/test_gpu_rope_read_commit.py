"""bkv_rope_append, bkv_kv_read and bkv_kv_commit against plain torch (64 bits where values are computed), and the
whole of a speculative step: append a draft, attend, commit, go on."""
import math

import pytest
import torch

from bonsai_vk_amd import KvCache, Rope, tree_mask
from tests.gpu_util import say
from tests.tree_util import F16, HD, Q8, arrays, attention, check_rows, gen, make_cache, parents, same, scribble, slots, tolerance, values

pytestmark = pytest.mark.gpu
FORMATS = [(Q8, Q8), (F16, Q8), (Q8, F16), (F16, F16)]
EPS = 1e-5


def rotated(x, w, rope, at):
    """fp64 rows [n][heads][HD], and per element the absolute sum of its terms."""
    p = rope.params
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    half = p.nrot // 2
    turns = torch.tensor(list(p.turns)[:half], dtype=torch.float64, device="cuda")
    a = at.double()[:, None, None] * turns * (2 * math.pi)
    c, s = torch.cos(a) * p.mscale, torch.sin(a) * p.mscale
    i = torch.arange(half, device="cuda")
    lo, hi = (i, i + half) if p.layout == 0 else (2 * i, 2 * i + 1)
    y, size = x.clone(), x.abs()
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    size[..., lo] = size[..., hi] = (x[..., lo].abs() + x[..., hi].abs()) * p.mscale
    return y, size


def inputs(n, nh, nkv, seed):
    g = gen(seed)
    q, k, v = (torch.randn(n, h, HD, generator=g, device="cuda") * 2 for h in (nh, nkv, nkv))
    w = [1 + 0.1 * torch.randn(HD, generator=g, device="cuda") for _ in range(2)]
    return q, k, v, w


def check_append(c, layer, pos0, q, k, v, w, rope, positions, q_out):
    """q within the fp32 arithmetic's own error, K and V as quantising these rows gives."""
    n = k.shape[0]
    at = torch.arange(pos0, pos0 + n, device="cuda") if positions is None else positions
    qn, kn = w if w else (None, None)
    # the norm: squares, 10 sums, a division, a root and two products, 16 roundings of 2^-24; the angle's sine and
    # cosine, the products and the sum 5 more; fp64 angles of positions to 2^31 lose 2^-20 turns * 2^-2 .. 2^-53 * 2^31
    rnd = 2.0 ** -24 * (16 if w else 0) + 2.0 ** -24 * 5 + 2.0 ** -52 * float(at.double().abs().max()) * 7
    if q is not None:
        want, size = rotated(q, qn, rope, at)
        check_rows(q_out, want, size * rnd + 1e-37)
    for which, x, fmt in (("k", rotated(k, kn, rope, at), c.k_fmt), ("v", (v.double(), v.double().abs() * 0), c.v_fmt)):
        x, size = x
        err = size * (rnd if which == "k" else 0)
        got = values(c, which, layer, pos0, n)
        if fmt == F16:
            check_rows(got, x, err * (1 + 2.0 ** -10) + x.abs() * 2.0 ** -11 + 2.0 ** -25)
        else:
            # half a step d = amax / 127 of the block, the scale's own rounding to fp16 on a byte of at most 127, and
            # the fp32 quotient and product before the rounding (3 roundings of at most 127 steps)
            b = x.unflatten(-1, (8, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2) / 127
            check_rows(got, x, b * (0.5 + 127 * 2.0 ** -11 + 127 * 3 * 2.0 ** -24) + 2 * err.amax(-1, keepdim=True) + 2.0 ** -25 * 127)


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("nrot,layout", [(64, "half"), (20, "half"), (256, "half"), (2, "half"), (64, "interleaved"), (6, "interleaved"), (256, "interleaved"), (0, "half")])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_append(kf, vf, nrot, layout, norm):
    say(f"rope kf {kf} vf {vf} nrot {nrot} {layout} norm {norm}")
    n, pos0 = 13, 41
    c = make_cache(pos0 + n + 3, kf, vf, page=16 if nrot == 64 else 0)
    scribble(c, 3)
    before = [a.clone() for a in arrays(c)]
    q, k, v, w = inputs(n, 16, 4, nrot)
    w = w if norm else None
    rope = Rope(nrot, layout=layout, freq_base=1e4)
    got = c.rope_append(0, pos0, q, k, v, rope, qn_w=w and w[0], kn_w=w and w[1], eps=EPS)
    check_append(c, 0, pos0, q, k, v, w, rope, None, got)
    mine = torch.zeros(c.cap, dtype=torch.bool, device="cuda")
    mine[slots(c, 0, pos0, n)] = True
    for a, b in zip(arrays(c), before):            # no other slot is touched
        assert same(a[0][~mine], b[0][~mine])


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scaled_and_far_positions(scaling, layout):
    n = 11
    c = make_cache(n, F16, F16)
    q, k, v, w = inputs(n, 16, 4, 5)
    rope = Rope(128, layout=layout, freq_base=1e6, scaling=scaling, factor=8.0, trained_ctx=8192)
    at = torch.tensor([0, 1, 5, 5, 5, 131071, 1048577, 16777217, 2**31 - 1, -1, -70000], dtype=torch.int32, device="cuda")
    got = c.rope_append(0, 0, q, k, v, rope, positions=at)
    check_append(c, 0, 0, q, k, v, None, rope, at, got)
    if scaling != "yarn":
        assert same(got[0], q[0])                  # position 0 turns nothing


@pytest.mark.parametrize("nkv,group,n", [(1, 1, 1), (3, 5, 7), (16, 4, 2), (2, 16, 65), (4, 4, 1), (4, 4, 700)])
def test_head_counts_and_strides(nkv, group, n):
    nh = nkv * group
    q, k, v, w = inputs(n, nh, nkv, n)
    rope = Rope(64, freq_base=1e7)
    a, b, d = (make_cache(n, Q8, Q8, nkv=nkv, group=group) for _ in range(3))
    want = a.rope_append(0, 0, q, k, v, rope, qn_w=w[0], kn_w=w[1], eps=EPS)
    check_append(a, 0, 0, q, k, v, w, rope, None, want)
    fused = torch.cat([q, k, v], 1).contiguous()
    got = b.rope_append(0, 0, fused[:, :nh], fused[:, nh:nh + nkv], fused[:, nh + nkv:], rope, qn_w=w[0], kn_w=w[1], eps=EPS)
    assert same(got, want) and all(same(x, y) for x, y in zip(arrays(a), arrays(b)))
    qg = torch.cat([q, torch.randn_like(q)], 2)
    inplace = q.clone()
    assert same(d.rope_append(0, 0, qg[..., :HD], k, v, rope, qn_w=w[0], kn_w=w[1], eps=EPS), want)
    assert same(d.rope_append(0, 0, inplace, k, v, rope, qn_w=w[0], kn_w=w[1], eps=EPS, q_out=inplace), want) and same(inplace, want)
    assert d.rope_append(0, 0, None, k, v, rope, qn_w=w[0], kn_w=w[1], eps=EPS) is None
    assert all(same(x, y) for x, y in zip(arrays(a), arrays(d)))


@pytest.mark.parametrize("kf,vf", FORMATS)
def test_rope_append_writes_what_append_writes(kf, vf):
    """Without norm and rotation the bytes are bkv_kv_append's, for ordinary, tiny, zero, huge and non-finite rows."""
    n = 9
    k, v = (torch.randn(n, 4, HD, generator=gen(i), device="cuda") for i in range(2))
    for x in (k, v):
        x[1] *= 1e-38
        x[2] = 0
        x[3] *= 1e30
        x[4, :, 3] = math.inf
        x[5, :, 100] = math.nan
        x[6] *= 1e-7
        x[7, :, :32] = 1e-36
    a, b = make_cache(n, kf, vf), make_cache(n, kf, vf)
    a.append(0, 0, k, v)
    b.rope_append(0, 0, None, k, v, Rope(0))
    for x, y in zip(arrays(a), arrays(b)):
        assert same(x, y)


def test_rope_append_agrees_with_the_reference_front_end():
    n = 33
    q, k, v, w = inputs(n, 16, 4, 8)
    a, b = make_cache(500 + n, F16, Q8), make_cache(500 + n, F16, Q8)
    x = a.norm_rope_append(0, 500, q, k, v, w[0], w[1], nrot=64, eps=EPS, freq_base=1e7)
    y = b.rope_append(0, 500, q, k, v, Rope(64, freq_base=1e7), qn_w=w[0], kn_w=w[1], eps=EPS)
    # the front end's serial sum of 256 squares (256 roundings, halved by the root) and its fp32 angle (2^-24 of at
    # most 533 radians, twice)
    assert bool(((x - y).abs() <= (x.abs().amax(-1, keepdim=True) * 2) * (2.0 ** -24 * (128 + 2 * 533 + 16))).all())
    assert same(a.v_data, b.v_data) and same(a.v_scales, b.v_scales)


def test_rope_append_refusals_and_bad_pages():
    c = make_cache(64, Q8, Q8, page=16)
    q, k, v, w = inputs(5, 16, 4, 1)
    rope = Rope()
    with pytest.raises(ValueError):
        c.rope_append(0, 0, q[:4], k, v, rope)
    with pytest.raises(ValueError):
        c.rope_append(0, 0, q, k, v[:4], rope)
    with pytest.raises(ValueError):
        c.rope_append(0, 0, q, k, v, rope, positions=torch.zeros(5, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        c.rope_append(0, 0, None, k, v, rope, q_out=q)
    with pytest.raises(Exception, match="EINVAL"):
        c.rope_append(0, 0, q, k, v, rope, qn_w=w[0])
    with pytest.raises(Exception, match="ECAP"):
        c.rope_append(0, 60, q, k, v, rope)
    good = c.rope_append(0, 30, q, k, v, rope)
    keep = [a.clone() for a in arrays(c)]
    for bad in (-1, 2**31 - 1, c.cap // 16):
        c.block_table[0, 1] = bad                  # positions 16 .. 31: the first two tokens
        got = c.rope_append(0, 30, q, k, v, rope)
        assert same(got, good) and all(same(x, y) for x, y in zip(arrays(c), keep))
        kk, vv = c.read(0, 28, 6)
        assert not bool(kk[:4].any()) and not bool(vv[:4].any()) and bool(kk[4:].any())
        before = [a.clone() for a in arrays(c)]
        c.commit(30, 5, torch.tensor([2, 3, 0, 1], dtype=torch.int32, device="cuda"))
        for x, y in zip(arrays(c), before):        # neither into nor out of a page that is not there
            assert same(x, y)


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,nkv,pos0,n", [(0, 4, 0, 1), (16, 3, 5, 70), (48, 1, 100, 33), (0, 16, 3, 517)])
def test_read(kf, vf, dtype, page, nkv, pos0, n):
    c = make_cache(pos0 + n, kf, vf, page=page, nkv=nkv, layers=2)
    scribble(c, n)
    for layer in range(2):
        k, v = c.read(layer, pos0, n, dtype)
        # fp16 entries and f16(scale) * int8 are exact in fp32 (19 bits), so one rounding is all there is
        for got, which in ((k, "k"), (v, "v")):
            want = values(c, which, layer, pos0, n).float().to(dtype)
            ok = (got == want) | (torch.isnan(got) & torch.isnan(want))
            assert got.shape == (n, nkv, HD) and got.dtype == dtype and bool(ok.all())


def test_read_into_given_rows():
    c = make_cache(90, Q8, F16)
    scribble(c, 1)
    c.v_data.view(torch.int16).bitwise_and_(0x3BFF)
    c.k_scales.view(torch.int16).bitwise_and_(0x3BFF)
    k, v = c.read(0, 7, 50)
    heads = torch.full((4, 60, HD), 9.0, device="cuda")
    a, b = c.read(0, 7, 50, k_out=heads[:, 5:55].transpose(0, 1))
    assert b is None and same(a, k) and bool((heads[:, :5] == 9).all()) and bool((heads[:, 55:] == 9).all())
    wide = torch.full((2, 50, 4, HD + 8), 9.0, device="cuda")
    c.read(0, 7, 50, k_out=wide[0, ..., :HD], v_out=wide[1, ..., :HD])
    assert same(wide[0, ..., :HD], k) and same(wide[1, ..., :HD], v) and bool((wide[..., HD:] == 9).all())
    a, b = c.read(0, 7, 50, v_out=wide[1, ..., :HD])
    assert a is None and same(b, v)
    assert c.read(0, 7, 0)[0].shape == (0, 4, HD)
    for bad in (dict(k_out=k.cpu()), dict(k_out=k[:49]), dict(k_out=k.double()), dict(k_out=k, v_out=wide[1, ..., :HD]), dict(k_out=k, v_out=v.half())):
        with pytest.raises(ValueError):
            c.read(0, 7, 50, **bad)
    with pytest.raises(Exception, match="EINVAL"):
        c.read(0, 7, 50, k_out=torch.empty(1, 4, HD, device="cuda").expand(50, 4, HD))
    with pytest.raises(Exception, match="ECAP"):
        c.read(0, 41, 50)


# ------------------------------------------------------------------ commit
def moved(c, pos0, n, idx):
    """The arrays after a commit, by plain indexing."""
    out = [a.clone() for a in arrays(c)]
    for layer in range(c.n_layers):
        src = [(i, int(j)) for i, j in enumerate(idx.tolist()) if 0 <= j < n]
        if not src:
            continue
        at = slots(c, layer, pos0, n)
        to, frm = at[[i for i, _ in src]], at[[j for _, j in src]]
        for a, o in zip(arrays(c), out):
            o[layer, to] = a[layer, frm]
    return out


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("page,nkv,layers", [(0, 4, 8), (16, 3, 2), (48, 1, 3)])
@pytest.mark.parametrize("n,keep", [(1, 1), (8, 3), (64, 64), (65, 65), (300, 257), (1024, 1024), (1000, 5)])
def test_commit(kf, vf, page, nkv, layers, n, keep):
    pos0 = 21
    c = make_cache(pos0 + n + 9, kf, vf, page=page, nkv=nkv, layers=layers)
    g = torch.Generator().manual_seed(n + keep)
    cases = [torch.sort(torch.randperm(n, generator=g)[:keep]).values, torch.randperm(n, generator=g)[:keep], torch.arange(n - 1, n - 1 - keep, -1),
             torch.full((keep,), n - 1), torch.randint(-3, n + 3, (keep,), generator=g), torch.full((keep,), -2**31)]
    for i, idx in enumerate(cases):
        scribble(c, 10 * i)
        want = moved(c, pos0, n, idx)
        c.commit(pos0, n, idx.int().cuda())
        assert all(same(a, b) for a, b in zip(arrays(c), want)), i


def test_commit_refusals():
    c = make_cache(64, Q8, Q8)
    for bad in (torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(ValueError):
            c.commit(0, 8, bad)
    with pytest.raises(Exception, match="EINVAL"):
        c.commit(0, 2, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(Exception, match="ECAP"):
        c.commit(60, 8, torch.zeros(3, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("page", [0, 16])
def test_speculative_steps(kf, vf, page):
    """Three steps of a speculating program over two layers: each appends a draft at its tree positions, attends, keeps
    a path of it, and goes on from there. The cache ends bit for bit as one that only ever appended the kept tokens,
    and the attention of every kept token is as over that cache."""
    layers, n, room = 2, 14, 200
    c, plain = (make_cache(room, kf, vf, page=page, layers=layers, seed=s) for s in (1, 2))
    rope = Rope(64, layout="interleaved", freq_base=1e5)
    g = gen(4)
    pos = 37
    k, v = (torch.randn(pos, 4, HD, generator=g, device="cuda") for _ in range(2))
    for layer in range(layers):
        for x in (c, plain):
            x.rope_append(layer, 0, None, k, v, rope)
    for step in range(3):
        parent = parents(n, 30 + step)
        mask, depth = tree_mask(parent)
        path, j = [], n - 1
        while j >= 0:
            path.insert(0, j)
            j = parent[j]
        at = (pos + depth).int().cuda()
        for layer in range(layers):
            q, k, v, w = inputs(n, 16, 4, 50 * step + layer)
            qr = c.rope_append(layer, pos, q, k, v, rope, positions=at, qn_w=w[0], kn_w=w[1])
            out, _ = c.attn_tree(layer, pos, qr, mask.cuda())
            kept = torch.tensor(path, device="cuda")
            qp = plain.rope_append(layer, pos, q[kept], k[kept], v[kept], rope, qn_w=w[0], kn_w=w[1])
            assert same(qr[kept], qp)
            want, _, size = attention(plain, layer, pos, qp, None)
            check_rows(out[kept], want, tolerance(size, pos + n))
        c.commit(pos, n, torch.tensor(path + [-1] * 2, dtype=torch.int32, device="cuda")[: min(n, len(path) + 2)])
        pos += len(path)
        for layer in range(layers):
            for a, b in zip(c.read(layer, 0, pos), plain.read(layer, 0, pos)):
                assert same(a, b)
            dq = torch.randn(16, HD, generator=g, device="cuda")
            assert same(c.decode(layer, pos, dq)[0], plain.decode(layer, pos, dq)[0])


def test_a_step_in_a_graph():
    """append + attention + commit captured once, replayed with other drafts, eager work and synchronisation between."""
    n, pos0 = 12, 100
    c, e = make_cache(pos0 + n, Q8, Q8), make_cache(pos0 + n, Q8, Q8)
    rope = Rope()
    base = inputs(pos0, 16, 4, 1)
    for x in (c, e):
        x.rope_append(0, 0, None, base[1], base[2], rope)
    c.tree_workspace()
    q, k, v, _ = inputs(n, 16, 4, 2)
    at, mask, idx = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, 1, dtype=torch.int64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    qr, out = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.rope_append(0, pos0, q, k, v, rope, positions=at, q_out=qr)
        c.attn_tree(0, pos0, qr, mask, out=out)
        c.commit(pos0, n, idx)
    for step in range(4):
        new = inputs(n, 16, 4, 10 + step)
        for dst, src in zip((q, k, v), new):
            dst.copy_(src)
        m, depth = tree_mask(parents(n, step))
        at.copy_((depth + pos0).int())
        mask.copy_(m)
        idx.copy_(torch.tensor([0, 3, 5, -1], dtype=torch.int32))
        graph.replay()
        eq = e.rope_append(0, pos0, q, k, v, rope, positions=at)
        eo, _ = e.attn_tree(0, pos0, eq, mask)
        e.commit(pos0, n, idx)
        torch.cuda.synchronize()
        assert same(qr, eq) and same(out, eo) and all(same(a, b) for a, b in zip(arrays(c), arrays(e)))


def test_streams():
    """Each call on a stream that is not the default one, ordered by events alone."""
    c = KvCache(n_layers=1, cap=80, k_fmt=Q8, v_fmt=Q8)
    q, k, v, w = inputs(80, 16, 4, 3)
    rope = Rope()
    want_q = c.rope_append(0, 0, q, k, v, rope)
    want = c.read(0, 0, 80)
    torch.cuda.synchronize()
    for a in arrays(c):
        a.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got_q = c.rope_append(0, 0, q, k, v, rope)
        got = c.read(0, 0, 80)
        c.commit(70, 10, torch.tensor([5, 6], dtype=torch.int32, device="cuda"))
        after = c.read(0, 70, 2)
    s.synchronize()
    assert same(got_q, want_q) and all(same(a, b) for a, b in zip(got, want))
    assert all(same(a, b[75:77]) for a, b in zip(after, want))
