"""bkv_attn_tree against its formula in 64 bits: formats, pages, head counts, lengths, masks, strides, values at the
edges of the formats, streams and graphs."""
import math

import pytest
import torch

from tests.gpu_util import say
from tests.tree_util import (F16, HD, Q8, attention, check_rows, gen, make_cache, put, rel, same, scribble, seen, slots, some_mask,
                             tolerance, values)

pytestmark = pytest.mark.gpu
FORMATS = [(Q8, Q8), (F16, Q8), (Q8, F16), (F16, F16)]
# drafts that 16 rows, 128 rows (of them 60, and more than two tiles) and 256 rows a workgroup are chosen for
KERNELS = [(9, 801), (15, 20000), (70, 6001), (1000, 4011)]


def filled(n, kf, vf, seed=1, **kw):
    c = make_cache(n, kf, vf, seed=seed, **kw)
    g = gen(seed)
    k = torch.randn(n, c.nkv, HD, generator=g, device="cuda")
    k[..., :3] *= 6
    v = torch.randn(n, c.nkv, HD, generator=g, device="cuda") * 0.5
    if c.nh == 4 * c.nkv:
        for layer in range(c.n_layers):
            c.append(layer, 0, k, v)
    else:
        from bonsai_vk_amd import Rope
        for layer in range(c.n_layers):
            c.rope_append(layer, 0, None, k, v, Rope(0))
    return c


def rows(n, nh, seed, scale=1.0):
    g = gen(1000 + seed)
    return torch.randn(n, nh, HD, generator=g, device="cuda") * scale, torch.randn(n, nh, HD, generator=g, device="cuda") * 2


def check(c, pos0, n, kind, seed=3, qscale=1.0, gate=True, layer=0, accurate=True):
    q, g = rows(n, c.nh, seed, qscale)
    mask = some_mask(kind, n, seed)
    out, og = c.attn_tree(layer, pos0, q, mask, g if gate else None)
    want, wg, size = attention(c, layer, pos0, q, mask, g)
    tol = tolerance(size, pos0 + n)
    check_rows(out, want, tol)
    if gate:
        # the sigmoid: exp, a sum and a division in fp32, 2^-21 together
        check_rows(og, wg, tol + wg.abs() * 2.0 ** -21)
    r = rel(out, want)
    say(f"  n {n} pos0 {pos0} {kind}: rel {r:.2e}")
    if accurate:
        # roundings are independent, so the whole is far nearer than the bound of each element: scores of a few
        # units carry about 2^-24 * 8 each, the sums of p v as much again
        assert r < 4e-6
    return out, want


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("page", [0, 16, 48])
@pytest.mark.parametrize("n,pos0,kind", [(1, 0, "chain"), (1, 1, "chain"), (1, 333, "tree"), (3, 30, "tree"), (4, 31, "tree"), (5, 64, "chain"),
                                         (16, 500, "tree"), (17, 1, "tree"), (33, 700, "padded"), (70, 95, "tree"), (130, 0, "chain")])
def test_small(kf, vf, page, n, pos0, kind):
    say(f"tree kf {kf} vf {vf} page {page}")
    check(filled(pos0 + n, kf, vf, page=page), pos0, n, kind)


@pytest.mark.parametrize("nkv,group", [(1, 1), (3, 1), (2, 2), (3, 5), (1, 8), (2, 16), (16, 4), (1, 33)])
@pytest.mark.parametrize("kf,vf", [(Q8, Q8), (F16, F16)])
def test_head_counts(nkv, group, kf, vf):
    say(f"tree heads {nkv} x {group}")
    check(filled(300, kf, vf, nkv=nkv, group=group, page=16), 277, 23, "tree")
    check(filled(150, kf, vf, nkv=nkv, group=group), 0, 150, "tree")


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("n,pos0", [(1, 5000), (2, 4097), (9, 6000), (25, 4000), (65, 3001), (200, 2000), (513, 1500), (1024, 100)])
def test_longer(kf, vf, n, pos0):
    say(f"tree kf {kf} vf {vf}")
    check(filled(pos0 + n, kf, vf), pos0, n, "tree", gate=False)


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("page", [0, 48, 64])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_each_kernel(kf, vf, page, n, pos0):
    say(f"tree kf {kf} vf {vf} page {page}")
    check(filled(pos0 + n, kf, vf, page=page), pos0, n, "padded")


@pytest.mark.parametrize("kf,vf", [(Q8, Q8), (F16, F16)])
@pytest.mark.parametrize("nkv", [1, 2, 3])
@pytest.mark.parametrize("n,pos0", [(1, 20000), (40, 30000)])
def test_few_heads_many_ranges(kf, vf, nkv, n, pos0):
    """Up to 128 ranges of the keys, and numbers of ranges and row blocks that 8 does not divide."""
    say(f"tree heads {nkv} kf {kf}")
    check(filled(pos0 + n, kf, vf, nkv=nkv), pos0, n, "tree")


@pytest.mark.parametrize("kf,vf", [(Q8, Q8), (F16, F16)])
@pytest.mark.parametrize("nkv,group,n", [(3, 5, 41), (5, 3, 43), (16, 4, 65), (1, 33, 31), (16, 8, 600), (8, 8, 1024)])
def test_places(kf, vf, nkv, group, n):
    """Row blocks shared out over the XCDs, and more workgroups than one round of them."""
    say(f"tree heads {nkv} x {group} n {n}")
    check(filled(700 + n, kf, vf, nkv=nkv, group=group), 700, n, "tree", gate=False)


@pytest.mark.parametrize("vf", [Q8, F16])
@pytest.mark.parametrize("page", [0, 48, 64])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_each_kernel_with_values_that_are_not_finite(vf, page, n, pos0):
    """NaN in a drafted token's V that most rows do not see, and Inf in its K."""
    c = filled(pos0 + n, F16, vf, page=page)
    q, _ = rows(n, c.nh, 5, 0.1)
    mask = some_mask("tree", n, 9)
    mask[torch.arange(n, device="cuda") != 1, 0] &= ~2                 # (only token 1 sees token 1)
    want, _, size = attention(c, 0, pos0, q, mask)
    others = torch.arange(n, device="cuda") != 1
    for bad in (math.inf, math.nan):
        x = torch.full((4, HD), bad, device="cuda")
        put(c, "v", 0, pos0 + 1, x if vf == F16 else (torch.full((4, HD), 3, device="cuda"), torch.full((4, 8), bad, device="cuda")))
        put(c, "k", 0, pos0 + 1, x)
        out, _ = c.attn_tree(0, pos0, q, mask)
        check_rows(out[others], want[others], tolerance(size, pos0 + n)[others])
        assert bool(torch.isnan(out[1]).any())


@pytest.mark.parametrize("page", [48, 64])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_each_kernel_with_bad_pages(page, n, pos0):
    """As if the positions of a page outside the pool were absent, in the context and among the drafted tokens."""
    c = make_cache(pos0 + n, Q8, Q8, page=page)
    k, v = (torch.randn(pos0 + n, 4, HD, generator=gen(2 + i), device="cuda") for i in range(2))
    c.append(0, 0, k, v)
    q, _ = rows(n, c.nh, 4, 0.1)
    mask = some_mask("tree", n, 2)
    c.block_table[0, 3], c.block_table[0, 5] = -1, c.cap // page
    out, _ = c.attn_tree(0, pos0, q, mask)
    keep = torch.ones(pos0 + n, dtype=torch.bool, device="cuda")
    keep[3 * page:4 * page] = keep[5 * page:6 * page] = False
    d = make_cache(int(keep.sum()), Q8, Q8)
    d.append(0, 0, k[keep], v[keep])
    want, _, size = attention(d, 0, int(keep[:pos0].sum()), q, mask)
    check_rows(out, want, tolerance(size, pos0 + n))
    # nothing but the drafted tokens' own pages, and no page at all
    first = pos0 // page
    keep[:first * page], keep[first * page:] = False, True
    c.block_table[0, :first] = -1
    out, _ = c.attn_tree(0, pos0, q, mask)
    d = make_cache(int(keep.sum()), Q8, Q8)
    d.append(0, 0, k[keep], v[keep])
    want, _, size = attention(d, 0, pos0 - first * page, q, mask)
    check_rows(out, want, tolerance(size, pos0 + n))
    c.block_table[0, :] = -1
    assert not bool(c.attn_tree(0, pos0, q, mask)[0].any())


@pytest.mark.parametrize("kf,vf", [(Q8, Q8), (F16, F16)])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 127, 300])
@pytest.mark.parametrize("pos0", [0, 7])
def test_any_mask(kf, vf, n, pos0):
    """Any bits, rows without any, bits past the last token: rows that see nothing are 0 (and gated 0)."""
    say(f"tree mask n {n} pos0 {pos0}")
    c = filled(pos0 + n, kf, vf)
    out, _ = check(c, pos0, n, "random", accurate=n > 8)
    none = ~seen(some_mask("random", n, 3), n).any(1)
    if pos0 == 0:
        assert bool(none.any()) and not bool(out[none].any())


@pytest.mark.parametrize("kf,vf", FORMATS)
def test_what_a_row_does_not_see_has_no_effect(kf, vf):
    """Inf and NaN in the K and V of drafted tokens: the rows that do not see them are as without them, bit for bit
    where no other row of theirs does either."""
    pos0, n = 70, 20
    c = filled(pos0 + n + 40, kf, vf)
    q, g = rows(n, c.nh, 5)
    mask = some_mask("tree", n, 9)
    see = seen(mask, n)
    want, _, size = attention(c, 0, pos0, q, mask)
    for bad in (math.inf, -math.inf, math.nan):
        for j, which in ((n - 1, "v"), (n - 1, "k"), (3, "v"), (7, "k")):
            d = filled(pos0 + n + 40, kf, vf)
            fmt = kf if which == "k" else vf
            x = values(d, which, 0, pos0 + j, 1)[0].float()
            x[:, ::5] = bad
            if fmt == F16:
                put(d, which, 0, pos0 + j, x)
            else:
                s = torch.full((4, 8), 0.01, device="cuda")
                s[:, ::2] = bad
                put(d, which, 0, pos0 + j, (torch.full((4, HD), 3, device="cuda"), s))
            out, _ = d.attn_tree(0, pos0, q, mask)
            others = ~see[:, j]
            assert bool(others.any())
            check_rows(out[others], want[others], tolerance(size, pos0 + n)[others])
            mine, _, _ = attention(d, 0, pos0, q, mask)
            check_rows(out[~others], mine[~others], torch.full_like(mine[~others], 1e-4))


@pytest.mark.parametrize("kf,vf", FORMATS)
def test_positions_past_the_last_are_not_read(kf, vf):
    """Whatever lies behind the drafted tokens, in their own page and in the next, changes no bit."""
    pos0, n = 37, 6
    for page in (0, 16, 64):
        c = make_cache(200, kf, vf, page=page)
        scribble(c, 5)
        k, v = (torch.randn(pos0 + n, 4, HD, generator=gen(2 + i), device="cuda") for i in range(2))
        c.append(0, 0, k, v)
        q, g = rows(n, c.nh, 4)
        a, _ = c.attn_tree(0, pos0, q, some_mask("tree", n, 1))
        keep = [x.clone() for x in (c.k_data, c.v_data)]
        scribble(c, 77)
        c.append(0, 0, k, v)
        b, _ = c.attn_tree(0, pos0, q, some_mask("tree", n, 1))
        assert same(a, b) and bool(torch.isfinite(a).all()) and len(keep) == 2


@pytest.mark.parametrize("kf", [Q8, F16])
@pytest.mark.parametrize("scale", [2.0 ** -24, 2.0 ** -20, 1e-5, 1e-3, 1.0, 60.0, 700.0, 6e4])
def test_v_scales_over_their_whole_range(kf, scale):
    """q8_0 V from the smallest fp16 scale to the largest, all of one size and mixed with ordinary ones."""
    pos0, n = 200, 9
    c = filled(pos0 + n, kf, Q8)
    g = gen(8)
    c.v_data.copy_(torch.randint(-127, 128, c.v_data.shape, generator=g, device="cuda").to(torch.int8).view(torch.uint8))
    sc = torch.full((1, pos0 + n, 4 * 8), scale, device="cuda").half()
    c.v_scales.copy_(sc.view(torch.uint8).reshape(c.v_scales.shape))
    say(f"V scale {scale}")
    check(c, pos0, n, "tree")
    sc[:, ::2] *= 0.37
    sc[:, 5:60, :9] = 0.01
    sc[:, 100:120] = 0.0
    c.v_scales.copy_(sc.view(torch.uint8).reshape(c.v_scales.shape))
    check(c, pos0, n, "tree", accurate=False)


def far_larger(n, pos0, usual, big):
    c = filled(pos0 + n, Q8, Q8)
    v = torch.randn(pos0 + n, 4, HD, generator=gen(4), device="cuda") * usual
    v[pos0 + 1] *= big / usual
    c.append(0, 0, torch.randn(pos0 + n, 4, HD, generator=gen(5), device="cuda"), v)
    q, _ = rows(n, c.nh, 6, 0.01)
    mask = some_mask("tree", n, 9)
    mask[torch.arange(n, device="cuda") != 1, 0] &= ~2                 # (only token 1 sees token 1)
    out, _ = c.attn_tree(0, pos0, q, mask)
    want, _, size = attention(c, 0, pos0, q, mask)
    others = torch.arange(n, device="cuda") != 1
    say(f"usual {usual} big {big}: rel {rel(out[others], want[others]):.2e}")
    check_rows(out, want, tolerance(size, pos0 + n))
    assert rel(out[others], want[others]) < 4e-6
    # the same in the context, where every row sees it with next to no weight: the 2^-34 of sum |v| is the bound then
    k = torch.randn(pos0 + n, 4, HD, generator=gen(5), device="cuda")
    k[7] = -40.0
    v[pos0 + 1] *= usual / big
    v[7] *= big / usual
    c.append(0, 0, k, v)
    q = q.abs() * 100
    out, _ = c.attn_tree(0, pos0, q, mask)
    want, _, size = attention(c, 0, pos0, q, mask)
    # (6e6: most blocks' scales are above fp16's largest, Inf. The weight of e^-500 is not 0 in 64 bits, so Inf is the
    # sum there; it is far below 2^-149, fp32's smallest, and 0 * Inf is NaN)
    fin = torch.isfinite(want)
    assert not bool(torch.isfinite(out[~fin]).any()) and (big > 1e6 or bool(fin.all()))
    tol = tolerance(size, pos0 + n)
    check_rows(out[fin], want[fin], tol[fin])
    assert rel(out[fin], want[fin]) < 4e-6


@pytest.mark.parametrize("n", [3, 8, 30, 70])
@pytest.mark.parametrize("usual,big", [(1e-3, 100.0), (2e-2, 100.0), (1e-3, 2e4), (1.0, 2e4), (0.05, 1e6), (0.05, 6e6)])
def test_a_far_larger_v_among_ordinary_ones(n, usual, big):
    """A drafted token's q8_0 V, and one of the context with hardly any weight, 10^4 to 10^8 times the others': the
    rows that do not see it keep their precision. Scores are small, so that tolerance() is about 2^-19 of sum p |v|; the
    2-norm's bound is check()'s."""
    far_larger(n, 300, usual, big)


@pytest.mark.parametrize("usual,big", [(2e-2, 100.0), (1e-3, 2e4), (0.05, 1e6)])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_a_far_larger_v_in_each_kernel(n, pos0, usual, big):
    far_larger(n, pos0, usual, big)


def test_fp16_values_over_their_whole_range():
    pos0, n = 130, 5
    for mul in (6e-8, 1e-6, 1e-4, 1.0, 6e4):
        c = filled(pos0 + n, F16, F16)
        v = (torch.rand(pos0 + n, 4, HD, generator=gen(3), device="cuda") * 2 - 1) * mul
        c.v_data[0] = v.half().view(torch.uint8).reshape(pos0 + n, -1)
        say(f"V size {mul}")
        check(c, pos0, n, "tree")


@pytest.mark.parametrize("kf,vf", FORMATS)
@pytest.mark.parametrize("qscale", [0.0, 1e-6, 0.1, 8.0, 60.0])
def test_flat_and_peaked_scores(kf, vf, qscale):
    check(filled(1500, kf, vf), 1490, 10, "tree", qscale=qscale, accurate=qscale <= 1.0)


def test_growing_scores():
    """Every key beats the ones before it, so the reference is lifted all along; and the other way round."""
    for flip in (False, True):
        c = make_cache(1300, F16, Q8)
        ramp = torch.linspace(0, 30, 1300, device="cuda")
        if flip:
            ramp = ramp.flip(0)
        k = torch.randn(1300, 4, HD, generator=gen(1), device="cuda") * 0.05
        k[..., 0] = ramp[:, None]
        c.append(0, 0, k, torch.randn(1300, 4, HD, generator=gen(2), device="cuda"))
        q = torch.randn(8, 16, HD, generator=gen(3), device="cuda") * 0.1
        q[..., 0] = 40.0                           # scores 0 .. 75
        out, _ = c.attn_tree(0, 1292, q, some_mask("tree", 8, 2))
        want, _, size = attention(c, 0, 1292, q, some_mask("tree", 8, 2))
        check_rows(out, want, tolerance(size, 1300))


def test_scores_that_are_not_finite():
    """A visible key with a score of -Inf counts for nothing; +Inf or NaN makes its rows NaN, and only those."""
    c = filled(50, F16, F16)
    k = values(c, "k", 0, 45, 1)[0].float()
    k[0, 0] = math.inf
    put(c, "k", 0, 45, k)                          # drafted token 5, KV head 0
    q = torch.randn(10, 16, HD, generator=gen(3), device="cuda")
    q[:, :, 0] = q[:, :, 0].abs() + 0.1
    q[:, 1, 0] *= -1                               # head 1: -Inf
    mask = some_mask("tree", 10, 4)
    out, _ = c.attn_tree(0, 40, q, mask)
    want, _, size = attention(c, 0, 40, q, mask)
    sees = seen(mask, 10)[:, 5]
    assert bool(torch.isnan(out[sees][:, [0, 2, 3]]).all()) and bool(torch.isfinite(out[~sees]).all())
    assert bool(torch.isfinite(out[:, 4:]).all()) and bool(torch.isfinite(out[:, 1]).all())
    good = torch.isfinite(want)
    t = (want.abs() + 1.0) * 1e-4                  # (this test is about which rows are finite)
    check_rows(out[good], want[good], t[good])


def test_axes_of_one_may_have_any_stride():
    """One token, or one head, whose stride is whatever a view left there."""
    for nkv, group, n in ((4, 4, 1), (1, 1, 5)):
        c = filled(64, Q8, Q8, nkv=nkv, group=group)
        q, g = rows(n, c.nh, 4)
        want = c.attn_tree(0, 50, q, None, g)
        odd = [x.as_strided(x.shape, (1, HD, 1) if n == 1 else (HD, 3, 1)) for x in (q, g)]
        got = c.attn_tree(0, 50, odd[0], None, odd[1])
        assert all(same(a, b) for a, b in zip(want, got))


def test_positions_of_more_than_32_bits_are_refused():
    """They would be taken modulo 2^32."""
    c = filled(64, Q8, Q8)
    q, _ = rows(2, c.nh, 4)
    kv = torch.zeros(2, 4, HD, device="cuda")
    from bonsai_vk_amd import Rope
    before = [x.clone() for x in (c.k_data, c.v_data)]
    for pos0 in (2 ** 32, 2 ** 32 + 5, -2 ** 32 + 5, -1):
        for call in (lambda: c.attn_tree(0, pos0, q), lambda: c.read(0, pos0, 2), lambda: c.rope_append(0, pos0, None, kv, kv, Rope(0)),
                     lambda: c.commit(pos0, 2, torch.zeros(1, dtype=torch.int32, device="cuda"))):
            with pytest.raises(ValueError):
                call()
    assert same(before[0], c.k_data) and same(before[1], c.v_data)


def test_strided_rows():
    """q beside its gate ([nh][2 hd] per token), rows of a fused buffer, and copies where rows cannot be taken in place."""
    c = filled(400, Q8, Q8)
    n, pos0 = 12, 388
    q, g = rows(n, 16, 6)
    mask = some_mask("tree", n, 2)
    want = c.attn_tree(0, pos0, q, mask, g)
    qg = torch.cat([q, g], 2)
    fused = torch.randn(n, 16 * HD + 40 + 16 * HD, device="cuda")
    fq, fg = fused[:, :16 * HD].view(n, 16, HD), fused[:, 16 * HD + 40:].view(n, 16, HD)
    fq.copy_(q), fg.copy_(g)
    odd = torch.zeros(n, 16, HD + 1, device="cuda")
    odd[..., 1:] = q
    for a, b in ((qg[..., :HD], qg[..., HD:]), (fq, fg), (odd[..., 1:], g.transpose(0, 1).contiguous().transpose(0, 1)), (q.double(), g.half().float())):
        ga = b
        got = c.attn_tree(0, pos0, a, mask, ga)
        assert same(got[0], want[0])
        if b.dtype == torch.float32 and torch.equal(b, g):
            assert same(got[1], want[1])
    one = q[:1].expand(n, 16, HD)                  # (a token stride of 0)
    assert same(c.attn_tree(0, pos0, one, mask)[0], c.attn_tree(0, pos0, one.contiguous(), mask)[0])


def test_given_outputs_and_refusals():
    c = filled(100, Q8, Q8)
    q, g = rows(5, 16, 1)
    mask = some_mask("tree", 5, 1)
    out, og = torch.full((7, 16, HD), 7.0, device="cuda"), torch.full((7, 16, HD), 7.0, device="cuda")
    a = c.attn_tree(0, 90, q, mask, g, out=out[1:6], out_gated=og[1:6])
    b = c.attn_tree(0, 90, q, mask, g)
    assert same(a[0], b[0]) and same(a[1], b[1]) and a[0].data_ptr() == out[1:].data_ptr()
    for t in (out, og):                            # rows around the call's own stay as they were
        assert bool((t[0] == 7).all()) and bool((t[6] == 7).all())
    empty = c.attn_tree(0, 90, q[:0], None)
    assert empty[0].shape == (0, 16, HD)
    for bad in (dict(mask=mask.cpu()), dict(mask=mask.int()), dict(mask=mask[:4]), dict(gate=g[:4]), dict(out=out[:4]), dict(out_gated=og[:5]),
                dict(out=out[:5].transpose(0, 1)), dict(gate=g, out_gated=og[:5].double())):
        with pytest.raises(ValueError):
            c.attn_tree(0, 90, q, **{"mask": mask, **bad})
    with pytest.raises(ValueError):
        c.attn_tree(0, 90, q[:, :8])
    with pytest.raises(Exception, match="ECAP"):
        c.attn_tree(0, 96, q, mask)


def test_bad_pages_are_not_followed():
    """Table entries outside the pool: no row sees their positions, the others' results are as if they were absent."""
    c = make_cache(100, Q8, F16, page=16)
    k, v = (torch.randn(100, 4, HD, generator=gen(2 + i), device="cuda") for i in range(2))
    c.append(0, 0, k, v)
    q, _ = rows(7, 16, 4)
    mask = some_mask("tree", 7, 2)
    good = c.block_table.clone()
    for bad in (-1, c.cap // 16, 2**31 - 1, -2**31):
        c.block_table.copy_(good)
        c.block_table[0, 2] = bad                  # positions 32 .. 47
        out, _ = c.attn_tree(0, 93, q, mask)
        keep = torch.cat([torch.arange(0, 32), torch.arange(48, 100)]).cuda()
        c.block_table.copy_(good)
        d = make_cache(84, Q8, F16)
        d.append(0, 0, k[keep], v[keep])
        want, _, size = attention(d, 0, 77, q, mask)
        check_rows(out, want, tolerance(size, 100))
    c.block_table[0, :] = -1
    out, _ = c.attn_tree(0, 93, q, mask)
    assert not bool(out.any())


def test_offsets_past_32_bits():
    """An fp16 cache of more than 4 GiB per array: pages at its end."""
    nkv, page = 16, 64
    cap = 600064
    c = make_cache(1, F16, F16, nkv=nkv, cap=64)
    from bonsai_vk_amd import KvCache
    table = (cap // page - 1 - torch.arange(8)).int()[None]
    d = KvCache(n_layers=1, nh=64, nkv=nkv, cap=cap, k_fmt=F16, v_fmt=F16, page_tokens=page, max_pages=8, block_table=table)
    e = KvCache(n_layers=1, nh=64, nkv=nkv, cap=512, k_fmt=F16, v_fmt=F16)
    k, v = (torch.randn(500, nkv, HD, generator=gen(2 + i), device="cuda") for i in range(2))
    q, _ = rows(6, 64, 4)
    mask = some_mask("tree", 6, 2)
    for x in (d, e):
        x.append(0, 0, k, v)
    assert same(d.attn_tree(0, 494, q, mask)[0], e.attn_tree(0, 494, q, mask)[0]) and c.cap == 64
    for a, b in zip(d.read(0, 0, 500, torch.float16), e.read(0, 0, 500, torch.float16)):
        assert same(a, b)


def test_the_same_call_twice_and_other_layers():
    c = filled(900, Q8, Q8, layers=3, page=64)
    q, g = rows(20, 16, 2)
    mask = some_mask("tree", 20, 5)
    a = [c.attn_tree(layer, 880, q, mask, g)[1] for layer in range(3)]
    b = [c.attn_tree(layer, 880, q, mask, g)[1] for layer in range(3)]
    assert all(same(x, y) for x, y in zip(a, b))
    want = attention(c, 2, 880, q, mask, g)
    check_rows(a[2], want[1], tolerance(want[2], 900) + want[1].abs() * 2.0 ** -21)


def test_on_another_stream_and_in_a_graph():
    c = filled(2000, Q8, Q8)
    pos0, n = 1950, 17
    q, g = rows(n, 16, 2)
    mask = some_mask("tree", n, 5)
    want = c.attn_tree(0, pos0, q, mask, g)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = c.attn_tree(0, pos0, q, mask, g)
    s.synchronize()
    assert same(got[0], want[0]) and same(got[1], want[1])
    # two graphs on one workspace, replayed in turn with eager calls between them
    q2 = torch.randn_like(q)
    outs = [torch.empty_like(q) for _ in range(4)]
    graphs = []
    for qq, o, og in ((q, outs[0], outs[1]), (q2, outs[2], outs[3])):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.attn_tree(0, pos0, qq, mask, g, out=o, out_gated=og)
        graphs.append(graph)
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=gen(step), device="cuda"))
        q2.copy_(torch.randn(q.shape, generator=gen(100 + step), device="cuda"))
        for o in outs:
            o.zero_()
        for graph in graphs:
            graph.replay()
        eager = c.attn_tree(0, pos0, q, mask, g) + c.attn_tree(0, pos0, q2, mask, g)
        torch.cuda.synchronize()
        assert all(same(o, e) for o, e in zip(outs, eager))
    fresh = filled(100, Q8, Q8)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="tree_workspace"):
        with torch.cuda.graph(graph):
            fresh.attn_tree(0, 90, q[:5])


def test_workspace_serves_decodes_too():
    """One workspace of BKV_OP_TREE under both calls, in turn: neither changes the other's results."""
    c = filled(3000, Q8, Q8)
    ws = c.tree_workspace()
    from bonsai_vk_amd._lib import check as ok, lib
    ok(lib().bkv_workspace_init(c.desc, ws.data_ptr(), ws.numel(), c._stream()), "init")
    q, _ = rows(9, 16, 2)
    want = c.decode(0, 2500, q[0])[0]
    tree = c.attn_tree(0, 2991, q)[0]
    c.workspace = ws
    for _ in range(3):
        assert same(c.decode(0, 2500, q[0])[0], want)
        assert same(c.attn_tree(0, 2991, q)[0], tree)
    c.check_workspace()


@pytest.mark.parametrize("kf,vf", FORMATS)
def test_agrees_with_decode(kf, vf):
    """A chain's rows are the decodes at their positions, but for the rounding of the decodes' probabilities to fp16
    (half a step of 2^-11 each, so 2^-11 of sum p |v|)."""
    c = filled(700, kf, vf)
    q, g = rows(5, 16, 2)
    out, og = c.attn_tree(0, 695, q, None, g)
    _, _, size = attention(c, 0, 695, q, None)
    for i in range(5):
        d, dg = c.decode(0, 696 + i, q[i], g[i])
        assert bool(((out[i] - d).abs().double() <= size[0][i] * 2.0 ** -11 + tolerance(size, 700)[i]).all())
    assert bool(torch.isfinite(og).all()) and slots(c, 0, 0, 1).numel() == 1
