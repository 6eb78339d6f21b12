"""bkv_attn_tree with V of very different sizes in different dims, held to the formula in 64 bits dim by dim: a row's
large outputs say nothing about its small ones."""
import math
import random

import pytest
import torch

from tests.gpu_util import say
from tests.test_gpu_tree import KERNELS, filled, rows
from tests.tree_util import F16, HD, Q8, attention, check_rows, gen, rel, seen, some_mask, tolerance, values

pytestmark = pytest.mark.gpu
SMALL = {0: 1e-5, 9: 1e-6, 66: 1e-6, 130: 1e-7, 131: 2.0 ** -24, 250: 1e-7}   # dims and the size of their V


def put_v(c, v):
    """v [n][nkv][HD] as the fp16 V of the first n positions, unrounded by any append."""
    c.v_data[0, :v.shape[0]] = v.half().view(torch.uint8).reshape(v.shape[0], -1)


def small_dims(v):
    for d, size in SMALL.items():
        v[..., d] *= size / 0.5
    return v


def check_dims(c, pos0, n, q, mask, dims):
    out, _ = c.attn_tree(0, pos0, q, mask)
    want, _, size = attention(c, 0, pos0, q, mask)
    worst = max(rel(out[..., d], want[..., d]) for d in dims)
    say(f"  n {n} pos0 {pos0}: worst dim {worst:.2e}")
    check_rows(out, want, tolerance(size, pos0 + n))
    # A dim's outputs are as precise as a whole row's: its products and sums are its own. 4e-6 as for whole rows, the
    # scores being smaller here.
    assert worst < 4e-6
    return out, want


def largest_weight(c, pos0, q, mask):
    """The largest probability of each row, [n][nh][1], in 64 bits."""
    n, group = q.shape[0], c.nh // c.nkv
    k = values(c, "k", 0, 0, pos0 + n)
    see = torch.cat([torch.ones(n, pos0, dtype=torch.bool, device="cuda"), seen(mask, n)], 1)
    top = []
    for h in range(c.nh):
        s = (q[:, h].half().double() @ k[:, h // group].t().contiguous()) * c.scale
        top.append(torch.softmax(s.masked_fill(~see, -math.inf), 1).max(1).values)
    return torch.stack(top, 1)[..., None]


def by_key(nk):
    """What rows that are computed key by key add to a 2-norm: the sums of p and of p v are up to nk fp32 additions, one
    after another, each off by 2^-24 of what the sum comes to."""
    return 2 * nk * 2.0 ** -24


def check_tiny(c, pos0, n, q, mask):
    """Values that are left subnormal: up to 2^-36 of the largest weight for each position (bkv_attn_tree's bound)."""
    out, _ = c.attn_tree(0, pos0, q, mask)
    want, _, size = attention(c, 0, pos0, q, mask)
    check_rows(out, want, tolerance(size, pos0 + n) + (pos0 + n) * 2.0 ** -36 * largest_weight(c, pos0, q, mask))
    assert rel(out, want) < 4e-6


@pytest.mark.parametrize("kf", [Q8, F16])
@pytest.mark.parametrize("page", [0, 48, 64])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_dims_of_small_fp16_values(kf, page, n, pos0):
    """V of 1e-5 to fp16's smallest in a few dims, ordinary in the others."""
    c = filled(pos0 + n, kf, F16, page=page)
    v = small_dims(torch.randn(pos0 + n, 4, HD, generator=gen(6), device="cuda") * 0.5)
    c.append(0, 0, torch.randn(pos0 + n, 4, HD, generator=gen(7), device="cuda"), v)
    q, _ = rows(n, 16, 3, 0.5)
    check_dims(c, pos0, n, q, some_mask("tree", n, 3), SMALL)


@pytest.mark.parametrize("kf", [Q8, F16])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_dims_of_small_fp16_values_beside_large_ones(kf, n, pos0):
    """The same with values of 100 and more: in two dims of every key, and in all of two keys."""
    for where in ("dims", "keys"):
        c = filled(pos0 + n, kf, F16)
        v = torch.randn(pos0 + n, 4, HD, generator=gen(6), device="cuda") * 0.5
        if where == "dims":
            v[..., 7] *= 400.0
            v[..., 200] *= 60000.0
        else:
            v[5] *= 1000.0
            v[pos0 - 3] *= 30000.0
        small_dims(v)
        put_v(c, v.clamp(-6e4, 6e4))
        q, _ = rows(n, 16, 3, 0.5)
        check_tiny(c, pos0, n, q, some_mask("tree", n, 3))


@pytest.mark.parametrize("kf", [Q8, F16])
@pytest.mark.parametrize("page", [0, 48])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_dims_that_are_small_in_some_steps(kf, page, n, pos0):
    """Runs of 1 to 5 steps of 32 keys whose small dims come and go, in each quarter of the dims by itself: the outputs
    change their unit back and forth."""
    c = filled(pos0 + n, kf, F16, page=page)
    nk = pos0 + n
    v = torch.randn(nk, 4, HD, generator=gen(6), device="cuda") * 0.5
    r = random.Random(n)
    for quarter in range(4):
        at, on = 0, False
        while at < nk:
            end = at + 32 * r.randint(1, 5)
            if on:
                v[at:end, :, 64 * quarter + 5:64 * quarter + 64:13] *= 1e-7 / 0.5
            at, on = end, not on
    put_v(c, v) if not page else c.append(0, 0, torch.randn(nk, 4, HD, generator=gen(7), device="cuda"), v)
    q, _ = rows(n, 16, 3, 0.5)
    check_dims(c, pos0, n, q, some_mask("tree", n, 3), range(5, HD, 13))


@pytest.mark.parametrize("kf", [Q8, F16])
def test_steps_with_and_without_large_values(kf):
    """Large values in some keys of many: the outputs change their unit back and forth, in each half of the dims."""
    for n, pos0 in KERNELS:
        c = filled(pos0 + n, kf, F16)
        v = torch.randn(pos0 + n, 4, HD, generator=gen(6), device="cuda") * 0.5
        v[::77, :, :100] *= 300.0
        v[::50, :, 150:] *= 500.0
        put_v(c, v)
        q, _ = rows(n, 16, 3, 0.5)
        check_dims(c, pos0, n, q, some_mask("padded", n, 3), range(0, HD, 15))


@pytest.mark.parametrize("vf", [F16, Q8])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_small_values_behind_a_zero_of_a_large_weight(vf, n, pos0):
    """One key with nearly all of the weight has V = 0, the others the type's smallest: the result is theirs, not 0."""
    c = filled(pos0 + n, F16, vf)
    k = torch.randn(pos0 + n, 4, HD, generator=gen(7), device="cuda") * 0.01
    v = torch.full((pos0 + n, 4, HD), 2.0 ** -24, device="cuda")
    q = torch.randn(n, 16, HD, generator=gen(8), device="cuda") * 0.01
    q[..., 0] = 1.0
    k[3, :, 0] = 16 * 9.7                          # a score of 9.7, e^9.7 = 2^14
    v[3] = 0.0
    c.append(0, 0, k, v)
    if vf == F16:
        put_v(c, v)
    else:                                          # (bytes of 1 with fp16's smallest scale)
        c.v_data.fill_(1)
        c.v_scales.copy_(torch.full((c.v_scales.numel() // 2,), 2.0 ** -24, device="cuda").half().view(torch.uint8).view(c.v_scales.shape))
        c.v_data[0, 3] = 0
    mask = some_mask("tree", n, 3)
    out, _ = c.attn_tree(0, pos0, q, mask)
    want, _, size = attention(c, 0, pos0, q, mask)
    check_rows(out, want, tolerance(size, pos0 + n))
    assert float(want.min()) > 0 and rel(out, want) < 4e-6 + by_key(pos0 + n)


def q8_rows(c, n, scales):
    """Small whole numbers in every dim, under scales [n][4][8]."""
    b = torch.randint(-2, 3, (n, 4, HD), generator=gen(11), device="cuda")
    c.v_data[0, :n] = b.to(torch.int8).view(torch.uint8).reshape(n, -1)
    c.v_scales[0, :n] = scales.half().view(torch.uint8).reshape(n, -1)


@pytest.mark.parametrize("kf", [Q8, F16])
@pytest.mark.parametrize("big", [0.3, 1.0, 100.0, 300.0, 6e4])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_blocks_of_small_q8_0_scales_beside_large_ones(kf, big, n, pos0):
    """q8_0 blocks whose values are fp16's smallest beside blocks of ordinary and of large ones, in every key; and as
    much of each in some keys only, beside others whose blocks in the same place are large."""
    for some in (False, True):
        c = filled(pos0 + n, kf, Q8)
        g = gen(9)
        sc = torch.full((pos0 + n, 4, 8), 0.01, device="cuda")
        small = 2.0 ** -24 * torch.randint(1, 4, (pos0 + n, 4, 2), generator=g, device="cuda")
        sc[..., 1::4] = small
        sc[..., 2] = big
        if some:
            sc[::3, :, 1::4] = 0.02
            sc[1::5, :, 2] = 0.01
        q8_rows(c, pos0 + n, sc)
        q, _ = rows(n, 16, 3, 0.5)
        mask = some_mask("tree", n, 3)
        check_tiny(c, pos0, n, q, mask)


@pytest.mark.parametrize("vf", [F16, Q8])
@pytest.mark.parametrize("n,pos0", KERNELS)
def test_rows_that_are_small_as_a_whole(vf, n, pos0):
    """V of 1e-6 in every dim beside one key of 100 that no row but its own sees, and V of 0.5 with next to no weight
    beside keys of 1e-6: such rows are computed key by key where the products would be subnormal."""
    for case in ("all", "some"):
        c = filled(pos0 + n, F16, vf)
        k = torch.randn(pos0 + n, 4, HD, generator=gen(7), device="cuda") * 0.01
        v = torch.randn(pos0 + n, 4, HD, generator=gen(8), device="cuda") * (1e-6 if case == "all" else 0.5)
        q = torch.randn(n, 16, HD, generator=gen(9), device="cuda") * 0.01
        mask = some_mask("tree", n, 3)
        if case == "all":
            v[pos0 + 1] *= 1e8
            mask[torch.arange(n, device="cuda") != 1, 0] &= ~2
        else:
            q[..., 0] = 4.0
            k[3::20, :, 0] = 72.0 + 4 * torch.randn(k[3::20].shape[0], 4, generator=gen(10), device="cuda")   # scores about 18
            v[3::20] *= 2e-6
        c.append(0, 0, k, v)
        if vf == F16:
            put_v(c, v)
        out, _ = c.attn_tree(0, pos0, q, mask)
        want, _, size = attention(c, 0, pos0, q, mask)
        check_rows(out, want, tolerance(size, pos0 + n) + size[0] * by_key(pos0 + n))
        # (scores of 18 are off by 18 * 1.44 * 2^-23 = 3e-6 at most, each for itself)
        others = torch.arange(n, device="cuda") != 1
        assert rel(out[others], want[others]) < 4e-6 + by_key(pos0 + n)


def test_v_of_zeros_is_zero():
    for vf in (F16, Q8):
        for n, pos0 in KERNELS:
            c = filled(pos0 + n, F16, vf)
            c.v_data.zero_()
            out, _ = c.attn_tree(0, pos0, rows(n, 16, 3)[0], some_mask("tree", n, 3))
            assert not bool(out.any())
