"""Caches with known contents, and the drafted-token operators in 64 bits (on the GPU, in plain torch)."""
import math
import random

import numpy as np
import torch

from bonsai_vk_amd import BKV_F16, BKV_Q8_0, KvCache, tree_mask

HD = 256
Q8, F16 = BKV_Q8_0, BKV_F16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_cache(n, kf, vf, page=0, nkv=4, group=4, layers=1, seed=0, spare=2, cap=None):
    """A cache of room for n positions; paged: shuffled pages of a pool with `spare` more than are needed."""
    if not page:
        return KvCache(n_layers=layers, nh=nkv * group, nkv=nkv, cap=cap or n, k_fmt=kf, v_fmt=vf)
    pages = -(-n // page)
    pool = pages + spare
    table = torch.stack([torch.randperm(pool, generator=torch.Generator().manual_seed(seed + i))[:pages] for i in range(layers)])
    return KvCache(n_layers=layers, nh=nkv * group, nkv=nkv, cap=pool * page, k_fmt=kf, v_fmt=vf, page_tokens=page,
                   max_pages=pages, block_table=table.int())


def slots(c, layer, first, n):
    p = torch.arange(first, first + n, device="cuda")
    if c.block_table is None:
        return p
    return c.block_table[layer].long()[p // c.page_tokens] * c.page_tokens + p % c.page_tokens


def arrays(c):
    return [a for a in (c.k_data, c.k_scales, c.v_data, c.v_scales) if a is not None]


def scribble(c, seed):
    """Random bytes everywhere (NaN and Inf patterns of fp16 among them)."""
    for i, a in enumerate(arrays(c)):
        a.copy_(torch.randint(0, 256, a.shape, generator=gen(seed + i), device="cuda", dtype=torch.uint8))


def values(c, which, layer, first, n):
    """Positions first .. of K or V in 64 bits, [n][nkv][HD]."""
    at = slots(c, layer, first, n)
    data, scales = (c.k_data, c.k_scales) if which == "k" else (c.v_data, c.v_scales)
    d = data[layer][at]
    if scales is None:
        return d.view(torch.float16).view(n, c.nkv, HD).double()
    s = scales[layer][at].view(torch.float16).view(n, c.nkv, HD // 32, 1).double()
    return (d.view(torch.int8).view(n, c.nkv, HD // 32, 32).double() * s).flatten(-2)


def put(c, which, layer, pos, x):
    """Raw fp16 values of an fp16 array at one position, or (bytes, scales) of a q8_0 one."""
    at = slots(c, layer, pos, 1)[0]
    data, scales = (c.k_data, c.k_scales) if which == "k" else (c.v_data, c.v_scales)
    if scales is None:
        data[layer, at] = x.half().contiguous().view(torch.uint8).reshape(-1)
    else:
        q, s = x
        data[layer, at] = q.to(torch.int8).contiguous().view(torch.uint8).reshape(-1)
        scales[layer, at] = s.half().contiguous().view(torch.uint8).reshape(-1)


def parents(n, seed):
    r = random.Random(seed)
    return [-1 if i == 0 or r.random() < 0.1 else r.randint(max(0, i - 5), i - 1) for i in range(n)]


def some_mask(kind, n, seed):
    """int64 mask words on the GPU, or None for a chain."""
    if kind == "chain":
        return None
    if kind == "random":                           # any bits, some rows without any, bits past n set
        g = gen(seed)
        w = torch.randint(-2**62, 2**62, (n, -(-n // 64)), generator=g, device="cuda")
        w[::3] = 0
        return w
    mask = tree_mask(parents(n, seed))[0]
    if kind == "padded":
        mask[n - n // 3:] = 0
    return mask.cuda()


def seen(mask, n):
    j = torch.arange(n, device="cuda")
    if mask is None:
        return j[None] <= j[:, None]
    return (mask[:, j // 64] >> (j % 64)) & 1 != 0


def attention(c, layer, pos0, q, mask, gate=None):
    """(out, out_gated, what tolerance() takes): bkv_attn_tree in 64 bits. The last is, per row and dim, sum p |v| over
    the visible keys, the largest score's absolute sum, and sum |v|."""
    n, nk, group = q.shape[0], pos0 + q.shape[0], c.nh // c.nkv
    k, v = values(c, "k", layer, 0, nk), values(c, "v", layer, 0, nk)
    kb, ks = k, None
    if c.k_scales is not None:                     # the path's q8_0 scores: per block the scale times the bytes' sum
        at = slots(c, layer, 0, nk)
        kb = c.k_data[layer][at].view(torch.int8).view(nk, c.nkv, HD).double()
        ks = c.k_scales[layer][at].view(torch.float16).view(nk, c.nkv, HD // 32).double()
    see = torch.cat([torch.ones(n, pos0, dtype=torch.bool, device="cuda"), seen(mask, n)], 1)
    out = torch.zeros(n, c.nh, HD, dtype=torch.float64, device="cuda")
    size, top, every = torch.zeros_like(out), 0.0, torch.zeros_like(out)
    for h in range(c.nh):
        kh, vh = k[:, h // group].contiguous(), v[:, h // group].contiguous()
        q16 = q[:, h].half().double()
        if ks is None:
            s = (q16 @ kh.t().contiguous()) * c.scale
        else:
            s = 0
            for b in range(HD // 32):
                s = s + (q16[:, 32 * b:32 * b + 32] @ kb[:, h // group, 32 * b:32 * b + 32].t().contiguous()) * ks[:, h // group, b]
            s = s * c.scale
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        fin = torch.where(see, (q16.abs() @ kh.abs().t().contiguous()) * c.scale, torch.zeros_like(s))
        top = max(top, float(fin[torch.isfinite(fin)].max()))
        some = see.any(1)
        p = torch.softmax(s[some], 1)
        if bool(torch.isfinite(vh).all()):
            out[some, h], size[some, h] = p @ vh, p @ vh.abs()
            every[some, h] = see[some].double() @ vh.abs()
            continue
        for i, row in zip(torch.nonzero(some).flatten().tolist(), p):
            m = see[i]
            out[i, h] = row[m] @ vh[m]
            size[i, h] = row[m] @ vh[m].abs()
            every[i, h] = vh[m].abs().sum(0)
    g = None if gate is None else out * torch.sigmoid(gate.double())
    return out, g, (size, top, every)


def tolerance(sizes, nk):
    """What fp32 arithmetic of the kernels may add to each output, per element.
    A score is 8 products of 32 terms on the matrix cores and 8 fp32 steps; the cores may cut instead of round, so
    each of at most 40 steps is off by 2^-23 of the terms' absolute sum A at most, the products with the softmax
    scale and log2(e) by 2^-23 A more; a probability is off by twice the largest score error (its own and the
    sum's) and 2^-21 for exp2 and its split in two; P V takes nk / 32 * 3 steps at most, one after another, and 8 to
    join, each cut by 2^-23 of the sum of p |v|.
    A probability enters as two fp16 of 2^9 times its ratio to a reference. The second one's last place is 2^-24 at
    least (fp16 has no smaller), so a ratio is off by up to 2^-25 / 2^9 whatever its size, and as the key that set the
    reference has the ratio 1, the sum that divides is 1 at least: 2^-34 of sum |v|. (Beside one key far above all
    others the sum of p |v| can be smaller than that, where that key's v is 0.)"""
    size, top, every = sizes
    return size * (2.0 ** -23 * (2 * 42 * top + 8 + nk / 32 * 3 + 8) + 2.0 ** -20) + every * 2.0 ** -34 + 1e-37


def check_rows(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    bad &= ~(torch.isnan(got) & torch.isnan(want)) & ~(got.double() == want)
    assert not bool(bad.any()), (torch.nonzero(bad)[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())


def rel(got, want):
    """2-norm of the difference over the 2-norm of the result."""
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-300))


def bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy().tobytes() if t.numel() else b""


def same(a, b):
    return bool(np.array_equal(np.frombuffer(bits(a), np.uint8), np.frombuffer(bits(b), np.uint8)))
