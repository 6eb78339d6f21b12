"""The host side of the drafted-token calls: masks and depths of a draft, rotary tables, and every refusal that the
C ABI makes before anything is launched (no GPU is touched)."""
import ctypes
import math
import random

import numpy as np
import pytest

from bonsai_vk_amd import BkvError, Rope, _lib, tree_mask
from tests.test_abi import call, desc

OK, EINVAL, ECAP, EALIGN, EWORKSPACE, EUNSUPPORTED = 0, -1, -3, -4, -5, -7
Z = 0x600000


def rows(p=Z, tok=4096, head=256):
    return _lib.BkvRows(p, tok, head)


# ------------------------------------------------------------------ masks
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 130, 1024])
def test_tree_mask_follows_the_parents(n):
    r = random.Random(n)
    parents = [r.randint(-1, i - 1) if r.random() < 0.9 else -1 for i in range(n)]
    mask, depth = tree_mask(parents)
    assert mask.shape == (n, -(-n // 64)) and depth.shape == (n,)
    words = mask.numpy().view(np.uint64)
    for i in range(n):
        chain, j = {i}, parents[i]
        while j >= 0:
            chain.add(j)
            j = parents[j]
        got = {64 * w + b for w in range(words.shape[1]) for b in range(64) if int(words[i, w]) >> b & 1}
        assert got == chain
        assert int(depth[i]) == len(chain) - 1


def test_tree_mask_refuses_what_is_no_tree():
    for parents in ([0], [-1, 1], [-1, 2, 0], [-2], [-1] * 1025):
        with pytest.raises(BkvError, match="EINVAL"):
            tree_mask(parents)
    assert call("bkv_tree_mask", None, 1, None, None) == EINVAL
    p = (ctypes.c_int32 * 2)(-1, 0)
    assert call("bkv_tree_mask", p, -1, None, None) == EINVAL
    assert call("bkv_tree_mask", p, 2, None, None) == OK           # (neither output asked for: a check)


# ------------------------------------------------------------------ rotary tables
def turns(r, n):
    return [r.params.turns[p] * 2 * math.pi for p in range(n)]


@pytest.mark.parametrize("nrot", [2, 20, 64, 256])
def test_rope_tables(nrot):
    # every step is a few fp64 operations: 1e-13 leaves 450 roundings (half an ulp each is 1.1e-16)
    half, base = nrot // 2, 1e6
    plain = [base ** (-2.0 * p / nrot) for p in range(half)]
    r = Rope(nrot, freq_base=base)
    assert r.params.mscale == 1.0 and r.params.nrot == nrot and r.params.layout == 0
    assert np.allclose(turns(r, half), plain, rtol=1e-13, atol=0)
    assert np.allclose(turns(Rope(nrot, freq_base=base, scaling="linear", factor=4.0), half), np.array(plain) / 4, rtol=1e-13, atol=0)
    if nrot > 2:
        b = base * 8.0 ** (nrot / (nrot - 2))
        assert np.allclose(turns(Rope(nrot, freq_base=base, scaling="ntk", factor=8.0), half),
                           [b ** (-2.0 * p / nrot) for p in range(half)], rtol=1e-12, atol=0)
    y = Rope(nrot, layout="interleaved", freq_base=base, scaling="yarn", factor=4.0, trained_ctx=4096)
    assert y.params.layout == 1 and abs(y.params.mscale - (1 + 0.1 * math.log(4))) < 2.0 ** -23
    got = turns(y, half)
    for p, t in enumerate(plain):
        assert t / 4 * (1 - 1e-12) <= got[p] <= t * (1 + 1e-12)
        # a pair that turns more than beta_fast times keeps its angle (one whole pair is the ramp's rounding), one
        # that turns less than beta_slow times is interpolated
        if p + 1 < half and 4096 * plain[p + 1] / (2 * math.pi) >= 32:
            assert got[p] == pytest.approx(t, rel=1e-12)
        if p >= 1 and 4096 * plain[p - 1] / (2 * math.pi) <= 1:
            assert got[p] == pytest.approx(t / 4, rel=1e-12)
    assert Rope(nrot, freq_base=base, scaling="yarn", factor=0.5, trained_ctx=4096).params.mscale == 1.0


@pytest.mark.parametrize("kw", [
    dict(nrot=7), dict(nrot=-2), dict(nrot=258), dict(freq_base=1.0), dict(freq_base=math.inf), dict(freq_base=math.nan),
    dict(scaling="linear", factor=0.0), dict(scaling="ntk", factor=-1.0), dict(scaling="ntk", nrot=2, factor=2.0),
    dict(scaling="yarn", factor=2.0), dict(scaling="yarn", factor=2.0, trained_ctx=4096, beta_fast=1.0, beta_slow=1.0),
    dict(scaling="yarn", factor=math.inf, trained_ctx=4096), dict(scaling="ntk", factor=1e300)])
def test_rope_refuses(kw):
    with pytest.raises(BkvError, match="EINVAL"):
        Rope(**kw)


def test_rope_names():
    with pytest.raises(ValueError):
        Rope(layout="neither")
    with pytest.raises(ValueError):
        Rope(scaling="other")
    assert call("bkv_rope_init", None, 64, 0, 1e4, 0, 1.0, 0.0, 0.0, 0.0) == EINVAL
    p = _lib.BkvRope()
    assert call("bkv_rope_init", p, 64, 2, 1e4, 0, 1.0, 0.0, 0.0, 0.0) == EINVAL
    assert call("bkv_rope_init", p, 64, 0, 1e4, 4, 1.0, 0.0, 0.0, 0.0) == EINVAL
    assert call("bkv_rope_init", p, 0, 0, 1e4, 3, 2.0, 64.0, 32.0, 1.0) == OK


# ------------------------------------------------------------------ refusals before a launch
def tree(d, layer=0, pos0=100, n=8, q=rows(), mask=None, gate=None, out=Z, og=None, ws=Z, size=1 << 40):
    return call("bkv_attn_tree", d, layer, pos0, n, q, mask, gate, out, og, ws, size, None)


def test_attn_tree_refusals():
    d = desc()
    assert tree(desc(hd=128)) == EUNSUPPORTED
    assert tree(desc(nh=15)) == -2
    assert tree(desc(nh=1 << 22), n=1024) == EUNSUPPORTED          # (rows are counted in 32 bits)
    assert tree(d, layer=8) == EINVAL and tree(d, layer=-1) == EINVAL
    assert tree(d, n=-1) == EINVAL and tree(d, n=1025) == EINVAL
    assert tree(d, n=0, q=None, out=None, ws=None) == OK
    assert tree(d, pos0=4089) == ECAP and tree(d, pos0=2**32 - 1, n=1) == ECAP
    assert tree(d, q=None) == EINVAL and tree(d, q=rows(p=None)) == EINVAL and tree(d, out=None) == EINVAL
    assert tree(d, q=rows(tok=-4)) == EINVAL and tree(d, q=rows(head=-256)) == EINVAL
    assert tree(d, q=rows(tok=4097)) == EALIGN and tree(d, q=rows(p=Z + 4)) == EALIGN and tree(d, out=Z + 8) == EALIGN
    assert tree(d, gate=rows()) == EINVAL and tree(d, og=Z) == EINVAL
    assert tree(d, gate=rows(head=258), og=Z) == EALIGN and tree(d, gate=rows(), og=Z + 4) == EALIGN
    assert tree(d, mask=Z + 4) == EALIGN
    assert tree(d, ws=None) == EWORKSPACE and tree(d, ws=Z + 16) == EALIGN
    paged = desc(page_tokens=64, max_pages=3, block_table=0x500000)
    assert tree(paged, pos0=185) == ECAP
    # a block table of more positions than 32 bits hold
    wide = desc(page_tokens=4096, max_pages=1 << 21, block_table=0x500000)
    assert call("bkv_max_positions", wide) == 1 << 33
    assert tree(wide, pos0=2**32 - 64, n=8) == ECAP and tree(wide, pos0=2**32 - 200, n=8, ws=None) == EWORKSPACE
    assert rope_call(wide, pos0=2**32 - 4) == ECAP and read(wide, pos0=2**32 - 8) == ECAP
    assert call("bkv_kv_commit", wide, 2**32 - 8, 8, 4, Z, None) == ECAP


def test_tree_workspace_does_not_depend_on_the_context():
    for kw in (dict(), dict(nh=4), dict(nh=32), dict(nh=20), dict(nh=3, nkv=1)):
        d = desc(cap=1 << 20, n_layers=1, **kw)
        need = call("bkv_workspace_bytes", d, 2, 1)
        assert need > call("bkv_workspace_bytes", d, 0, 1 << 20) and need == call("bkv_workspace_bytes", d, 2, 1 << 20)
        assert call("bkv_workspace_bytes", d, 2, 0) == 0
        # a workspace for decodes is refused
        assert tree(d, size=call("bkv_workspace_bytes", d, 0, 1 << 20)) == EWORKSPACE
    assert call("bkv_workspace_bytes", desc(), 3, 1) == 0


def rope_call(d, rope=None, layer=0, pos0=0, n=4, q=rows(), k=rows(), v=rows(), qn=None, kn=None, eps=1e-6, pos=None, out=Z):
    return call("bkv_rope_append", d, layer, pos0, n, rope or Rope().params, q, k, v, qn, kn, eps, pos, out, None)


def test_rope_append_refusals():
    d = desc()
    assert rope_call(desc(hd=128)) == EUNSUPPORTED
    assert call("bkv_rope_append", d, 0, 0, 4, None, rows(), rows(), rows(), None, None, 1e-6, None, Z, None) == EINVAL
    assert rope_call(d, layer=8) == EINVAL and rope_call(d, n=-1) == EINVAL and rope_call(d, n=0) == OK
    assert rope_call(d, pos0=4093) == ECAP
    for change in (dict(nrot=3), dict(nrot=300), dict(nrot=-2), dict(layout=2), dict(mscale=math.nan)):
        p = Rope().params
        for key, value in change.items():
            setattr(p, key, value)
        assert rope_call(d, rope=p) == EINVAL
    p = Rope().params
    p.turns[31] = math.inf
    assert rope_call(d, rope=p) == EINVAL
    p.turns[31], p.turns[32] = 0.1, math.inf                   # (past nrot / 2: not read)
    assert rope_call(d, rope=p, n=0) == OK
    assert rope_call(d, qn=Z) == EINVAL and rope_call(d, qn=Z, kn=Z, eps=-1.0) == EINVAL
    assert rope_call(d, qn=Z, kn=Z, eps=math.nan) == EINVAL and rope_call(d, qn=Z + 4, kn=Z) == EALIGN
    assert rope_call(d, out=None) == EINVAL and rope_call(d, q=None) == EINVAL
    assert rope_call(d, k=None) == EINVAL and rope_call(d, v=rows(p=None)) == EINVAL
    assert rope_call(d, v=rows(tok=2)) == EALIGN and rope_call(d, out=Z + 4) == EALIGN and rope_call(d, pos=Z + 2) == EALIGN


def read(d, layer=0, pos0=0, n=8, t=0, k=Z, v=Z, tok=1024, head=256):
    return call("bkv_kv_read", d, layer, pos0, n, t, k, v, tok, head, None)


def test_read_refusals():
    d = desc()
    assert read(desc(hd=128)) == EUNSUPPORTED
    assert read(d, layer=9) == EINVAL and read(d, n=-1) == EINVAL and read(d, n=0) == OK
    assert read(d, t=3) == EINVAL and read(d, t=-1) == EINVAL
    assert read(d, pos0=4089) == ECAP and read(d, k=None, v=None) == EINVAL
    # rows that overlap: tokens inside a token's heads, heads inside a head's tokens
    assert read(d, tok=1020) == EINVAL and read(d, head=252) == EINVAL and read(d, tok=256, head=2044) == EINVAL
    assert read(d, tok=-1024) == EINVAL and read(d, tok=0) == EINVAL and read(d, head=0) == EINVAL
    assert read(d, tok=2**62, head=2**62) == EINVAL
    assert read(d, tok=1026) == EALIGN and read(d, tok=1028, t=1) == EALIGN and read(d, k=Z + 8) == EALIGN and read(d, v=Z + 4) == EALIGN


def test_commit_refusals():
    d = desc()

    def commit(d, pos0=0, n=8, keep=4, idx=Z):
        return call("bkv_kv_commit", d, pos0, n, keep, idx, None)

    assert commit(desc(hd=128)) == EUNSUPPORTED
    assert commit(d, n=-1) == EINVAL and commit(d, n=1025) == EINVAL and commit(d, keep=9) == EINVAL and commit(d, keep=-1) == EINVAL
    assert commit(d, keep=0, idx=None) == OK and commit(d, idx=None) == EINVAL and commit(d, idx=Z + 2) == EALIGN
    assert commit(d, pos0=4089) == ECAP


def test_library_names():
    assert _lib.BKV_TREE_MAX_Q == 1024
    assert ctypes.sizeof(_lib.BkvRope) == 16 + 128 * 8 and ctypes.sizeof(_lib.BkvRows) == 24
