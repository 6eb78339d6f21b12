"""What the calls for several sequences refuse, before any GPU work, and the host parts of them: axes, workspace sizes, the
4-bit geometry. (No counterpart in the reference. No GPU: every call here is refused or has nothing to do.)"""
import ctypes

import numpy as np
import pytest

from bonsai_vk_amd import BkvError, RopeAxes
from bonsai_vk_amd._lib import BKV_Q4_0, BKV_Q8_0, BkvCacheDesc, BkvRope, BkvRopeAxes, BkvRows, BkvSeqs, lib

from seqs_util import q4_pack, q4_quantise, q4_values

EINVAL, ESHAPE, ECAP, EALIGN, EWORKSPACE, EUNSUPPORTED = -1, -2, -3, -4, -5, -7
PTR = 0x7F0000000000                               # (an address that is never followed: every call below ends before)


def desc(page=16, **kw):
    d = BkvCacheDesc()
    d.n_layers, d.nh, d.nkv, d.hd, d.cap = 2, 16, 4, 256, 1024
    d.k_fmt = d.v_fmt = BKV_Q4_0
    d.scale = 0.0625
    d.k_data, d.k_scales, d.v_data, d.v_scales = (PTR + i * (1 << 24) for i in range(4))
    for i, sb in enumerate((512, 64, 512, 64)):
        d.layer_stride_bytes[i] = 2 * sb * 1024
    if page:
        d.page_tokens, d.max_pages, d.block_table = page, 8, PTR
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def seqs(n_seq=3, n_tok=7, q_start=PTR, len=PTR, tables=PTR, max_q=0, reserved=0):
    return BkvSeqs(n_seq, n_tok, max_q, reserved, q_start, len, tables)


def rows(p=PTR, tok=4096, head=256):
    return BkvRows(p, tok, head)


def rope(nrot=64):
    r = BkvRope()
    assert lib().bkv_rope_init(ctypes.byref(r), nrot, 0, 1e7, 0, 1.0, 0.0, 32.0, 1.0) == 0
    return r


def axes(pairs=(12, 10, 10), order=1):
    x = BkvRopeAxes()
    assert lib().bkv_rope_axes_init(ctypes.byref(x), len(pairs), (ctypes.c_int32 * len(pairs))(*pairs), order) == 0
    return x


def attn(d=None, layer=0, s=None, q=None, gate=None, out=PTR, gated=None, ws=PTR, ws_bytes=1 << 40):
    return lib().bkv_seqs_attn(d or desc(), layer, s or seqs(), q or rows(), gate, out, gated, ws, ws_bytes, None)


def test_attention_refuses():
    L = lib()
    assert L.bkv_seqs_attn(None, 0, seqs(), rows(), None, PTR, None, PTR, 1 << 40, None) == EINVAL
    assert L.bkv_seqs_attn(desc(), 0, None, rows(), None, PTR, None, PTR, 1 << 40, None) == EINVAL
    assert L.bkv_seqs_attn(desc(), 0, seqs(), None, None, PTR, None, PTR, 1 << 40, None) == EINVAL
    assert attn(desc(hd=128)) == EUNSUPPORTED and attn(desc(hd=96)) == ESHAPE and attn(desc(nh=15)) == ESHAPE
    for bad in (dict(k_fmt=BKV_Q8_0), dict(v_fmt=BKV_Q8_0), dict(k_fmt=0), dict(v_fmt=0)):
        d = desc(**bad)
        for i in range(4):
            d.layer_stride_bytes[i] = 1 << 24
        assert attn(d) == EUNSUPPORTED, bad
    assert attn(desc(k_scales=None)) == EINVAL and attn(desc(v_scales=None)) == EINVAL and attn(desc(k_fmt=3)) == EINVAL
    assert attn(layer=-1) == EINVAL and attn(layer=2) == EINVAL
    for s in (seqs(n_seq=-1), seqs(n_seq=1025), seqs(n_tok=-1), seqs(len=None), seqs(tables=None), seqs(max_q=-1), seqs(reserved=1),
              seqs(n_seq=8, n_tok=7, q_start=None)):
        assert attn(s=s) == EINVAL
    assert attn(desc(page=0), s=seqs(n_seq=2, tables=None)) == EINVAL
    for s in (seqs(q_start=PTR + 2), seqs(len=PTR + 1), seqs(tables=PTR + 2)):
        assert attn(s=s) == EALIGN
    assert attn(s=seqs(n_tok=2**31 - 1)) == EUNSUPPORTED
    assert attn(q=rows(p=None)) == EINVAL and attn(q=rows(tok=-4)) == EINVAL
    assert attn(q=rows(p=PTR + 4)) == EALIGN and attn(q=rows(head=254)) == EALIGN
    assert attn(out=None) == EINVAL and attn(gated=PTR) == EINVAL and attn(gate=rows()) == EINVAL
    assert attn(out=PTR + 8) == EALIGN and attn(gate=rows(), gated=PTR + 4) == EALIGN and attn(gate=rows(head=2), gated=PTR) == EALIGN
    need = lib().bkv_seqs_workspace_bytes(desc(), 3, 7)
    assert need > 0
    assert attn(ws=None) == EWORKSPACE and attn(ws_bytes=need - 1) == EWORKSPACE and attn(ws=PTR + 16) == EALIGN


def test_nothing_to_do():
    assert attn(s=seqs(n_seq=0)) == 0 and attn(s=seqs(n_tok=0)) == 0
    L = lib()
    assert L.bkv_seqs_rope_append(desc(), 0, seqs(n_tok=0), rope(), None, None, rows(), rows(), None, None, 0.0, None, None, None) == 0
    assert L.bkv_seqs_read(desc(), 0, seqs(n_seq=0), 0, None, None, 0, 0, None) == 0
    assert L.bkv_pages_fork(desc(), 0, PTR, PTR, None, None, None) == 0


def test_append_refuses():
    def call(d=None, layer=0, s=None, r=None, x=None, q=None, k=None, v=None, qw=None, kw=None, eps=1e-6, at=PTR, out=None):
        return lib().bkv_seqs_rope_append(d or desc(), layer, s or seqs(), r or rope(), x, q, k or rows(), v or rows(), qw, kw, eps, at, out, None)
    assert lib().bkv_seqs_rope_append(desc(), 0, seqs(), None, None, None, rows(), rows(), None, None, 0.0, None, None, None) == EINVAL
    assert call(desc(hd=128)) == EUNSUPPORTED and call(layer=2) == EINVAL and call(s=seqs(n_seq=1025)) == EINVAL
    bad = rope()
    bad.nrot = 63
    assert call(r=bad) == EINVAL
    bad = rope()
    bad.turns[5] = float("nan")
    assert call(r=bad) == EINVAL
    assert call(x=axes((12, 10, 11))) == EINVAL                         # (33 pairs for 32)
    assert call(x=axes(), at=None) == EINVAL                            # (several axes and no positions)
    bad = axes()
    bad.axis[31] = 3
    assert call(x=bad) == EINVAL
    bad = axes()
    bad.n_axes = 9
    assert call(x=bad) == EINVAL
    assert call(q=rows()) == EINVAL and call(out=PTR) == EINVAL
    assert call(qw=PTR) == EINVAL and call(qw=PTR, kw=PTR, eps=-1.0) == EINVAL and call(qw=PTR, kw=PTR, eps=float("nan")) == EINVAL
    assert call(k=rows(p=PTR + 4)) == EALIGN and call(v=rows(tok=2)) == EALIGN and call(q=rows(head=1), out=PTR) == EALIGN
    assert call(at=PTR + 2) == EALIGN and call(q=rows(), out=PTR + 4) == EALIGN and call(qw=PTR + 4, kw=PTR) == EALIGN


def test_read_refuses():
    def call(d=None, layer=0, s=None, kind=0, k=PTR, v=PTR, tok=1024, head=256):
        return lib().bkv_seqs_read(d or desc(), layer, s or seqs(), kind, k, v, tok, head, None)
    assert call(layer=5) == EINVAL and call(kind=3) == EINVAL and call(k=None, v=None) == EINVAL
    assert call(tok=256) == EINVAL and call(head=128) == EINVAL and call(k=PTR + 4) == EALIGN and call(tok=1026) == EALIGN
    assert call(s=seqs(len=None)) == EINVAL and call(desc(hd=64)) == EUNSUPPORTED


def test_axes_refuse():
    L, x = lib(), BkvRopeAxes()

    def call(pairs, order=0, n=None):
        return L.bkv_rope_axes_init(ctypes.byref(x), len(pairs) if n is None else n, (ctypes.c_int32 * max(1, len(pairs)))(*pairs), order)
    assert call([]) == EINVAL and call([1] * 9) == EINVAL and call([5, -1]) == EINVAL and call([100, 29]) == EINVAL
    assert call([2**31 - 1, 2**31 - 1]) == EINVAL and call([4], order=2) == EINVAL and call([4], order=-1) == EINVAL
    assert L.bkv_rope_axes_init(None, 1, (ctypes.c_int32 * 1)(1), 0) == EINVAL and L.bkv_rope_axes_init(ctypes.byref(x), 1, None, 0) == EINVAL
    assert call([100, 28]) == 0 and x.n_pairs == 128 and list(x.axis[99:101]) == [0, 1]
    with pytest.raises(BkvError):
        RopeAxes([])
    with pytest.raises(ValueError):
        RopeAxes([4, 4], order="mixed")
    assert RopeAxes([3, 1, 2], "dealt").axis == [0, 1, 2, 0, 2, 0] and RopeAxes([3, 1, 2]).axis == [0, 0, 0, 1, 2, 2]


def test_pages_refuse():
    L = lib()
    need = L.bkv_pages_workspace_bytes(desc())
    assert need > 0 and L.bkv_pages_workspace_bytes(desc(page=0)) == 0

    def fork(d=None, n=3, tables=PTR, refs=PTR, len=None, parent=PTR):
        return L.bkv_pages_fork(d or desc(), n, tables, refs, len, parent, None)

    def extend(d=None, n=3, tables=PTR, refs=PTR, len=PTR, n_new=PTR, lack=PTR, ws=PTR, ws_bytes=need):
        return L.bkv_pages_extend(d or desc(), n, tables, refs, len, n_new, lack, ws, ws_bytes, None)

    def compact(d=None, n=3, tables=PTR, refs=PTR, to=PTR, refs_to=PTR, ws=PTR, ws_bytes=need):
        return L.bkv_pages_compact(d or desc(), n, tables, refs, to, refs_to, ws, ws_bytes, None)
    for f in (fork, extend, compact):
        assert f(desc(page=0)) == EINVAL and f(n=-1) == EINVAL and f(n=1025) == EINVAL and f(tables=None) == EINVAL and f(refs=None) == EINVAL
        assert f(tables=PTR + 2) == EALIGN and f(refs=PTR + 1) == EALIGN
        assert f(desc(max_pages=1 << 29)) == EUNSUPPORTED and f(desc(nh=3)) == ESHAPE
    assert fork(parent=None) == EINVAL and fork(parent=PTR + 2) == EALIGN and fork(len=PTR + 2) == EALIGN
    assert extend(len=None) == EINVAL and extend(n_new=None) == EINVAL and extend(lack=None) == EINVAL and extend(lack=PTR + 2) == EALIGN
    assert compact(to=None) == EINVAL and compact(refs_to=None) == EINVAL and compact(to=PTR + 2) == EALIGN
    for f in (extend, compact):
        assert f(ws=None) == EWORKSPACE and f(ws_bytes=need - 1) == EWORKSPACE and f(ws=PTR + 8) == EALIGN


def test_four_bit_geometry():
    L = lib()
    d = desc(page=0)
    assert L.bkv_geom_check(d) == 0 and [L.bkv_slot_bytes(d, i) for i in range(4)] == [512, 64, 512, 64]
    assert L.bkv_max_positions(d) == 1024 and L.bkv_decode_path(d, 10) == -1
    assert L.bkv_workspace_bytes(d, 0, 100) == L.bkv_workspace_bytes(d, 1, 100) == L.bkv_workspace_bytes(d, 2, 100) == 0
    assert L.bkv_attn_decode(d, 0, 5, PTR, None, PTR, None, PTR, 1 << 40, None) == EUNSUPPORTED
    assert L.bkv_attn_prefill_chunk(d, 0, 5, 2, PTR, None, PTR, None, PTR, 1 << 40, None) == EUNSUPPORTED
    assert L.bkv_attn_tree(d, 0, 5, 2, rows(), None, None, PTR, None, PTR, 1 << 40, None) == EUNSUPPORTED


def test_workspace_grows():
    L = lib()
    for nkv, nh in ((1, 1), (4, 16), (3, 15), (600, 1200)):
        last = 0
        for n_seq, n_tok in ((1, 1), (1, 5), (4, 5), (4, 400), (100, 400), (1024, 70000)):
            need = L.bkv_seqs_workspace_bytes(desc(nkv=nkv, nh=nh, layer_stride_bytes=(ctypes.c_uint64 * 4)(*[1 << 32] * 4)), n_seq, n_tok)
            assert need >= last > -1 and need > 0
            last = need
    assert L.bkv_seqs_workspace_bytes(desc(), 0, 5) == L.bkv_seqs_workspace_bytes(desc(), 3, 0) == L.bkv_seqs_workspace_bytes(desc(), 1025, 5) == 0
    assert L.bkv_seqs_workspace_bytes(desc(), 3, 2**31 - 1) == 0


def test_the_format_in_numpy():
    """The oracle itself: exact values in fp16, half a step's error, the extremes' codes."""
    r = np.random.default_rng(0)
    x = (r.standard_normal((500, 256)) * np.exp(r.uniform(-6, 6, (500, 1)))).astype(np.float32)
    c, d = q4_quantise(x)
    y = q4_values(q4_pack(c), d)
    assert np.array_equal(y.astype(np.float16).astype(np.float64), y) and np.array_equal(y, y.astype(np.float16))
    assert int((d & 7).max()) == 0 and int(c.min()) >= 0 and int(c.max()) <= 15
    step = np.abs(d.view(np.float16).astype(np.float64)).repeat(32, -1).reshape(500, 256)
    b = x.reshape(500, 8, 32)
    far = np.where(b.max(-1) >= -b.min(-1), b.max(-1), b.min(-1))[..., None].repeat(32, -1).reshape(500, 256)
    inside = np.sign(x) == np.sign(far)
    assert (np.abs(y - x)[inside] <= step[inside] * (0.5 + 8 * 2.0 ** -8)).all()
    assert (np.abs(y - x) <= step * (1.0 + 8 * 2.0 ** -8)).all()
