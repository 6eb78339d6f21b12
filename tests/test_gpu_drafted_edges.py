"""Calls at the edges of the drafted-token operators' ranges: outputs whose axes of one have any stride, and caches
whose offsets pass 32 bits in each attention kernel."""
import pytest
import torch

from bonsai_vk_amd import KvCache
from tests.tree_util import F16, HD, Q8, attention, check_rows, gen, make_cache, same, some_mask, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nkv,n", [(4, 1), (1, 5), (1, 1), (4, 0)])
def test_read_into_rows_with_axes_of_one(nkv, n):
    """One position, or one head: the stride of that axis means nothing, and need not be the same for K and V."""
    c = make_cache(16, Q8, F16, nkv=nkv)
    k, v = (torch.randn(16, nkv, HD, generator=gen(i), device="cuda") for i in range(2))
    from bonsai_vk_amd import Rope
    c.rope_append(0, 0, None, k, v, Rope(0))
    want = c.read(0, 3, n)
    shape = (n, nkv, HD)
    odd = (7 if n <= 1 else nkv * HD, 3 if nkv == 1 else HD, 1)
    ko = torch.zeros(6 * nkv * HD, device="cuda").as_strided(shape, odd)
    vo = torch.zeros(6 * nkv * HD, device="cuda").as_strided(shape, (nkv * HD, HD, 1))
    for a, b in ((ko, vo), (vo, ko), (ko, None), (None, ko)):
        for t in (ko, vo):
            t.fill_(-1.0)
        c.read(0, 3, n, k_out=a, v_out=b)
        for t, w in zip((a, b), want):
            assert t is None or same(t, w)


def test_read_refuses_other_layouts():
    c = make_cache(16, Q8, Q8)
    a = torch.zeros(5, 4, HD, device="cuda")
    wide = torch.zeros(5, 4, 2 * HD, device="cuda")
    for k, v in ((a, wide[..., :HD]), (a, torch.zeros(4, 5, HD, device="cuda").transpose(0, 1)), (wide[..., ::2], wide[..., 1::2]),
                 (a.transpose(0, 1), None), (a[0], None), (a, a.half())):
        with pytest.raises(ValueError):
            c.read(0, 0, 5, k_out=k, v_out=v)


# drafts of 16 KV heads that 16, 128 and 256 rows a workgroup are chosen for
FAR = [(6, 1000), (200, 900), (600, 600)]


@pytest.mark.parametrize("page", [48, 64])
@pytest.mark.parametrize("n,pos0", FAR)
def test_offsets_past_32_bits_in_each_kernel(n, pos0, page):
    """An fp16 cache of more than 4 GiB per array, its positions in the pages at its end, bit for bit as in the same
    pages of a small one: a slot of its own per key, and whole steps."""
    nkv, used = 16, -(-1200 // page)
    pool = 600000 // page                          # 8 KiB a slot
    small, far = (KvCache(n_layers=1, nh=64, nkv=nkv, cap=pages * page, k_fmt=F16, v_fmt=F16, page_tokens=page, max_pages=used,
                          block_table=(pages - 1 - torch.arange(used)).int()[None]) for pages in (used, pool))
    k, v = (torch.randn(pos0 + n, nkv, HD, generator=gen(2 + i), device="cuda") for i in range(2))
    q = torch.randn(n, 64, HD, generator=gen(4), device="cuda")
    mask = some_mask("tree", n, 2)
    for c in (small, far):
        c.append(0, 0, k, v)
    assert far.k_data.numel() > 2 ** 32 and not bool(far.k_data[0, :(pool - used) * page].any())
    assert same(far.attn_tree(0, pos0, q, mask)[0], small.attn_tree(0, pos0, q, mask)[0])
    idx = torch.tensor([n - 1, 0], dtype=torch.int32, device="cuda")
    for c in (small, far):
        c.commit(pos0, n, idx)
    for a, b in zip(far.read(0, 0, pos0 + n), small.read(0, 0, pos0 + n)):
        assert same(a, b)


# the same of 64 KV heads without groups
FAR_CONTIGUOUS = [(3, 139000), (100, 139000), (600, 139000)]


@pytest.mark.parametrize("n,pos0", FAR_CONTIGUOUS)
def test_offsets_past_32_bits_without_pages(n, pos0):
    """32 KiB a position: the last 300 of the context and the drafted ones lie past 4 GiB. Their scores are about 40, the
    others' 0 with V = 0: their weight is 139000 e^-40 = 6e-13, so the result is that of the last ones alone."""
    c = KvCache(n_layers=1, nh=64, nkv=64, cap=pos0 + n, k_fmt=F16, v_fmt=F16)
    near = KvCache(n_layers=1, nh=64, nkv=64, cap=300 + n, k_fmt=F16, v_fmt=F16)
    k, v = (torch.randn(300 + n, 64, HD, generator=gen(2 + i), device="cuda") * 0.3 for i in range(2))
    k[..., 0] = 640.0
    q = torch.randn(n, 64, HD, generator=gen(4), device="cuda")
    q[..., 0] = 1.0
    from bonsai_vk_amd import Rope
    c.rope_append(0, pos0 - 300, None, k, v, Rope(0))
    near.rope_append(0, 0, None, k, v, Rope(0))
    assert c.k_data[0, :pos0 - 300].numel() > 2 ** 32
    mask = some_mask("tree", n, 2)
    out, _ = c.attn_tree(0, pos0, q, mask)
    want, _, (size, top, every) = attention(near, 0, 300, q, mask)
    check_rows(out, want, tolerance((size, top, every), pos0 + n) + size * 1e-12)
    for a, b in zip(c.read(0, pos0 - 300, 300 + n), near.read(0, 0, 300 + n)):
        assert same(a, b)
