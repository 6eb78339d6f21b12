"""Calls at the edges of the drafted-token operators' ranges: outputs whose axes of one have any stride, and caches
whose offsets pass 32 bits in each attention kernel."""
import pytest
import torch

from bonsai_vk_amd import KvCache
from tests.tree_util import F16, HD, Q8, gen, make_cache, same, some_mask

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
