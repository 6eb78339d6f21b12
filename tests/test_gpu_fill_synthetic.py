"""bkv_kv_fill_synthetic at every head_dim that the geometry allows: each array whole, and nothing beside it."""
import ctypes

import pytest
import torch

from bonsai_vk_amd import BKV_F16, BKV_Q4_0, BKV_Q8_0, BkvCacheDesc, lib

pytestmark = pytest.mark.gpu
GUARD = 4096                                       # bytes before, between the layers and behind


@pytest.mark.parametrize("hd", [64, 128, 192, 256, 512])
@pytest.mark.parametrize("nkv", [1, 3])
@pytest.mark.parametrize("k_fmt, v_fmt", [(BKV_Q8_0, BKV_Q4_0), (BKV_Q4_0, BKV_Q8_0), (BKV_F16, BKV_Q8_0), (BKV_F16, BKV_F16)])
def test_whole_arrays_and_nothing_else(hd, nkv, k_fmt, v_fmt):
    cap, layers = 44, 3
    d = BkvCacheDesc()
    d.n_layers, d.nh, d.nkv, d.hd, d.cap, d.k_fmt, d.v_fmt, d.scale = layers, 2 * nkv, nkv, hd, cap, k_fmt, v_fmt, 0.125
    names, held = ("k_data", "k_scales", "v_data", "v_scales"), []
    for i, name in enumerate(names):
        size = cap * lib().bkv_slot_bytes(ctypes.byref(d), i)
        stride = size + (-size) % 16 + GUARD
        t = torch.full((GUARD + layers * stride,), 0x77, dtype=torch.uint8, device="cuda")
        setattr(d, name, t.data_ptr() + GUARD)     # (an array that the format does not have is not written, wherever it points)
        d.layer_stride_bytes[i] = stride
        held.append((t, size, stride))
    assert lib().bkv_kv_fill_synthetic(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    for t, size, stride in held:
        want = torch.full_like(t, 0x77)
        for layer in range(layers):
            at = GUARD + layer * stride
            want[at:at + size] = torch.tensor([0x00, 0x3C, 0x00, 0x3C], dtype=torch.uint8, device="cuda").repeat(size // 4)
        assert torch.equal(t, want)
