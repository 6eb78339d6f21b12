"""Workspaces as calls grow: of KvSeqs.attn all that were handed out stay, of KvCache's prefills those that a call was captured
with, since a captured call has its workspace's address. (No counterpart in the reference.)"""
import weakref

import pytest
import torch

import bonsai_vk_amd.cache as cache_module
import bonsai_vk_amd.seqs as module
from bonsai_vk_amd import BKV_Q4_0, BKV_Q8_0, BkvError, KvCache, KvSeqs
from bonsai_vk_amd._lib import lib

from seqs_util import device_ints, fill, make


class Host:
    """The library's host parts; bkv_workspace_init, the one call of workspace() that needs a GPU, is only noted."""

    def __init__(self):
        self.made, self.answer = [], 0

    def bkv_workspace_init(self, desc, ws, size, stream):
        self.made.append((ws, size))
        return self.answer

    def __getattr__(self, name):
        return getattr(lib(), name)


@pytest.fixture
def host(monkeypatch):
    host = Host()
    monkeypatch.setattr(module, "lib", lambda: host)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    cache = KvCache(n_layers=1, nh=16, nkv=4, cap=64, k_fmt=BKV_Q4_0, v_fmt=BKV_Q4_0, page_tokens=16, max_pages=4,
                    block_table=torch.full((1, 4), -1), device="cpu")
    cache._my_stream = lambda: 0
    return host, KvSeqs(cache, 3)


def test_an_outgrown_workspace_lives_on(host):
    host, seqs = host
    first = seqs.workspace(3)
    alive, address = weakref.ref(first), first.data_ptr()
    del first
    larger = seqs.workspace(3000)
    assert larger.data_ptr() != address and alive() is not None and alive().data_ptr() == address
    assert seqs.workspace(3) is larger and seqs.workspace(0) is larger


def test_all_together_are_bounded(host):
    """A row more at every call: a workspace is at least twice the one before."""
    host, seqs = host
    for n in range(1, 30000, 7):
        need = lib().bkv_seqs_workspace_bytes(seqs.desc, 3, n)
        assert seqs.workspace(n).numel() >= need
    sizes = [size for _, size in host.made]
    assert len(sizes) > 2 and all(b >= 2 * a for a, b in zip(sizes, sizes[1:])) and sum(sizes) < 2 * sizes[-1]
    assert sizes[-1] < 2 * need


def test_one_that_was_not_made_ready_is_not_used(host):
    host, seqs = host
    host.answer = -6
    with pytest.raises(BkvError):
        seqs.workspace(3)
    host.answer = 0
    assert seqs.workspace(3).data_ptr() == host.made[-1][0] and len(host.made) == 2


def test_a_prefill_workspace_that_was_captured_lives_on(monkeypatch):
    capturing = [False]
    monkeypatch.setattr(cache_module, "lib", lambda host=Host(): host)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(KvCache, "_stream", lambda self: 0)
    cache = KvCache(n_layers=1, nh=16, nkv=4, cap=8192, k_fmt=BKV_Q8_0, v_fmt=BKV_Q8_0, device="cpu")
    seen, sizes = [], (600, 2000, 4000)
    for ctx in sizes:
        seen.append(weakref.ref(cache.prefill_workspace(ctx)))
        capturing[0] = ctx == 2000                 # (the call of that context captured, twice)
        for _ in range(2):
            assert cache.prefill_workspace(ctx) is seen[-1]()
        capturing[0] = False
    assert seen[0]() is None and seen[1]() is not None and seen[2]() is cache.prefill_workspace(600)
    assert len(cache._captured) == 1


@pytest.mark.gpu
def test_a_captured_call_beside_larger_ones():
    """A captured step of single tokens, then prompts that need more, and other tensors of the workspace's size: every replay gives
    what an eager call does, and what is in the others' memory stays."""
    cache, seqs = make([900, 500, 700], 32, room=1000)
    fill(cache)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    q, large = torch.randn(3, 16, 256, generator=g, device="cuda"), torch.randn(700, 16, 256, generator=g, device="cuda")
    starts, many = device_ints([0, 1, 2, 3]), device_ints([0, 200, 690, 700])
    size = seqs.workspace(3).numel()
    out = torch.zeros(3, 16, 256, device="cuda")
    seqs.attn(0, q, starts, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seqs.attn(0, q, starts, out=out)
    want = seqs.attn(0, large, many)[0].clone()
    others = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(4)]
    for step in range(4):
        q.normal_()
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, seqs.attn(0, q, starts)[0])
        assert torch.equal(seqs.attn(0, large, many)[0], want)
        assert all(bool((x == 0x5A).all()) for x in others)
