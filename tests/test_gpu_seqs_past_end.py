"""Sequences whose length is past what the cache holds: the tokens whose positions are in it are appended, read back and attend
as if the others were not there; those see all that is there. (No counterpart in the reference.)"""
import pytest
import torch

from bonsai_vk_amd import Rope

from seqs_util import attention, device_ints, fill, make, starts_of

pytestmark = pytest.mark.gpu
SCALE = 1.0 / 16.0


def expected(seqs, q, n, lens):
    """(out, bound) of seqs_util.attention, whose lengths are within the cache: the rows of positions that are there are a chunk
    that ends where the cache does, each of the others is a single token at that end."""
    held = seqs.cache.max_positions
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")

    def part(s, a, b, length):
        x = attention(seqs, 0, q[a:b], [0] * (s + 1) + [b - a], [0] * s + [length], SCALE)
        out[a:b], bound[a:b] = x
    at = starts_of(n)
    for s, length in enumerate(lens):
        past = min(max(length - held, 0), n[s])
        inside = at[s] + n[s] - past
        if inside > at[s]:
            part(s, at[s], inside, min(length, held))
        for r in range(inside, at[s + 1]):
            part(s, r, r + 1, held)
    return out, bound


def filled(room, page, sequences=1, nkv=4, grp=4):
    cache, seqs = make([room] * sequences, page, nkv, grp, seed=page + room)
    fill(cache, room)
    return cache, seqs


def queries(n, nh, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(n, nh, 256, generator=g, device="cuda")


@pytest.mark.parametrize("page", [0, 16, 32, 48])
@pytest.mark.parametrize("room, n, past", [(96, 10, 6), (96, 1, 1), (96, 3, 2**31 - 1 - 96), (96, 10, 10), (96, 40, 39), (1008, 17, 5), (480, 300, 150),
                                           (960, 64, 33), (480, 200, 2**31 - 1 - 480)])
def test_a_sequence_past_the_cache(page, room, n, past):
    """10 tokens of which 6 are outside, one outside, all far outside; row blocks and tiles."""
    if page and room % page:
        room += page - room % page
    cache, seqs = filled(room, page)
    length = min(room + past, 2**31 - 1)
    seqs.len.copy_(device_ints([length]))
    q = queries(n, 16, n)
    g = queries(n, 16, n + 1)
    out, gated = seqs.attn(0, q, device_ints([0, n]), g)
    want, bound = expected(seqs, q, [n], [length])
    assert bool(((out.double() - want).abs() <= bound).all())
    gate = out.double() * torch.sigmoid(g.double())
    assert float((gated.double() - gate).abs().max()) <= 2.0 ** -21 * float(gate.abs().max()) + 1e-30


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("max_q", [0, 1])
def test_sequences_past_the_cache_beside_others(page, max_q):
    """Single tokens, chunks by row blocks and chunks by tiles, inside and past it in one call."""
    cache, seqs = filled(320, page, 7)
    lens, n = [320, 321, 325, 400, 90, 352, 5], [1, 1, 9, 200, 60, 64, 3]
    seqs.len.copy_(device_ints(lens))
    q = queries(sum(n), 16, 5)
    out, _ = seqs.attn(0, q, device_ints(starts_of(n)), max_q=max_q)
    want, bound = expected(seqs, q, n, lens)
    assert bool(((out.double() - want).abs() <= bound).all())


def test_many_tiles_past_the_cache():
    """More tiles than pieces of a KV head."""
    cache, seqs = filled(640, 64, 3, 2, 16)
    lens, n = [900, 640, 700], [600, 640, 300]
    seqs.len.copy_(device_ints(lens))
    q = queries(sum(n), 32, 6)
    out, _ = seqs.attn(0, q, device_ints(starts_of(n)))
    want, bound = expected(seqs, q, n, lens)
    assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("page", [0, 16])
def test_append_read_and_attention_agree(page):
    """A token is written where it is read, and its own key, which takes all of its softmax, is among those that it sees."""
    cache, seqs = filled(64, page, 1, 1, 2)
    seqs.len.copy_(device_ints([70]))
    starts = device_ints([0, 10])
    k, v = torch.zeros(10, 1, 256, device="cuda"), torch.zeros(10, 1, 256, device="cuda")
    for i in range(10):
        k[i, 0, 16 * i], v[i, 0, 0] = 56.0, -8.0 * (i + 1)   # (exact in 4 bits: -8 steps)
    k = -k
    q = seqs.rope_append(0, queries(10, 2, 7) * 0.01, k, v, Rope(0), starts)
    q = q.clone()
    for i in range(10):
        q[i, :, 16 * i] = -1000.0                            # (its own key: a score past all others' by far)
    got_k, got_v = seqs.read(0, starts, 10)
    assert torch.equal(got_k[:4], k[:4]) and torch.equal(got_v[:4], v[:4])
    assert not bool(got_k[4:].any()) and not bool(got_v[4:].any())
    out, _ = seqs.attn(0, q, starts)
    want, bound = expected(seqs, q, [10], [70])
    assert bool(((out.double() - want).abs() <= bound).all())
    for i in range(4):
        assert float((out[i, :, 0] - v[i, 0, 0]).abs().max()) < 1e-3
