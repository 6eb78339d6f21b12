"""A step whose pool is exhausted does nothing: with lengths and starts that follow extend's lack, sequences that share a page keep
its bytes, and the step succeeds once a sequence is given up. (No counterpart in the reference.)"""
import textwrap

import pytest
import torch

import bonsai_vk_amd.seqs as module
from bonsai_vk_amd import Rope, RopeAxes

from seqs_util import arrays, attention, device_ints, make, random_bytes, starts_of

pytestmark = pytest.mark.gpu
SCALE = 1.0 / 16.0


def step(seqs, n_new, starts, q, k, v, out):
    """A step as it is documented: nothing read back."""
    lack = seqs.extend(n_new)
    have = (lack == 0).all()
    seqs.len += n_new * have
    q_start = starts * have
    for layer in range(seqs.cache.n_layers):
        turned = seqs.rope_append(layer, q, k, v, Rope(64), q_start)
        seqs.attn(layer, turned, q_start, out=out[layer])
    return have, turned, q_start


def state(seqs):
    return [x.clone() for x in (*arrays(seqs.cache), seqs.tables, seqs.refs, seqs.len)]


def shared(page, fmt="q4_0"):
    """Two layers; four sequences that are one prompt's, whose last page is partly filled, and two free pages where three are
    wanted (the last one of four keeps the shared page)."""
    cache, seqs = make([0] * 4, page, 2, 4, k=fmt, v=fmt, layers=2, cap=page * 5, room=4 * page)
    random_bytes(cache, page)
    first = device_ints([2 * page + 5, 0, 0, 0])
    assert seqs.extend(first).tolist() == [0, 0]
    seqs.len += first
    seqs.fork(device_ints([0, 0, 0, 0]))
    return cache, seqs


def rows(n, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(n, h, 256, generator=g, device="cuda") for h in (8, 2, 2)]


@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("n", [[1, 1, 1, 1], [3, 1, 60, 2], [0, 1, 300, 0]])
def test_an_exhausted_pool_after_a_fork(page, n):
    cache, seqs = shared(page)
    before = state(seqs)
    q, k, v = rows(sum(n), 1)
    out = torch.full((2, sum(n), 8, 256), 7.0, device="cuda")
    have, _, _ = step(seqs, device_ints(n), device_ints(starts_of(n)), q, k, v, out)
    for a, b in zip(state(seqs), before):
        assert torch.equal(a, b)
    assert not bool(have) and bool((out == 7.0).all())
    # one given up: three that share, two of which get a page
    seqs.fork(device_ints([0, 1, 2, -1]))
    n = [1, 1, 1, 0]
    have, turned, starts = step(seqs, device_ints(n), device_ints(starts_of(n)), q[:3], k[:3], v[:3], out[:, :3])
    assert bool(have) and seqs.len.tolist() == [2 * page + 6] * 3 + [0] and starts.tolist() == starts_of(n)
    want, bound = attention(seqs, 1, turned, starts_of(n), seqs.len.tolist(), SCALE)
    assert bool(((out[1, :3].double() - want).abs() <= bound).all())
    held = seqs.tables[:3, :, 2]
    assert all(len(set(held[:, layer].tolist())) == 3 for layer in range(2))


def test_replays_of_a_captured_step_that_lacks_pages_and_then_does_not():
    cache, seqs = shared(16)
    n_new, starts = device_ints([1, 1, 1, 1]), device_ints([0, 1, 2, 3, 4])
    q, k, v = rows(4, 2)
    out = torch.full((2, 4, 8, 256), 7.0, device="cuda")
    seqs.workspace(4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        have, turned, q_start = step(seqs, n_new, starts, q, k, v, out)
    before = state(seqs)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert not bool(have) and bool((out == 7.0).all())
        for a, b in zip(state(seqs), before):
            assert torch.equal(a, b)
    seqs.fork(device_ints([0, 1, 2, -1]))
    n_new.copy_(device_ints([1, 1, 1, 0]))
    starts.copy_(device_ints([0, 1, 2, 3, 3]))
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert bool(have) and seqs.len.tolist() == [38 + i] * 3 + [0]
        got = out.clone()
        assert bool((got[:, 3] == 7.0).all())
        want, bound = attention(seqs, 1, turned[:3], [0, 1, 2, 3, 3], seqs.len.tolist(), SCALE)
        assert bool(((got[1, :3].double() - want).abs() <= bound).all())


def test_the_documented_step():
    """The module's own example, as it stands there."""
    example = textwrap.dedent("\n".join(line for line in module.__doc__.splitlines() if line.startswith("    ")))
    assert "seqs.extend" in example and "seqs.attn" in example
    cache, seqs = make([37, 0, 0, 0], 16, 2, 4, cap=16 * 5, room=64)
    random_bytes(cache)
    seqs.fork(device_ints([0, 0, 0, 0]))
    before = state(seqs)
    q, k, v = rows(4, 3)
    names = dict(seqs=seqs, layer=0, q=q, k=k, v=v, rope=Rope(32), positions=torch.zeros(2, 4, dtype=torch.int32, device="cuda"),
                 axes=RopeAxes([8, 8]), gate=q.clone(), longest=1, n_new=device_ints([1, 1, 1, 1]), starts=device_ints([0, 1, 2, 3, 4]))
    exec(example, names)
    for a, b in zip(state(seqs), before):
        assert torch.equal(a, b)
    seqs.fork(device_ints([0, 1, 2, -1]))
    names.update(q=q, k=k, v=v, n_new=device_ints([1, 1, 1, 0]), starts=device_ints([0, 1, 2, 3, 3]))
    exec(example, names)
    assert seqs.len.tolist() == [38, 38, 38, 0]
    want, bound = attention(seqs, 0, names["q"][:3], [0, 1, 2, 3, 3], [38, 38, 38, 0], SCALE)
    assert bool(((names["out"][:3].double() - want).abs() <= bound).all())
