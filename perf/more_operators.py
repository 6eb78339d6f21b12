"""Timed cases of several sequences served from one cache held in 4 bits: attention of a ragged batch, rotary positions of
one or three axes with the quantising append, and the pages under it: branching (fork and copy on write) and compacting.

Default shape: the reference's (16 query heads, 4 KV heads, head_dim 256, 8 attention layers); other head counts come with
the drawn cases. K ~ N(0, 1) with 3 channels per KV head scaled x8, V ~ N(0, 0.5), as in bench.py; Q ~ N(0, 1).

q4_0: blocks of 32 values with a scale d, value = d * q, q = -8 .. 7. d is the value furthest from 0 (the positive one
where both signs are as far) times -1/8, rounded to fp16, then to that number's upper 13 bits (8 significant ones), at
most 2048; q = x / d rounded to the nearest. Word w of a row holds elements 8 w + i as q + 8, i = 2 s + h at bit 16 h + 4 s.

A case is a dict:
  op     "attend"  attention of the tokens of `seqs` sequences of lo .. hi positions: "one" token each, a "chunk" of n
                   tokens each, or "mixed": a sixth of them with chunks of up to n tokens, the others with one
         "append"  the same tokens' projections rotated and appended, then read back
         "branch"  every one of `seqs` sequences goes on from a chosen one (as beams and samples of one prompt do): pages
                   shared, then one more token each, which gives each its own copy of a page that is not full
         "compact" a pool of `pool` pages, `full` per cent of them used by `seqs` sequences here and there, moved together
  kf, vf cache formats of K and V: "q4_0", "q8_0" or "f16"; page: tokens per page, 0 = contiguous (one sequence)
  rows   "append": the projections' rows are "own" arrays, one "fused" q|k|v buffer, or "qg" (q beside its gate)
"""
import math
import random

import numpy as np
import torch

own = False

HD, BLK = 256, 32
BASE, EPS = 1e7, 1e-6
ROW = {"f16": HD * 2, "q8_0": HD, "q4_0": HD // 2}       # bytes of a head row's values


def _case(name, op, seqs, lo, hi, kf="q4_0", vf="q4_0", page=64, nkv=4, group=4, layers=1, **more):
    c = {"op": op, "seqs": seqs, "lo": lo, "hi": hi, "kf": kf, "vf": vf, "page": page, "nkv": nkv, "group": group,
         "layers": layers, **more}
    return dict(c, name=name) if name else c


def _attend(name, seqs, lo, hi, n=1, kind="one", gate=True, **more):
    return _case(name, "attend", seqs, lo, hi, n=n, kind=kind, gate=gate, **more)


def _append(name, seqs, lo, hi, n=1, kind="one", axes=3, order="blocks", nrot=64, layout="half", scaling="none", norm=True,
            rows="own", **more):
    return _case(name, "append", seqs, lo, hi, n=n, kind=kind, axes=axes, order=order, nrot=nrot, layout=layout,
                 scaling=scaling, norm=norm, rows=rows, **more)


def listed():
    return [
        # a chat's first words, one token
        _attend("attend_1_at_600", 1, 600, 600, page=0),
        # one token at the headline context
        _attend("attend_1_at_32k", 1, 32768, 32768, page=0),
        # an odd batch of conversations of all lengths, a token each
        _attend("attend_29_ragged", 29, 40, 12000),
        # a chunk of a prompt: the standard 512 queries onto 8192 positions
        _attend("attend_chunk_512_at_8k", 1, 8704, 8704, n=512, kind="chunk", gate=False, page=256),
        # a server's step: running conversations and the prompts that just came in, small pages of an odd size
        _attend("attend_mixed_15", 15, 700, 3500, n=400, kind="mixed", page=48),
        # one token of text on its way into the cache
        _append("append_1_at_4k", 1, 4097, 4097),
        # a picture's tokens, from one fused projection buffer, positions of three axes dealt out in turn
        _append("append_image_1201", 1, 3001, 3001, n=1201, kind="chunk", order="dealt", nrot=128, layout="interleaved",
                norm=False, rows="fused"),
        # a server's step, pictures among it, positions scaled past the trained context
        _append("append_mixed_61", 61, 300, 9000, n=130, kind="mixed", scaling="yarn", rows="qg", page=16),
        # a step of a beam search, all layers
        _case("branch_8_beams", "branch", 8, 2000, 2000, layers=8),
        # many samples of one long prompt, larger pages
        _case("branch_200_samples", "branch", 200, 5000, 5000, page=128, layers=8),
        # a small pool after a few conversations ended
        _case("compact_77_pages", "compact", 5, 0, 0, pool=77, full=60, page=16, layers=8),
        # a large pool, two thirds of it in use
        _case("compact_2000_pages", "compact", 96, 0, 0, pool=2000, full=66, layers=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the listed ranges: 1 to 200 sequences of 1 to 60000 positions, chunks of 1 to 700 tokens, 1 to 8 KV
    heads with 1 to 8 query heads each, contiguous (one sequence) and pages of 16 to 256."""
    op = rng.choice(["attend", "attend", "attend", "append", "append", "branch", "compact"])
    page = rng.choice([16, 48, 64, 64, 100, 256])
    nkv = rng.choice([4, 4, 4, 1, 2, 3, 8])
    group = rng.choice([4, 4, 4, 1, 2, 5, 8])
    if op in ("branch", "compact"):
        kf, vf = rng.choice([("q4_0", "q4_0"), ("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q8_0", "q8_0"), ("f16", "f16")])
        shape = dict(kf=kf, vf=vf, page=page, nkv=nkv, group=group, layers=rng.choice([1, 4, 8]))
        # (at most 64 MB a layer)
        room = int(64e6 / (nkv * page * (ROW[kf] + ROW[vf] + 32)))
        if op == "compact":
            pool = _log(rng, 10, min(room, 3000))
            return _case(None, op, _log(rng, 1, 100), 0, 0, pool=pool, full=rng.randint(5, 95), **shape)
        seqs, at = _log(rng, 2, 200), _log(rng, 1, 6000)
        at = min(at, (room - 2 * seqs - 4) * page) if room > 2 * seqs + 4 else 1
        return _case(None, op, min(seqs, max(2, room // 3)), at, at, **shape)
    shape = dict(page=page, nkv=nkv, group=group)
    kind = rng.choice(["one", "one", "chunk", "mixed"])
    seqs = _log(rng, 1, 100 if kind == "one" else 24)
    if kind == "mixed" and seqs < 6:
        kind = "chunk"
    n = 1 if kind == "one" else _log(rng, 2, 700)
    if seqs == 1 and rng.random() < 0.5:
        shape["page"] = 0
    if op == "append":
        kf, vf = rng.choice([("q4_0", "q4_0"), ("q4_0", "q4_0"), ("q8_0", "q4_0"), ("f16", "q8_0")])
        if kind == "chunk":
            n = max(2, min(n, 3000 // (seqs * nkv)))
        lo = _log(rng, n, n + 20000 // seqs)
        return _append(None, seqs, lo, lo + _log(rng, 1, 4000), n, kind, axes=rng.choice([3, 3, 1, 2]),
                       order=rng.choice(["blocks", "dealt"]), nrot=rng.choice([64, 64, 32, 128, 256, 20]),
                       layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                       norm=rng.random() < 0.5, rows=rng.choice(["own", "fused", "qg"]), kf=kf, vf=vf, **shape)
    # at most the largest listed case's query-key pairs, and what its plain form holds
    many = seqs if kind == "chunk" else 1 if kind == "one" else -(-seqs // 6)
    if kind != "one":
        n = max(1, min(n, 2048 // (many * nkv * group) * 4 + 3))
    pairs = 512 * 8704 * 16 / (nkv * group * (many * n if kind != "one" else seqs))
    wide = 3.2e8 / (seqs * nkv * max(group * n, 256))
    room = int(min(60000, pairs, wide))
    hi = max(n, _log(rng, 2, max(3, room)))
    lo = hi if rng.random() < 0.3 else max(1, hi // rng.choice([2, 10, 100]))
    return _attend(None, seqs, lo, hi, n, kind, gate=rng.random() < 0.5, **shape)


def _lens(c):
    """(positions, tokens of this call) of every sequence: the same for every seed."""
    r = random.Random(1000 * c["seqs"] + c["hi"])
    lens = [int(round(math.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"]))))) for _ in range(c["seqs"])]
    lens[0] = c["hi"]
    if c["kind"] == "one":
        return lens, [1] * c["seqs"]
    if c["kind"] == "chunk":
        n = [c["n"]] + [r.randint(1, c["n"]) for _ in range(c["seqs"] - 1)]
    else:
        n = [r.randint(max(1, c["n"] // 2), c["n"]) if s % 6 == 0 else 1 for s in range(c["seqs"])]
    return lens, [min(a, b) for a, b in zip(n, lens)]


def _slot_bytes(c):
    """Bytes of one position of one layer: K and V, data and scales."""
    return sum(c["nkv"] * (ROW[f] + (0 if f == "f16" else HD // BLK * 2)) for f in (c["kf"], c["vf"]))


def _max_pages(c):
    return -(-(c["hi"] + 1) // c["page"]) + 1


def _pool(c):
    if c["op"] == "compact":
        return c["pool"]
    if c["op"] == "branch":                         # the prompt's pages, and two of each sequence's own
        return -(-c["lo"] // c["page"]) + 2 * c["seqs"] + 2
    return sum(-(-x // c["page"]) for x in _lens(c)[0]) + 5


def _parents(c):
    r = random.Random(31 * c["seqs"] + c["lo"])
    return [r.randrange(c["seqs"]) for _ in range(c["seqs"])]


def _moved(c):
    """Pages that a compaction moves, in all layers, as the inputs are made."""
    used = round(c["pool"] * c["full"] / 100)
    return round(used * (1 - used / c["pool"])) * c["layers"]


def work(case):
    c, sb = case, _slot_bytes(case)
    if c["op"] == "branch":
        # the tables and counts in and out; each sequence's positions in a page that is not full, where it is no parent's last
        copies = c["seqs"] - len(set(_parents(c)))
        rem = c["lo"] % c["page"]
        tables = 2 * c["seqs"] * c["layers"] * _max_pages(c) * 4
        return {"bytes": tables + 2 * 4 * c["layers"] * _pool(c) + 2 * copies * rem * sb * c["layers"], "flops": 0}
    if c["op"] == "compact":
        tables = 2 * c["seqs"] * c["layers"] * c["pool"] * 4
        return {"bytes": tables + 2 * 4 * c["layers"] * c["pool"] + 2 * _moved(c) * c["page"] * sb, "flops": 0}
    lens, n = _lens(c)
    nh, nkv, tok = c["nkv"] * c["group"], c["nkv"], sum(n)
    if c["op"] == "attend":
        pairs = sum(q * (x - q) + q * (q + 1) // 2 for x, q in zip(lens, n))
        return {"bytes": sum(lens) * sb + tok * nh * HD * 4 * (4 if c["gate"] else 2), "flops": 4 * HD * nh * pairs}
    # projections in, q out; the cache written and read again, the values out
    return {"bytes": tok * ((2 * nh + 2 * nkv) * HD * 4 + 2 * sb + 2 * nkv * HD * 2), "flops": tok * (nh + 2 * nkv) * HD * 6}


# ------------------------------------------------------------------ inputs
def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 7919 * stream + 1)
    return g


def _quantise4(x):
    """q4_0 of fp32 [..][HD]: whole numbers -8 .. 7 [..][HD / 32][32] and fp16 scales [..][HD / 32]."""
    b = x.unflatten(-1, (HD // BLK, BLK))
    hi, lo = b.amax(-1), b.amin(-1)
    h = (torch.where(hi >= -lo, hi, lo) * -0.125).half().view(torch.int16).int()
    m = h & 0x7FFF
    m = ((m + 3 + (m >> 3 & 1)) & 0x7FF8).clamp(max=0x6800)
    d = torch.where(m > 0, m | (h & 0x8000), m).short().view(torch.float16)
    inv = torch.where(d != 0, 1.0 / d.float(), torch.zeros_like(d, dtype=torch.float32))
    return (b * inv[..., None]).round().clamp(-8, 7), d


def _quantise8(x):
    b = x.unflatten(-1, (HD // BLK, BLK))
    amax = b.abs().amax(-1)
    d = torch.where(amax > 1e-35, amax / 127.0, torch.zeros_like(amax))
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return (b * inv[..., None]).round().clamp(-127, 127), d.half()


def _bytes(t):
    return t.contiguous().view(torch.uint8).reshape(*t.shape[:-2], -1)


def _bits():
    i = torch.arange(8, device="cuda", dtype=torch.int32)
    return 16 * (i % 2) + 4 * (i // 2)


def _packed(q):
    """The words of whole numbers -8 .. 7 [..][HD / 32][32], as bytes [..][heads * HD / 2]."""
    w = ((q.long() + 8).unflatten(-1, (4, 8)) << _bits()).sum(-1)
    return _bytes(torch.where(w >= 2**31, w - 2**32, w).int().flatten(-2))


def _slots(st, layer):
    """The cache slot of every sequence's every position, [seqs][longest] (behind a sequence's end: of its last)."""
    p = torch.arange(max(st["lens"]), device="cuda")[None].minimum(st["len"].long()[:, None] - 1)
    if st["tables"] is None:
        return p
    page = st["case"]["page"]
    return st["tables"][:, layer].long().gather(1, p // page) * page + p % page


def _fill(st, seed):
    """Positions 0 .. len - 1 of every sequence, in layer 0."""
    c, g = st["case"], _gen(seed, 100)
    slots = _slots(st, 0)
    big = torch.ones(c["nkv"], HD, device="cuda")
    big.scatter_(1, torch.stack([torch.randperm(HD, generator=g, device="cuda")[:3] for _ in range(c["nkv"])]), 8.0)
    for s, n in enumerate(st["lens"]):
        for a in range(0, n, 16384):
            at = slots[s, a:min(n, a + 16384)]
            for name, mul in (("k", big), ("v", 0.5)):
                q, d = _quantise4(torch.randn(len(at), c["nkv"], HD, generator=g, device="cuda") * mul)
                st[name + "_data"][0, at] = _packed(q)
                st[name + "_scales"][0, at] = _bytes(d)


FACTOR, TRAINED, FAST, SLOW = 4.0, 32768, 32.0, 1.0


def _angles(c):
    """Radians per position of each pair, and the factor on cosines and sines."""
    nrot, half = c["nrot"], c["nrot"] // 2
    base, scaling = BASE, c["scaling"]
    if scaling == "ntk":
        base *= FACTOR ** (nrot / (nrot - 2))
    th = [base ** (-2.0 * p / nrot) for p in range(half)]
    if scaling == "linear":
        th = [t / FACTOR for t in th]
    if scaling == "yarn":
        at = [nrot * math.log(TRAINED / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (FAST, SLOW)]
        lo, hi = max(0, math.floor(at[0])), min(nrot - 1, math.ceil(at[1]))
        ramp = [min(1.0, max(0.0, (p - lo) / max(hi - lo, 1e-3))) for p in range(half)]
        th = [t * (1 - r) + t / FACTOR * r for t, r in zip(th, ramp)]
    return th, 0.1 * math.log(FACTOR) + 1.0 if scaling == "yarn" else 1.0


def _sections(c):
    """Pairs of each axis."""
    pairs, n = c["nrot"] // 2, c["axes"]
    return [pairs - (n - 1) * (pairs // n)] + [pairs // n] * (n - 1)


def _axis_of_pair(c):
    left, got = _sections(c), []
    if c["order"] == "blocks":
        return [a for a, k in enumerate(left) for _ in range(k)]
    while sum(left):                                # dealt out in turn to the axes that still want some
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def _positions(c, lens, n):
    """[axes][tokens]: text has one position on all axes, a chunk is a picture of some width after a few words."""
    rows = []
    for x, q in zip(lens, n):
        first, wide = x - q, max(1, math.isqrt(q))
        for i in range(q):
            text = min(i, 5)
            rows.append([first + text] + [first + text + (max(0, i - 5) // wide if a == 1 else max(0, i - 5) % wide)
                                          for a in range(1, c["axes"])])
    return torch.tensor(rows, dtype=torch.int32, device="cuda").t().contiguous()


def _scattered(st, seed):
    """A pool whose used pages lie here and there, some shared by two sequences: tables and counts."""
    c, r = st["case"], random.Random(int(seed) * 7 + 3)
    used = round(c["pool"] * c["full"] / 100)
    tables = np.full((c["seqs"], c["layers"], c["pool"]), -1, dtype=np.int32)
    refs = np.zeros((c["layers"], c["pool"]), dtype=np.int32)
    for layer in range(c["layers"]):
        at = [0] * c["seqs"]
        for pg in r.sample(range(c["pool"]), used):
            for s in {r.randrange(c["seqs"]) for _ in range(2 if r.random() < 0.2 else 1)}:
                tables[s, layer, at[s]] = pg
                at[s] += 1
                refs[layer, pg] += 1
    st["tables"], st["refs"] = torch.from_numpy(tables).cuda(), torch.from_numpy(refs).cuda()


def prepare(case, seed):
    c = dict(case)
    nkv, nh, page, layers = c["nkv"], c["nkv"] * c["group"], c["page"], c["layers"]
    st, g = {"case": c, "tables": None, "refs": None}, _gen(seed, 1)
    pages = _pool(c) if page else 0
    if c["op"] in ("attend", "append"):
        st["lens"], st["n"] = _lens(c)
        st["len"] = torch.tensor(st["lens"], dtype=torch.int32, device="cuda")
        starts = [0] + list(np.cumsum(st["n"]))
        st["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        tok = starts[-1]
        if page:
            st["tables"] = torch.full((c["seqs"], layers, _max_pages(c)), -1, dtype=torch.int32, device="cuda")
            ids = torch.randperm(pages, generator=g, device="cuda").int()
            for s, x in enumerate(st["lens"]):
                k = -(-x // page)
                st["tables"][s, 0, :k], ids = ids[:k], ids[k:]
    cap = pages * page if page else c["hi"]
    for name, fmt in (("k", c["kf"]), ("v", c["vf"])):
        make = torch.zeros
        if c["op"] in ("branch", "compact"):
            def make(*shape, **kw):
                return torch.randint(0, 256, shape, generator=g, **kw)
        st[name + "_data"] = make(layers, cap, nkv * ROW[fmt], dtype=torch.uint8, device="cuda")
        st[name + "_scales"] = None if fmt == "f16" else make(layers, cap, nkv * HD // BLK * 2, dtype=torch.uint8, device="cuda")
    if c["op"] == "branch":
        s = c["seqs"]
        st["tables"] = torch.full((s, layers, _max_pages(c)), -1, dtype=torch.int32, device="cuda")
        st["refs"] = torch.zeros(layers, pages, dtype=torch.int32, device="cuda")
        # the pool's numbers in use are the prompt's, in any order, then every sequence's own last page
        k = -(-c["lo"] // page)
        prompt = torch.stack([torch.randperm(k, generator=g, device="cuda") for _ in range(layers)]).int()
        st["tables"][:, :, :k] = prompt[None]
        st["refs"].scatter_(1, prompt.long(), s)
        st["len"] = torch.full((s,), c["lo"], dtype=torch.int32, device="cuda")
        st["n_new"] = torch.ones(s, dtype=torch.int32, device="cuda")
        st["parent"] = torch.tensor(_parents(c), dtype=torch.int32, device="cuda")
        _extend(st)
    if c["op"] == "compact":
        _scattered(st, seed)
    if own:
        # the objects that a user's program keeps, their arrays in the place of the plain ones
        from bonsai_vk_amd import BKV_F16, BKV_Q4_0, BKV_Q8_0, KvCache, KvSeqs
        fmt = {"f16": BKV_F16, "q8_0": BKV_Q8_0, "q4_0": BKV_Q4_0}
        per = st["tables"].shape[2] if page else 0
        st["cache"] = KvCache(n_layers=layers, nh=nh, nkv=nkv, cap=cap, k_fmt=fmt[c["kf"]], v_fmt=fmt[c["vf"]],
                              page_tokens=page, max_pages=per,
                              block_table=torch.full((layers, per), -1, dtype=torch.int32) if page else None)
        st["seqs"] = KvSeqs(st["cache"], c["seqs"])
        for name in ("k_data", "k_scales", "v_data", "v_scales"):
            if st[name] is not None:
                getattr(st["cache"], name).copy_(st[name])
            st[name] = getattr(st["cache"], name)
        for name in ("tables", "refs", "len"):
            if st.get(name) is not None:
                getattr(st["seqs"], name).copy_(st[name])
                st[name] = getattr(st["seqs"], name)
        if c["op"] == "compact":
            st["to"] = (torch.empty_like(st["tables"]), torch.empty_like(st["refs"]))
    if c["op"] == "attend":
        _fill(st, seed)
        st["q"] = torch.randn(tok, nh, HD, generator=g, device="cuda")
        st["gate"] = torch.randn(tok, nh, HD, generator=g, device="cuda") if c["gate"] else None
    if c["op"] == "append":
        rows = torch.randn(tok, 2 * nh + 2 * nkv, HD, generator=g, device="cuda") * 2.0
        if c["rows"] == "fused":
            st["q"], st["k"], st["v"] = rows[:, :nh], rows[:, nh:nh + nkv], rows[:, nh + nkv:nh + 2 * nkv]
        elif c["rows"] == "qg":
            st["q"] = rows[:, :2 * nh].contiguous().view(tok, nh, 2 * HD)[:, :, :HD]
            st["k"], st["v"] = rows[:, 2 * nh:2 * nh + nkv].contiguous(), rows[:, 2 * nh + nkv:].contiguous()
        else:
            st["q"], st["k"], st["v"] = (rows[:, a:b].contiguous() for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
        st["qn_w"] = st["kn_w"] = None
        if c["norm"]:
            st["qn_w"], st["kn_w"] = (1.0 + 0.1 * torch.randn(HD, generator=g, device="cuda") for _ in range(2))
        st["positions"] = _positions(c, st["lens"], st["n"])
        th, st["mscale"] = _angles(c)
        st["theta"] = torch.tensor(th, dtype=torch.float64, device="cuda")
        st["axis"] = torch.tensor(_axis_of_pair(c), device="cuda")
        if own:
            from bonsai_vk_amd import Rope, RopeAxes
            st["rope"] = Rope(c["nrot"], layout=c["layout"], freq_base=BASE, scaling=c["scaling"], factor=FACTOR,
                              trained_ctx=TRAINED, beta_fast=FAST, beta_slow=SLOW)
            st["axes"] = RopeAxes(_sections(c), order=c["order"])
    return st


# ------------------------------------------------------------------ one pass
def _values(st, name, slots):
    """What the 4-bit cache holds at slots [..], as fp32 [..][nkv][HD]."""
    nkv = st["case"]["nkv"]
    w = st[name + "_data"][0][slots].view(torch.int32).unflatten(-1, (nkv, HD // BLK, BLK // 8))
    q = ((w[..., None] >> _bits()) & 15) - 8
    d = st[name + "_scales"][0][slots].view(torch.float16).float().unflatten(-1, (nkv, HD // BLK))
    return (q.flatten(-2).float() * d[..., None]).flatten(-2)


def _attended(st):
    c = st["case"]
    nkv, group, lens, n = c["nkv"], c["group"], st["len"].long(), (st["q_start"][1:] - st["q_start"][:-1]).long()
    most, tok = max(st["n"]), st["q"].shape[0]
    slots = _slots(st, 0)
    k, v = (_values(st, x, slots).transpose(1, 2).contiguous() for x in "kv")           # [seqs][nkv][keys][HD]
    i = torch.arange(most, device="cuda")
    rows = (st["q_start"][:-1, None] + i).clamp(max=tok - 1).long()
    q = st["q"].half().float()[rows].view(-1, most, nkv, group, HD).permute(0, 2, 3, 1, 4).reshape(-1, nkv, group * most, HD)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(-1, nkv, group, most, slots.shape[1]) * HD ** -0.5
    seen = torch.arange(slots.shape[1], device="cuda") <= (lens - n)[:, None, None] + i[:, None]        # [seqs][most][keys]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(-1, nkv, group * most, slots.shape[1]), v).view(-1, nkv, group, most, HD) / total
    mine = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n, output_size=tok)
    at = torch.arange(tok, device="cuda") - st["q_start"].long()[mine]
    out = out[mine, :, :, at].reshape(tok, nkv * group, HD)
    return (out,) if st["gate"] is None else (out, out / (1.0 + torch.exp(-st["gate"])))


def _rotate(st, x, w):
    """Norm (where there are weights) and rotation of fp32 rows [n][heads][HD]."""
    c = st["case"]
    nrot, half = c["nrot"], c["nrot"] // 2
    if w is not None:
        x = x * (1.0 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float() * w
    a = st["positions"].double()[st["axis"]].t()[:, None] * st["theta"]
    cs, sn = (torch.cos(a) * st["mscale"]).float(), (torch.sin(a) * st["mscale"]).float()
    if c["layout"] == "half":
        lo, hi = x[..., :half], x[..., half:nrot]
        return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn, x[..., nrot:]], -1)
    lo, hi = x[..., :nrot:2], x[..., 1:nrot:2]
    return torch.cat([torch.stack([lo * cs - hi * sn, hi * cs + lo * sn], -1).flatten(-2), x[..., nrot:]], -1)


def _stored(x, fmt):
    if fmt == "f16":
        return x.half()
    q, d = _quantise4(x) if fmt == "q4_0" else _quantise8(x)
    return (q * d.float()[..., None]).flatten(-2).half()


def _fork(st):
    refs, old = st["refs"], st["tables"]
    new = old[st["parent"].long()]
    for t, one in ((old, -1), (new, 1)):
        t = t.transpose(0, 1).flatten(1)
        refs.scatter_add_(1, t.clamp(min=0).long(), torch.where(t >= 0, one, 0).int())
    old.copy_(new)
    st["len"].copy_(st["len"][st["parent"].long()])


def _extend(st):
    """Pages for n_new more tokens of every sequence (one at most here, so one page), whose own they are."""
    c, refs, tables = st["case"], st["refs"], st["tables"]
    page, pages = c["page"], refs.shape[1]
    seqs, layers = tables.shape[:2]
    at = (st["len"].long() // page)[:, None].expand(seqs, layers)
    want = (st["n_new"] > 0)[:, None].expand(seqs, layers).t()                          # [layers][seqs]
    entry = tables.gather(2, at[..., None]).squeeze(-1).t().long()
    there = want & (entry >= 0)
    shared = there & (refs.gather(1, entry.clamp(min=0)) > 1)
    # of those that share a page and all want it, the last keeps it
    order = torch.arange(seqs, device="cuda").expand(layers, seqs)
    to = torch.where(shared, entry, pages)
    wants = torch.zeros(layers, pages + 1, dtype=torch.int32, device="cuda").scatter_add_(1, to, shared.int())
    last = torch.full((layers, pages + 1), -1, device="cuda").scatter_reduce_(1, to, order, "amax")
    keep = shared & (wants.gather(1, to) == refs.gather(1, entry.clamp(min=0))) & (last.gather(1, to) == order)
    fresh = want & (~there | (shared & ~keep))
    free = torch.argsort((refs > 0).int(), dim=1, stable=True)
    short = (fresh.sum(1) - (refs == 0).sum(1)).clamp(min=0)
    fresh &= short.sum() == 0
    new = free.gather(1, (fresh.long().cumsum(1) - 1).clamp(min=0))
    layer, s = fresh.nonzero().unbind(1)
    src, dst, p = entry[layer, s], new[layer, s], at[s, 0]
    tables[s, layer, p] = dst.int()
    refs[layer, dst] = 1
    copy = src >= 0
    layer, s, src, dst = layer[copy], s[copy], src[copy], dst[copy]
    refs.view(-1).scatter_add_(0, layer * pages + src, torch.full_like(src, -1, dtype=torch.int32))
    held = (torch.arange(page, device="cuda") < (st["len"].long() % page)[s][:, None])[..., None]
    for a in ("k_data", "k_scales", "v_data", "v_scales"):
        if st[a] is not None:
            x = st[a].view(layers, pages, page, -1)
            x[layer, dst] = torch.where(held, x[layer, src], x[layer, dst])
    return short.int()


def _compacted(st):
    refs, tables = st["refs"], st["tables"]
    layers, pages = refs.shape
    used, at = refs > 0, torch.arange(pages, device="cuda")
    most = used.sum(1, keepdim=True)
    layer, src = (used & (at >= most)).nonzero().unbind(1)
    dst = (~used & (at < most)).nonzero()[:, 1]     # (as many in every layer, in the same order)
    to = at.int().repeat(layers, 1)
    to[layer, src] = dst.int()
    new = to.gather(1, tables.clamp(min=0).transpose(0, 1).flatten(1).long()).view(layers, -1, tables.shape[2]).transpose(0, 1)
    counts = refs.clone()
    counts[layer, dst] = refs[layer, src]
    counts[layer, src] = 0
    for a in ("k_data", "k_scales", "v_data", "v_scales"):
        if st[a] is not None:
            x = st[a].view(layers, pages, -1)
            x[layer, dst] = x[layer, src]
    return torch.where(tables >= 0, new, tables).contiguous(), counts


def _arrays(st):
    return [st[a] for a in ("k_data", "k_scales", "v_data", "v_scales") if st[a] is not None]


def run(state):
    st, c = state, state["case"]
    if c["op"] == "attend":
        if own:
            out, gated = st["seqs"].attn(0, st["q"], st["q_start"], gate=st["gate"], max_q=max(st["n"]))
            return (out,) if gated is None else (out, gated)
        return _attended(st)
    if c["op"] == "append":
        if own:
            q = st["seqs"].rope_append(0, st["q"], st["k"], st["v"], st["rope"], st["q_start"], positions=st["positions"],
                                       axes=st["axes"], qn_w=st["qn_w"], kn_w=st["kn_w"], eps=EPS)
            k, v = st["seqs"].read(0, st["q_start"], q.shape[0], dtype=torch.float16)
            return {"q": q, "k": k, "v": v}
        return {"q": _rotate(st, st["q"], st["qn_w"]), "k": _stored(_rotate(st, st["k"], st["kn_w"]), c["kf"]),
                "v": _stored(st["v"], c["vf"])}
    if c["op"] == "branch":
        if own:
            st["seqs"].fork(st["parent"])
            short = st["seqs"].extend(st["n_new"])
        else:
            _fork(st)
            short = _extend(st)
        return [st["tables"], st["refs"], short] + _arrays(st)
    if own:
        tables, refs = st["seqs"].compact(*st["to"])
    else:
        tables, refs = _compacted(st)
    return [tables, refs] + _arrays(st)


# ------------------------------------------------------------------ in 64 bits
def _held(st, name, s):
    """What the cache's bytes stand for at sequence s's positions, [positions][nkv][HD] in 64 bits."""
    c, n = st["case"], st["lens"][s]
    if st["tables"] is None:
        at = torch.arange(n)
    else:
        row, page = st["tables"][s, 0].tolist(), c["page"]
        at = torch.tensor([row[p // page] * page + p % page for p in range(n)])
    b = st[name + "_data"][0].index_select(0, at.cuda()).view(n, c["nkv"], HD // 8, 4)
    v = torch.empty(n, c["nkv"], HD // 8, 8, dtype=torch.float64, device="cuda")
    for j in range(4):                              # byte j of a word: elements 4 (j % 2) + j / 2, and that + 2
        v[..., 4 * (j % 2) + j // 2] = b[..., j].bitwise_and(15).double() - 8
        v[..., 4 * (j % 2) + j // 2 + 2] = b[..., j].div(16, rounding_mode="floor").double() - 8
    d = st[name + "_scales"][0].index_select(0, at.cuda()).view(torch.float16).double().view(n, c["nkv"], HD // BLK)
    return v.reshape(n, c["nkv"], HD) * d.repeat_interleave(BLK, dim=2)


def _exact_attend(st):
    c = st["case"]
    outs = []
    for s, (x, n) in enumerate(zip(st["lens"], st["n"])):
        k, v = (_held(st, name, s) for name in "kv")
        first = int(st["q_start"][s])
        q = st["q"][first:first + n].half().double()
        hide = torch.triu(torch.ones(n, x, dtype=torch.bool, device="cuda"), diagonal=x - n + 1)
        out = torch.empty(n, c["nkv"] * c["group"], HD, dtype=torch.float64, device="cuda")
        for h in range(c["nkv"] * c["group"]):
            logits = q[:, h].mm(k[:, h // c["group"]].t()).div(math.sqrt(HD))
            out[:, h] = torch.softmax(logits.masked_fill(hide, -math.inf), 1).mm(v[:, h // c["group"]])
        outs.append(out)
    out = torch.cat(outs)
    return (out,) if st["gate"] is None else (out, out * torch.sigmoid(st["gate"].double()))


def _exact_append(st):
    c = st["case"]
    nrot, tok = c["nrot"], st["q"].shape[0]
    p = np.arange(nrot // 2)
    base = BASE * FACTOR ** (nrot / (nrot - 2)) if c["scaling"] == "ntk" else BASE
    freq = np.exp(-2.0 * p / nrot * np.log(base))
    mul = 1.0
    if c["scaling"] == "linear":
        freq = freq / FACTOR
    elif c["scaling"] == "yarn":
        def pair_of(turns):
            return nrot / 2 * np.log(TRAINED / (2 * np.pi * turns)) / np.log(BASE)
        lo, hi = max(np.floor(pair_of(FAST)), 0), min(np.ceil(pair_of(SLOW)), nrot - 1)
        part = np.clip((p - lo) / max(hi - lo, 1e-3), 0, 1)
        freq = freq * (1 - part + part / FACTOR)
        mul = 1 + 0.1 * np.log(FACTOR)
    sizes = np.array(_sections(c))
    if c["order"] == "blocks":
        axis = np.searchsorted(np.cumsum(sizes), p, side="right")
    else:                                           # the j-th pair of axis a comes in round j, behind the lower axes'
        axis = np.array([a for _, a in sorted((j, a) for a, k in enumerate(sizes) for j in range(k))], dtype=int)
    at = st["positions"].cpu().numpy()
    turn = torch.from_numpy(np.exp(1j * at[axis].T * freq) * mul).cuda()[:, None]          # [tokens][1][pairs]
    first = torch.arange(nrot // 2, device="cuda") * (1 if c["layout"] == "half" else 2)
    second = first + (nrot // 2 if c["layout"] == "half" else 1)

    def rotated(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(2, keepdim=True) + EPS) * w.double()
        y = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def kept(x, fmt):
        if fmt == "f16":
            return x
        b = x.reshape(tok, c["nkv"], HD // BLK, BLK)
        if fmt == "q8_0":
            d = b.abs().amax(3, keepdim=True) / 127
            return (torch.round(b / torch.where(d > 0, d, torch.ones_like(d))) * d.half().double()).reshape(x.shape)
        far = torch.where(b.amax(3, keepdim=True) + b.amin(3, keepdim=True) >= 0, b.amax(3, keepdim=True), b.amin(3, keepdim=True))
        m, e = torch.frexp((far / -8).half().double())     # (every scale here is a normal fp16 number)
        d = torch.ldexp(torch.round(m * 256) / 256, e)
        return (torch.round(b / torch.where(d != 0, d, torch.ones_like(d))).clamp(-8, 7) * d).reshape(x.shape)

    return {"q": rotated(st["q"], st["qn_w"]), "k": kept(rotated(st["k"], st["kn_w"]), c["kf"]),
            "v": kept(st["v"].double(), c["vf"])}


def exact(case, seed):
    if case["op"] not in ("attend", "append"):
        return None                                 # whole numbers and bytes
    st = prepare(case, seed)
    return _exact_attend(st) if case["op"] == "attend" else _exact_append(st)
