"""Timed cases of the speculative-decoding operators around the KV cache: attention for a tree of drafted
tokens, rotary positions with the quantising append, reading the cache back, and keeping the accepted path.

Default shape: the reference's (16 query heads, 4 KV heads, head_dim 256, 8 attention layers); other head
counts come with the drawn cases. K ~ N(0, 1) with 3 channels per KV head scaled x8, V ~ N(0, 0.5), as in
bench.py; Q ~ N(0, 1).

A case is a dict:
  op     "tree"    attention of `n` drafted tokens, cached at ctx .. ctx + n - 1, over the ctx positions before
                   them and over their own ancestors (mask "tree"), over each other in order ("chain"), or as
                   "tree" with the last rows of the batch left over: padding that sees no drafted token
         "rope"    `n` projected tokens rotated and appended at ctx .., then read back
         "read"    positions ctx .. ctx + n - 1 read back as `dtype`
         "commit"  of `n` drafted tokens at ctx .., `keep` moved to ctx .. ctx + keep - 1, in every layer
  kf, vf cache formats of K and V, "q8_0" or "f16"; page: tokens per page, 0 = contiguous
  rows   "rope": the projections' rows are "own" arrays, one "fused" q|k|v buffer, or "qg" (q beside its gate)
"""
import math
import random

import numpy as np
import torch

own = False

HD, BLK = 256, 32
BASE, EPS = 1e7, 1e-6
CHUNK = 8192            # tokens per generated piece of a cache
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, n, ctx, kf="q8_0", vf="q8_0", page=0, nkv=4, group=4, layers=1, **more):
    c = {"op": op, "n": n, "ctx": ctx, "kf": kf, "vf": vf, "page": page, "nkv": nkv, "group": group,
         "layers": layers, **more}
    return dict(c, name=name) if name else c


def _tree(name, n, ctx, mask="tree", gate=True, **more):
    return _case(name, "tree", n, ctx, mask=mask, gate=gate, **more)


def _rope(name, n, ctx, nrot=64, layout="half", scaling="none", norm=True, rows="own", tree=False, **more):
    return _case(name, "rope", n, ctx, nrot=nrot, layout=layout, scaling=scaling, norm=norm, rows=rows, tree=tree,
                 **more)


def listed():
    return [
        # a chat's first words checked against a small draft, in the reference's cache format
        _tree("tree_7_at_600_ref", 7, 600, kf="f16"),
        # an ordinary draft of a few branches in a running conversation
        _tree("tree_25_at_8k", 25, 8192),
        # a single token at the headline context
        _tree("tree_1_at_32k", 1, 32768),
        # a wide draft at the headline context
        _tree("tree_64_at_32k", 64, 32768),
        # a wide draft over a long document in fp16, 256-token pages of a shared pool, an odd count
        _tree("tree_63_at_64k_paged_f16", 63, 65536, kf="f16", vf="f16", page=256, gate=False),
        # a chunk of a prompt: the standard 512 queries onto 8192 keys, in order
        _tree("chain_512_at_8k", 512, 8192, mask="chain", gate=False),
        # one token's projections on their way into the cache, and back for a check
        _rope("rope_1_at_4k", 1, 4096),
        # a draft's worth of tokens, several at the same depth, from one fused projection buffer, with
        # interleaved pairs and positions scaled past the trained context
        _rope("rope_501_yarn_fused", 501, 40000, nrot=128, layout="interleaved", scaling="yarn", norm=False,
              rows="fused", tree=True, kf="f16"),
        # a layer of a long cache read back for another engine
        _case("read_32k_bf16", "read", 32768, 0, dtype="bf16"),
        # a few pages read back exactly
        _case("read_777_paged_f32", "read", 777, 300, kf="f16", vf="f16", page=64, dtype="f32"),
        # the accepted path of a draft, all layers
        _case("commit_5_of_64", "commit", 64, 2000, keep=5, layers=8),
        # many kept tokens of a large draft, fp16 in pages
        _case("commit_300_of_900_paged_f16", "commit", 900, 100, keep=300, kf="f16", vf="f16", page=16, layers=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the listed ranges: trees of 1 to 700 tokens onto none to 128K cached ones, 1 to 16 KV
    heads with 1 to 8 query heads each, every format pair, contiguous and paged."""
    op = rng.choice(["tree", "tree", "tree", "rope", "rope", "read", "commit"])
    kf, vf = rng.choice([("q8_0", "q8_0"), ("q8_0", "q8_0"), ("f16", "q8_0"), ("q8_0", "f16"), ("f16", "f16")])
    page = rng.choice([0, 0, 16, 48, 64, 256])
    nkv = rng.choice([4, 4, 4, 1, 2, 3, 8, 16])
    group = rng.choice([4, 4, 4, 1, 2, 5, 8])
    shape = dict(kf=kf, vf=vf, page=page, nkv=nkv, group=group)
    if op == "tree":
        n = _log(rng, 1, 700)
        # at most the largest listed case's query-key pairs and cached bytes
        room = int(min(512 * 8448 * 16 / (nkv * group * n) - n, 131072 * 4 / nkv / (2 if "f16" in (kf, vf) else 1)))
        ctx = rng.choice([0, 1, 31]) if room < 64 or rng.random() < 0.15 else _log(rng, 32, room)
        return _tree(None, n, ctx, mask=rng.choice(["tree", "tree", "tree", "chain", "padded"]),
                     gate=rng.random() < 0.6, **shape)
    if op == "rope":
        return _rope(None, _log(rng, 1, 2000 // nkv), _log(rng, 1, 200000) - 1, nrot=rng.choice([64, 64, 32, 128, 256, 20]),
                     layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                     norm=rng.random() < 0.5, rows=rng.choice(["own", "fused", "qg"]), tree=rng.random() < 0.5,
                     **dict(shape, page=0))
    if op == "read":
        return _case(None, "read", _log(rng, 1, 100000 // nkv), _log(rng, 1, 10000) - 1,
                     dtype=rng.choice(["f32", "f16", "bf16"]), **shape)
    n = _log(rng, 2, 1000)
    return _case(None, "commit", n, _log(rng, 1, 2000), keep=rng.randint(1, max(1, n // 2)), layers=rng.choice([1, 4, 8]),
                 **shape)


def _slot_bytes(c):
    """Bytes of one position of one layer: K and V, data and scales."""
    return sum(c["nkv"] * (HD * 2 if f == "f16" else HD + HD // BLK * 2) for f in (c["kf"], c["vf"]))


def work(case):
    n, ctx, nkv = case["n"], case["ctx"], case["nkv"]
    nh, sb = nkv * case["group"], _slot_bytes(case)
    if case["op"] == "tree":
        # q and out, the gate and the gated output; every row sees the context and at least itself
        pairs = n * (ctx + 1) if case["mask"] != "chain" else n * ctx + n * (n + 1) // 2
        return {"bytes": (ctx + n) * sb + n * nh * HD * 4 * (4 if case["gate"] else 2), "flops": 4 * HD * nh * pairs}
    if case["op"] == "rope":
        # projections in, q out; the cache written and read again, the values out
        return {"bytes": n * ((2 * nh + 2 * nkv) * HD * 4 + 2 * sb + 2 * nkv * HD * 2),
                "flops": n * (nh + 2 * nkv) * HD * 6}
    if case["op"] == "read":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * (sb + 2 * nkv * HD * size), "flops": n * 2 * nkv * HD}
    return {"bytes": 2 * case["keep"] * case["layers"] * sb, "flops": 0}


# ------------------------------------------------------------------ inputs
def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 7919 * stream + 1)
    return g


def _quantise(x):
    """q8_0 of fp32 [..][HD]: bytes, and one fp16 scale per 32 elements (d = amax / 127, q = rne(x * (1 / d)))."""
    b = x.unflatten(-1, (HD // BLK, BLK))
    amax = b.abs().amax(-1, keepdim=True)
    d = torch.where(amax > 1e-35, amax / 127.0, torch.zeros_like(amax))
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    q = (b * inv).round().clamp(-127, 127)
    return q.to(torch.int8).flatten(-2), d.squeeze(-1).half()


def _bytes(t):
    return t.contiguous().view(torch.uint8).reshape(*t.shape[:-2], -1)


def _slots(st, layer, first, n):
    """The cache slots of positions first .. first + n - 1."""
    p = torch.arange(first, first + n, device="cuda")
    if st["table"] is None:
        return p
    page = st["case"]["page"]
    return st["table"][layer].long()[p // page] * page + p % page


def _fill(st, seed):
    """Every layer's cache with positions 0 .. ctx + n - 1 written."""
    c = st["case"]
    nkv, end = c["nkv"], c["ctx"] + c["n"]
    for layer in range(c["layers"]):
        g = _gen(seed, 100 + layer)
        ch = torch.stack([torch.randperm(HD, generator=g, device="cuda")[:3] for _ in range(nkv)])
        big = torch.ones(nkv, HD, device="cuda").scatter_(1, ch, 8.0)
        for s in range(0, end, CHUNK):
            m = min(CHUNK, end - s)
            at = _slots(st, layer, s, m)
            for name, fmt, mul in (("k", c["kf"], big), ("v", c["vf"], 0.5)):
                x = torch.randn(m, nkv, HD, generator=g, device="cuda") * mul
                if fmt == "f16":
                    st[name + "_data"][layer, at] = _bytes(x.half())
                else:
                    q, d = _quantise(x)
                    st[name + "_data"][layer, at] = _bytes(q)
                    st[name + "_scales"][layer, at] = _bytes(d)


def _parents(n, r):
    """A draft in the order in which it grew: each token follows one of the last few, or the context."""
    return [-1 if i == 0 or r.random() < 0.05 else r.randint(max(0, i - 6), i - 1) for i in range(n)]


def _ancestors(parents):
    """Per token the bits of itself and the tokens that it follows, as a whole number, and its depth."""
    bits, depth = [], []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return bits, depth


def _mask_words(bits, n):
    words = -(-n // 64)
    u = np.array([[(b >> 64 * w) & (2**64 - 1) for w in range(words)] for b in bits], dtype=np.uint64)
    return torch.from_numpy(u.view(np.int64)).cuda()


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
        # pairs that turn FAST times or more in the trained context keep their angle, those that turn SLOW
        # times or fewer are interpolated, a ramp over the pairs' numbers joins the two
        at = [nrot * math.log(TRAINED / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (FAST, SLOW)]
        lo, hi = max(0, math.floor(at[0])), min(nrot - 1, math.ceil(at[1]))
        ramp = [min(1.0, max(0.0, (p - lo) / max(hi - lo, 1e-3))) for p in range(half)]
        th = [t * (1 - r) + t / FACTOR * r for t, r in zip(th, ramp)]
    return th, 0.1 * math.log(FACTOR) + 1.0 if scaling == "yarn" else 1.0


def prepare(case, seed):
    c = dict(case)
    nkv, nh, n, ctx, page = c["nkv"], c["nkv"] * c["group"], c["n"], c["ctx"], c["page"]
    st, g, r = {"case": c, "table": None}, _gen(seed, 1), random.Random(int(seed) * 7 + 3)
    cap, pages = ctx + n, 0
    if page:
        pages = -(-cap // page)
        pool = pages + 3
        st["table"] = torch.stack([torch.randperm(pool, generator=g, device="cuda")[:pages].int() for _ in range(c["layers"])])
        cap = pool * page
    for name, fmt in (("k", c["kf"]), ("v", c["vf"])):
        st[name + "_data"] = torch.zeros(c["layers"], cap, nkv * HD * (2 if fmt == "f16" else 1), dtype=torch.uint8, device="cuda")
        st[name + "_scales"] = None if fmt == "f16" else torch.zeros(c["layers"], cap, nkv * HD // BLK * 2, dtype=torch.uint8, device="cuda")
    if own:
        # the cache object that a user's program keeps, its arrays in the place of the plain ones
        from bonsai_vk_amd import BKV_F16, BKV_Q8_0, KvCache
        fmt = {"f16": BKV_F16, "q8_0": BKV_Q8_0}
        st["cache"] = KvCache(n_layers=c["layers"], nh=nh, nkv=nkv, cap=cap, k_fmt=fmt[c["kf"]], v_fmt=fmt[c["vf"]],
                              page_tokens=page, max_pages=pages, block_table=st["table"])
        for name in ("k_data", "k_scales", "v_data", "v_scales"):
            st[name] = getattr(st["cache"], name)
    if c["op"] != "rope":
        _fill(st, seed)
    if c["op"] == "tree":
        st["q"] = torch.randn(n, nh, HD, generator=g, device="cuda")
        st["gate"] = torch.randn(n, nh, HD, generator=g, device="cuda") if c["gate"] else None
        if c["mask"] == "chain":
            st["mask"] = None
        else:
            bits, _ = _ancestors(_parents(n, r))
            if c["mask"] == "padded":
                bits = bits[: n - n // 3] + [0] * (n // 3)
            st["mask"] = _mask_words(bits, n)
    if c["op"] == "rope":
        rows = torch.randn(n, 2 * nh + 2 * nkv, HD, generator=g, device="cuda") * 2.0
        if c["rows"] == "fused":
            st["q"], st["k"], st["v"] = rows[:, :nh], rows[:, nh:nh + nkv], rows[:, nh + nkv:nh + 2 * nkv]
        elif c["rows"] == "qg":
            st["q"] = rows[:, :2 * nh].contiguous().view(n, nh, 2 * HD)[:, :, :HD]
            st["k"], st["v"] = rows[:, 2 * nh:2 * nh + nkv].contiguous(), rows[:, 2 * nh + nkv:].contiguous()
        else:
            st["q"], st["k"], st["v"] = (rows[:, a:b].contiguous() for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
        st["qn_w"] = st["kn_w"] = None
        if c["norm"]:
            st["qn_w"], st["kn_w"] = (1.0 + 0.1 * torch.randn(HD, generator=g, device="cuda") for _ in range(2))
        depth = _ancestors(_parents(n, r))[1]
        st["positions"] = torch.tensor([ctx + d for d in depth], dtype=torch.int32, device="cuda") if c["tree"] else None
        th, st["mscale"] = _angles(c)
        st["theta"] = torch.tensor(th, dtype=torch.float64, device="cuda")
        if own:
            from bonsai_vk_amd import Rope
            st["rope"] = Rope(c["nrot"], layout=c["layout"], freq_base=BASE, scaling=c["scaling"], factor=FACTOR,
                              trained_ctx=TRAINED, beta_fast=FAST, beta_slow=SLOW)
    if c["op"] == "commit":
        # a path from the root: its first tokens stay where they are, the others come from behind what is kept
        keep = c["keep"]
        stay = r.randint(0, keep) if 2 * keep <= n else keep
        tail = sorted(r.sample(range(keep, n), keep - stay))
        st["idx"] = torch.tensor(list(range(stay)) + tail, dtype=torch.int32, device="cuda")
    return st


# ------------------------------------------------------------------ one pass
def _read(st, name, layer, first, n):
    """Positions first .. of K or V as fp32 [n][nkv][HD]."""
    c, at = st["case"], _slots(st, layer, first, n)
    data = st[name + "_data"][layer][at]
    if st[name + "_scales"] is None:
        return data.view(torch.float16).view(n, c["nkv"], HD).float()
    d = st[name + "_scales"][layer][at].view(torch.float16).view(n, c["nkv"], HD // BLK, 1).float()
    return (data.view(torch.int8).view(n, c["nkv"], HD // BLK, BLK).float() * d).flatten(-2)


def _attend(st):
    c = st["case"]
    n, ctx, nkv, group = c["n"], c["ctx"], c["nkv"], c["group"]
    k, v = (_read(st, x, 0, 0, ctx + n).transpose(0, 1).contiguous() for x in "kv")    # [nkv][keys][HD]
    q = st["q"].half().float().view(n, nkv, group, HD).permute(1, 2, 0, 3).reshape(nkv, group * n, HD)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).view(nkv, group, n, ctx + n) * HD ** -0.5
    j = torch.arange(n, device="cuda")
    seen = j[None] <= j[:, None] if st["mask"] is None else (st["mask"][:, j // 64] >> (j % 64)) & 1 != 0
    s[..., ctx:].masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(nkv, group * n, ctx + n), v).view(nkv, group, n, HD)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    out = out.permute(2, 0, 1, 3).reshape(n, nkv * group, HD)
    return (out,) if st["gate"] is None else (out, out / (1.0 + torch.exp(-st["gate"])))


def _rotate(st, x, w):
    """Norm (where there are weights) and rotation of fp32 rows [n][heads][HD]."""
    c = st["case"]
    nrot, half = c["nrot"], c["nrot"] // 2
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    at = torch.arange(c["ctx"], c["ctx"] + c["n"], device="cuda") if st["positions"] is None else st["positions"]
    a = at.double()[:, None, None] * st["theta"]
    cs, sn = (torch.cos(a) * st["mscale"]).float(), (torch.sin(a) * st["mscale"]).float()
    if c["layout"] == "half":
        lo, hi = x[..., :half], x[..., half:nrot]
        return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn, x[..., nrot:]], -1)
    lo, hi = x[..., :nrot:2], x[..., 1:nrot:2]
    return torch.cat([torch.stack([lo * cs - hi * sn, hi * cs + lo * sn], -1).flatten(-2), x[..., nrot:]], -1)


def _stored(x, fmt):
    if fmt == "f16":
        return x.half()
    q, d = _quantise(x)
    return (q.unflatten(-1, (HD // BLK, BLK)).float() * d.float()[..., None]).flatten(-2).half()


def _commit(st):
    c, arrays = st["case"], [st[a] for a in ("k_data", "k_scales", "v_data", "v_scales") if st[a] is not None]
    layer = torch.arange(c["layers"], device="cuda")[:, None]
    src = (st["idx"] + c["ctx"]).long().expand(c["layers"], -1)
    dst = torch.arange(c["ctx"], c["ctx"] + c["keep"], device="cuda").expand(c["layers"], -1)
    if st["table"] is not None:
        src, dst = (st["table"].long().gather(1, p // c["page"]) * c["page"] + p % c["page"] for p in (src, dst))
    for a in arrays:
        a[layer, dst] = a[layer, src]
    return arrays


def run(state):
    st, c = state, state["case"]
    n, ctx, op = c["n"], c["ctx"], c["op"]
    if op == "tree":
        if own:
            out, gated = st["cache"].attn_tree(0, ctx, st["q"], st["mask"], st["gate"])
            return (out,) if gated is None else (out, gated)
        return _attend(st)
    if op == "rope":
        if own:
            q = st["cache"].rope_append(0, ctx, st["q"], st["k"], st["v"], st["rope"], positions=st["positions"],
                                        qn_w=st["qn_w"], kn_w=st["kn_w"], eps=EPS)
            k, v = st["cache"].read(0, ctx, n, dtype=torch.float16)
            return {"q": q, "k": k, "v": v}
        return {"q": _rotate(st, st["q"], st["qn_w"]), "k": _stored(_rotate(st, st["k"], st["kn_w"]), c["kf"]),
                "v": _stored(st["v"], c["vf"])}
    if op == "read":
        if own:
            return st["cache"].read(0, ctx, n, dtype=DTYPE[c["dtype"]])
        return tuple(_read(st, x, 0, ctx, n).to(DTYPE[c["dtype"]]) for x in "kv")
    if own:
        st["cache"].commit(ctx, n, st["idx"])
        return [st[a] for a in ("k_data", "k_scales", "v_data", "v_scales") if st[a] is not None]
    return _commit(st)


# ------------------------------------------------------------------ in 64 bits
def _stored_values(st, name, first, n):
    """What the cache's bytes stand for, [n][nkv][HD] in 64 bits."""
    c = st["case"]
    pos = range(first, first + n)
    if st["table"] is None:
        at = torch.tensor(list(pos))
    else:
        row, page = st["table"][0].tolist(), c["page"]
        at = torch.tensor([row[p // page] * page + p % page for p in pos])
    data = st[name + "_data"][0].index_select(0, at.cuda())
    if c["kf" if name == "k" else "vf"] == "f16":
        return data.view(torch.float16).double().reshape(n, c["nkv"], HD)
    d = st[name + "_scales"][0].index_select(0, at.cuda()).view(torch.float16).double()
    return (data.view(torch.int8).double() * d.repeat_interleave(BLK, dim=1)).reshape(n, c["nkv"], HD)


def _exact_tree(st):
    c = st["case"]
    n, ctx, group = c["n"], c["ctx"], c["group"]
    k, v = (_stored_values(st, x, 0, ctx + n) for x in "kv")
    see = torch.ones(n, ctx + n, dtype=torch.bool)
    words = None if st["mask"] is None else st["mask"].cpu().numpy().view(np.uint64)
    for i in range(n):
        row = list(range(n)) if words is None else [int(w) >> b & 1 for w in words[i] for b in range(64)]
        see[i, ctx:] = torch.tensor([j <= i if words is None else bool(row[j]) for j in range(n)])
    see = see.cuda()
    out = torch.zeros(n, c["nkv"] * group, HD, dtype=torch.float64, device="cuda")
    for h in range(c["nkv"] * group):
        logits = st["q"][:, h].half().double().mm(k[:, h // group].t()) / math.sqrt(HD)
        logits = logits.masked_fill(~see, -math.inf)
        some = see.any(1)
        p = torch.softmax(logits[some], 1)
        out[some, h] = p.mm(v[:, h // group])
    if st["gate"] is None:
        return (out,)
    return out, out * torch.sigmoid(st["gate"].double())


def _exact_rope(st):
    c = st["case"]
    nrot, n = c["nrot"], c["n"]
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
    at = np.arange(c["ctx"], c["ctx"] + n) if st["positions"] is None else st["positions"].cpu().numpy()
    turn = torch.from_numpy(np.exp(1j * np.outer(at, freq)) * mul).cuda()[:, None]      # [n][1][pairs]
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
        b = x.reshape(n, c["nkv"], HD // BLK, BLK)
        d = b.abs().amax(3, keepdim=True) / 127
        return (torch.round(b / torch.where(d > 0, d, torch.ones_like(d))) * d.half().double()).reshape(x.shape)

    return {"q": rotated(st["q"], st["qn_w"]), "k": kept(rotated(st["k"], st["kn_w"]), c["kf"]),
            "v": kept(st["v"].double(), c["vf"])}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(st)
    if case["op"] == "rope":
        return _exact_rope(st)
    if case["op"] == "read":
        return tuple(_stored_values(st, x, case["ctx"], case["n"]) for x in "kv")
    return None
