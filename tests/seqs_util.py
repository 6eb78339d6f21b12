"""Plain 64-bit counterparts of the calls for several sequences (bkv_seqs_*, bkv_pages_*) and of the 4-bit format, and
caches to run them on. (No counterpart in the reference.)"""
import numpy as np
import torch

from bonsai_vk_amd import BKV_F16, BKV_Q4_0, BKV_Q8_0, KvCache, KvSeqs

HD = 256
FMT = {"f16": BKV_F16, "q8_0": BKV_Q8_0, "q4_0": BKV_Q4_0}


# ------------------------------------------------------------------ the format
def q4_quantise(x):
    """(codes 0 .. 15 [..][256], scale words uint16 [..][8]) of fp32 [..][256]."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], 8, 32)
    with np.errstate(all="ignore"):
        hi, lo = np.fmax.reduce(b, -1), np.fmin.reduce(b, -1)
        h = (np.where(hi >= -lo, hi, lo) * np.float32(-0.125)).astype(np.float16).view(np.uint16).astype(np.uint32)
        m = h & 0x7FFF
        m = np.minimum((m + 3 + (m >> 3 & 1)) & 0x7FF8, 0x6800)
        d = np.where(m > 0, m | (h & 0x8000), 0).astype(np.uint16)
        f = d.view(np.float16).astype(np.float32)
        inv = np.where(f != 0, np.float32(1) / f, np.float32(0)).astype(np.float32)
        q = np.rint(b * inv[..., None])
    q = np.where(np.isnan(q), 0, np.clip(q, -8, 7)).astype(np.int64)
    return (q + 8).reshape(x.shape), d


def q4_pack(codes):
    """Bytes [..][128] of codes [..][256]."""
    c = codes.reshape(*codes.shape[:-1], 32, 8).astype(np.uint32)
    w = np.zeros(c.shape[:-1], np.uint32)
    for e in range(8):
        w |= c[..., e] << np.uint32(16 * (e % 2) + 4 * (e // 2))
    return np.ascontiguousarray(w).view(np.uint8).reshape(*codes.shape[:-1], 128)


def q4_values(data, scales):
    """Values in 64 bits of bytes [..][128] and scale words uint16 [..][8]."""
    w = np.ascontiguousarray(data).view(np.uint32)
    c = np.stack([w >> np.uint32(16 * (e % 2) + 4 * (e // 2)) & np.uint32(15) for e in range(8)], -1).reshape(*data.shape[:-1], 8, 32)
    s = scales.astype(np.uint32)
    f = ((np.minimum(s & 0x7FF8, 0x6800) | (s & 0x8000)).astype(np.uint16)).view(np.float16).astype(np.float64)
    return ((c.astype(np.float64) - 8) * f[..., None]).reshape(*data.shape[:-1], 256)


# ------------------------------------------------------------------ caches
def make(lens, page, nkv=4, grp=4, k="q4_0", v="q4_0", layers=1, spare=3, seed=0, cap=None, room=None, hd=256):
    """(KvCache, KvSeqs) of sequences that have `lens` positions, their pages anywhere in the pool (every layer its own);
    room: positions that a sequence can have."""
    r = np.random.default_rng(seed)
    if page:
        per = [-(-n // page) for n in lens]
        pool = sum(per) + spare if cap is None else cap // page
        most = max(1, -(-(room or max(lens)) // page), *per)
        cache = KvCache(n_layers=layers, nh=nkv * grp, nkv=nkv, hd=hd, cap=pool * page, k_fmt=FMT[k], v_fmt=FMT[v], page_tokens=page,
                        max_pages=most, block_table=torch.full((layers, most), -1))
    else:
        cache = KvCache(n_layers=layers, nh=nkv * grp, nkv=nkv, cap=cap or max(max(lens), 1), k_fmt=FMT[k], v_fmt=FMT[v])
    seqs = KvSeqs(cache, len(lens))
    seqs.len.copy_(torch.tensor(lens, dtype=torch.int32))
    if page:
        for layer in range(layers):
            ids = r.permutation(pool)
            at = 0
            for s, n in enumerate(per):
                seqs.tables[s, layer, :n] = torch.from_numpy(ids[at:at + n].astype(np.int32))
                seqs.refs[layer, ids[at:at + n]] = 1
                at += n
    return cache, seqs


def fill(cache, seed=0, k_mul=1.0, v_mul=0.5):
    """Random values in every slot of every layer of a 4-bit cache (through the numpy format)."""
    r = np.random.default_rng(seed)
    for name, mul in (("k", k_mul), ("v", v_mul)):
        data, scales = getattr(cache, name + "_data"), getattr(cache, name + "_scales")
        x = (r.standard_normal((cache.n_layers, cache.cap, cache.nkv, HD)) * mul).astype(np.float32)
        c, d = q4_quantise(x)
        data.copy_(torch.from_numpy(q4_pack(c).reshape(cache.n_layers, cache.cap, -1)))
        scales.copy_(torch.from_numpy(np.ascontiguousarray(d).view(np.uint8).reshape(cache.n_layers, cache.cap, -1)))


def slots(seqs, layer, s, n):
    """Slots of sequence s's first n positions, -1 where the page is outside the pool."""
    p = np.arange(n)
    if seqs.tables is None:
        return p
    page, pool = seqs.cache.page_tokens, seqs.refs.shape[1]
    row = seqs.tables[s, layer].cpu().numpy()[p // page]
    return np.where((row >= 0) & (row < pool), row * page + p % page, -1)


def held(seqs, layer, s, n):
    """K and V of sequence s's first n positions in 64 bits [n][nkv][256] on the GPU, and which of them are there."""
    c, at = seqs.cache, slots(seqs, layer, s, n)
    out = []
    for name in "kv":
        d = getattr(c, name + "_data")[layer].cpu().numpy()[np.maximum(at, 0)].reshape(n, c.nkv, 128)
        sc = getattr(c, name + "_scales")[layer].cpu().numpy()[np.maximum(at, 0)].reshape(n, c.nkv, 16)
        out.append(torch.from_numpy(q4_values(d, np.ascontiguousarray(sc).view(np.uint16).reshape(n, c.nkv, 8))).cuda())
    return out[0], out[1], torch.from_numpy(at >= 0).cuda()


# ------------------------------------------------------------------ attention
def attention(seqs, layer, q, starts, lens, scale):
    """(out, bound) in 64 bits [n_tok][nh][256]; bound: what an output may be off by, for the roundings counted here, with
    eps = 2^-24 and per row A = scale * the largest sum |q k|:
      the score's products are exact, 256 of them are added: 256 eps A; times scale * log2(e), less m: 2 eps (A + 16)
      (the last in units of log2; a score is at most A and a reference at most 15 above the largest)
      exp2: 2 eps; p to ph + pl: 2^-22 of it, or, where that is more, half of fp16's smallest step: p is 2^9 2^(x - m) there,
      so 2^-25 / 2^9 = 2^-34 of the largest p (whose x is m or more) for each key: 2^-34 sum |v|; each output's sum, 3 adds a key of a step, then over steps, waves, pieces: the steps'
      number + 128 + 32 roundings; the division and the sum of p: as many again."""
    nh, nkv = seqs.cache.nh, seqs.cache.nkv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    eps = 2.0 ** -24
    for s, n_pos in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        n = b - a
        if n <= 0 or n_pos <= 0:
            continue
        k, v, there = held(seqs, layer, s, n_pos)
        i = torch.arange(n, device="cuda")
        see = (torch.arange(n_pos, device="cuda")[None] <= (n_pos - n + i)[:, None]) & there[None]
        some = see.any(1)
        for h in range(nh):
            qd, kd, vd = q[a:b, h].half().double(), k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
            x = (qd @ kd.t() * scale).masked_fill(~see, float("-inf"))
            p = torch.softmax(x[some], 1)
            size = (qd.abs() @ kd.abs().t() * scale).masked_fill(~see, 0.0).amax(1)[some]
            o = torch.zeros(n, HD, dtype=torch.float64, device="cuda")
            o[some] = p @ vd
            out[a:b, h] = o
            off = 2 * (256 * eps * size + 2 * eps * (size + 16) * 0.7 + 2 * eps + 2.0 ** -22) + 2 * (n_pos / 32 + 160) * eps
            w = torch.zeros(n, HD, dtype=torch.float64, device="cuda")
            w[some] = off[:, None] * (p @ vd.abs()) + 2.0 ** -34 * (see[some].double() @ vd.abs()) + 2.0 ** -36
            bound[a:b, h] = w
    return out, bound


def starts_of(n):
    return [0] + [int(x) for x in np.cumsum(n)]


def device_ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ pages
class Pages:
    """tables, refs and len as Python numbers, and the calls on them one page after another."""

    def __init__(self, seqs):
        self.tables, self.refs = seqs.tables.cpu().numpy().copy(), seqs.refs.cpu().numpy().copy()
        self.len, self.page = seqs.len.cpu().numpy().copy(), seqs.cache.page_tokens

    def valid(self, e):
        return 0 <= e < self.refs.shape[1]

    def fork(self, parent):
        n = len(parent)
        new = np.stack([self.tables[p] if 0 <= p < n else np.full_like(self.tables[0], -1) for p in parent])
        for t, one in ((self.tables, -1), (new, 1)):
            for layer in range(t.shape[1]):
                for e in t[:, layer].reshape(-1):
                    if self.valid(e):
                        self.refs[layer, e] += one
        self.tables = new
        self.len = np.array([self.len[p] if 0 <= p < n else 0 for p in parent], np.int32)

    def extend(self, n_new):
        """(lack per layer, copies as (layer, from, to, positions held))"""
        seqs, layers, most = self.tables.shape
        lack, plan = [], []
        for layer in range(layers):
            refs = self.refs[layer]
            wants, over = [], 0
            for s in range(seqs):
                have, n = max(int(self.len[s]), 0), max(int(n_new[s]), 0)
                for p in range(have // self.page, -(-(have + n) // self.page)) if n else ():
                    if p >= most:
                        over += 1
                    else:
                        wants.append((s, p))
            who = {}
            for s, p in wants:
                who.setdefault(int(self.tables[s, layer, p]), []).append(s)
            todo = []
            for s, p in wants:
                e = int(self.tables[s, layer, p])
                if not self.valid(e):
                    todo.append((s, p, -1))
                elif refs[e] > 1 and not (len(who[e]) == refs[e] and s == max(who[e])):
                    todo.append((s, p, e))
            free = [p for p in range(len(refs)) if refs[p] == 0]
            lack.append(max(0, len(todo) - len(free)) + over)
            plan.append(list(zip(todo, free)))
        copies = []
        if not any(lack):
            for layer, todo in enumerate(plan):
                for (s, p, e), to in todo:
                    self.tables[s, layer, p] = to
                    self.refs[layer, to] = 1
                    if e >= 0:
                        self.refs[layer, e] -= 1
                        held = int(self.len[s]) % self.page if p == int(self.len[s]) // self.page else 0
                        copies.append((layer, e, to, held))
        return lack, copies

    def compact(self):
        copies = []
        for layer, refs in enumerate(self.refs):
            used = int((refs > 0).sum())
            moved = [p for p in range(len(refs)) if refs[p] > 0 and p >= used]
            into = [p for p in range(used) if refs[p] <= 0]
            to = dict(zip(moved, into))
            for a, b in to.items():
                copies.append((layer, a, b, self.page))
                refs[b], refs[a] = refs[a], 0
            t = self.tables[:, layer]
            self.tables[:, layer] = np.vectorize(lambda e: to.get(e, e), otypes=[np.int32])(t)
        return copies


def arrays(cache):
    return [a for a in (cache.k_data, cache.k_scales, cache.v_data, cache.v_scales) if a is not None]


def copied(before, copies, page):
    """The arrays' bytes after the copies, every source read before."""
    after = [a.clone() for a in before]
    for a, b in zip(before, after):
        for layer, src, dst, n in copies:
            b[layer, dst * page:dst * page + n] = a[layer, src * page:src * page + n]
    return after


def random_bytes(cache, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for a in arrays(cache):
        a.copy_(torch.randint(0, 256, a.shape, dtype=torch.uint8, device="cuda", generator=g))
