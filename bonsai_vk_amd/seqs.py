"""Several sequences over one KvCache (no counterpart in the reference, which runs one): who has which pages
(bkv_pages_fork, bkv_pages_extend, bkv_pages_compact), their tokens' way into the cache (bkv_seqs_rope_append) and back
(bkv_seqs_read), and attention over a 4-bit cache (bkv_seqs_attn).

A step of a server, everything on the device and nothing read back:

    lack = seqs.extend(n_new)                # pages for the new tokens, copied where others share them
    have = (lack == 0).all()                 # else nothing was changed, and the step must not happen:
    seqs.len += n_new * have                 # no sequence gets longer,
    q_start = starts * have                  # none has rows in this call
    q = seqs.rope_append(layer, q, k, v, rope, q_start, positions, axes)
    out, gated = seqs.attn(layer, q, q_start, gate, max_q=longest)   # (tokens of the sequence that has most)

Without `have`, a pool that is exhausted would leave sequences that share a page all writing their new tokens into it. Whoever
takes the step's results reads `have` with them; a server then gives up a sequence (fork) and takes the step again.
"""
import ctypes

import torch

from ._lib import BKV_SEQS_MAX, BkvCacheDesc, BkvRopeAxes, BkvSeqs, check, lib
from .cache import _OUT_TYPES


class RopeAxes:
    """bkv_rope_axes_init: positions of several axes, pairs[i] of the rotated pairs turned by axis i's; order "blocks" (the
    first axis' pairs, then the second's) or "dealt" (in turn to the axes that still want some)."""

    def __init__(self, pairs, order="blocks"):
        orders = ("blocks", "dealt")
        if order not in orders:
            raise ValueError(f"order is one of {orders}")
        self.params, n = BkvRopeAxes(), len(pairs)
        check(lib().bkv_rope_axes_init(ctypes.byref(self.params), n, (ctypes.c_int32 * max(n, 1))(*pairs), orders.index(order)),
              "bkv_rope_axes_init")

    @property
    def n_axes(self):
        return self.params.n_axes

    @property
    def axis(self):
        """The axis of each pair."""
        return list(self.params.axis[:self.params.n_pairs])


class KvSeqs:
    """Up to n_seq sequences over `cache` (a KvCache, whose block table is not used). Tensors on its device:
      len     int32 [n_seq]                        positions that each has; the caller's to advance
      tables  int32 [n_seq][n_layers][max_pages]   their pages, -1 where there is none (paged only)
      refs    int32 [n_layers][pages]              how many table entries name a page (paged only)
    Others of the same kind may be put in their places (compact's, say); captured calls go on with those that were there.
    A contiguous cache has one sequence, and no pages to give out."""

    def __init__(self, cache, n_seq):
        if not 1 <= n_seq <= BKV_SEQS_MAX:
            raise ValueError(f"1 .. {BKV_SEQS_MAX} sequences, got {n_seq}")
        if not cache.page_tokens and n_seq != 1:
            raise ValueError("a contiguous cache holds one sequence")
        self.cache, self.n_seq, self._dev = cache, n_seq, cache._dev
        self._per, self._starts = torch.Size((n_seq,)), torch.Size((n_seq + 1,))
        self.len = torch.zeros(n_seq, dtype=torch.int32, device=self._dev)
        self._tables = self._refs = None
        self.desc = BkvCacheDesc()
        ctypes.memmove(ctypes.byref(self.desc), ctypes.byref(cache.desc), ctypes.sizeof(BkvCacheDesc))
        if cache.page_tokens:
            self._tables = torch.full((n_seq, cache.n_layers, cache.max_pages), -1, dtype=torch.int32, device=self._dev)
            self._refs = torch.zeros((cache.n_layers, cache.cap // cache.page_tokens), dtype=torch.int32, device=self._dev)
            self.desc.block_table = self._tables.data_ptr()
            need = lib().bkv_pages_workspace_bytes(ctypes.byref(self.desc))
            self._pws = torch.empty(need, dtype=torch.uint8, device=self._dev)
            self._pws_bytes = need
        self._ws, self._ws_bytes, self._held = None, 0, []

    # (looked at when they are set: the calls hand their addresses on as they are)
    @property
    def tables(self):
        return self._tables

    @tables.setter
    def tables(self, t):
        self._paged()
        self._tables = self.cache._on_device(t, torch.int32, self._tables.shape)
        self.desc.block_table = t.data_ptr()

    @property
    def refs(self):
        return self._refs

    @refs.setter
    def refs(self, t):
        self._paged()
        self._refs = self.cache._on_device(t, torch.int32, self._refs.shape)

    # ---------------------------------------------------------------- helpers
    def _paged(self):
        if self._tables is None:
            raise ValueError("a contiguous cache has no pages")

    def _per_seq(self, t):
        return self.cache._on_device(t, torch.int32, self._per).data_ptr()

    def _seqs(self, n_tok, q_start, max_q=0):
        if q_start is not None:
            q_start = self.cache._on_device(q_start, torch.int32, self._starts).data_ptr()
        elif n_tok < self.n_seq:
            raise ValueError(f"a token of each of {self.n_seq} sequences is wanted without q_start, got {n_tok}")
        return BkvSeqs(self.n_seq, n_tok, 1 if q_start is None else max_q, 0, q_start, self._per_seq(self.len),
                       None if self._tables is None else self._tables.data_ptr())

    def workspace(self, n_tok):
        """The workspace of attn for n_tok rows, made where the one there is smaller; a program that captures that call into a
        graph asks for it before. All of this object's attn calls (and replays) share it: they run one after another, on one
        stream or on streams that wait for one another. One that was ever handed out lives as long as this object: captured
        calls have its address, and a stream may still be at work in it."""
        need = lib().bkv_seqs_workspace_bytes(self.desc, self.n_seq, n_tok) if n_tok else 0
        if need > self._ws_bytes:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call workspace(n_tok) before the capture: memory of a graph's own pool would not outlive it")
            need = max(need, 2 * self._ws_bytes)   # (all that were outgrown together are no larger than the one there)
            ws = torch.empty(need, dtype=torch.uint8, device=self._dev)
            check(lib().bkv_workspace_init(self.desc, ws.data_ptr(), need, self.cache._my_stream()), "bkv_workspace_init")
            self._held.append(ws)
            self._ws, self._ws_bytes = ws, need
        return self._ws

    # ---------------------------------------------------------------- pages
    def fork(self, parent):
        """bkv_pages_fork: sequence s goes on from what parent[s] (int32 [n_seq] on the cache's device) was, len too; a parent
        outside 0 .. n_seq - 1 empties it."""
        if self.cache._elsewhere():
            with torch.cuda.device(self._dev):
                return self.fork(parent)
        self._paged()
        rc = lib().bkv_pages_fork(self.desc, self.n_seq, self._tables.data_ptr(), self._refs.data_ptr(), self._per_seq(self.len),
                                  self._per_seq(parent), self.cache._my_stream())
        if rc:
            check(rc, "bkv_pages_fork")

    def extend(self, n_new, lack=None):
        """bkv_pages_extend: pages for n_new[s] (int32 [n_seq] on the cache's device) more positions than len[s]. Returns lack,
        int32 [n_layers] on the device: the pages that each layer is short of; where any is, nothing was changed, and the new
        positions must not be written (a page there may still be several sequences'): len stays, and no sequence has rows in
        the step's calls (a q_start of 0s)."""
        if self.cache._elsewhere():
            with torch.cuda.device(self._dev):
                return self.extend(n_new, lack)
        self._paged()
        if lack is None:
            lack = torch.empty(self.cache.n_layers, dtype=torch.int32, device=self._dev)
        else:
            self.cache._on_device(lack, torch.int32, (self.cache.n_layers,))
        rc = lib().bkv_pages_extend(self.desc, self.n_seq, self._tables.data_ptr(), self._refs.data_ptr(), self._per_seq(self.len),
                                    self._per_seq(n_new), lack.data_ptr(), self._pws.data_ptr(), self._pws_bytes, self.cache._my_stream())
        if rc:
            check(rc, "bkv_pages_extend")
        return lack

    def compact(self, tables=None, refs=None):
        """bkv_pages_compact: the pages in use moved to the lowest numbers. The new tables and counts go to `tables` and `refs`
        where they are given (the old ones then still name the old pages), else in place. Returns them."""
        if self.cache._elsewhere():
            with torch.cuda.device(self._dev):
                return self.compact(tables, refs)
        self._paged()
        if (tables is None) != (refs is None):
            raise ValueError("tables and refs, or neither")
        tables = self._tables if tables is None else self.cache._on_device(tables, torch.int32, self._tables.shape)
        refs = self._refs if refs is None else self.cache._on_device(refs, torch.int32, self._refs.shape)
        rc = lib().bkv_pages_compact(self.desc, self.n_seq, self._tables.data_ptr(), self._refs.data_ptr(), tables.data_ptr(),
                                     refs.data_ptr(), self._pws.data_ptr(), self._pws_bytes, self.cache._my_stream())
        if rc:
            check(rc, "bkv_pages_compact")
        return tables, refs

    # ---------------------------------------------------------------- tokens
    def rope_append(self, layer, q, k, v, rope, q_start=None, positions=None, axes=None, qn_w=None, kn_w=None, eps=1e-6,
                    q_out=None):
        """bkv_seqs_rope_append: q [n_tok][nh][hd] (or None), k and v [n_tok][nkv][hd] as the projections left them (strided
        rows are taken in place), sequence s's tokens in rows q_start[s] .. (int32 [n_seq + 1] on the cache's device; None:
        one each), normed where qn_w and kn_w are given, rotated by `rope` at positions (int32 [n_axes][n_tok], or [n_tok] for
        one axis; None: those in the cache) with the pairs shared out by `axes` (RopeAxes), written as the last of len[s]
        positions. Returns the rotated Q; rows that are no sequence's are left as they are in q_out."""
        c = self.cache
        if c._elsewhere():
            with torch.cuda.device(self._dev):
                return self.rope_append(layer, q, k, v, rope, q_start, positions, axes, qn_w, kn_w, eps, q_out)
        n, keep = k.shape[0], []
        kr, vr, qr = c._rows(k, c.nkv, keep), c._rows(v, c.nkv, keep), None
        if v.shape[0] != n or (q is not None and q.shape[0] != n):
            raise ValueError("q, k and v of as many tokens are wanted")
        if q is not None:
            qr, q_out = c._rows(q, c.nh, keep), c._out(q_out, n)
        elif q_out is not None:
            raise ValueError("q_out without q")
        qw = None if qn_w is None else c._f32(qn_w, (c.hd,))
        kw = None if kn_w is None else c._f32(kn_w, (c.hd,))
        n_axes = 1 if axes is None else axes.n_axes
        if positions is not None:
            c._on_device(positions, torch.int32, (n,) if n_axes == 1 and positions.dim() == 1 else (n_axes, n))
        rc = lib().bkv_seqs_rope_append(self.desc, layer, self._seqs(n, q_start), rope.params, None if axes is None else axes.params,
                                        qr, kr, vr, c._ptr(qw), c._ptr(kw), eps, c._ptr(positions), c._ptr(q_out), c._my_stream())
        if rc:
            check(rc, "bkv_seqs_rope_append")
        return q_out

    def read(self, layer, q_start, n_tok, dtype=torch.float32):
        """bkv_seqs_read: (K, V) of the call's tokens as values, [n_tok][nkv][hd] of dtype (float32, float16 or bfloat16);
        rows that are no sequence's are not written."""
        c = self.cache
        if c._elsewhere():
            with torch.cuda.device(self._dev):
                return self.read(layer, q_start, n_tok, dtype)
        if dtype not in _OUT_TYPES:
            raise ValueError(f"{dtype} is none of {list(_OUT_TYPES)}")
        k, v = torch.empty((2, n_tok, c.nkv, c.hd), dtype=dtype, device=self._dev).unbind(0)
        rc = lib().bkv_seqs_read(self.desc, layer, self._seqs(n_tok, q_start), _OUT_TYPES[dtype], k.data_ptr(), v.data_ptr(),
                                 c.nkv * c.hd, c.hd, c._my_stream())
        if rc:
            check(rc, "bkv_seqs_read")
        return k, v

    def attn(self, layer, q, q_start=None, gate=None, out=None, out_gated=None, max_q=0):
        """bkv_seqs_attn: attention of the tokens' queries (q [n_tok][nh][hd], rotated), each over its sequence's positions up to
        its own, K and V both in 4 bits. q and gate may be strided rows. max_q: tokens that no sequence has more of (0: not
        known), by which the kernels are chosen (64 single tokens at 1000 positions: 20.9 us, 25.1 without it). Returns (out, out_gated); out_gated is None without a gate. Rows that are no sequence's are left
        as they are."""
        c = self.cache
        if c._elsewhere():
            with torch.cuda.device(self._dev):
                return self.attn(layer, q, q_start, gate, out, out_gated, max_q)
        n, keep = q.shape[0], []
        qr, gr = c._rows(q, c.nh, keep), None
        if gate is not None:
            gr = c._rows(gate, c.nh, keep)
            if gate.shape[0] != n:
                raise ValueError(f"a gate of {n} tokens is wanted, got {gate.shape[0]}")
            out_gated = c._out(out_gated, n)
        elif out_gated is not None:
            raise ValueError("out_gated without a gate")
        out, seqs = c._out(out, n), self._seqs(n, q_start, max_q)
        ws = self.workspace(n)
        rc = lib().bkv_seqs_attn(self.desc, layer, seqs, qr, gr, out.data_ptr(), c._ptr(out_gated), c._ptr(ws), self._ws_bytes,
                                 c._my_stream())
        if rc:
            check(rc, "bkv_seqs_attn")
        return out, out_gated
