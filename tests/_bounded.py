"""Sequences in bounded caches: pools whose bytes are built on the host, and what the operators are to give in 64 bits."""
import numpy as np
import torch

import _inputs as I
import _oracle as O
from _gpu import dev


def values(kv_type, raw, D):
    """[..., head bytes] uint8 -> [..., D] float64: what the bytes stand for"""
    raw = np.ascontiguousarray(raw)
    if kv_type == O.KV_F16:
        return raw.view(np.float16).astype(np.float64)
    nb = D // 32
    if kv_type == O.KV_Q8_0:
        d = np.ascontiguousarray(raw[..., :2 * nb]).view(np.float16).astype(np.float64)
        q = np.ascontiguousarray(raw[..., 2 * nb:]).view(np.int8).astype(np.float64)
        return (q.reshape(*d.shape, 32) * d[..., None]).reshape(*raw.shape[:-1], D)
    b = raw.reshape(*raw.shape[:-1], nb, 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (q * d).reshape(*raw.shape[:-1], D)


class Cache:
    """K and V pools of one layer [pages][positions][Hkv][head bytes] (rows of `extra` more bytes a page), the sequences' pages in random order; every
    position of a sequence's pages holds a value. stray: page-table entries past a sequence's pages (never to be followed)."""

    def __init__(self, p1a, kv_type, Hkv, D, psh, lens, seed, extra=0, stray=1 << 28, max_pages=None, paged=True):
        self.p1a, self.type, self.Hkv, self.D, self.psh, self.lens = p1a, kv_type, Hkv, D, psh, list(lens)
        g = I.rng(seed)
        page = 1 << psh
        self.page = page
        per = [max((n + page - 1) // page, 1) for n in lens]
        self.max_pages = max_pages or max(per) + 1
        self.n_pages = sum(per) + 2
        order = g.permutation(self.n_pages) if paged else np.arange(self.n_pages)
        self.table = np.full((len(lens), self.max_pages), stray, np.int32)
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at:at + n]
            at += n
        hb = O.row_bytes(kv_type, 1, D)
        self.hb = hb
        self.pstride = page * Hkv * hb + extra
        self.host = {}
        for w in "kv":
            x = I.normal(g, (self.n_pages * page, Hkv, D))
            if w == "k":
                x = x / np.sqrt((x * x).mean(-1, keepdims=True))
            c = O.HostKV.contiguous(kv_type, len(x), Hkv, D)
            O.kv_append_rows(c, x, x, np.arange(len(x)))
            raw = np.zeros((self.n_pages, self.pstride), np.uint8)
            raw[:, :page * Hkv * hb] = c.k.reshape(self.n_pages, -1)
            self.host[w] = raw
        self.upload()
        self.dtable = dev(self.table.reshape(-1))
        self.offsets = dev((np.arange(len(lens)) * self.max_pages).astype(np.int32))
        n_ctx = self.max_pages * page if paged else per[0] * page
        if paged:
            self.kv = p1a.KVCache(kv_type, n_ctx, Hkv, D, self.k.data_ptr(), self.v.data_ptr(), pt=self.dtable, rtab=self.offsets, psh=psh, pstride=self.pstride)
        else:
            self.kv = p1a.KVCache(kv_type, n_ctx, Hkv, D, self.k.data_ptr(), self.v.data_ptr())

    def upload(self):
        self.k, self.v = dev(self.host["k"].reshape(-1)), dev(self.host["v"].reshape(-1))

    def raw(self, w, s, n, pool=None):
        """bytes of the first n positions of sequence s: [n][Hkv][head bytes]"""
        pool = self.host[w] if pool is None else pool.reshape(self.n_pages, self.pstride)
        j = np.arange(n)
        rows = pool[:, :self.page * self.Hkv * self.hb].reshape(self.n_pages, self.page, self.Hkv, self.hb)
        return rows[self.table[s][j // self.page], j % self.page]

    def heads(self, w, s, n, pool=None):
        return values(self.type, self.raw(w, s, n, pool), self.D)


def seen(p, n, window, n_sink):
    """[rows][n]: what rows at positions p see"""
    p, j = np.asarray(p)[:, None], np.arange(n)[None]
    m = (j <= p) & (p >= 0)
    if window:
        m &= (j > p - window) | (j < n_sink)
    return m


def rows_exact(q, k, v, see, scale):
    """float64: out [T][Hq][D], lse [T][Hq], weights [T][Hq][n], the weighted sum of |v| and the largest sum of |q k| of a row. q [T][Hq][D], k, v [n][Hkv][D]"""
    q, k, v = (torch.from_numpy(np.ascontiguousarray(x, np.float64)) for x in (q, k, v))
    T, Hq, D = q.shape
    n, Hkv = k.shape[:2]
    grp = Hq // Hkv
    kk, vv = (x.repeat_interleave(grp, 1).permute(1, 2, 0) for x in (k, v))      # [Hq][D][n]
    x = torch.matmul(q.permute(1, 0, 2), kk) * scale
    see = torch.from_numpy(see)[None].expand(Hq, -1, -1)
    x = torch.where(see, x, -torch.inf)
    lse = torch.logsumexp(x, -1) if n else torch.full((Hq, T), -torch.inf, dtype=torch.float64)
    w = torch.where(see, (x - torch.where(lse.isinf(), 0, lse)[..., None]).exp(), 0)
    out = torch.matmul(w, vv.transpose(1, 2))
    size = torch.matmul(w, vv.abs().transpose(1, 2))
    qk = (torch.matmul(q.abs().permute(1, 0, 2), kk.abs()) * abs(scale) * see).amax(-1) if n else torch.zeros(Hq, T)
    f = lambda t: t.transpose(0, 1).contiguous().numpy()  # noqa: E731
    return f(out), f(lse), f(w), f(size), f(qk)


def bf16(x):
    """float array -> the bf16 tensor nearest to it, and what it holds"""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16)
    return t.cuda() if torch.cuda.is_available() else t, t.float().numpy().astype(np.float64)


def gated(x, gate):
    return x if gate is None else x / (1 + np.exp(-gate.astype(np.float64).reshape(x.shape)))
