"""Attention of several sequences' chunks with windows and sinks, attention weight per position, eviction - each against its formula in 64 bits, and a
session that runs through all of them.

How far results may be off, from the arithmetic alone. f32 results: q and P are cut into two halves of 11 bits (2^-22 each), products of two low halves are
left out (2^-22), sums are fp32 - a few 2^-24 of the summed magnitudes each, signs at random: 1e-5 in the 2-norm is what the header says. bf16 results: one
rounding of the result (2^-8 of it), q, P and quantized K and V rounded to f16 once (2^-11 each): a score is off by at most 2 * 2^-11 * sum |q k| scale,
a weight by twice that much of itself, the result by that, P's and V's of the weighted sum of |v|."""
import numpy as np
import pytest
import torch

import _inputs as I
import _oracle as O
from _bounded import Cache, bf16, gated, rows_exact, seen
from _gpu import dev

pytestmark = pytest.mark.gpu

KVS = {"f16": O.KV_F16, "q8_0": O.KV_Q8_0, "q4_0": O.KV_Q4_0}
REL = 1e-5


def rows_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


class Call:
    """One call's inputs and, sequence by sequence, what it is to give"""

    def __init__(self, p1a, cache, Hq, counts, pos0, window=0, n_sink=0, q_bf16=False, gate=False, seed=1, scale=None, spare=0, max_n=0, max_rows=None, row0=True):
        g = I.rng(seed)
        T, D = int(sum(counts)), cache.D
        self.cache, self.Hq, self.T, self.scale = cache, Hq, T, D ** -0.5 if scale is None else scale
        q = I.normal(g, (T + spare, Hq, D))
        q /= np.sqrt((q * q).mean(-1, keepdims=True))
        self.q, self.q64 = bf16(q) if q_bf16 else (dev(q), q.astype(np.float64))
        self.gate = I.normal(g, (T + spare, Hq * D)) if gate else None
        self.dgate = dev(self.gate) if gate else None
        self.first, self.counts, self.pos0 = rows_of(counts), list(counts), list(pos0)
        self.row0, self.dpos = dev(self.first) if row0 else None, dev(np.asarray(pos0, np.int32))
        self.rows = p1a.Rows(T + spare, n_seq=len(counts), row0=self.row0, pos0=self.dpos, max_rows=max(counts) if max_rows is None else max_rows, max_n=max_n,
                             window=window, n_sink=n_sink)
        n_ctx = cache.kv.n_ctx
        self.want = []
        for s, (c, p0) in enumerate(zip(counts, pos0)):
            p = p0 + np.arange(c)
            p = np.where((p >= 0) & (p < n_ctx), p, -1)
            n = int(p.max(initial=-1)) + 1
            self.want.append(rows_exact(self.q64[self.first[s]:self.first[s + 1]], cache.heads("k", s, n), cache.heads("v", s, n), seen(p, n, window, n_sink), self.scale))

    def all(self, i):
        return np.concatenate([w[i] for w in self.want])

    def chunk(self, p1a, out_bf16=False, lse=True, scratch=None):
        out = torch.full((self.q.shape[0], self.Hq, self.cache.D), 77.0, dtype=torch.bfloat16 if out_bf16 else torch.float32, device="cuda")
        z = torch.full((self.q.shape[0], self.Hq), 77.0, device="cuda") if lse else None
        p1a.attn_chunk(self.q, self.cache.kv, out, self.rows, self.Hq, self.scale, gate=self.dgate, lse=z, scratch=scratch)
        torch.cuda.synchronize()
        assert (out[self.T:] == 77).all() and (z is None or (z[self.T:] == 77).all()), "rows of no sequence were written"
        return out[:self.T].float().cpu().numpy().astype(np.float64), None if z is None else z[:self.T].cpu().numpy().astype(np.float64)

    def check(self, p1a, out_bf16=False, lse=True, quantized=None):
        got, z = self.chunk(p1a, out_bf16, lse)
        gate = None if self.gate is None else self.gate[:self.T]
        want, size, qk = gated(self.all(0), gate), gated(self.all(3), gate), self.all(4)
        assert np.isfinite(got).all()
        if out_bf16:
            tol = 2.0 ** -8 * np.abs(want) + (2 * (2 * 2.0 ** -11) * qk[..., None] * 1.01 + 2 * 2.0 ** -11) * size + 1e-6 * size
            assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) - tol).max())
        else:
            assert np.linalg.norm(got - want) <= REL * np.linalg.norm(want), np.linalg.norm(got - want) / np.linalg.norm(want)
            assert np.abs(got - want).max(initial=0) <= 40 * REL * max(size.max(initial=0), 1e-30)
        if z is not None:
            ref = self.all(1)
            live = np.isfinite(ref)
            assert np.array_equal(z == -np.inf, ~live)
            # a score is off by some 2^-22 of sum |q k|, the logarithm and its factor by 2^-24 of themselves
            assert (np.abs(z - np.where(live, ref, 0))[live] <= (REL * qk + 2.0 ** -22 * (np.abs(np.where(live, ref, 0)) + 16))[live]).all()


SHAPES = [(4, 1, 64), (12, 2, 256), (32, 8, 128), (8, 8, 64), (5, 5, 128), (16, 1, 64), (40, 1, 128), (64, 1, 64)]


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", list(KVS))
def test_ragged_chunks(p1a, kv, D, out_bf16):
    """sequences of no rows, of one and of hundreds, over whole contexts, through windows, with sinks; gates; rows behind the last sequence"""
    lens = [130, 1, 611, 64, 300]
    counts = [130, 0, 77, 1, 33]
    cache = Cache(p1a, KVS[kv], 2, D, 4, lens, 5)
    for window, n_sink in ((0, 0), (100, 0), (64, 5), (1, 0), (37, 70), (5000, 4)):
        Call(p1a, cache, 12, counts, [n - c for n, c in zip(lens, counts)], window, n_sink, gate=window == 64, spare=3).check(p1a, out_bf16, lse=not out_bf16)


@pytest.mark.parametrize("Hq, Hkv, D", SHAPES)
@pytest.mark.parametrize("kv", list(KVS))
def test_single_tokens(p1a, kv, Hq, Hkv, D):
    """decode: one token a sequence, from the first position on; bf16 in, f32 out and the other way round"""
    lens = [1, 2, 17, 64, 65, 500, 1500]
    cache = Cache(p1a, KVS[kv], Hkv, D, 5, lens, 6)
    for window, n_sink in ((0, 0), (128, 4), (3, 1)):
        call = Call(p1a, cache, Hq, [1] * len(lens), [n - 1 for n in lens], window, n_sink, q_bf16=window == 3, row0=window != 3)
        call.check(p1a)
        call.check(p1a, out_bf16=True, lse=False)


@pytest.mark.parametrize("psh, extra", [(0, 0), (1, 16), (2, 0), (3, 48), (6, 0), (8, 16)])
def test_pages(p1a, psh, extra):
    """pages of one position and more, tiles that end inside a page and pages inside a tile, page strides of more than the page"""
    lens, counts = [333, 70], [45, 70]
    for kv in KVS:
        cache = Cache(p1a, KVS[kv], 2, 128, psh, lens, 7, extra=extra)
        Call(p1a, cache, 6, counts, [n - c for n, c in zip(lens, counts)], 50, 9).check(p1a)


def test_contiguous_and_host_position(p1a):
    """a cache without pages; the position of the only sequence from the host"""
    for kv in KVS:
        cache = Cache(p1a, KVS[kv], 4, 64, 4, [400], 8, paged=False)
        call = Call(p1a, cache, 8, [90], [310], 77, 3)
        want, z = call.chunk(p1a)
        call.check(p1a)
        call.rows = p1a.Rows(90, p0=310, window=77, n_sink=3)
        got, zz = call.chunk(p1a)
        assert np.allclose(got, want, rtol=1e-5, atol=1e-6) and np.allclose(z, zz, rtol=1e-5)
        call.check(p1a)


def test_rows_that_see_nothing(p1a):
    """positions below zero and past the descriptor's n_ctx: results 0, log-sum-exp -inf, gate or not; their neighbours as ever"""
    cache = Cache(p1a, O.KV_Q8_0, 2, 64, 4, [64, 64, 64], 9, max_pages=4)
    assert cache.kv.n_ctx == 64
    for window in (0, 20):
        call = Call(p1a, cache, 8, [10, 10, 10], [-4, 60, -2000000000], window, 2 if window else 0, gate=True)
        call.check(p1a)
        got, z = call.chunk(p1a)
        assert (got[:4] == 0).all() and (got[14:] == 0).all() and (z[20:] == -np.inf).all()
    call = Call(p1a, cache, 8, [10, 10, 10], [2147483640, 64, 2], 0, 0)
    got, z = call.chunk(p1a)
    assert (got[:20] == 0).all() and (got[20:] != 0).any(-1).all()


@pytest.mark.parametrize("kv", list(KVS))
def test_what_no_row_sees_is_not_read(p1a, kv):
    """behind a window: page-table entries that lead nowhere, and rows of NaN in pages that are partly seen; past the last position likewise"""
    D, lens, counts, window, n_sink = 128, [700, 300], [40, 1], 90, 3
    cache = Cache(p1a, KVS[kv], 2, D, 4, lens, 10)
    call = Call(p1a, cache, 4, counts, [n - c for n, c in zip(lens, counts)], window, n_sink)
    clean, z = call.chunk(p1a)
    for s, n in enumerate(lens):
        low = n - counts[s] - window + 1
        for j in list(range(n_sink, low)) + list(range(n, -(-n // 16) * 16)):
            for w in "kv":
                cache.host[w][cache.table[s, j // 16]].reshape(16, -1)[j % 16] = 0xff     # NaN as f16, as scale and as code
        cache.table[s, -(-n_sink // 16):low // 16] = 1 << 28
    cache.upload()
    cache.kv.k, cache.kv.v = cache.k.data_ptr(), cache.v.data_ptr()
    cache.dtable.copy_(torch.from_numpy(cache.table.reshape(-1)))
    got, zz = call.chunk(p1a)
    assert np.array_equal(got, clean) and np.array_equal(z, zz)
    mass = [torch.zeros(2, 2, 704, device="cuda") for _ in range(2)]
    for m in mass:
        p1a.attn_mass(call.q, cache.kv, torch.from_numpy(z.astype(np.float32)).cuda(), m, call.rows, 4, call.scale)
    assert torch.isfinite(mass[0]).all() and torch.equal(*mass)


def test_large_and_small_numbers(p1a):
    """queries far outside f16's range on either side, a negative scale, a scale of zero"""
    cache = Cache(p1a, O.KV_Q8_0, 2, 64, 4, [200], 11)
    for size, scale in ((1e6, 1e-7), (3e-7, 4e5), (1.0, -0.125), (1.0, 0.0), (1e-30, 0.125)):
        call = Call(p1a, cache, 4, [30], [170], 0, 0)
        call.q = call.q * size
        call.q64, call.scale = call.q.cpu().numpy().astype(np.float64), scale
        call.want = [rows_exact(call.q64, cache.heads("k", 0, 200), cache.heads("v", 0, 200), seen(170 + np.arange(30), 200, 0, 0), scale)]
        call.check(p1a)


def test_scores_far_apart(p1a):
    """rows whose maximum grows by hundreds along the keys (the running reference moves), and falls (it does not)"""
    for order in (1, -1):
        cache = Cache(p1a, O.KV_F16, 1, 64, 4, [640], 12)
        k = cache.heads("k", 0, 640) * np.linspace(0.01, 20, 640)[::order][:, None, None]
        for j in range(640):
            cache.host["k"][cache.table[0, j // 16]].reshape(16, -1)[j % 16] = k[j].astype(np.float16).view(np.uint8).reshape(-1)
        cache.upload()
        cache.kv.k, cache.kv.v = cache.k.data_ptr(), cache.v.data_ptr()
        call = Call(p1a, cache, 4, [100], [540], 0, 0, scale=1.0)
        got, z = call.chunk(p1a)
        # (weights are e^s: a score of size 400 in fp32 is off by 2^-24 * 3 D of it at most, some 1e-4)
        assert np.abs(got - call.all(0)).max() <= 1e-3 and np.abs(z - call.all(1)).max() <= 1e-3


@pytest.mark.parametrize("counts, lens, window", [([1], [9000], 0), ([3, 1], [5000, 2], 0), ([20], [4100], 2500), ([40, 9], [2600, 2600], 0)])
def test_splits(p1a, counts, lens, window):
    """few rows over many keys: split and merged; partials in the library's memory and the caller's give the same bits, the rows behind are left"""
    cache = Cache(p1a, O.KV_Q4_0, 1, 128, 6, lens, 13)
    call = Call(p1a, cache, 8, counts, [n - c for n, c in zip(lens, counts)], window, 4 if window else 0, gate=True, spare=2)
    need = p1a.chunk_scratch_bytes(cache.kv, call.rows, 8)
    assert need > 0
    call.check(p1a)
    call.check(p1a, out_bf16=True, lse=False)
    a = call.chunk(p1a)
    for extra in (0, -256):                                    # (less than it needs: the library's)
        scratch = torch.full((need + extra,), 255, dtype=torch.uint8, device="cuda")
        b = call.chunk(p1a, scratch=scratch)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_many_sequences(p1a):
    """more sequences than a wave has lanes, ragged"""
    g = I.rng(14)
    counts = [int(x) for x in g.integers(0, 5, 150)]
    lens = [c + int(x) for c, x in zip(counts, g.integers(0, 40, 150))]
    cache = Cache(p1a, O.KV_F16, 1, 64, 4, [max(n, 1) for n in lens], 14)
    Call(p1a, cache, 2, counts, [n - c for n, c in zip(lens, counts)], 16, 2, spare=1).check(p1a)


def test_device_numbers_out_of_line(p1a):
    """row0 past T, running backwards, sequences of more rows than max_rows: nothing outside the tensors is touched, whole sequences come out right"""
    cache = Cache(p1a, O.KV_F16, 2, 64, 4, [40, 40, 40, 40], 15)
    q = torch.randn(30, 4, 64, device="cuda")
    for row0 in ([0, 10, 5, 20, 30], [0, 10, 20, 30, 1000], [-7, 10, 20, 30, 30], [30, 0, 0, 0, 0]):
        out, z = torch.full((30, 4, 64), 7.0, device="cuda"), torch.full((30, 4), 7.0, device="cuda")
        rows = p1a.Rows(30, n_seq=4, row0=torch.tensor(row0, dtype=torch.int32, device="cuda"), pos0=torch.zeros(4, dtype=torch.int32, device="cuda"), max_rows=12)
        p1a.attn_chunk(q, cache.kv, out, rows, 4, 0.125, lse=z)
        mass = torch.zeros(4, 2, 48, device="cuda")
        p1a.attn_mass(q, cache.kv, torch.zeros(30, 4, device="cuda"), mass, rows, 4, 0.125)
        torch.cuda.synchronize()
        assert torch.isfinite(out).all() and torch.isfinite(mass).all()


def test_far_pages(p1a):
    """pages whose bytes lie past 4 GB from the base"""
    D, Hkv, page = 128, 2, 64
    stride = page * Hkv * D * 2
    far = (5 << 30) // stride
    pool = torch.zeros((far + 8) * stride, dtype=torch.uint8, device="cuda")
    cache = Cache(p1a, O.KV_F16, Hkv, D, 6, [200], 16)
    old = cache.table[0, :4].copy()
    new = np.array([far + 3, 1, far + 6, far + 1], np.int32)
    table = torch.from_numpy(new).cuda()
    vpool = torch.zeros_like(pool)
    for o, n in zip(old, new):
        pool[int(n) * stride:(int(n) + 1) * stride] = dev(cache.host["k"][o])
        vpool[int(n) * stride:(int(n) + 1) * stride] = dev(cache.host["v"][o])
    call = Call(p1a, cache, 4, [60], [140], max_n=200)          # (the two descriptors' n_ctx differ; this is what the work is dealt out by)
    want = call.chunk(p1a)
    call.cache.kv = p1a.KVCache(p1a.KV_F16, 256, Hkv, D, pool.data_ptr(), vpool.data_ptr(), pt=table, rtab=torch.zeros(1, dtype=torch.int32, device="cuda"), psh=6, pstride=stride)
    got = call.chunk(p1a)
    assert np.array_equal(want[0], got[0])
    m = torch.zeros(1, Hkv, 200, device="cuda")
    p1a.attn_mass(call.q, call.cache.kv, torch.from_numpy(got[1].astype(np.float32)).cuda(), m, call.rows, 4, call.scale)
    assert abs(float(m.sum()) - 60 * 4) < 1e-2
    keep = torch.tensor([[[0, 130, 199], [5, 6, 140]]], dtype=torch.int32, device="cuda")
    p1a.kv_compact(call.cache.kv, keep)
    torch.cuda.synchronize()
    at = lambda p, j, h: p[int(new[j // page]) * stride + (j % page) * Hkv * D * 2 + h * D * 2:][:D * 2].cpu().numpy()  # noqa: E731
    for h, idx in enumerate(keep[0].tolist()):
        for k, j in enumerate(idx):
            assert np.array_equal(at(pool, k, h).view(np.float16), cache.heads("k", 0, 200)[j, h].astype(np.float16)), (h, k, j)
            assert np.array_equal(at(vpool, k, h).view(np.float16), cache.heads("v", 0, 200)[j, h].astype(np.float16)), (h, k, j)


# ---- attention weight per position ----
def mass_want(call, cache, mass, ld):
    got = mass.astype(np.float64).copy()
    for s, w in enumerate(call.want):
        n = min(w[2].shape[-1], ld)
        if n and len(w[2]):
            got[s, :, :n] += w[2].reshape(len(w[2]), cache.Hkv, -1, w[2].shape[-1]).sum((0, 2))[:, :n]
    return got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", list(KVS))
def test_mass(p1a, kv, D):
    """decode steps, ragged chunks, windows and sinks, rows of the total longer and shorter than the sequences; twice: the total doubles; the same bits each time.
    A weight e^(s - lse) is off by a few 2^-22 of sum |q k| and 2^-23 of |s| + |lse| (some 20): 1e-5 in the 2-norm"""
    lens, counts = [130, 1, 611, 64, 300], [130, 0, 77, 1, 33]
    cache = Cache(p1a, KVS[kv], 2, D, 4, lens, 21)
    for window, n_sink, ld in ((0, 0, 611), (100, 0, 700), (64, 5, 611), (1, 0, 611), (37, 70, 400), (0, 0, 33)):
        call = Call(p1a, cache, 12, counts, [n - c for n, c in zip(lens, counts)], window, n_sink, q_bf16=window == 100, spare=2)
        lse = dev(np.concatenate([call.all(1), np.full((2, 12), np.nan)]).astype(np.float32))
        start = np.abs(I.normal(I.rng(3), (5, 2, ld))) * 0.01
        m, again = dev(start), dev(start)
        p1a.attn_mass(call.q, cache.kv, lse, m, call.rows, 12, call.scale)
        p1a.attn_mass(call.q, cache.kv, lse, again, call.rows, 12, call.scale)
        assert torch.equal(m, again)
        want = mass_want(call, cache, start, ld)
        got = m.cpu().numpy().astype(np.float64)
        assert np.linalg.norm(got - want) <= REL * np.linalg.norm(want - start) + 2.0 ** -24 * np.linalg.norm(want), (window, n_sink, ld)
        untouched = want == start.astype(np.float64)
        assert np.array_equal(got[untouched], start[untouched].astype(np.float64))
        p1a.attn_mass(call.q, cache.kv, lse, m, call.rows, 12, call.scale)
        want2 = mass_want(call, cache, got.astype(np.float32), ld)
        assert np.linalg.norm(m.cpu().numpy() - want2) <= REL * np.linalg.norm(want2 - got) + 2.0 ** -24 * np.linalg.norm(want2)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", list(KVS))
def test_mass_rows_by_the_tile(p1a, kv, D):
    """33 to 385 rows under a kv head - two to thirteen times 32, every place that rows take in turn -, several blocks of keys, positions that come to lie on
    their ends; the tolerance is test_mass's"""
    counts = [9, 16, 24, 25, 40, 49, 57, 64, 97]
    lens = [9, 256, 257, 511, 513, 49, 1030, 64, 700]
    cache = Cache(p1a, KVS[kv], 1, D, 4, lens, 25)
    call = Call(p1a, cache, 4, counts, [n - c for n, c in zip(lens, counts)])
    m = torch.zeros(9, 1, 1030, device="cuda")
    p1a.attn_mass(call.q, cache.kv, dev(call.all(1).astype(np.float32)), m, call.rows, 4, call.scale)
    want = mass_want(call, cache, np.zeros((9, 1, 1030), np.float32), 1030)
    got = m.cpu().numpy()
    for s in range(9):
        assert np.linalg.norm(got[s] - want[s]) <= REL * np.linalg.norm(want[s]), s
        assert not got[s, :, lens[s]:].any()


@pytest.mark.parametrize("Hq, Hkv, D", SHAPES)
def test_mass_single_tokens(p1a, Hq, Hkv, D):
    lens = [1, 2, 33, 64, 129, 500, 1500]
    for kv in KVS:
        cache = Cache(p1a, KVS[kv], Hkv, D, 4, lens, 22)
        call = Call(p1a, cache, Hq, [1] * 7, [n - 1 for n in lens], 0, 0, max_n=100, row0=False)      # (max_n understated: the same totals)
        m = torch.zeros(7, Hkv, 1500, device="cuda")
        p1a.attn_mass(call.q, cache.kv, dev(call.all(1).astype(np.float32)), m, call.rows, Hq, call.scale)
        want = mass_want(call, cache, np.zeros((7, Hkv, 1500), np.float32), 1500)
        assert np.linalg.norm(m.cpu().numpy() - want) <= REL * np.linalg.norm(want)


# ---- which positions stay ----
def keep_want(mass, n, budget, n_sink, n_recent):
    keep = np.full(mass.shape[:2] + (budget,), -1, np.int32)
    for s in range(mass.shape[0]):
        ns = min(max(int(n[s]), 0), mass.shape[2])
        for h in range(mass.shape[1]):
            if ns <= budget:
                keep[s, h, :ns] = np.arange(ns)
                continue
            m = mass[s, h, :ns].astype(np.float64)
            m = np.where(np.isnan(m), -np.inf, m)
            nan = np.isnan(mass[s, h, :ns])
            mid = np.arange(n_sink, ns - n_recent)
            best = mid[np.lexsort((mid, -m[mid], nan[mid]))][:budget - n_sink - n_recent]
            keep[s, h] = np.sort(np.concatenate([np.arange(n_sink), best, np.arange(ns - n_recent, ns)]))
    return keep


@pytest.mark.parametrize("values", ["spread", "equal", "few", "signs", "odd"])
@pytest.mark.parametrize("ld, n, budget, n_sink, n_recent", [(100, [100, 50, 51, 0, 200], 50, 4, 10), (1000, [1000, 999, 501, 3, -5], 500, 0, 0), (17, [17, 16, 9, 1, 2], 8, 3, 5),
                                                            (40001, [40001, 16385, 16390, 30000, 20000], 16384, 16, 1000), (50000, [50000, 33333, 2, 49999, 7], 7, 0, 2),
                                                            (2000, [2000, 1500, 1, 1001, 1000], 1000, 1000, 0), (9, [9, 9, 9, 9, 9], 1, 0, 0)])
def test_select(p1a, ld, n, budget, n_sink, n_recent, values):
    """ties go to the lowest position, NaN below everything, infinities where they belong; budgets met exactly, all sinks, all recent"""
    g = I.rng(31 + ld)
    m = np.exp(2 * I.normal(g, (5, 3, ld))).astype(np.float32)
    if values == "equal":
        m[:] = 0.25
    elif values == "few":
        m = g.integers(0, 4, m.shape).astype(np.float32)
    elif values == "signs":
        m = (I.normal(g, m.shape) * (g.random(m.shape) < 0.5)).astype(np.float32)
        m[..., ::7] = -0.0
    elif values == "odd":
        m[g.random(m.shape) < 0.2] = np.nan
        m[g.random(m.shape) < 0.1] = np.inf
        m[g.random(m.shape) < 0.1] = -np.inf
    keep = torch.full((5, 3, budget), -9, dtype=torch.int32, device="cuda")
    p1a.evict_select(dev(m), dev(np.asarray(n, np.int32)), keep, n_sink=n_sink, n_recent=n_recent)
    assert np.array_equal(keep.cpu().numpy(), keep_want(m, n, budget, n_sink, n_recent))


# ---- moving what stays ----
@pytest.mark.parametrize("kv, Hkv, D, psh, extra", [("f16", 2, 64, 4, 0), ("f16", 4, 256, 6, 0), ("f16", 3, 96, 0, 2), ("q8_0", 2, 256, 4, 0), ("q8_0", 5, 128, 3, 8), ("q8_0", 1, 64, 8, 4),
                                                    ("q4_0", 2, 256, 5, 16), ("q4_0", 3, 32, 4, 2), ("q4_0", 1, 512, 2, 0)])
def test_compact(p1a, kv, Hkv, D, psh, extra):
    """every byte: kept rows at the front in order, everything from the budget on as it was; totals moved into another tensor and in place"""
    lens = [700, 90, 1, 333, 401]
    budget, n_sink, n_recent = 200, 5, 40
    cache = Cache(p1a, KVS[kv], Hkv, D, psh, lens, 41, extra=extra, stray=0)
    ld = 720
    m = np.exp(2 * I.normal(I.rng(42), (5, Hkv, ld))).astype(np.float32)
    keep = keep_want(m, lens, budget, n_sink, n_recent)
    dm, out, place = dev(m), torch.full((5, Hkv, ld), 9.0, device="cuda"), dev(m)
    p1a.kv_compact(cache.kv, dev(keep), mass=dm, mass_out=out)
    torch.cuda.synchronize()
    for w, pool in (("k", cache.k), ("v", cache.v)):
        want = cache.host[w].copy()
        old = {s: cache.raw(w, s, n) for s, n in enumerate(lens)}
        rows = want[:, :cache.page * Hkv * cache.hb].reshape(cache.n_pages, cache.page, Hkv, cache.hb)
        for s in range(5):
            for h in range(Hkv):
                for k, j in enumerate(keep[s, h]):
                    if j > k:
                        rows[cache.table[s, k // cache.page], k % cache.page, h] = old[s][j, h]
        assert np.array_equal(pool.cpu().numpy().reshape(want.shape), want), w
    want = np.zeros_like(m)
    for s in range(5):
        for h in range(Hkv):
            live = keep[s, h] >= 0
            want[s, h, :budget][live] = m[s, h][keep[s, h][live]]
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(dm.cpu().numpy(), m)
    p1a.kv_compact(cache.kv, torch.full_like(dev(keep), -1))                     # (nothing to move: nothing moves)
    p1a.kv_compact(cache.kv, dev(keep), mass=place, mass_out=place)
    assert np.array_equal(place.cpu().numpy(), want)


def test_compact_ignores_entries_out_of_line(p1a):
    """entries below their own index, negative or past n_ctx move nothing"""
    cache = Cache(p1a, O.KV_F16, 1, 64, 4, [64], 43, stray=0)
    keep = torch.tensor([[[0, 0, 1, -1, 3, 1 << 30, 80, 2147483647, 9]]], dtype=torch.int32, device="cuda")
    assert cache.kv.n_ctx == 80
    p1a.kv_compact(cache.kv, keep)
    want = cache.raw("k", 0, 64)
    want[8] = want[9]
    assert np.array_equal(cache.raw("k", 0, 64, cache.k.cpu().numpy()), want)


# ---- together ----
@pytest.mark.parametrize("kv", list(KVS))
def test_a_session_in_a_bounded_cache(p1a, kv):
    """two sequences of a pool: prompts through attn_prep and one ragged call, the weights their last tokens give, eviction to a budget, pages given back; then
    new tokens at the next slots with their true positions as rotary ones, decoded over what was kept, their weights added. Every step against 64 bits on
    the bytes the cache then holds"""
    Hq, Hkv, D, psh, n_ctx, n_rot = 8, 2, 64, 4, 512, 32
    lens, budget, n_sink, n_recent = [300, 170], 64, 4, 16
    pool = p1a.Pool(KVS[kv], 1, Hkv, D, psh, n_ctx, 4, 2048)
    ids = [pool.seq_create() for _ in lens]
    g = I.rng(51)
    T = sum(lens)
    gate = torch.empty(T, Hq * D, device="cuda")
    q = torch.empty(T, Hq, D, device="cuda")
    first = rows_of(lens)

    def prep(a, b, cache, p0, pos, mrope=None):
        n = b - a
        qg, k, v = (dev(I.normal(g, s)) for s in ((n, Hq, 2 * D), (n, Hkv, D), (n, Hkv, D)))
        p1a.attn_prep(qg, k, v, None, None, dev(np.asarray(pos, np.int32)), q[a:b], gate[a:b], cache, p0, n, Hq, n_rot, 1e4, 1e-6, mrope=mrope)

    for s, i in enumerate(ids):
        pool.seq_advance(i, list(range(lens[s])))
        prep(first[s], first[s + 1], pool.cache_seq(0, i), 0, np.arange(lens[s]))
    pool.set_rows(ids)
    cache = pool.cache_rows(0)
    kvd = cache.struct()
    pages = 2048 >> psh
    pblk = (1 << psh) * p1a.kv_row_bytes(KVS[kv], Hkv, D)

    def heads(i, n):
        """K and V of the first n slots of a sequence as the pool holds them now: appended to f32 through an identity of the oracle's reader"""
        from _bounded import values
        torch.cuda.synchronize()
        host = np.empty(2 * n_pages(i) * pblk, np.uint8)
        buf = torch.empty(len(host), dtype=torch.uint8, pin_memory=True)
        pool.pages_out(i, 0, n_pages(i), buf.data_ptr())
        torch.cuda.synchronize()
        x = buf.numpy().reshape(n_pages(i), 2, 1 << psh, Hkv, -1)
        return [values(KVS[kv], x[:, w].reshape(-1, Hkv, x.shape[-1])[:n], D) for w in (0, 1)]

    def n_pages(i):
        return pool.seq_pages(i)

    dfirst, zero = dev(first), torch.zeros(2, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(T, Hq, D, device="cuda"), torch.empty(T, Hq, device="cuda")
    p1a.attn_chunk(q, cache, out, p1a.Rows(T, n_seq=2, row0=dfirst, pos0=zero, max_rows=300, max_n=300), Hq, 0.125, gate=gate, lse=lse)
    want = []
    for s, i in enumerate(ids):
        k, v = heads(i, lens[s])
        want.append(rows_exact(q[first[s]:first[s + 1]].cpu().numpy(), k, v, seen(np.arange(lens[s]), lens[s], 0, 0), 0.125))
        ref = gated(want[s][0], gate[first[s]:first[s + 1]].cpu().numpy())
        got = out[first[s]:first[s + 1]].cpu().numpy()
        assert np.linalg.norm(got - ref) <= REL * np.linalg.norm(ref)
    # the weights of each prompt's last 16 tokens
    mass = torch.zeros(2, Hkv, n_ctx, device="cuda")
    tail = torch.cat([torch.arange(first[s + 1] - 16, first[s + 1]) for s in range(2)]).cuda()
    p1a.attn_mass(q[tail].contiguous(), cache, lse[tail].contiguous(), mass,
                  p1a.Rows(32, n_seq=2, pos0=dev(np.array([n - 16 for n in lens], np.int32)), max_n=300), Hq, 0.125)
    total = mass.cpu().numpy()
    for s in range(2):
        ref = want[s][2][-16:].reshape(16, Hkv, -1, lens[s]).sum((0, 2))
        assert np.linalg.norm(total[s, :, :lens[s]] - ref) <= REL * np.linalg.norm(ref) and (total[s, :, lens[s]:] == 0).all()
    before = [heads(i, n) for i, n in zip(ids, lens)]
    keep = torch.empty(2, Hkv, budget, dtype=torch.int32, device="cuda")
    p1a.evict_select(mass, dev(np.array(lens, np.int32)), keep, n_sink=n_sink, n_recent=n_recent)
    p1a.kv_compact(cache, keep, mass=mass, mass_out=mass)
    kept = keep.cpu().numpy()
    assert np.array_equal(kept, keep_want(total, lens, budget, n_sink, n_recent))
    free = pool.free_pages
    for s, i in enumerate(ids):
        pool.seq_evict(i, budget)
        assert pool.seq_len(i) == budget and pool.seq_tokens(i) == [-1] * budget
        for a, b in zip(heads(i, budget), before[s]):
            assert np.array_equal(a, np.stack([b[kept[s, h], h] for h in range(Hkv)], 1))
    assert pool.free_pages == free + sum(-(-n // 16) - 4 for n in lens)
    # new tokens: slots budget, budget + 1, ...; rotary positions go on where the prompts ended
    for step in range(3):
        for i in ids:
            pool.seq_advance(i, None, 1)
        slots = dev(np.full(2, budget + step, np.int32))
        place = dev(np.array([n + step for n in lens] * 3, np.int32).reshape(3, 2))
        prep(0, 2, cache, -1, [budget + step] * 2, mrope=(place, 2, (1, 0, 0), 1))
        z = torch.empty(2, Hq, device="cuda")
        rows = p1a.Rows(2, n_seq=2, pos0=slots, max_n=budget + step + 1)
        o = torch.empty(2, Hq, D, device="cuda")
        p1a.attn_chunk(q[:2], cache, o, rows, Hq, 0.125, gate=gate[:2], lse=z)
        o2 = torch.empty_like(o)
        p1a.attn_decode_rows(q[:2], cache, o2, 2, slots, Hq, 0.125, gate=gate[:2])
        p1a.attn_mass(q[:2], cache, z, mass, rows, Hq, 0.125)
        n = budget + step + 1
        for s, i in enumerate(ids):
            k, v = heads(i, n)
            w = rows_exact(q[s:s + 1].cpu().numpy(), k, v, np.ones((1, n), bool), 0.125)
            ref = gated(w[0], gate[s:s + 1].cpu().numpy())
            assert np.linalg.norm(o[s].cpu().numpy() - ref) <= REL * np.linalg.norm(ref)
            assert np.abs(o2[s].cpu().numpy() - ref).max() <= I.MAX_ABS_TOL          # (the decode call's own tolerance)
            assert abs(float(mass[s].sum()) - (total[s].astype(np.float64)[np.arange(Hkv)[:, None], kept[s]].sum() + (step + 1) * Hq)) <= 1e-3
    assert kvd.n_ctx == n_ctx and pages
    pool.close()


def test_captured_and_replayed(p1a):
    """the step of a bounded cache in a graph - attention, weights, choice, move - replayed with other positions and queries in the same memory, eager work
    between the replays: the bits of the eager calls; a call whose partials would have to be allocated is refused under capture"""
    cache, twin = (Cache(p1a, O.KV_Q8_0, 2, 64, 4, [1500, 1200], 61) for _ in range(2))
    pos, q = torch.tensor([1499, 1199], dtype=torch.int32, device="cuda"), torch.zeros(2, 8, 64, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    rows = p1a.Rows(2, n_seq=2, pos0=pos, window=1000, n_sink=4)
    bufs = [[torch.zeros(2, 8, 64, device="cuda"), torch.zeros(2, 8, device="cuda"), torch.zeros(2, 2, 1536, device="cuda"), torch.zeros(2, 2, 128, dtype=torch.int32, device="cuda"),
             torch.zeros(2, 2, 1536, device="cuda")] for _ in range(2)]

    def step(c, b, scratch=None):
        p1a.attn_chunk(q, c.kv, b[0], rows, 8, 0.125, lse=b[1], scratch=scratch)
        p1a.attn_mass(q, c.kv, b[1], b[2], rows, 8, 0.125)
        p1a.evict_select(b[2], n, b[3], n_sink=4, n_recent=16)
        p1a.kv_compact(c.kv, b[3], mass=b[2], mass_out=b[4])

    need = p1a.chunk_scratch_bytes(cache.kv, rows, 8)
    assert need > 0
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        big = p1a.Rows(2, n_seq=2, pos0=pos)
        with torch.cuda.graph(graph, stream=s):
            step(cache, bufs[0], scratch=torch.empty(need, dtype=torch.uint8, device="cuda"))
            with pytest.raises(p1a.P1AError, match="capture"):
                p1a.attn_chunk(q, cache.kv, bufs[0][0], big, 8, 0.125)
    for i in range(4):
        q.normal_()
        pos.copy_(torch.tensor([1499 - 50 * i, 1199 - 7 * i]))
        n.copy_(pos + 1)
        for x in (0, 1):
            bufs[x][2].fill_(0.001 * i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(twin, bufs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*bufs)), i
        assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)


def test_two_streams(p1a):
    """calls on two streams at once, each with partials of its own"""
    caches = [Cache(p1a, O.KV_F16, 1, 64, 4, [6000], 71 + i) for i in range(2)]
    calls = [Call(p1a, c, 4, [2], [5998]) for c in caches]
    want = [c.chunk(p1a) for c in calls]
    outs = [torch.empty(2, 4, 64, device="cuda") for _ in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        for c, o, s in zip(calls, outs, streams):
            with torch.cuda.stream(s):
                p1a.attn_chunk(c.q, c.cache.kv, o, c.rows, 4, c.scale)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o.cpu().numpy().astype(np.float64), w[0])
