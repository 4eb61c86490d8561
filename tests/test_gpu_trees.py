"""Drafted trees on the GPU: masks from parents, attention of the nodes' rows, verification, the accepted path's move - each against its formula in 64 bits -
and steps that run through all of them.

How far attention may be off is what tests/test_gpu_bounded.py derives: with f32 results 1e-5 in the 2-norm (halves of 2^-22, fp32 sums); with bf16 results one
rounding of the result, 2^-8 of it, and q, P, K and V rounded to f16 once, 2^-11 each. Verification's sums are of 64 bits: its whole numbers are equal."""
import numpy as np
import pytest
import torch

import _inputs as I
import _oracle as O
import _trees as R
from _bounded import Cache, bf16, gated, rows_exact
from _gpu import dev

pytestmark = pytest.mark.gpu

KVS = {"f16": O.KV_F16, "q8_0": O.KV_Q8_0, "q4_0": O.KV_Q4_0}
REL = 1e-5


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


class Call:
    """One call's inputs and, sequence by sequence, what it is to give. see: per sequence [nodes][nodes] (None: of random trees)"""

    def __init__(self, p1a, cache, Hq, counts, pos0, window=0, n_sink=0, q_bf16=False, gate=False, seed=1, spare=0, max_n=0, see=None, junk=False, scale=None, row0=True, words=None):
        g = I.rng(seed)
        T, D = int(sum(counts)), cache.D
        self.cache, self.Hq, self.T, self.scale = cache, Hq, T, D ** -0.5 if scale is None else scale
        q = I.normal(g, (T + spare, Hq, D))
        q /= np.sqrt((q * q).mean(-1, keepdims=True))
        self.q, self.q64 = bf16(q) if q_bf16 else (dev(q), q.astype(np.float64))
        self.gate = I.normal(g, (T + spare, Hq * D)) if gate else None
        self.dgate = dev(self.gate) if gate else None
        self.see = [R.paths(R.tree(g, n))[0] for n in counts] if see is None else see
        most = max(max(counts), 1)
        words = words or (most + 31) // 32
        mask = np.zeros((T + spare, words), np.int32)
        first = starts(counts)
        for s, m in enumerate(self.see):
            mask[first[s]:first[s + 1]] = R.words_of(m, words)
            if junk:                                           # (bits of nodes that the sequence does not have)
                all_bits = R.words_of(np.ones((1, 32 * words), bool), words) & ~R.words_of(np.ones((1, counts[s]), bool), words)
                mask[first[s]:first[s + 1]] |= all_bits
        self.mask, self.first, self.counts, self.pos0 = dev(mask), first, list(counts), list(pos0)
        self.row0, self.dpos = dev(first) if row0 else None, dev(np.asarray(pos0, np.int32))
        self.rows = p1a.Rows(T + spare, n_seq=len(counts), row0=self.row0, pos0=self.dpos, max_rows=most, max_n=max_n, window=window, n_sink=n_sink)
        self.want = []
        for s, (m, p0) in enumerate(zip(self.see, pos0)):
            sees = R.sees(m, p0, cache.kv.n_ctx, window, n_sink)
            n = sees.shape[1]
            self.want.append(rows_exact(self.q64[first[s]:first[s + 1]], cache.heads("k", s, n), cache.heads("v", s, n), sees, self.scale))

    def all(self, i):
        return np.concatenate([w[i] for w in self.want])

    def run(self, p1a, out_bf16=False, lse=True, scratch=None):
        out = torch.full((self.q.shape[0], self.Hq, self.cache.D), 77.0, dtype=torch.bfloat16 if out_bf16 else torch.float32, device="cuda")
        z = torch.full((self.q.shape[0], self.Hq), 77.0, device="cuda") if lse else None
        p1a.attn_tree(self.q, self.cache.kv, out, self.rows, self.mask, self.Hq, self.scale, gate=self.dgate, lse=z, scratch=scratch)
        torch.cuda.synchronize()
        assert (out[self.T:] == 77).all() and (z is None or (z[self.T:] == 77).all()), "rows of no sequence were written"
        return out[:self.T].float().cpu().numpy().astype(np.float64), None if z is None else z[:self.T].cpu().numpy().astype(np.float64)

    def check(self, p1a, out_bf16=False, lse=True):
        got, z = self.run(p1a, out_bf16, lse)
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
            assert (np.abs(z - np.where(live, ref, 0))[live] <= (REL * qk + 2.0 ** -22 * (np.abs(np.where(live, ref, 0)) + 16))[live]).all()
        return got


# ---- masks and positions ----
@pytest.mark.parametrize("counts", [[1], [8], [0, 5, 0, 33, 1], [32, 64, 31, 65], [1024, 3], [300, 0, 1000]])
def test_rows_from_parents(p1a, counts):
    g = I.rng(sum(counts))
    parents = [R.tree(g, n, 4) for n in counts]
    if len(counts) > 2:                                        # parents that are none: a node without one
        parents[1] = [7, 0, 5, -3, 3][:counts[1]] + parents[1][5:]
    if 1024 in counts:                                         # a chain of all nodes
        parents[0] = list(range(-1, 1023))
    T, words = sum(counts), (max(counts) + 31) // 32 + 1 if max(counts) < 1000 else 32
    pos0 = np.array([100 * s + 7 for s in range(len(counts))], np.int32)
    spare = 2
    rows = p1a.Rows(T + spare, n_seq=len(counts), row0=dev(starts(counts)), pos0=dev(pos0), max_rows=max(counts))
    parent = dev(np.array(sum(parents, []) + [0] * spare, np.int32))
    mask, pos, slot = (torch.full((T + spare, k), 77, dtype=torch.int32, device="cuda") for k in (words, 1, 1))
    p1a.tree_rows(parent, rows, mask, pos=pos, slot=slot)
    again = torch.full_like(mask, 77)
    p1a.tree_rows(parent, rows, again)
    want = [R.paths(p) for p in parents]
    m = np.concatenate([R.words_of(see, words) for see, _ in want])
    assert np.array_equal(mask[:T].cpu().numpy(), m) and torch.equal(mask, again)
    assert np.array_equal(pos[:T, 0].cpu().numpy(), np.concatenate([p + d for p, (_, d) in zip(pos0, want)]))
    assert np.array_equal(slot[:T, 0].cpu().numpy(), np.concatenate([p + np.arange(n) for p, n in zip(pos0, counts)]))
    assert (mask[T:] == 77).all() and (pos[T:] == 77).all() and (slot[T:] == 77).all()


# ---- attention ----
SHAPES = [(4, 1, 64), (12, 2, 256), (32, 8, 128), (8, 8, 64), (5, 5, 128), (16, 1, 64), (40, 1, 128), (64, 1, 64), (24, 4, 256)]


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv", list(KVS))
def test_ragged_trees(p1a, kv, D, out_bf16):
    """sequences of no nodes, of one and of more than a hundred - one group of blocks of columns and several -, whole contexts and windows, gates; rows behind the last sequence"""
    lens, counts = [730, 1, 611, 64, 300, 40], [70, 0, 133, 1, 33, 40]
    cache = Cache(p1a, KVS[kv], 2, D, 4, lens, 5)
    for window, n_sink in ((0, 0), (100, 0), (64, 5), (1, 0), (37, 70), (5000, 4)):
        Call(p1a, cache, 12, counts, [n - c for n, c in zip(lens, counts)], window, n_sink, gate=window == 64, spare=3).check(p1a, out_bf16, lse=not out_bf16)


@pytest.mark.parametrize("Hq, Hkv, D", SHAPES)
@pytest.mark.parametrize("kv", list(KVS))
def test_small_trees(p1a, kv, Hq, Hkv, D):
    """one node and a few, from the first position on; bf16 in, f32 out and the other way round"""
    lens, counts = [1, 9, 17, 64, 65, 500, 1500], [1, 9, 3, 8, 2, 11, 5]
    cache = Cache(p1a, KVS[kv], Hkv, D, 5, lens, 6)
    for window, n_sink in ((0, 0), (128, 4), (3, 1)):
        call = Call(p1a, cache, Hq, counts, [n - c for n, c in zip(lens, counts)], window, n_sink, q_bf16=window == 3)
        call.check(p1a)
        call.check(p1a, out_bf16=True, lse=False)


@pytest.mark.parametrize("count", [1, 2, 3, 4, 5, 6, 8, 10, 11, 12, 13, 16, 17, 22, 32, 43])
def test_every_number_of_blocks(p1a, count):
    """one tile of columns and two, one to four blocks of a group, two groups and three, streams of keys shared by one, two and four waves"""
    for kv, D, Hq in (("q8_0", 256, 6), ("f16", 64, 8), ("q4_0", 128, 3)):
        cache = Cache(p1a, KVS[kv], 1, D, 4, [300 + count, 40 + count], 60 + count)
        call = Call(p1a, cache, Hq, [count, count], [300, 40], row0=False)
        call.check(p1a)
        call.check(p1a, out_bf16=True, lse=False)


@pytest.mark.parametrize("psh, extra", [(0, 0), (1, 16), (2, 0), (3, 48), (6, 0), (8, 16)])
def test_pages(p1a, psh, extra):
    """pages of one position and more, trees that lie across pages and tiles, page strides of more than the page"""
    lens, counts = [333, 70], [45, 70]
    for kv in KVS:
        cache = Cache(p1a, KVS[kv], 2, 128, psh, lens, 7, extra=extra)
        Call(p1a, cache, 6, counts, [n - c for n, c in zip(lens, counts)], 50, 9).check(p1a)


def test_every_place_of_a_tree_in_a_tile(p1a):
    for kv in KVS:
        cache = Cache(p1a, KVS[kv], 1, 64, 4, [200], 71)
        for p0 in list(range(60, 100, 3)) + [0, 1, 31, 32, 33]:
            Call(p1a, cache, 4, [37], [p0], seed=p0 + 1).check(p1a)


def test_contiguous_and_host_position(p1a):
    """a cache without pages; the position of the only sequence from the host"""
    for kv in KVS:
        cache = Cache(p1a, KVS[kv], 4, 64, 4, [400], 8, paged=False)
        call = Call(p1a, cache, 8, [20], [380])
        want = call.check(p1a)
        rows = p1a.Rows(20, p0=380)
        out = torch.empty(20, 8, 64, device="cuda")
        p1a.attn_tree(call.q, cache.kv, out, rows, call.mask, 8, call.scale)
        assert np.linalg.norm(out.cpu().numpy() - want) <= 2 * REL * np.linalg.norm(want)


@pytest.mark.parametrize("kv", list(KVS))
def test_any_mask(p1a, kv):
    """masks that are no trees: rows that see all nodes, those behind them, none of the tree, nothing at all; bits of nodes that are not there"""
    g = I.rng(9)
    counts = [40, 7, 64]
    see = [g.random((n, n)) < 0.3 for n in counts]
    see[0][3] = True
    see[0][4] = False
    see[1][:] = False
    see[2][5:9] = False
    for D, out_bf16 in ((64, False), (128, True), (256, False)):
        cache = Cache(p1a, KVS[kv], 2, D, 4, [240, 7, 64], 10)
        call = Call(p1a, cache, 8, counts, [200, 0, 0], see=see, junk=True, words=4)
        got = call.check(p1a, out_bf16, lse=not out_bf16)
        assert (got[40:47] == 0).all() and (got[47 + 5:47 + 9] == 0).all()
        Call(p1a, cache, 8, counts, [200, 0, 0], 20, 3, see=see, junk=True, words=2).check(p1a, out_bf16, lse=not out_bf16)


def test_slots_that_are_none(p1a):
    """nodes in front of position 0 and behind the cache's last see nothing, and are not seen"""
    cache = Cache(p1a, O.KV_F16, 2, 64, 4, [64, 64], 11, max_pages=4)
    Call(p1a, cache, 4, [20, 20], [50, -7], gate=True).check(p1a)
    Call(p1a, cache, 4, [20, 20], [64, -20]).check(p1a)
    Call(p1a, cache, 4, [20, 20], [63, -19], 5, 2).check(p1a)


def test_what_is_not_a_number_stays_where_it_is(p1a):
    """NaN in K and V of positions that no row sees, and in the K of nodes that a row does not see; in a row of q: that row's result alone"""
    cache = Cache(p1a, O.KV_F16, 1, 64, 4, [200], 12)
    see, _ = R.paths([-1, 0, 0, 1, 2, 2])
    clean = Call(p1a, cache, 4, [6], [150], 32, 2, see=[see])
    want = clean.check(p1a)
    for w in "kv":
        raw = cache.host[w].reshape(cache.n_pages, 16, 64 * 2)
        for j in [*range(2, 119), *range(156, 200)]:           # out of the window, behind the tree
            raw[cache.table[0][j // 16], j % 16].view(np.float16)[:] = np.nan
    k = cache.host["k"].reshape(cache.n_pages, 16, 128)
    k[cache.table[0][155 // 16], 155 % 16].view(np.float16)[:] = np.nan      # node 5: only its own row sees it
    cache.upload()
    cache.kv.k, cache.kv.v = cache.k.data_ptr(), cache.v.data_ptr()
    got, z = clean.run(p1a)
    assert np.array_equal(got[:5], want[:5]) and np.isnan(got[5]).all() and np.isnan(z[5]).all()
    q = clean.q.clone()
    q[2, 1, 7], q[3, 0, 0] = float("nan"), float("inf")
    clean.q = q
    got, z = clean.run(p1a)
    bad = np.zeros((5, 4), bool)
    bad[2, 1] = bad[3, 0] = True
    assert np.isnan(got[:5][bad]).all() and np.isnan(z[:5][bad]).all() and np.array_equal(got[:5][~bad], want[:5][~bad])


@pytest.mark.parametrize("kv", list(KVS))
def test_a_chain_is_a_chunk(p1a, kv):
    """the tree without branches gives what attn_chunk gives for the same rows"""
    lens, counts = [900, 77], [23, 9]
    cache = Cache(p1a, KVS[kv], 2, 128, 4, lens, 13)
    see = [np.tril(np.ones((n, n), bool)) for n in counts]
    for window, n_sink in ((0, 0), (40, 3), (5, 0)):
        # (a window inside the tree is the mask's business: wide enough here, or the chain's last `window` nodes)
        seen = [m & ~np.tril(np.ones_like(m), -window) if window else m for m in see]
        if window and window < max(counts):
            continue
        call = Call(p1a, cache, 8, counts, [n - c for n, c in zip(lens, counts)], window, n_sink, see=seen)
        got = call.check(p1a)
        out = torch.empty(call.T, 8, 128, device="cuda")
        p1a.attn_chunk(call.q, cache.kv, out, call.rows, 8, call.scale)
        assert np.linalg.norm(out.cpu().numpy() - got) <= 2 * REL * np.linalg.norm(got)


def test_scales_and_their_signs(p1a):
    cache = Cache(p1a, O.KV_Q8_0, 1, 128, 4, [300], 14)
    for scale in (-0.1, 0.0, 1.0):
        Call(p1a, cache, 4, [9], [291], scale=scale).check(p1a)


def test_scratch_streams_and_repeats(p1a):
    """the caller's scratch, another stream and a second run give the same bits; too little scratch is not used"""
    cache = Cache(p1a, O.KV_Q8_0, 4, 256, 8, [9000, 500], 15)
    call = Call(p1a, cache, 24, [16, 9], [8984, 491], gate=True, max_n=9000)
    first, z = call.run(p1a)
    need = p1a.tree_scratch_bytes(cache.kv, call.rows, 24)
    assert need > 0
    room = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    for scratch in (room, room[:need - 1], None):
        again, z2 = call.run(p1a, scratch=scratch)
        assert np.array_equal(first, again) and np.array_equal(z, z2)
    assert (room[need:] == 255).all()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again, z2 = call.run(p1a)
    assert np.array_equal(first, again) and np.array_equal(z, z2)


def test_long_contexts(p1a):
    """32768 positions and more, split among many workgroups; a sequence of a few beside it"""
    cache = Cache(p1a, O.KV_Q4_0, 2, 64, 8, [40000, 33], 16)
    for out_bf16 in (False, True):
        Call(p1a, cache, 8, [48, 12], [39952, 21]).check(p1a, out_bf16, lse=not out_bf16)
        Call(p1a, cache, 8, [3, 1], [39997, 32]).check(p1a, out_bf16, lse=not out_bf16)


def test_the_largest_tree(p1a):
    cache = Cache(p1a, O.KV_F16, 1, 64, 6, [1500], 17)
    Call(p1a, cache, 3, [1024], [476]).check(p1a)


def test_more_sequences_than_lanes(p1a):
    counts = [(s * 7) % 5 for s in range(150)]
    lens = [40 + (s * 13) % 90 for s in range(150)]
    cache = Cache(p1a, O.KV_F16, 1, 64, 3, lens, 18)
    Call(p1a, cache, 4, counts, [n - c for n, c in zip(lens, counts)]).check(p1a)


def test_wide_page_strides(p1a):
    """rows more than 2^32 bytes behind the cache's base"""
    page, D, n = 16, 64, 40
    stride = 3 << 30
    pool = torch.zeros((stride * 2 + page * D * 2) // 2, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    order = [2, 0, 1]
    k = torch.randn(48, D, generator=g, device="cuda").half()
    for i, pg in enumerate(order):
        pool[pg * stride // 2: pg * stride // 2 + page * D] = k[16 * i:16 * i + 16].flatten()
    pt = torch.tensor(order, dtype=torch.int32, device="cuda")
    kv = p1a.KVCache(1, 48, 1, D, pool.data_ptr(), pool.data_ptr(), pt=pt, psh=4, pstride=stride)
    see, _ = R.paths([-1, 0, 0, 1])
    q = torch.randn(4, 2, D, generator=g, device="cuda")
    out = torch.empty_like(q)
    p1a.attn_tree(q, kv, out, p1a.Rows(4, p0=n - 4), dev(R.words_of(see, 1)), 2, 0.125)
    x = k[:n, None].double().cpu().numpy()
    want = rows_exact(q.double().cpu().numpy(), x, x, R.sees(see, n - 4, 48, 0, 0), 0.125)[0]
    assert np.linalg.norm(out.cpu().numpy() - want) <= REL * np.linalg.norm(want)


# ---- verification ----
class Batch:
    """Sequences to verify: logits (or probabilities), the draft's probabilities, tokens drawn from them, random numbers"""

    def __init__(self, seed, counts, V, branch=3, draft="iid", logits=True, dtype=torch.float32, draft_dtype=torch.float32, spread=2.0, noise=0.7, temps=True, pad=0, shift=0, parents=None, chains=False):
        g = self.g = np.random.default_rng(seed)
        self.counts, self.V, self.branch, self.how, self.logits, self.first = list(counts), V, branch, draft, logits, starts(counts)
        T = self.T = int(sum(counts))
        self.parents = parents or [list(range(-1, n - 1)) if chains else R.tree(g, n, branch) for n in counts]
        self.chains = chains
        l = (g.normal(size=(T, V)) * spread).astype(np.float32)
        self.temp = np.where(g.random(len(counts)) < 0.25, 0, 0.5 + g.random(len(counts))).astype(np.float32) if temps and logits else None
        q = R.softmax(l.astype(np.float64) + noise * g.normal(size=(T, V)))
        q = q.astype(np.float32) if draft_dtype == torch.float32 else R.bf16_values(q)
        p = l if logits else R.softmax(l.astype(np.float64)).astype(np.float32)
        self.target = p if dtype == torch.float32 else R.bf16_values(p)
        self.draft = None if draft == "none" else q
        self.token = np.zeros(T, np.int32)
        for s, parent in enumerate(self.parents):
            kid = {}
            for i, r in enumerate(parent):
                if r < 0:
                    continue
                w = q[self.first[s] + r].astype(np.float64)
                if r not in kid:
                    k = min(branch, V)
                    enough = np.count_nonzero(w) >= k
                    kid[r] = list(g.choice(V, k, replace=draft == "iid" or not enough, p=w / w.sum()))
                self.token[self.first[s] + i] = kid[r].pop(0) if kid[r] else 0
        self.u, self.u_next = g.random(T).astype(np.float32), g.random(len(counts)).astype(np.float32)
        self.dtype, self.draft_dtype, self.pad, self.shift = dtype, draft_dtype, pad, shift

    def rows_on_gpu(self, x, dtype):
        """rows `pad` numbers further apart than they are long, `shift` numbers behind an aligned place"""
        t = torch.full((self.T * (self.V + self.pad) + self.shift,), float("nan"), dtype=dtype, device="cuda")
        v = t[self.shift:].view(self.T, self.V + self.pad)[:, :self.V]
        v.copy_(torch.from_numpy(x))
        return v

    def expect(self, width, kids=None):
        n, path, nxt = [], np.full((len(self.counts), width), -1, np.int32), []
        for s, c in enumerate(self.counts):
            a, b = self.first[s], self.first[s + 1]
            p, x = R.verify(self.target[a:b].reshape(c, self.V), self.token[a:b], self.parents[s], self.u[a:b], self.u_next[s], None if self.draft is None else self.draft[a:b],
                            1.0 if self.temp is None else self.temp[s], self.logits, kids or self.branch, self.how == "distinct")
            n.append(len(p))
            path[s, :min(len(p), width)] = p[:width]
            nxt.append(x)
        return np.array(n), path, np.array(nxt)

    def call(self, p1a, width=None, kids=None, scratch=None, spare=0):
        S = len(self.counts)
        width = width or max(max(self.counts), 1)
        self.dt, self.dd = self.rows_on_gpu(self.target, self.dtype), None if self.draft is None else self.rows_on_gpu(self.draft, self.draft_dtype)
        self.rows = p1a.Rows(self.T, n_seq=S, row0=dev(self.first), max_rows=max(self.counts))
        n, nxt = (torch.full((S + spare,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        path = torch.full((S + spare, width), 77, dtype=torch.int32, device="cuda")
        self.kept = [dev(x) for x in (self.token, self.u, self.u_next, np.array(sum(self.parents, []), np.int32))]
        token, u, u_next, parent = self.kept
        p1a.tree_verify(self.dt, token, self.rows, u, u_next, n, path, nxt, parent=None if self.chains else parent, draft=self.dd, temp=None if self.temp is None else dev(self.temp),
                        logits=self.logits, max_children=kids or self.branch, distinct=self.how == "distinct", scratch=scratch)
        torch.cuda.synchronize()
        assert (n[S:] == 77).all() and (nxt[S:] == 77).all() and (path[S:] == 77).all()
        return n[:S].cpu().numpy(), path[:S].cpu().numpy(), nxt[:S].cpu().numpy()

    def check(self, p1a, width=None, kids=None, **more):
        got, want = self.call(p1a, width, kids, **more), self.expect(width or max(max(self.counts), 1), kids)
        for name, a, b in zip(("n_accept", "path", "next"), got, want):
            assert np.array_equal(a, b), (name, a, b)
        return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("draft", ["none", "iid", "distinct"])
def test_verify(p1a, draft, logits, dtype):
    """vocabularies of one token to several stretches of 4096, trees of no node to a hundred, chains; strides and starts off their alignment"""
    for i, (V, counts) in enumerate([(1, [3, 1]), (2, [9, 4, 0]), (7, [20, 0, 1, 33]), (100, [40, 100]), (4095, [6, 12]), (4096, [9]), (4097, [5, 7, 3]), (20011, [12, 1, 30])]):
        Batch(10 * i, counts, V, draft=draft, logits=logits, dtype=dtype, pad=i % 3, shift=i % 4).check(p1a)
        Batch(10 * i + 1, counts, V, 1, draft=draft, logits=logits, dtype=dtype, chains=True, draft_dtype=torch.bfloat16 if i % 2 else torch.float32).check(p1a, spare=2)
        Batch(10 * i + 2, counts, V, 5, draft=draft, logits=logits, dtype=dtype, noise=0.05, spread=6.0).check(p1a)


@pytest.mark.parametrize("draft", ["none", "iid", "distinct"])
def test_verify_many_draws(p1a, draft):
    """hundreds of small trees at once: every kind of outcome, by the number"""
    b = Batch(77, [1 + s % 9 for s in range(400)], 50, 4, draft=draft, noise=1.0)
    n, _, _ = b.check(p1a)
    assert n.min() == 0 and n.max() >= 3


def test_verify_wide_and_deep(p1a):
    Batch(5, [1024], 33, 1, draft="iid", chains=True, noise=0.0).check(p1a)                 # (p = q but for a rounding: long paths)
    Batch(6, [1024, 2], 33, 1023, draft="none", parents=[[-1] + [0] * 1023, [-1, 0]], noise=3.0).check(p1a)
    Batch(7, [65, 65], 500, 64, draft="distinct", parents=[[-1] + [0] * 64, [-1] + [0] * 64], noise=3.0).check(p1a)
    Batch(8, [12], 160001, 4, draft="iid", dtype=torch.bfloat16).check(p1a)


def test_verify_cuts(p1a):
    """fewer children than there are, paths that do not fit"""
    b = Batch(21, [30, 41, 8, 1], 60, 4, noise=1.5)
    for kids in (1, 2, 3, 4, 9):
        b.check(p1a, kids=kids)
    b = Batch(22, [20] * 30, 40, 2, noise=0.1)
    n, _, _ = b.check(p1a, width=2)
    assert n.max() > 2


def test_verify_rows_without_weight(p1a):
    """NaN, infinite and missing logits; probabilities that are none; tokens out of the vocabulary; the same token twice; u of 0 and next to 1"""
    inf, nan = np.inf, np.nan
    for draft in ("none", "iid"):
        b = Batch(31, [4] * 12, 6, 3, draft=draft, parents=[[-1, 0, 0, 0]] * 12)
        b.target[0] = -inf
        b.target[4] = nan
        b.target[8, :3] = nan
        b.target[12, 2] = inf
        b.target[16, [1, 4]] = inf
        b.target[20, 1:] = -inf
        b.target[24] = 3.0
        b.token[[29, 33]] = -1, 6
        b.token[37:40] = 2
        b.u[:] = np.where(np.arange(48) % 4 == 1, 0, b.u)
        b.u_next[::3], b.u_next[1::3] = 0, np.float32(1 - 2.0 ** -24)
        got = b.check(p1a)
        assert got[2][0] == -1 and got[2][1] == -1 and got[0][0] == 0
        b.temp = np.zeros(12, np.float32)
        b.check(p1a)
        b.temp = np.array([nan, -1, inf] * 4, np.float32)
        b.target[:16] = 1.0                                    # (infinite temperature over infinite logits is no one's)
        b.check(p1a)
        b = Batch(32, [4] * 6, 6, 3, draft=draft, logits=False, parents=[[-1, 0, 0, 0]] * 6)
        b.target[0], b.target[4, :3], b.target[8, 1:], b.target[12] = 0, -0.5, 0, nan
        assert b.check(p1a)[2][0] == -1


def test_verify_what_was_drafted_from_the_target_stands(p1a):
    """p = q exactly: everything is accepted; and nothing of what the target cannot give"""
    b = Batch(41, [6] * 8, 4, 1, logits=False, chains=True)
    b.target[:] = [0.5, 0.25, 0.125, 0.125]
    b.draft[:] = b.target
    b.token[:] = np.arange(48) % 4
    n, path, nxt = b.check(p1a)
    assert (n == 5).all()
    b.target[:] = [0, 0.5, 0.25, 0.25]
    b.token[:], b.u[:] = 0, 0
    assert (b.check(p1a)[0] == 0).all()


def test_verify_greedy_is_verify_accept(p1a):
    """temperature 0 over chains: the engine's bookkeeping of greedily verified drafts"""
    for draft in ("none", "iid"):
        b = Batch(51, [5] * 40, 7, 1, draft=draft, chains=True, noise=0.3)
        b.temp = np.zeros(40, np.float32)
        n, path, nxt = b.check(p1a)
        for s in range(40):
            greedy = b.target[5 * s:5 * s + 5].argmax(-1)
            q, accepted, token = p1a.verify_accept([int(x) for x in b.token[5 * s:5 * s + 5]], [int(x) for x in greedy], 1 << 20)
            assert (accepted, token) == (n[s], nxt[s]) and q == n[s] + 1
            assert list(path[s][:n[s]]) == list(range(1, n[s] + 1))


def test_verify_scratch_and_repeats(p1a):
    b = Batch(61, [9, 14, 3], 9001, 3)
    want = b.check(p1a)
    need = p1a.verify_scratch_bytes(b.rows, b.V)
    room = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    for scratch in (room, room[:need - 1], None):
        for a, c in zip(want, b.call(p1a, scratch=scratch)):
            assert np.array_equal(a, c)
    assert (room[need:] == 255).all()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for a, c in zip(want, b.call(p1a)):
            assert np.array_equal(a, c)


def test_verify_sequences_that_share_rows(p1a):
    """row0 that does not ascend: two sequences hold some of the same rows - nobody's results, but numbers of nodes and tokens that there are, and an end"""
    for seed in range(6):
        b = Batch(70 + seed, [12, 12, 12, 12], 9000, 4, draft="distinct", noise=2.0)
        rows = p1a.Rows(48, n_seq=5, row0=dev(np.array([0, 24, 12, 40, 30, 48], np.int32)), max_rows=48)
        held = [24, 0, 28, 0, 18]
        n, nxt = (torch.full((5,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        path = torch.full((5, 48), 77, dtype=torch.int32, device="cuda")
        p1a.tree_verify(b.rows_on_gpu(b.target, torch.float32), dev(b.token), rows, dev(b.u), dev(np.resize(b.u_next, 5)), n, path, nxt, parent=dev(np.array(sum(b.parents, []), np.int32)),
                        draft=b.rows_on_gpu(b.draft, torch.float32), max_children=4, distinct=True)
        torch.cuda.synchronize()
        for s, count in enumerate(held):
            k = int(n[s])
            got = path[s].tolist()
            assert 0 <= k < max(count, 1) and got[k:] == [-1] * (48 - k) and all(0 < i < count for i in got[:k]) and got[:k] == sorted(set(got[:k]))
            assert 0 <= int(nxt[s]) < 9000 if count else int(nxt[s]) == -1


@pytest.mark.parametrize("how", ["none", "iid", "distinct"])
def test_verify_keeps_the_target_s_distribution(p1a, how):
    """the first token behind node 0 has the target's distribution, whatever was drafted: 40000 trees of three children"""
    g = np.random.default_rng(5)
    V, N = 6, 40000
    p, q = R.softmax(g.normal(size=V) * 1.5), R.softmax(g.normal(size=V) * 1.5)
    gen = torch.Generator(device="cuda").manual_seed(3)
    dq = torch.tensor(q, dtype=torch.float32, device="cuda")
    kids = torch.multinomial(dq.expand(N, V), 3, replacement=how == "iid", generator=gen).int()
    if how == "none":
        kids = torch.argsort(-dq)[:3].int().expand(N, 3)
    token = torch.cat([torch.zeros(N, 1, dtype=torch.int32, device="cuda"), kids], 1).contiguous()
    parent = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda").repeat(N)
    target = torch.tensor(np.log(p), dtype=torch.float32, device="cuda").expand(4 * N, V).contiguous()
    n, nxt, path = (torch.empty(N, w, dtype=torch.int32, device="cuda") for w in (1, 1, 3))
    p1a.tree_verify(target, token.flatten(), p1a.Rows(4 * N, n_seq=N), torch.rand(4 * N, generator=gen, device="cuda"), torch.rand(N, generator=gen, device="cuda"), n, path, nxt, parent=parent,
                    draft=None if how == "none" else dq.expand(4 * N, V).contiguous(), max_children=3, distinct=how == "distinct")
    first = torch.where(n[:, 0] > 0, token.gather(1, path[:, :1].long().clamp_min(0))[:, 0], nxt[:, 0])
    seen = torch.bincount(first.long(), minlength=V).double().cpu().numpy() / N
    assert (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / N)).all(), (seen, p)


# ---- the accepted path ----
def moved(cache, raw, s, p0, path, n_ctx, count):
    """bytes of sequence s after its path has moved: [positions][Hkv][head bytes]"""
    for k, node in enumerate(path):
        if node > k + 1 and node < count and p0 + 1 + k >= 0 and p0 + node < n_ctx:
            raw[p0 + 1 + k] = raw[p0 + node]
    return raw


@pytest.mark.parametrize("psh, extra", [(0, 2), (2, 0), (4, 2), (6, 48), (8, 0)])
@pytest.mark.parametrize("kv", list(KVS))
def test_commit(p1a, kv, psh, extra):
    """three layers at once, sequences that accepted nothing, all of a chain, nodes far apart; entries that are none"""
    counts, lens, g = [40, 5, 9, 1, 70, 0], [300, 21, 9, 50, 111, 30], I.rng(3)
    layers = [Cache(p1a, KVS[kv], 2, 64, psh, lens, 20 + i, extra=extra) for i in range(3)]
    for c in layers[1:]:                                       # (one page table for all layers)
        c.table = layers[0].table
        c.kv.pt, c.kv.rtab = layers[0].kv.pt, layers[0].kv.rtab
    paths = [[2, 5, 9, 17, 38], [1, 2, 3, 4], [3, 2, 9, 8, 77], [], sorted(g.choice(np.arange(1, 70), 66, replace=False).tolist()), [3]]
    width = 66
    path = np.full((6, width), -1, np.int32)
    for s, p in enumerate(paths):
        path[s, :len(p)] = p
    n = np.array([5, 4, 5, -3, 99, 1], np.int32)
    pos0 = [a - b for a, b in zip(lens, counts)]
    rows = p1a.Rows(sum(counts), n_seq=6, row0=dev(starts(counts)), pos0=dev(np.array(pos0, np.int32)), max_rows=70)
    p1a.tree_commit(p1a.Layers([c.kv for c in layers]), rows, dev(n), dev(path))
    torch.cuda.synchronize()
    for c in layers:
        for w, t in (("k", c.k), ("v", c.v)):
            got = t.cpu().numpy()
            want = c.host[w].copy()
            view = want[:, :c.page * c.Hkv * c.hb].reshape(c.n_pages, c.page, c.Hkv, c.hb)
            for s in range(6):
                raw = moved(c, c.raw(w, s, lens[s]), s, pos0[s], paths[s][:max(int(n[s]), 0)], c.kv.n_ctx, counts[s])
                for j in range(lens[s]):
                    view[c.table[s][j // c.page], j % c.page] = raw[j]
            assert np.array_equal(got.reshape(want.shape), want)


def test_commit_contiguous_and_edges(p1a):
    """a cache without pages, a position from the host; slots in front of the cache and behind it move nothing"""
    for p0 in (-4, 0, 90, 97):
        c = Cache(p1a, O.KV_Q4_0, 3, 64, 0, [100], 30, paged=False)
        c.kv.n_ctx = 100
        rows = p1a.Rows(8, p0=p0)
        path = [3, 4, 6, 7]
        p1a.tree_commit([c.kv], rows, dev(np.array([4], np.int32)), dev(np.array([path], np.int32)))
        got = c.k.cpu().numpy().reshape(c.n_pages, -1)
        want = c.host["k"].copy()
        raw = c.raw("k", 0, 100)
        for k, node in enumerate(path):
            if p0 + 1 + k >= 0 and p0 + node < 100:
                raw[p0 + 1 + k] = raw[p0 + node]
        want.reshape(-1)[:raw.size] = raw.reshape(-1)
        assert np.array_equal(got, want), p0


# ---- steps that run through all of it ----
@pytest.mark.parametrize("kv", list(KVS))
def test_a_session_in_trees(p1a, kv):
    """Two sequences drafted in trees, three steps, two layers: masks and positions, prep into the nodes' slots, attention, verification, the move. In the end the caches hold the
    bytes, and attention gives the results, of the accepted tokens run one after the other."""
    Hq, Hkv, D, V, psh, n_rot = 4, 2, 64, 50, 4, 32
    g = I.rng(41)
    lens, page, max_pages = [37, 5], 16, 8
    table = dev(g.permutation(16).astype(np.int32))
    offsets = dev(np.array([0, max_pages], np.int32))
    rowb = p1a.kv_row_bytes(KVS[kv], Hkv, D)

    def caches():
        mem = [torch.zeros(16 * page * rowb, dtype=torch.uint8, device="cuda") for _ in range(4)]
        return mem, [p1a.KVCache(KVS[kv], max_pages * page, Hkv, D, mem[2 * i].data_ptr(), mem[2 * i + 1].data_ptr(), pt=table, rtab=offsets, psh=psh, pstride=page * rowb) for i in range(2)]
    embed = dev(I.normal(g, (V, 2, (2 * Hq + 2 * Hkv) * D)))    # of a token: q and gate, k, v of both layers
    head = dev(I.normal(g, (Hq * D, V)))
    qn, kn = (dev(1 + 0.1 * I.normal(g, (D,))) for _ in range(2))

    def prep(layer, c, token, pos, slot, of_row):
        x = embed[token.long(), layer]
        qg, k, v = (t.contiguous() for t in x.split([2 * Hq * D, Hkv * D, Hkv * D], 1))
        T = len(token)
        q, gate = torch.empty(T, Hq, D, device="cuda"), torch.empty(T, Hq * D, device="cuda")
        p1a.attn_prep(qg, k, v, qn, kn, slot, q, gate, c.with_rows(of_row), -1, T, Hq, n_rot, 1e4, 1e-6, mrope=(pos, T, (1, 0, 0), 1))
        return q, gate
    mem, layers = caches()
    ref_mem, ref_layers = caches()
    prompt = [g.integers(0, V, n).tolist() for n in lens]
    for s in range(2):                                         # (the prompts but for their last token)
        for L in (layers, ref_layers):
            for i, c in enumerate(L):
                m = lens[s] - 1
                t, at = dev(np.array(prompt[s][:m], np.int32)), dev(np.arange(m, dtype=np.int32))
                prep(i, c, t, at, at, offsets[s:s + 1].expand(m).contiguous())
    held, certain, told = [n - 1 for n in lens], [p[-1] for p in prompt], [[], []]
    outs = [[], []]
    for step in range(3):
        counts = [11, 6]
        parents = [R.tree(g, n) for n in counts]
        T = sum(counts)
        token = np.array([t for s in range(2) for t in [certain[s], *g.integers(0, V, counts[s] - 1)]], np.int32)
        dtok, parent = dev(token), dev(np.array(sum(parents, []), np.int32))
        rows = p1a.Rows(T, n_seq=2, row0=dev(starts(counts)), pos0=dev(np.array(held, np.int32)), max_rows=11)
        mask, pos, slot = (torch.empty(T, k, dtype=torch.int32, device="cuda").squeeze(-1) for k in (1, 1, 1))
        mask = mask.view(T, 1)
        p1a.tree_rows(parent, rows, mask, pos=pos, slot=slot)
        of_row = torch.repeat_interleave(offsets, torch.tensor(counts, device="cuda")).contiguous()
        total = 0
        for i, c in enumerate(layers):
            q, gate = prep(i, c, dtok, pos, slot, of_row)
            out = torch.empty(T, Hq, D, device="cuda")
            p1a.attn_tree(q, c, out, rows, mask, Hq, D ** -0.5, gate=gate)
            total = total + out.view(T, -1)
        logits = total @ head
        # (drafts that stand now and then: look-ups into what the target would say)
        for r in range(T):
            s = int(r >= counts[0])
            i = r - s * counts[0]
            if parents[s][i] >= 0 and g.random() < 0.8:
                dtok[r] = logits[s * counts[0] + parents[s][i]].argmax()
        n, nxt = (torch.empty(2, dtype=torch.int32, device="cuda") for _ in range(2))
        path = torch.empty(2, 11, dtype=torch.int32, device="cuda")
        # (the drafts were changed behind their attention: what is accepted goes through the step once more, with its K and V)
        for i, c in enumerate(layers):
            q, gate = prep(i, c, dtok, pos, slot, of_row)
            out = torch.empty(T, Hq, D, device="cuda")
            p1a.attn_tree(q, c, out, rows, mask, Hq, D ** -0.5, gate=gate)
            total = out.view(T, -1) if i == 0 else total + out.view(T, -1)
        p1a.tree_verify(total @ head, dtok, rows, torch.rand(T, device="cuda"), torch.rand(2, device="cuda"), n, path, nxt, parent=parent, temp=torch.zeros(2, device="cuda"))
        p1a.tree_commit(layers, rows, n, path)
        for s in range(2):
            nodes = [0] + path[s][:int(n[s])].tolist()
            told[s] += [int(dtok[s * counts[0] + i]) for i in nodes]
            outs[s] += [total[s * counts[0] + i].clone() for i in nodes]
            held[s] += len(nodes)
            certain[s] = int(nxt[s])
    assert max(len(t) for t in told) > 3
    for s in range(2):
        for k, t in enumerate(told[s]):
            at = dev(np.array([lens[s] - 1 + k], np.int32))
            total = 0
            for i, c in enumerate(ref_layers):
                q, gate = prep(i, c, dev(np.array([t], np.int32)), at, at, offsets[s:s + 1].contiguous())
                out = torch.empty(1, Hq, D, device="cuda")
                p1a.attn_chunk(q, c.with_rows(offsets[s:s + 1].contiguous()), out, p1a.Rows(1, pos0=at), Hq, D ** -0.5, gate=gate)
                total = total + out.view(-1)
            assert (total - outs[s][k]).norm() <= 4 * REL * total.norm()
    tab = table.cpu().numpy().reshape(2, max_pages)
    for a, b in zip(mem, ref_mem):
        a, b = (x.cpu().numpy().reshape(16, page, rowb) for x in (a, b))
        for s in range(2):
            j = np.arange(held[s])
            assert np.array_equal(a[tab[s][j // page], j % page], b[tab[s][j // page], j % page])


def test_a_recorded_step(p1a):
    """masks, attention, verification and the move in one graph: replays with other inputs give what eager calls give"""
    counts, lens, Hq, D, V = [20, 9], [3000, 300], 8, 128, 9000
    cache = Cache(p1a, O.KV_Q8_0, 2, D, 6, lens, 50)
    g = np.random.default_rng(1)
    pos0 = dev(np.array([n - c - 50 for n, c in zip(lens, counts)], np.int32))
    T = sum(counts)
    rows = p1a.Rows(T, n_seq=2, row0=dev(starts(counts)), pos0=pos0, max_rows=20)
    st = {"parent": dev(np.array(sum((R.tree(g, n) for n in counts), []), np.int32)), "token": dev(g.integers(0, V, T).astype(np.int32)), "q": torch.randn(T, Hq, D, device="cuda"),
          "target": 3 * torch.randn(T, V, device="cuda"), "draft": torch.softmax(3 * torch.randn(T, V, device="cuda"), -1), "u": torch.rand(T, device="cuda"), "u_next": torch.rand(2, device="cuda")}

    def step(scratch=None):
        mask = torch.empty(T, 1, dtype=torch.int32, device="cuda")
        out, n, path, nxt = torch.empty(T, Hq, D, device="cuda"), *(torch.empty(2, w, dtype=torch.int32, device="cuda") for w in (1, 20, 1))
        p1a.tree_rows(st["parent"], rows, mask)
        p1a.attn_tree(st["q"], cache.kv, out, rows, mask, Hq, 0.1, scratch=scratch)
        p1a.tree_verify(st["target"], st["token"], rows, st["u"], st["u_next"], n, path, nxt, parent=st["parent"], draft=st["draft"], max_children=3, scratch=scratch)
        p1a.tree_commit(layers, rows, n, path)
        return out, n, path, nxt
    layers = p1a.Layers([cache.kv])
    need = max(p1a.tree_scratch_bytes(cache.kv, rows, Hq), p1a.verify_scratch_bytes(rows, V))
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    k0, v0 = cache.k.clone(), cache.v.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()                                                 # (the library's own buffers of this stream)
    torch.cuda.synchronize()
    graphs = []
    for scratch in (None, room):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(scratch)
        graphs.append((graph, got))
    for seed in range(4):
        g = np.random.default_rng(100 + seed)
        st["parent"].copy_(dev(np.array(sum((R.tree(g, n) for n in counts), []), np.int32)))
        st["token"].copy_(dev(g.integers(0, V, T).astype(np.int32)))
        st["q"].normal_()
        st["target"].normal_().mul_(3)
        st["draft"].copy_(torch.softmax(st["target"] + torch.randn(T, V, device="cuda"), -1))
        st["u"].uniform_()
        pos0.add_(7)
        cache.k.copy_(k0)
        cache.v.copy_(v0)
        want = [x.clone() for x in step()]
        k, v = cache.k.clone(), cache.v.clone()
        for graph, got in graphs:
            cache.k.copy_(k0)
            cache.v.copy_(v0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(k, cache.k) and torch.equal(v, cache.v)


def test_two_streams_at_once(p1a):
    """calls on two streams that overlap have partials of their own"""
    cache = Cache(p1a, O.KV_F16, 4, 128, 6, [6000, 900], 51)
    calls = [Call(p1a, cache, 16, [12, 7], [5988, 893], seed=s) for s in (1, 2)]
    want = [c.run(p1a)[0] for c in calls]
    batches = [Batch(70 + s, [9, 5], 20000, 3) for s in (1, 2)]
    told = [b.check(p1a) for b in batches]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty(19, 16, 128, device="cuda") for _ in range(2)]
    ints = [[torch.empty(2, w, dtype=torch.int32, device="cuda") for w in (1, 9, 1)] for _ in range(2)]
    temps = [dev(b.temp) for b in batches]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, b, o, n, t, s in zip(calls, batches, outs, ints, temps, streams):
            with torch.cuda.stream(s):
                token, u, u_next, parent = b.kept
                p1a.attn_tree(c.q, cache.kv, o, c.rows, c.mask, 16, c.scale)
                p1a.tree_verify(b.dt, token, b.rows, u, u_next, *n, parent=parent, draft=b.dd, temp=t, max_children=3)
    torch.cuda.synchronize()
    for o, w, n, t in zip(outs, want, ints, told):
        assert np.array_equal(o.cpu().numpy().astype(np.float64), w)
        assert np.array_equal(n[0][:, 0].cpu().numpy(), t[0]) and np.array_equal(n[1].cpu().numpy(), t[1]) and np.array_equal(n[2][:, 0].cpu().numpy(), t[2])
