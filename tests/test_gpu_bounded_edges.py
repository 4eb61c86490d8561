"""Calls over bounded caches at the ends of what their documentation allows, each against its formula in 64 bits. Tolerances of f32 results are those derived in
test_gpu_bounded.py: 1e-5 in the 2-norm."""
import numpy as np
import pytest
import torch

import _inputs as I
import _oracle as O
from _bounded import Cache, rows_exact, seen
from _gpu import dev

pytestmark = pytest.mark.gpu

KVS = {"f16": O.KV_F16, "q8_0": O.KV_Q8_0, "q4_0": O.KV_Q4_0}
REL = 1e-5


@pytest.mark.parametrize("kv", ["f16", "q8_0"])
def test_rows_far_behind_the_first(p1a, kv):
    """few rows of a sequence behind 2^25 rows of nobody"""
    first, n, D = (1 << 25) + 3, 300, 64
    T = first + 2 + 5
    cache = Cache(p1a, KVS[kv], 1, D, 4, [n], 81)
    q = torch.empty(T, 1, D, dtype=torch.bfloat16, device="cuda")
    q[first:first + 2].normal_(generator=torch.Generator("cuda").manual_seed(82))
    lse = torch.empty(T, 1, device="cuda")
    rows = p1a.Rows(T, n_seq=1, row0=dev(np.array([first, first + 2], np.int32)), pos0=dev(np.array([n - 2], np.int32)), max_rows=2, max_n=n)
    out, z, w, _, _ = rows_exact(q[first:first + 2].float().cpu().numpy(), cache.heads("k", 0, n), cache.heads("v", 0, n), seen(np.array([n - 2, n - 1]), n, 0, 0), 0.125)
    lse[first:first + 2] = dev(z.astype(np.float32))
    mass = torch.zeros(1, 1, n, device="cuda")
    p1a.attn_mass(q, cache.kv, lse, mass, rows, 1, 0.125)
    want = w.sum((0, 1))
    assert np.linalg.norm(mass.cpu().numpy()[0, 0] - want) <= REL * np.linalg.norm(want)


@pytest.mark.parametrize("counts", [[1, 1], [40, 3]])
def test_a_cache_of_no_positions(p1a, counts):
    """n_ctx = 0: every row sees nothing, and totals stay as they are"""
    cache = Cache(p1a, O.KV_Q8_0, 2, 64, 4, [50, 50], 83)
    T = sum(counts)
    q, out, lse = torch.randn(T, 4, 64, device="cuda"), torch.full((T, 4, 64), 7.0, device="cuda"), torch.full((T, 4), 7.0, device="cuda")
    cache.kv.n_ctx = 0
    rows = p1a.Rows(T, n_seq=2, row0=dev(np.array([0, counts[0], T], np.int32)), pos0=dev(np.zeros(2, np.int32)), max_rows=max(counts))
    p1a.attn_chunk(q, cache.kv, out, rows, 4, 0.125, lse=lse)
    mass = torch.full((2, 2, 64), 3.0, device="cuda")
    p1a.attn_mass(q, cache.kv, torch.zeros(T, 4, device="cuda"), mass, rows, 4, 0.125)
    torch.cuda.synchronize()
    assert (out == 0).all() and (lse == -np.inf).all() and (mass == 3).all()


@pytest.mark.parametrize("times", [1, 10])                      # (up to 8 rows of four heads under a kv head: the kernel for few; ten times that: blocks)
@pytest.mark.parametrize("row0", [[0, 8, 3, 3, 3], [8, 8, 0, 5, 5], [7, 1, 4, 4, 2], [3, 0, 3, 8, 1], [0, 8, 2, 2, 0]])
def test_pairs_of_row0_that_run_backwards(p1a, row0, times):
    """... are empty sequences; the others' rows come out right where the call is split and merged too, and nobody's rows are left"""
    n, Hq, D, T = 5000, 4, 64, 9 * times
    cache = Cache(p1a, O.KV_Q8_0, 1, D, 6, [n] * 4, 84)
    first = np.array(row0, np.int32) * times
    q = I.normal(I.rng(85), (T, Hq, D))
    pos0 = np.array([n - 8 * times, n - 2000, n - 100 * times, 3000], np.int32)
    rows = p1a.Rows(T, n_seq=4, row0=dev(first), pos0=dev(pos0), max_rows=8 * times, max_n=n)
    assert p1a.chunk_scratch_bytes(cache.kv, rows, Hq) > 0
    out, z = torch.full((T, Hq, D), 7.0, device="cuda"), torch.full((T, Hq), 7.0, device="cuda")
    p1a.attn_chunk(dev(q), cache.kv, out, rows, Hq, 0.125, lse=z)
    out, z = out.cpu().numpy(), z.cpu().numpy()
    owned = np.zeros(T, bool)
    for s in range(4):
        a, b = first[s], first[s + 1]
        if b <= a:
            continue
        owned[a:b] = True
        p = pos0[s] + np.arange(b - a)
        m = int(p[-1]) + 1
        want, lse, _, _, qk = rows_exact(q[a:b].astype(np.float64), cache.heads("k", s, m), cache.heads("v", s, m), seen(p, m, 0, 0), 0.125)
        assert np.linalg.norm(out[a:b] - want) <= REL * np.linalg.norm(want), s
        assert (np.abs(z[a:b] - lse) <= REL * qk + 2.0 ** -22 * (np.abs(lse) + 16)).all(), s
    assert (out[~owned] == 7).all() and (z[~owned] == 7).all()


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("n", [40, 6000])                       # (unsplit, and split and merged)
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("kv", list(KVS))
def test_rows_of_nan_stay_nan(p1a, kv, T, n, D):
    """a row of q with a NaN or an infinity gives NaN under each head it is in, its log-sum-exp too, whatever the plan; its neighbours give what they do without it;
    its weights are NaN wherever it sees, under its kv head alone"""
    Hq, Hkv = 8, 2
    cache = Cache(p1a, KVS[kv], Hkv, D, 6, [n], 86)
    q = dev(I.normal(I.rng(87), (T, Hq, D)))
    bad = q.clone()
    bad[T // 2, 1, 5] = float("nan")
    bad[T - 1, 3, 0] = float("inf")
    hit = torch.zeros(T, Hq, dtype=torch.bool, device="cuda")
    hit[T // 2, 1] = hit[T - 1, 3] = True
    rows = p1a.Rows(T, p0=n - T)
    for out_bf16 in (False, True):
        got = []
        for x in (q, bad):
            out = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16 if out_bf16 else torch.float32, device="cuda")
            z = None if out_bf16 else torch.full((T, Hq), 7.0, device="cuda")
            p1a.attn_chunk(x, cache.kv, out, rows, Hq, D ** -0.5, lse=z)
            got.append((out, z))
        (clean, z0), (out, z) = got
        assert out[hit].isnan().all() and torch.equal(out[~hit], clean[~hit])
        if z is not None:
            assert z[T // 2, 1].isnan() and not z[T - 1, 3].isfinite() and z[T - 1, 3] != -np.inf and torch.equal(z[~hit], z0[~hit])
            masses = [torch.zeros(1, Hkv, n, device="cuda") for _ in range(2)]
            for m, x, zz in zip(masses, (q, bad), (z0, z)):
                p1a.attn_mass(x, cache.kv, zz, m, rows, Hq, D ** -0.5)
            assert masses[1][0, 0].isnan().all() and torch.equal(masses[1][0, 1], masses[0][0, 1])


@pytest.mark.parametrize("window, n_sink, ld, max_n", [(300, 70, 20000, 0), (1000, 0, 4500, 0), (64, 3, 2900, 100), (0, 0, 20000, 700), (5, 33, 20000, 0), (100, 4000, 20000, 0)])
@pytest.mark.parametrize("kv", ["f16", "q8_0"])
def test_partial_sums_of_weights(p1a, kv, window, n_sink, ld, max_n):
    """many rows shared among workgroups: rows of totals far longer than what is seen, shorter too, max_n understated; entries that no row sees are left"""
    lens, counts, Hq, D = [5000, 4000, 3001], [600, 41, 333], 4, 64
    cache = Cache(p1a, KVS[kv], 1, D, 5, lens, 88)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    pos0 = np.array([n - c for n, c in zip(lens, counts)], np.int32)
    q = I.normal(I.rng(89), (first[-1], Hq, D))
    rows = p1a.Rows(int(first[-1]), n_seq=3, row0=dev(first), pos0=dev(pos0), max_rows=600, max_n=max_n, window=window, n_sink=n_sink)
    need = p1a.mass_scratch_bytes(cache.kv, ld, rows, Hq)
    assert need > 0
    exact = []
    for s, n in enumerate(lens):
        p = pos0[s] + np.arange(counts[s])
        see = seen(p, n, window, n_sink)
        exact.append(rows_exact(q[first[s]:first[s + 1]].astype(np.float64), cache.heads("k", s, n), cache.heads("v", s, n), see, 0.125) + (see,))
    lse = dev(np.concatenate([e[1] for e in exact]).astype(np.float32))
    for scratch in (None, torch.full((need,), 255, dtype=torch.uint8, device="cuda")):
        mass = torch.full((3, 1, ld), 0.5, device="cuda")
        p1a.attn_mass(dev(q), cache.kv, lse, mass, rows, Hq, 0.125, scratch=scratch)
        got = mass.cpu().numpy().astype(np.float64)[:, 0]
        for s, e in enumerate(exact):
            n = min(lens[s], ld)
            want = e[2].sum((0, 1))[:n]
            assert np.linalg.norm(got[s, :n] - 0.5 - want) <= REL * np.linalg.norm(want) + 2.0 ** -24 * np.linalg.norm(want + 0.5), s
            untouched = np.ones(ld, bool)
            untouched[:n] = ~e[5].any(0)[:n]
            assert (got[s][untouched] == 0.5).all()


def test_sequences_of_two_layers_are_evicted_in_turn(p1a):
    """totals of each layer's own, one sequence shorter than the budget, and twice, over what was held each time: every layer keeps what its own totals say, the
    short sequence stays whole, pages come back from the long ones alone"""
    L, Hq, Hkv, D, psh, n_ctx, budget, n_sink, n_recent = 2, 8, 2, 64, 4, 512, 64, 4, 16
    hb = O.row_bytes(O.KV_Q8_0, 1, D)
    pool = p1a.Pool(p1a.KV_Q8_0, L, Hkv, D, psh, n_ctx, 4, 2048)
    held = [300, 40, 129]
    seqs = [pool.seq_create() for _ in held]
    g = I.rng(90)

    def raw(s):
        """[layer][K | V][position][Hkv][head bytes] of what sequence s holds"""
        torch.cuda.synchronize()
        n = pool.seq_pages(seqs[s])
        buf = torch.empty(n * 2 * L * (1 << psh) * Hkv * hb, dtype=torch.uint8, pin_memory=True)
        pool.pages_out(seqs[s], 0, n, buf.data_ptr())
        torch.cuda.synchronize()
        x = buf.numpy().reshape(n, 2, L, 1 << psh, Hkv, hb).transpose(2, 1, 0, 3, 4, 5)
        return np.ascontiguousarray(x).reshape(L, 2, n << psh, Hkv, hb)[:, :, :held[s]].copy()

    def add(counts):
        for s, c in enumerate(counts):
            pool.seq_advance(seqs[s], None, c)
            for layer in range(L):
                k, v = (dev(I.normal(g, (c, Hkv, D))) for _ in range(2))
                p1a.kv_append(pool.cache_seq(layer, seqs[s]), k, v, held[s], c)
            held[s] += c
        pool.set_rows(seqs)

    counts, held = held, [0, 0, 0]
    add(counts)
    layers = [pool.cache_rows(i) for i in range(L)]
    mass = [torch.zeros(3, Hkv, n_ctx, device="cuda") for _ in range(L)]
    keep = torch.empty(3, Hkv, budget, dtype=torch.int32, device="cuda")
    for turn in range(2):
        first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        T = int(first[-1])
        q = dev(I.normal(g, (T, Hq, D)))
        rows = p1a.Rows(T, n_seq=3, row0=dev(first), pos0=dev(np.array([h - c for h, c in zip(held, counts)], np.int32)), max_rows=max(counts), max_n=max(held))
        out, lse = torch.empty(T, Hq, D, device="cuda"), torch.empty(T, Hq, device="cuda")
        for i, (kv, m) in enumerate(zip(layers, mass)):
            p1a.attn_chunk(q * (1 + i), kv, out, rows, Hq, 0.125, lse=lse)
            p1a.attn_mass(q * (1 + i), kv, lse, m, rows, Hq, 0.125)
        before, totals = [raw(s) for s in range(3)], [m.cpu().numpy() for m in mass]
        n = dev(np.array(held, np.int32))
        lists = []
        for kv, m in zip(layers, mass):
            p1a.evict_select(m, n, keep, n_sink=n_sink, n_recent=n_recent)
            p1a.kv_compact(kv, keep, mass=m, mass_out=m)
            lists.append(keep.cpu().numpy())
        assert turn or not np.array_equal(lists[0][0], lists[1][0])      # (later on the old totals outweigh the new ones in both)
        free, was = pool.free_pages, list(held)
        for s, seq in enumerate(seqs):
            if held[s] > budget:
                pool.seq_evict(seq, budget)
            held[s] = min(held[s], budget)
            assert pool.seq_len(seq) == held[s]
        assert pool.free_pages - free == sum(-(-w // 16) - -(-h // 16) for w, h in zip(was, held))
        for s in range(3):
            now = raw(s)
            for i in range(L):
                kept = lists[i][s, :, :held[s]]
                t = totals[i][s]
                for h in range(Hkv):
                    if was[s] <= budget:
                        assert np.array_equal(kept[h], np.arange(was[s]))
                    else:
                        mid = np.arange(n_sink, was[s] - n_recent)
                        best = mid[np.lexsort((mid, -t[h][mid]))][:budget - n_sink - n_recent]
                        assert np.array_equal(kept[h], np.sort(np.concatenate([np.arange(n_sink), best, np.arange(was[s] - n_recent, was[s])])))
                    assert np.array_equal(now[i][:, :, h], before[s][i][:, kept[h], h])
                    assert np.array_equal(mass[i][s, h, :held[s]].cpu().numpy(), t[h][kept[h]]) and not mass[i][s, h, held[s]:].any()
        counts = [20, 3, 9]
        if turn == 0:
            add(counts)
    pool.close()


def test_partials_of_growing_calls(p1a):
    """calls that grow row by row, without scratch of their own, on a stream of theirs: none is refused, and what the library keeps for them stays within twice the
    largest one's (and as much again in buffers it replaced)"""
    n, D, most = 6000, 64, 700
    cache = Cache(p1a, O.KV_F16, 1, D, 6, [n], 91)
    q, out = torch.randn(most, 1, D, device="cuda"), torch.empty(most, 1, D, device="cuda")
    lse, mass = torch.empty(most, 1, device="cuda"), torch.zeros(1, 1, n, device="cuda")
    need = 0
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    with torch.cuda.stream(torch.cuda.Stream()):
        for T in range(33, most):
            rows = p1a.Rows(T, p0=n - T)
            need = max(need, p1a.chunk_scratch_bytes(cache.kv, rows, 1), p1a.mass_scratch_bytes(cache.kv, n, rows, 1))
            p1a.attn_chunk(q, cache.kv, out, rows, 1, 0.125, lse=lse)
            p1a.attn_mass(q, cache.kv, lse, mass, rows, 1, 0.125)
        torch.cuda.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= 4 * need + (64 << 20)             # (64 MB: what the runtime takes for a stream)


def test_sequences_by_the_ten_thousand(p1a):
    """40000 sequences, three of which have rows: nothing is refused, and they come out right"""
    n_seq, n, Hkv, D = 40000, 8192, 8, 64
    cache = Cache(p1a, O.KV_Q4_0, Hkv, D, 12, [n, n, n], 92)
    at, counts = {5: 0, 20000: 1, 39999: 2}, np.zeros(n_seq, np.int64)
    counts[list(at)] = [1, 3, 2]
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    pos0 = np.full(n_seq, n - 3, np.int32)
    table = np.zeros(n_seq, np.int32)
    for s, i in at.items():
        table[s] = i * cache.max_pages
    cache.kv.rtab = dev(table)
    q = I.normal(I.rng(93), (6, Hkv, D))
    rows = p1a.Rows(6, n_seq=n_seq, row0=dev(first), pos0=dev(pos0), max_rows=3, max_n=n)
    out, lse = torch.full((6, Hkv, D), 7.0, device="cuda"), torch.full((6, Hkv), 7.0, device="cuda")
    p1a.attn_chunk(dev(q), cache.kv, out, rows, Hkv, 0.125, lse=lse)
    for s, i in at.items():
        a, b = first[s], first[s + 1]
        p = n - 3 + np.arange(b - a)
        want, z, _, _, qk = rows_exact(q[a:b].astype(np.float64), cache.heads("k", i, n), cache.heads("v", i, n), seen(p, n, 0, 0), 0.125)
        assert np.linalg.norm(out[a:b].cpu().numpy() - want) <= REL * np.linalg.norm(want)
        assert (np.abs(lse[a:b].cpu().numpy() - z) <= REL * qk + 2.0 ** -22 * (np.abs(z) + 16)).all()
