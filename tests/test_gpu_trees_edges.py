"""Calls on drafted trees at the ends of what their documentation allows, each against its formula in 64 bits. Tolerances of attention are those of test_gpu_trees.py."""
import numpy as np
import pytest
import torch

import _inputs as I
import _oracle as O
from _bounded import Cache, rows_exact, seen
from _gpu import dev
from test_gpu_trees import Call

pytestmark = pytest.mark.gpu

KVS = {"f16": O.KV_F16, "q8_0": O.KV_Q8_0, "q4_0": O.KV_Q4_0}
REL = 1e-5


@pytest.mark.parametrize("Hq", [1, 12])                         # (20 columns: waves with keys of their own; 240: waves that share them)
@pytest.mark.parametrize("kv", list(KVS))
def test_masks_that_name_slots_past_the_cache(p1a, kv, Hq):
    """trees that reach past n_ctx, which ends inside a tile of keys: slots behind it are nobody's, whatever the masks say"""
    g = I.rng(91)
    some = [g.random((20, 20)) < 0.4 for _ in range(2)]
    some[0][0] = False
    some[0][0, [3, 12]] = True                                  # position 93 and, of a cache of 100, none
    every = [np.ones((20, 20), bool)] * 2
    for D, out_bf16 in ((64, False), (128, True), (256, False)):
        flat = Cache(p1a, KVS[kv], 1, D, 0, [100], 92, paged=False)
        paged = Cache(p1a, KVS[kv], 1, D, 4, [48, 48], 93, max_pages=3)
        assert flat.kv.n_ctx == 100 and paged.kv.n_ctx == 48
        for window, n_sink in ((0, 0), (30, 3)):
            for see in (some, every):
                Call(p1a, flat, Hq, [20], [90], window, n_sink, see=see[:1]).check(p1a, out_bf16, lse=not out_bf16)
                Call(p1a, paged, Hq, [20, 20], [40, 47], window, n_sink, see=see, junk=True, words=2).check(p1a, out_bf16, lse=not out_bf16)


@pytest.mark.parametrize("window", [(1 << 31) - 2, (1 << 31) - 7, (1 << 30) + 5, 1200])
@pytest.mark.parametrize("kv", list(KVS))
def test_windows_that_reach_past_everything(p1a, kv, window):
    """... hide nothing, whatever 32 bits hold of them: trees, chunks of few rows and of many, weight per position"""
    for D, Hq, count in ((64, 4, 3), (128, 12, 40)):
        cache = Cache(p1a, KVS[kv], 1, D, 4, [33 + count], 94)
        Call(p1a, cache, Hq, [count], [33], window, 2).check(p1a)
        chain = Call(p1a, cache, Hq, [count], [33], see=[np.tril(np.ones((count, count), bool))])
        want, lse = chain.run(p1a)
        n = 33 + count
        rows = p1a.Rows(count, pos0=chain.dpos, window=window, n_sink=2)
        out, z, mass = torch.empty_like(chain.q), torch.empty(count, Hq, device="cuda"), torch.zeros(1, 1, n, device="cuda")
        p1a.attn_chunk(chain.q, cache.kv, out, rows, Hq, chain.scale, lse=z)
        assert np.linalg.norm(out.cpu().numpy() - want) <= 2 * REL * np.linalg.norm(want)
        p1a.attn_mass(chain.q, cache.kv, z, mass, rows, Hq, chain.scale)
        weight = rows_exact(chain.q64, cache.heads("k", 0, n), cache.heads("v", 0, n), seen(33 + np.arange(count), n, 0, 0), chain.scale)[2].sum((0, 1))
        assert np.linalg.norm(mass.cpu().numpy()[0, 0] - weight) <= REL * np.linalg.norm(weight)


@pytest.mark.parametrize("count", [4, 40])
def test_gates_far_from_zero(p1a, count):
    """each gated result beside the one without a gate. The exponential and the reciprocal are 2^-23 of themselves off, the sum and the product 2^-24; g log2 e is rounded by 2^-24 of
    itself and log2 e by 0.22 2^-24, which moves the exponential by 1.22 |g| 2^-24 and the gate by that times 1 - gate"""
    g = I.rng(95)
    cache = Cache(p1a, O.KV_F16, 1, 64, 4, [300], 96)
    call = Call(p1a, cache, 6, [count], [260])
    plain, _ = call.run(p1a)
    for most in (1, 10, 30, 80):
        gate = (most * (2 * g.random((count, 6 * 64)) - 1)).astype(np.float32)
        call.dgate = dev(gate)
        got, _ = call.run(p1a)
        sigma = 1 / (1 + np.exp(-gate.astype(np.float64)))
        want, off = plain * sigma.reshape(plain.shape), ((6.01 + 1.22 * np.abs(gate) * (1 - sigma)) * 2.0 ** -24).reshape(plain.shape)
        assert (np.abs(got - want) <= off * np.abs(want)).all(), (most, float((np.abs(got - want) / (off * np.abs(want))).max()))
    call.dgate = dev(np.where(np.arange(6 * 64) % 2, np.inf, -np.inf).astype(np.float32) * np.ones((count, 1), np.float32))
    got, _ = call.run(p1a)
    assert np.array_equal(got.reshape(count, -1)[:, 1::2], plain.reshape(count, -1)[:, 1::2]) and (got.reshape(count, -1)[:, ::2] == 0).all()


def test_a_step_without_rows(p1a):
    """no row of any sequence: nothing accepted, no token"""
    cache, i = Cache(p1a, O.KV_F16, 1, 64, 4, [30], 97), torch.empty(0, 1, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 4, 64, device="cuda")
    p1a.tree_rows(i.flatten(), p1a.Rows(0), i, pos=i.flatten(), slot=i.flatten())
    p1a.attn_tree(q, cache.kv, q.clone(), p1a.Rows(0), i, 4, 0.125, lse=torch.empty(0, 4, device="cuda"))
    for draft in (None, torch.empty(0, 50, device="cuda")):
        rows = p1a.Rows(0, n_seq=3, row0=dev(np.zeros(4, np.int32)))
        i, f = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, device="cuda")
        n, nxt, path = (torch.full((3, w), 77, dtype=torch.int32, device="cuda") for w in (1, 1, 4))
        p1a.tree_verify(torch.empty(0, 50, device="cuda"), i, rows, f, torch.rand(3, device="cuda"), n, path, nxt, parent=i, draft=draft, max_children=3)
        assert (n == 0).all() and (nxt == -1).all() and (path == -1).all()


@pytest.mark.parametrize("kv", list(KVS))
def test_a_chain_behind_a_window_shorter_than_itself(p1a, kv):
    """the window cuts what is in front of the tree, never the path: rows whose window reaches back to the tree's first node give what attn_chunk gives, the others see more than a chunk's"""
    counts, lens, window, n_sink = [23, 40], [200, 60], 9, 2
    cache = Cache(p1a, KVS[kv], 2, 64, 4, lens, 98)
    call = Call(p1a, cache, 4, counts, [n - c for n, c in zip(lens, counts)], window, n_sink, see=[np.tril(np.ones((n, n), bool)) for n in counts])
    got = call.check(p1a)
    out = torch.empty(call.T, 4, 64, device="cuda")
    p1a.attn_chunk(call.q, cache.kv, out, call.rows, 4, call.scale)
    out = out.cpu().numpy()
    for s, c in enumerate(counts):
        a, b = call.first[s], call.first[s] + window
        assert np.linalg.norm(out[a:b] - got[a:b]) <= 2 * REL * np.linalg.norm(got[a:b])
        far = slice(b, call.first[s] + c)
        assert (np.abs(out[far] - got[far]).max((1, 2)) > 1e-3).all()


@pytest.mark.parametrize("kv", list(KVS))
def test_rounded_results_with_their_log_sum_exp(p1a, kv):
    """bf16 results beside an f32 log-sum-exp, whole and split: the results of f32 rounded once, the same log-sum-exp"""
    for D, Hq, lens, counts in ((64, 4, [300, 40], [3, 2]), (256, 12, [900, 70], [30, 8]), (128, 6, [5000], [4])):
        cache = Cache(p1a, KVS[kv], 2, D, 4, lens, 99)
        call = Call(p1a, cache, Hq, counts, [n - c for n, c in zip(lens, counts)], gate=True)
        got, lse = call.run(p1a)
        short, z = call.run(p1a, out_bf16=True)
        assert np.array_equal(z, lse) and np.array_equal(short, torch.from_numpy(got).to(torch.bfloat16).double().numpy())


@pytest.mark.parametrize("Hq, lens", [(2, [900, 60]), (12, [900, 60]), (12, [9000, 60])])
def test_sequences_longer_than_max_rows(p1a, Hq, lens):
    """rows past the first max_rows of a sequence are left as they are, and nobody sees them: masks, attention and verification as of trees that end there"""
    cache, counts, most, V = Cache(p1a, O.KV_Q8_0, 1, 64, 6, lens, 100), [13, 5], 7, 60
    pos0 = [n - 13 for n in lens]
    whole = Call(p1a, cache, Hq, counts, pos0)
    cut = Call(p1a, cache, Hq, [most, 5], pos0, see=[m[:most, :most] for m in whole.see])
    rows = p1a.Rows(18, n_seq=2, row0=whole.row0, pos0=whole.dpos, max_rows=most)
    out, lse = torch.full_like(whole.q, 77), torch.full((18, Hq), 77.0, device="cuda")
    p1a.attn_tree(whole.q, cache.kv, out, rows, whole.mask, Hq, whole.scale, lse=lse)
    assert (out[most:13] == 77).all() and (lse[most:13] == 77).all()
    keep = [*range(most), *range(13, 18)]
    cut.q = whole.q[keep].contiguous()
    want = torch.empty(most + 5, Hq, 64, device="cuda")
    p1a.attn_tree(cut.q, cache.kv, want, cut.rows, cut.mask, Hq, whole.scale)
    assert torch.equal(out[keep], want)
    parent = dev(np.array([*range(-1, 12), *range(-1, 4)], np.int32))
    mask, pos, slot = (torch.full((18, w), 77, dtype=torch.int32, device="cuda") for w in (1, 1, 1))
    p1a.tree_rows(parent, rows, mask, pos=pos, slot=slot)
    assert all((t[most:13] == 77).all() and (t[:most] != 77).all() for t in (mask, pos, slot))
    assert pos[:most, 0].tolist() == list(range(pos0[0], pos0[0] + most)) and (mask[:, 0][keep] == dev(np.array([(2 << i) - 1 for i in [*range(most), *range(5)]], np.int32))).all()
    n, nxt = (torch.empty(2, dtype=torch.int32, device="cuda") for _ in range(2))
    path = torch.empty(2, 12, dtype=torch.int32, device="cuda")
    target = torch.zeros(18, V, device="cuda")
    token = torch.arange(18, dtype=torch.int32, device="cuda")
    target[torch.arange(17), token[1:].long()] = 50             # (every draft is what the target says)
    p1a.tree_verify(target, token, rows, torch.rand(18, device="cuda"), torch.rand(2, device="cuda"), n, path, nxt, parent=parent)
    assert n.tolist() == [most - 1, 4] and path[0].tolist() == [*range(1, most)] + [-1] * (13 - most) and nxt[0] == most


def test_thousands_of_sequences(p1a):
    counts = [(s * 5) % 4 for s in range(3000)]
    lens = [20 + (s * 13) % 40 for s in range(3000)]
    cache = Cache(p1a, O.KV_F16, 1, 64, 4, lens, 101)
    Call(p1a, cache, 4, counts, [n - c for n, c in zip(lens, counts)]).check(p1a)


def test_masks_of_one_sequence_from_the_host(p1a):
    """the position of the only sequence is the host's; no positions and no slots asked for, or one of them"""
    parent = dev(np.array([-1, 0, 0, 2], np.int32))
    mask, at = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    p1a.tree_rows(parent, p1a.Rows(4, p0=70), mask)
    assert mask[:, 0].tolist() == [1, 3, 5, 13] and mask[:, 1].tolist() == [0] * 4
    p1a.tree_rows(parent, p1a.Rows(4, p0=70), mask, slot=at)
    assert at.tolist() == [70, 71, 72, 73]
    p1a.tree_rows(parent, p1a.Rows(4, p0=70), mask, pos=at)
    assert at.tolist() == [70, 71, 71, 72]


def test_commit_in_as_many_layers_as_a_call_takes(p1a):
    """128 layers; and a second commit of the same path, which moves what it finds"""
    layers, g = 128, torch.Generator("cuda").manual_seed(1)
    k, v = (torch.randint(0, 255, (layers, 20, 2 * 128), generator=g, dtype=torch.uint8, device="cuda") for _ in range(2))
    kv = [p1a.KVCache(1, 20, 2, 64, a.data_ptr(), b.data_ptr()) for a, b in zip(k, v)]
    rows, n, path = p1a.Rows(9, p0=8), dev(np.array([3], np.int32)), dev(np.array([[2, 5, 8]], np.int32))
    for _ in range(2):
        want = [t.clone() for t in (k, v)]
        for t in want:
            t[:, 9:12] = t[:, [10, 13, 16]].clone()
        p1a.tree_commit(kv, rows, n, path)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
