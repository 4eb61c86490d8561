"""Operators for trees of drafted tokens, as a server that verifies drafts of several sequences in one step calls them.

A step has, per sequence, the last token that is certain (node 0) and drafted tokens behind it, each with a parent among the nodes before it: a chain, or a
tree of alternatives. A case is one of four kinds of pass:

  "rows"    from the parents: which nodes of its tree a row sees (a bit each), its rotary position and its cache position.
  "tree"    attention of the nodes' rows over a paged cache: all positions in front of the tree (or a window of them and the first `sinks`), and of the
            tree the row's own path.
  "verify"  which drafted tokens stand, from the target's logits or probabilities, the draft's probabilities and given random numbers, and the token
            behind the last one that does.
  "commit"  the accepted nodes' rows of K and V moved behind node 0, in every layer.

Values of caches and queries are N(0, 1), keys and queries RMS-normed per head; logits N(0, 3^2), the draft's those and N(0, 0.7^2) more.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

KV_TYPES = {"f16": 1, "q4_0": 2, "q8_0": 8}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}
EPS = 1e-6


def _rows(name, seqs, nodes, branch, nodes_min=None):
    return {"name": name, "kind": "rows", "seqs": seqs, "nodes": nodes, "nodes_min": nodes if nodes_min is None else nodes_min, "branch": branch}


def _tree(name, kv, heads, kv_heads, dim, page, seqs, nodes, branch, ctx, nodes_min=None, ctx_min=None, window=0, sinks=0, gate=False, lse=False, q="f32", out="f32"):
    return {"name": name, "kind": "tree", "kv": kv, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": seqs, "nodes": nodes,
            "nodes_min": nodes if nodes_min is None else nodes_min, "branch": branch, "ctx": ctx, "ctx_min": ctx if ctx_min is None else ctx_min,
            "window": window, "sinks": sinks, "gate": gate, "lse": lse, "q": q, "out": out}


def _verify(name, seqs, nodes, branch, vocab, target, dtype, draft, nodes_min=None, greedy=False):
    return {"name": name, "kind": "verify", "seqs": seqs, "nodes": nodes, "nodes_min": nodes if nodes_min is None else nodes_min, "branch": branch,
            "vocab": vocab, "target": target, "type": dtype, "draft": draft, "greedy": greedy}


def _commit(name, layers, kv_heads, dim, page, seqs, nodes, branch, ctx, nodes_min=None, ctx_min=None):
    return {"name": name, "kind": "commit", "kv": "f16", "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": seqs, "nodes": nodes,
            "nodes_min": nodes if nodes_min is None else nodes_min, "branch": branch, "ctx": ctx, "ctx_min": ctx if ctx_min is None else ctx_min}


def listed():
    return [
        # one small tree: what making masks and positions costs at least, once a step
        _rows("rows_one", 1, 8, 2),
        # a full server with the widest trees
        _rows("rows64_wide", 64, 256, 8, nodes_min=33),
        # five drafted tokens of the smallest model the tests run: what a call costs when there is next to nothing to compute
        _tree("tree_one_d64_f16", "f16", 4, 1, 64, 16, 1, 6, 2, 700),
        # a step of 16 sequences of the 27B shape with small trees, contexts of every length, f32 rows and the gate as the engine has them
        _tree("tree16_27b_q8", "q8_0", 24, 4, 256, 256, 16, 16, 3, 32768, nodes_min=4, ctx_min=300, gate=True),
        # one chat far into a document, a large tree
        _tree("tree_long_27b_q8", "q8_0", 24, 4, 256, 256, 1, 63, 4, 32768, out="bf16"),
        # a full server, heads of 128, rows for bf16 products
        _tree("tree24_d128_f16", "f16", 32, 8, 128, 16, 24, 64, 4, 8000, nodes_min=3, ctx_min=500, q="bf16", out="bf16"),
        # trees wider than a mask's word through a window with sinks, statistics kept, everything in f32
        _tree("tree4_d128_q4_w2k", "q4_0", 32, 8, 128, 64, 4, 200, 6, 16000, nodes_min=40, ctx_min=900, window=2048, sinks=16, lse=True),
        # three tokens proposed by a look-up (no probabilities), one sequence: latency
        _verify("verify_one_lookup", 1, 4, 1, 32000, "logits", "bf16", "none"),
        # a step of 32 chats with four tokens each from a draft head, some of them decoded greedily
        _verify("verify32_chains", 32, 5, 1, 151936, "logits", "f32", "iid", greedy=True),
        # trees of sampled alternatives against probabilities that a sampler has filtered already
        _verify("verify8_trees", 8, 48, 4, 100003, "probs", "f32", "distinct", nodes_min=12),
        # the accepted path of one sequence, the 16 attention layers of the 27B shape
        _commit("commit_one_27b", 16, 4, 256, 256, 1, 16, 3, 700),
        # the same for a full server
        _commit("commit32_27b", 16, 4, 256, 16, 32, 64, 4, 400, nodes_min=5, ctx_min=70),
    ]


HEADS = [(4, 1), (24, 4), (16, 2), (32, 8), (8, 8), (16, 4)]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["rows", "tree", "tree", "tree", "tree", "verify", "verify", "verify", "commit"])
        seqs, branch = rng.choice([1, 1, 2, 4, 8, 16, 32]), rng.choice([1, 2, 3, 4, 8])
        nodes = _log_uniform(rng, 1, 64 if kind == "verify" else 256)
        nodes_min = max(1, nodes // rng.choice([1, 4, 16]))
        heads, kv_heads = rng.choice(HEADS)
        dim, page = rng.choice([64, 128, 256]), rng.choice([16, 64, 256])
        if kind == "rows":
            c = _rows("", seqs, nodes, branch, nodes_min)
        elif kind == "tree":
            ctx = _log_uniform(rng, max(16, nodes), 32768)
            window = rng.choice([0, 0, 0, _log_uniform(rng, 16, 8192)])
            c = _tree("", rng.choice(["f16", "q8_0", "q4_0"]), heads, kv_heads, dim, page, seqs, nodes, branch, ctx, nodes_min, max(1, ctx // rng.choice([1, 4, 16])), window,
                      rng.choice([0, 4, 64]) if window else 0, rng.random() < 0.5, rng.random() < 0.3, rng.choice(["f32", "f32", "bf16"]), rng.choice(["f32", "bf16"]))
        elif kind == "verify":
            c = _verify("", seqs, nodes, branch, _log_uniform(rng, 1000, 160001), rng.choice(["logits", "logits", "probs"]), rng.choice(["f32", "bf16"]),
                        rng.choice(["none", "iid", "distinct"]), nodes_min, rng.random() < 0.3)
        else:
            ctx = _log_uniform(rng, max(16, nodes), 700)
            c = _commit("", rng.choice([1, 4, 16]), kv_heads, dim, page, seqs, nodes, branch, ctx, nodes_min, max(1, ctx // rng.choice([1, 4])))
        del c["name"]
        if kind == "tree":
            pool = sum(_lengths(c)) * kv_heads * dim
            padded = seqs * max(_node_counts(c)) * heads * max(_lengths(c))
            fits = pool <= 1.3e8 and seqs * max(_lengths(c)) * kv_heads * dim <= 5.5e8 and padded <= 1.5e9 and work(c)["flops"] <= 1e11
        elif kind == "verify":
            fits = sum(_node_counts(c)) * c["vocab"] <= 3.7e7
        else:
            fits = kind == "rows" or c["layers"] * sum(_lengths(c)) * kv_heads * dim <= 1.3e8
        if fits:
            return c


def _spread(n, lo, hi, seed):
    """n whole numbers, evenly spread over the logarithm from lo to hi, in an order that is not sorted"""
    if n == 1:
        return [hi]
    at = random.Random(seed).sample(range(n), n)
    return [max(1, int(round(lo * (hi / lo) ** (a / (n - 1))))) for a in at]


def _node_counts(case):
    return _spread(case["seqs"], case["nodes_min"], case["nodes"], 1)


def _lengths(case):
    """the sequences' lengths, the nodes included"""
    return [max(a, b) for a, b in zip(_spread(case["seqs"], case["ctx_min"], case["ctx"], 2), _node_counts(case))]


def _parents(case):
    """per sequence the nodes' parents: a node takes one that has fewer than `branch` children, shallow ones more often"""
    rng, got = random.Random(3), []
    for n in _node_counts(case):
        parent, depth, kids = [-1], [0], [0]
        for i in range(1, n):
            free = [j for j in range(i) if kids[j] < case["branch"]]
            p = rng.choices(free, [0.75 ** depth[j] for j in free])[0]
            kids[p] += 1
            parent.append(p)
            depth.append(depth[p] + 1)
            kids.append(0)
        got.append(parent)
    return got


def _depths(parent):
    d = []
    for p in parent:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _accepted(case):
    """per sequence a path from node 0 down: to the deepest node, cut at two thirds of it"""
    got = []
    for parent in _parents(case):
        d = _depths(parent)
        i, path = d.index(max(d)), []
        while parent[i] >= 0:
            path.append(i)
            i = parent[i]
        got.append(path[::-1][: -(-2 * len(path) // 3)])
    return got


def _pairs(case):
    """visible (row, key) pairs, and keys that some row sees"""
    pairs = union = 0
    w, sinks = case["window"], case["sinks"]
    for n, parent in zip(_lengths(case), _parents(case)):
        m = len(parent)
        front = n - m
        for d in _depths(parent):
            low = max(0, min(front + d - w + 1, front)) if w else 0
            pairs += front - low + min(sinks, low) + d + 1
        low = max(0, min(front - w + 1, front)) if w else 0
        union += n - low + min(sinks, low)
    return pairs, union


def work(case):
    t = sum(_node_counts(case))
    if case["kind"] == "rows":
        words = -(-max(_node_counts(case)) // 32)
        return {"bytes": t * (4 + 4 * words + 8), "flops": 0}
    if case["kind"] == "verify":
        # every row of logits counts for its sum; probabilities, and the draft's, in the row that the last token is drawn from
        v, s, size = case["vocab"], case["seqs"], SIZES[case["type"]]
        b = t * v * size if case["target"] == "logits" else s * v * size
        return {"bytes": b + (0 if case["draft"] == "none" else 4 * s * v) + 16 * t, "flops": 0}
    if case["kind"] == "commit":
        moved = sum(sum(i != j + 1 for j, i in enumerate(path)) for path in _accepted(case))
        return {"bytes": moved * case["layers"] * 2 * 2 * case["kv_heads"] * 2 * case["dim"] + 8 * t, "flops": 0}
    hkv, d, hq = case["kv_heads"], case["dim"], case["heads"]
    pairs, union = _pairs(case)
    rows = t * hq * d * (SIZES[case["q"]] + SIZES[case["out"]] + (4 if case["gate"] else 0)) + (4 * t * hq if case["lse"] else 0)
    return {"bytes": rows + 2 * union * hkv * _head_bytes(case["kv"], d), "flops": 4 * hq * d * pairs}


# ---- the cache: rows of quantized or f16 heads in pages ----
def _head_bytes(kv, d):
    return {"f16": 2 * d, "q8_0": d // 32 * 34, "q4_0": d // 32 * 18}[kv]


def _encode(kv, x):
    """[..., D] f32 -> [..., head bytes] uint8"""
    if kv == "f16":
        return x.half().contiguous().view(torch.uint8)
    b = x.reshape(*x.shape[:-1], -1, 32)
    if kv == "q8_0":
        d = (b.abs().amax(-1) / 127).half()
        c = torch.where(d[..., None] > 0, b / d[..., None].float().clamp_min(1e-30), torch.zeros_like(b)).round().clamp(-127, 127).to(torch.int8)
        return torch.cat([d.view(torch.uint8), c.reshape(x.shape).view(torch.uint8)], -1)
    top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = (top / -8).half()
    c = torch.where(d != 0, b / d.float(), torch.zeros_like(b)).add(8.5).floor().clamp(0, 15).to(torch.uint8)
    return torch.cat([d.view(torch.uint8), c[..., :16] | c[..., 16:] << 4], -1).reshape(*x.shape[:-1], -1)


def _decode(kv, raw, d, t=torch.float32):
    """[..., head bytes] uint8 -> [..., D] numbers of type t"""
    if kv == "f16":
        return raw.contiguous().view(torch.float16).to(t)
    nb = d // 32
    if kv == "q8_0":
        s = raw[..., : 2 * nb].contiguous().view(torch.float16).to(t)
        c = raw[..., 2 * nb:].contiguous().view(torch.int8).to(t)
        return (c.unflatten(-1, (nb, 32)) * s[..., None]).flatten(-2)
    b = raw.unflatten(-1, (nb, 18))
    s = b[..., :2].contiguous().view(torch.float16).to(t)
    c = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).to(t) - 8
    return (c * s).flatten(-2)


def _normed(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, seqs = case["kind"], case["seqs"]
    parents, counts = _parents(case), _node_counts(case)
    t, most = sum(counts), max(counts)
    st = {"case": case, "t": t, "max_rows": most, "words": -(-most // 32), "deep": max(max(_depths(p)) for p in parents), "row0": _ints([0] + list(np.cumsum(counts))),
          "parent": _ints(sum(parents, []))}
    if kind == "rows":
        st["pos0"] = _ints([0]) + torch.randint(0, 30000, (seqs,), generator=g, device="cuda", dtype=torch.int32)
        st["mask"] = torch.empty(t, st["words"], dtype=torch.int32, device="cuda")
        st["pos"], st["slot"] = (torch.empty(t, dtype=torch.int32, device="cuda") for _ in range(2))
    elif kind == "verify":
        _prepare_verify(st, g)
    else:
        _prepare_cache(st, g, parents)
    if own:
        _own_plan(st)
    return st


def _prepare_cache(st, g, parents):
    case = st["case"]
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    hkv, d, page, seqs, kv = (case[k] for k in ("kv_heads", "dim", "page", "seqs", "kv"))
    lens, counts = _lengths(case), _node_counts(case)
    per = [-(-n // page) for n in lens]
    n_pages, max_pages = sum(per) + 2, max(per)
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.zeros(seqs, max_pages, dtype=torch.int32, device="cuda")
    at = 0
    for s, p in enumerate(per):
        table[s, :p] = order[at: at + p]
        at += p
    hb, layers = _head_bytes(kv, d), case.get("layers", 1)
    st["cache"] = torch.empty(layers, 2, n_pages, page, hkv, hb, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (page * hkv * d))
    for half in st["cache"]:
        for i in range(2):
            for a in range(0, n_pages, step):
                x = randn(min(step, n_pages - a), page, hkv, d)
                half[i, a: a + step] = _encode(kv, x if i else _normed(x))
    st["table"], st["offsets"] = table, (torch.arange(seqs, device="cuda") * max_pages).int()
    st["max_n"], st["pos0"] = max(lens), _ints([n - r for n, r in zip(lens, counts)])
    if case["kind"] == "commit":
        paths = _accepted(case)
        st["n_accept"], path = _ints([len(p) for p in paths]), np.full((seqs, max(1, st["deep"])), -1, np.int32)
        for s, p in enumerate(paths):
            path[s, : len(p)] = p
        st["path"] = torch.from_numpy(path).cuda()
        return
    hq, t = case["heads"], st["t"]
    mask = np.zeros((t, st["words"]), np.uint32)
    row = 0
    for parent in parents:
        for i, p in enumerate(parent):
            if p >= 0:
                mask[row + i] = mask[row + p]
            mask[row + i, i // 32] |= np.uint32(1 << (i % 32))
        row += len(parent)
    st["mask"] = torch.from_numpy(mask.view(np.int32)).cuda()
    st["q"] = _normed(randn(t, hq, d)).to(TYPES[case["q"]])
    st["scale"] = d ** -0.5
    st["gate"] = randn(t, hq * d) if case["gate"] else None
    st["out"] = torch.empty(t, hq, d, dtype=TYPES[case["out"]], device="cuda")
    st["lse"] = torch.empty(t, hq, device="cuda") if case["lse"] else None


def _prepare_verify(st, g):
    case = st["case"]
    t, v, seqs, branch = st["t"], case["vocab"], case["seqs"], case["branch"]
    temp = 0.6 + 0.6 * torch.rand(seqs, generator=g, device="cuda")
    if case["greedy"]:
        temp[::4] = 0
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), torch.tensor(_node_counts(case), device="cuda"), output_size=t)
    by = torch.where(temp > 0, 1 / temp, torch.ones_like(temp))[seq][:, None]
    logits = 3 * torch.randn(t, v, generator=g, device="cuda")
    q = torch.softmax((logits + 0.7 * torch.randn(t, v, generator=g, device="cuda")) * by, -1)
    # node i is drawn from the row of its parent, as its sibling's number says
    kid, seen = [], {}
    for s, parent in enumerate(_parents(case)):
        for p in parent:
            kid.append(seen.get((s, p), 0))
            seen[s, p] = kid[-1] + 1
    from_row = (st["row0"][:-1].long()[seq] + st["parent"].long().clamp_min(0))
    drawn = torch.multinomial(q, min(branch, v), replacement=case["draft"] == "iid", generator=g)
    st["token"] = drawn[from_row, torch.tensor(kid, device="cuda").clamp_max(branch - 1)].int()
    st["u"], st["u_next"] = torch.rand(t, generator=g, device="cuda"), torch.rand(seqs, generator=g, device="cuda")
    st["temp"] = temp
    if case["target"] == "probs":
        if case["greedy"]:                                     # (what a sampler makes of temperature 0)
            hot = torch.zeros_like(q).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
        p = torch.softmax(logits * by, -1)
        logits = torch.where(temp[seq][:, None] > 0, p, hot) if case["greedy"] else p
    st["target"] = logits.to(TYPES[case["type"]])
    st["draft"] = None if case["draft"] == "none" else q
    st["n_accept"], st["next"] = (torch.empty(seqs, dtype=torch.int32, device="cuda") for _ in range(2))
    st["path"] = torch.empty(seqs, max(1, st["deep"]), dtype=torch.int32, device="cuda")


# ---- the definitions in 64 bits, sequence by sequence ----
def exact(case, seed):
    st = prepare(case, seed)
    return {"rows": _exact_rows, "tree": _exact_tree, "verify": _exact_verify, "commit": _exact_commit}[case["kind"]](st)


def _exact_rows(st):
    mask, pos, slot = np.zeros((st["t"], st["words"]), np.uint32), [], []
    row = 0
    for s, parent in enumerate(_parents(st["case"])):
        p0 = int(st["pos0"][s])
        for i, d in enumerate(_depths(parent)):
            pos.append(p0 + d)
            slot.append(p0 + i)
            j = i
            while j >= 0:
                mask[row + i, j // 32] |= np.uint32(1 << (j % 32))
                j = parent[j]
        row += len(parent)
    return torch.from_numpy(mask.view(np.int32)).cuda(), _ints(pos), _ints(slot)


def _exact_tree(st):
    case = st["case"]
    hq, hkv, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    grp, outs, lses = hq // hkv, [], []
    row0, pos0 = st["row0"].tolist(), st["pos0"].tolist()
    for s, parent in enumerate(_parents(case)):
        r, front = len(parent), pos0[s]
        n = front + r
        path = np.zeros((r, r), bool)
        for i, p in enumerate(parent):
            if p >= 0:
                path[i] = path[p]
            path[i, i] = True
        at, j = torch.tensor(_depths(parent), device="cuda")[:, None] + front, torch.arange(front, device="cuda")[None]
        seen = torch.ones(r, front, dtype=torch.bool, device="cuda") if not case["window"] else (j > at - case["window"]) | (j < case["sinks"])
        seen = torch.cat([seen, torch.from_numpy(path).cuda()], 1)
        where = st["table"][s, : -(-n // page)].long()
        k, v = (_decode(case["kv"], st["cache"][0, i][where].flatten(0, 1)[:n], d, torch.float64) for i in range(2))
        q = st["q"][row0[s]: row0[s + 1]].double()
        out, lse = torch.empty(r, hq, d, dtype=torch.float64, device="cuda"), torch.empty(r, hq, dtype=torch.float64, device="cuda")
        for h in range(hkv):
            hs = slice(h * grp, (h + 1) * grp)
            x = torch.matmul(q[:, hs].reshape(-1, d), k[:, h].t().contiguous()).mul_(st["scale"]).view(r, grp, n)
            x.masked_fill_(~seen[:, None], -math.inf)
            lse[:, hs] = torch.logsumexp(x, -1)
            out[:, hs] = torch.matmul(x.sub_(lse[:, hs, None]).exp_().view(-1, n), v[:, h].contiguous()).view(r, grp, d)
        outs.append(out)
        lses.append(lse)
    out = torch.cat(outs)
    if case["gate"]:
        out = out / (1 + torch.exp(-st["gate"].double())).view_as(out)
    return (out, torch.cat(lses)) if case["lse"] else (out,)


def _exact_verify(st):
    case = st["case"]
    row0, token, u, u_next, temp = (st[k].tolist() for k in ("row0", "token", "u", "u_next", "temp"))
    width = st["path"].shape[1]
    got = []
    for s, parent in enumerate(_parents(case)):
        kids = [[] for _ in parent]
        for i, p in enumerate(parent):
            if p >= 0:
                kids[p].append(i)
        at, path = 0, []
        while True:
            p = st["target"][row0[s] + at].double().cpu().numpy()
            if case["target"] == "logits":
                if temp[s] > 0:
                    p = np.exp((p - p.max()) / temp[s])
                    p /= p.sum()
                else:
                    p = (np.arange(len(p)) == p.argmax()).astype(np.float64)
            q = None if st["draft"] is None else st["draft"][row0[s] + at].double().cpu().numpy()
            left, mass, gone, chosen = p.copy(), 1.0, 0.0, -1
            for c in kids[at]:
                x = token[row0[s] + c]
                share = 1.0 if q is None else q[x] / (1 - gone)
                if u[row0[s] + c] * share * mass < left[x]:
                    chosen = c
                    break
                if q is None:
                    mass -= left[x]
                    left[x] = 0
                else:
                    left = np.maximum(left - mass / (1 - gone) * q, 0)
                    mass = left.sum()
                    if case["draft"] == "distinct":
                        gone += q[x]
            if chosen < 0:
                break
            path.append(chosen)
            at = chosen
        if not left.sum() > 0:
            left = p
        total = np.cumsum(left)
        got.append((len(path), path + [-1] * (width - len(path)), int(np.searchsorted(total, u_next[s] * total[-1], side="right"))))
    return _ints([x[0] for x in got]), _ints([x[1] for x in got]), _ints([x[2] for x in got])


def _exact_commit(st):
    cache, page = st["cache"].view(torch.float16).double(), st["case"]["page"]
    table, pos0 = st["table"].tolist(), st["pos0"].tolist()
    for s, path in enumerate(_accepted(st["case"])):
        for j, i in enumerate(path):
            a, b = pos0[s] + i, pos0[s] + j + 1
            cache[:, :, table[s][b // page], b % page] = cache[:, :, table[s][a // page], a % page]
    return cache


# ---- one pass ----
def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"rows": _own_rows, "tree": _own_tree, "verify": _own_verify, "commit": _own_commit}[kind](st)
    return {"rows": _plain_rows, "tree": _plain_tree, "verify": _plain_verify, "commit": _plain_commit}[kind](st)


def _own_plan(st):
    """what a program keeps from step to step: the descriptors of its layers"""
    p1a = importlib.import_module("p100e-engine_amd")
    case = st["case"]
    if "cache" in st:
        page, width = case["page"], st["table"].shape[1]
        layers = [p1a.KVCache(KV_TYPES[case["kv"]], width * page, case["kv_heads"], case["dim"], kv[0].data_ptr(), kv[1].data_ptr(), pt=st["table"], rtab=st["offsets"],
                              psh=page.bit_length() - 1, pstride=kv.stride(1)) for kv in st["cache"]]
        st["layers"] = p1a.Layers(layers) if case["kind"] == "commit" else layers
    st["p1a"] = p1a


def _own_rows_of(st):
    p1a, case = st["p1a"], st["case"]
    return p1a.Rows(st["t"], n_seq=case["seqs"], row0=st["row0"], pos0=st.get("pos0"), max_rows=st["max_rows"], max_n=st.get("max_n", 0), window=case.get("window", 0),
                    n_sink=case.get("sinks", 0))


def _own_rows(st):
    if "p1a" not in st:
        _own_plan(st)
    st["p1a"].tree_rows(st["parent"], _own_rows_of(st), st["mask"], pos=st["pos"], slot=st["slot"])
    return st["mask"], st["pos"], st["slot"]


def _own_tree(st):
    if "p1a" not in st:
        _own_plan(st)
    st["p1a"].attn_tree(st["q"], st["layers"][0], st["out"], _own_rows_of(st), st["mask"], st["case"]["heads"], st["scale"], gate=st["gate"], lse=st["lse"])
    return (st["out"], st["lse"]) if st["lse"] is not None else (st["out"],)


def _own_verify(st):
    if "p1a" not in st:
        _own_plan(st)
    case = st["case"]
    st["p1a"].tree_verify(st["target"], st["token"], _own_rows_of(st), st["u"], st["u_next"], st["n_accept"], st["path"], st["next"],
                          parent=None if case["branch"] == 1 else st["parent"], draft=st["draft"], logits=case["target"] == "logits",
                          temp=st["temp"] if case["target"] == "logits" else None, max_children=case["branch"], distinct=case["draft"] == "distinct")
    return st["n_accept"], st["path"], st["next"]


def _own_commit(st):
    if "p1a" not in st:
        _own_plan(st)
    st["p1a"].tree_commit(st["layers"], _own_rows_of(st), st["n_accept"], st["path"])
    return st["cache"].view(torch.float16)


def _padded(st):
    """sequence by sequence, rows numbered from 0: which there are [seqs, rows], and where they stand among all rows"""
    row0 = st["row0"].long()
    i = torch.arange(st["max_rows"], device="cuda")
    return i[None] < (row0[1:] - row0[:-1])[:, None], (row0[:-1, None] + i[None]).clamp_max(st["t"] - 1)


def _plain_rows(st):
    live, at = _padded(st)
    seqs, r = live.shape
    parent = torch.where(live, st["parent"].long()[at], -1)
    up = torch.arange(r, device="cuda").expand(seqs, r)
    sees = torch.zeros(seqs, r, r + 1, dtype=torch.bool, device="cuda")       # (the last column takes what is above the top)
    depth = torch.zeros(seqs, r, dtype=torch.long, device="cuda")
    for _ in range(st["deep"] + 1):
        sees.scatter_(2, torch.where(up >= 0, up, r)[..., None], True)
        up = torch.where(up >= 0, parent.gather(1, up.clamp_min(0)), -1)
        depth += up >= 0
    bits = torch.zeros(seqs, r, 32 * st["words"], dtype=torch.long, device="cuda")
    bits[..., :r] = sees[..., :r]
    word = (bits.unflatten(-1, (-1, 32)) << torch.arange(32, device="cuda")).sum(-1)
    word = torch.where(word >= 1 << 31, word - (1 << 32), word).int()
    st["mask"].copy_(word[live])
    st["pos"].copy_((st["pos0"].long()[:, None] + depth)[live])
    st["slot"].copy_((st["pos0"].long()[:, None] + torch.arange(r, device="cuda"))[live])
    return st["mask"], st["pos"], st["slot"]


def _plain_tree(st):
    case = st["case"]
    hq, hkv, d, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "seqs"))
    n, r, grp = st["max_n"], st["max_rows"], hq // hkv
    live, at = _padded(st)
    where = st["table"].long()
    k, v = (_decode(case["kv"], st["cache"][0, i][where].flatten(1, 2)[:, :n], d).transpose(1, 2) for i in range(2))
    q = st["q"].float()[at].view(seqs, r, hkv, grp, d).transpose(1, 2).flatten(2, 3)
    bits = (st["mask"][at][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).bool().flatten(2)      # [seqs, rows, nodes]
    front, j = st["pos0"].long()[:, None, None], torch.arange(n, device="cuda")
    seen = j < front
    if case["window"]:
        p = front + bits.sum(-1, keepdim=True) - 1
        seen = seen & ((j > p - case["window"]) | (j < case["sinks"]))
    node = j - front
    inside = bits.gather(2, node.clamp(0, bits.shape[2] - 1).expand(seqs, r, n)) & (node >= 0) & (node < bits.shape[2])
    seen = (seen | inside) & live[..., None]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(st["scale"]).unflatten(2, (r, -1))
    x = x.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.flatten(2, 3), v.contiguous()).unflatten(2, (r, -1)) / total
    lse = (top + total.log()).squeeze(-1)
    out = out.transpose(1, 2).flatten(2, 3)[live]
    if case["gate"]:
        out = out / (1 + torch.exp(-st["gate"])).view_as(out)
    out = out.to(st["out"].dtype)
    return (out, lse.transpose(1, 2).flatten(2, 3)[live]) if case["lse"] else (out,)


def _plain_verify(st):
    """in 64 bits: a token is drawn where the running sum passes a number, next to a border for one of a thousand draws in 32"""
    case = st["case"]
    live, at = _padded(st)
    seqs, r = live.shape
    parent = torch.where(live, st["parent"].long()[at], -1)
    i = torch.arange(r, device="cuda")
    number = ((parent[:, :, None] == parent[:, None, :]) & (i[None, :] < i[:, None])).sum(-1)            # of a node among its siblings
    token, u = st["token"].long()[at], st["u"].double()[at]
    cur = torch.zeros(seqs, dtype=torch.long, device="cuda")
    done = torch.zeros(seqs, dtype=torch.bool, device="cuda")
    n_accept, nxt = torch.zeros_like(cur), torch.full_like(cur, -1)
    path = torch.full((seqs, st["path"].shape[1]), -1, device="cuda")
    for depth in range(st["deep"] + 1):
        row = at.gather(1, cur[:, None]).squeeze(1)
        p = st["target"][row].double()
        if case["target"] == "logits":
            t = st["temp"].double()[:, None]
            e = ((p - p.amax(-1, keepdim=True)) / torch.where(t > 0, t, 1.0)).exp()
            hot = torch.zeros_like(p).scatter_(1, p.argmax(-1, keepdim=True), 1.0)
            p = torch.where(t > 0, e / e.sum(-1, keepdim=True), hot)
        q = None if st["draft"] is None else st["draft"][row].double()
        left, mass, gone = p, torch.ones(seqs, 1, dtype=torch.float64, device="cuda"), torch.zeros(seqs, 1, dtype=torch.float64, device="cuda")
        chosen = torch.full_like(cur, -1)
        for k in range(case["branch"]):
            hit = (parent == cur[:, None]) & (number == k) & live
            c = hit.to(torch.uint8).argmax(1, keepdim=True)
            there = hit.any(1, keepdim=True) & (chosen < 0)[:, None]
            x = token.gather(1, c)
            share = torch.ones_like(mass) if q is None else q.gather(1, x) / (1 - gone)
            yes = there & (u.gather(1, c) * share * mass < left.gather(1, x))
            no = there & ~yes
            chosen = torch.where(yes.squeeze(1), c.squeeze(1), chosen)
            if q is None:
                mass = torch.where(no, mass - left.gather(1, x), mass)
                left = torch.where(no, left.scatter(1, x, 0.0), left)
            else:
                left = torch.where(no, (left - mass / (1 - gone) * q).clamp_min(0), left)
                mass = torch.where(no, left.sum(-1, keepdim=True), mass)
                if case["draft"] == "distinct":
                    gone = torch.where(no, gone + q.gather(1, x), gone)
        ends = ~done & (chosen < 0)
        total = torch.where(left.sum(-1, keepdim=True) > 0, left, p).cumsum(-1)
        pick = (total <= st["u_next"].double()[:, None] * total[:, -1:]).sum(-1)
        nxt = torch.where(ends, pick, nxt)
        done = done | ends
        goes = ~done
        if depth < path.shape[1]:
            path[:, depth] = torch.where(goes, chosen, -1)
        n_accept += goes
        cur = torch.where(goes, chosen, cur)
    st["n_accept"].copy_(n_accept)
    st["path"].copy_(path)
    st["next"].copy_(nxt)
    return st["n_accept"], st["path"], st["next"]


def _plain_commit(st):
    page, cache = st["case"]["page"], st["cache"]
    path, table = st["path"].long(), st["table"].long()
    j = torch.arange(path.shape[1], device="cuda")[None]
    moves = j < st["n_accept"][:, None]
    front = st["pos0"].long()[:, None]
    a, b = torch.where(moves, front + path, 0), torch.where(moves, front + 1 + j, 0)
    s = torch.arange(path.shape[0], device="cuda")[:, None].expand_as(a)[moves]
    a, b = a[moves], b[moves]
    cache[:, :, table[s, b // page], b % page] = cache[:, :, table[s, a // page], a % page]
    return cache.view(torch.float16)
