"""Operators for sequences in bounded caches, as a server that runs many long sessions calls them.

A case is one of three kinds of pass over a paged cache (pages of all sequences in random order in one pool), one layer:

  "chunk"  attention of the new tokens of several sequences - from one token each to whole prompts, ragged - over the keys each of them sees:
           all up to its own position, or the last `window` of them and the first `sinks` positions.
  "mass"   the attention weight that those rows give to every position, summed over rows and the heads of a kv head's group, added to a
           running total per (sequence, kv head, position).
  "evict"  per (sequence, kv head) the `budget` positions that stay - the first `sinks`, the last `recent`, and those of the largest total
           between - and the kept rows of K and V moved to the front of the sequence's pages, the totals with them.

Values are N(0, 1), keys and queries RMS-normed per head, totals log-normal.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

KV_TYPES = {"f16": 1, "q4_0": 2, "q8_0": 8}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def _chunk(name, kv, heads, kv_heads, dim, page, seqs, rows, ctx, rows_min=None, ctx_min=None, window=0, sinks=0, gate=False, lse=False, q="f32", out="f32"):
    return {"name": name, "kind": "chunk", "kv": kv, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": seqs, "rows": rows,
            "rows_min": rows if rows_min is None else rows_min, "ctx": ctx, "ctx_min": ctx if ctx_min is None else ctx_min, "window": window,
            "sinks": sinks, "gate": gate, "lse": lse, "q": q, "out": out}


def _mass(name, kv, heads, kv_heads, dim, page, seqs, rows, ctx, rows_min=None, ctx_min=None, window=0, sinks=0, q="f32"):
    c = _chunk(name, kv, heads, kv_heads, dim, page, seqs, rows, ctx, rows_min, ctx_min, window, sinks, q=q)
    for k in ("gate", "lse", "out"):
        del c[k]
    return dict(c, kind="mass")


def _evict(name, heads, kv_heads, dim, page, seqs, ctx, budget, ctx_min=None, sinks=4, recent=64):
    return {"name": name, "kind": "evict", "kv": "f16", "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "seqs": seqs, "ctx": ctx,
            "ctx_min": ctx if ctx_min is None else ctx_min, "budget": budget, "sinks": sinks, "recent": recent}


def listed():
    return [
        # one token of the smallest model the tests run, a short window: what a call costs when there is next to nothing to compute
        _chunk("one_d64_f16_w256", "f16", 4, 1, 64, 16, 1, 1, 700, window=256, sinks=4),
        # a full decode step of 32 long sessions of the 27B shape, each seeing 4096 positions and its first four
        _chunk("step32_27b_q8_w4k", "q8_0", 24, 4, 256, 256, 32, 1, 32768, ctx_min=300, window=4096, sinks=4, gate=True),
        # a serving step that mixes prompts' chunks with single tokens, whole contexts, heads of 128, results for a bf16 product
        _chunk("mixed24_d128_f16", "f16", 32, 8, 128, 16, 24, 500, 7000, rows_min=1, ctx_min=500, q="bf16", out="bf16"),
        # first prompts of eight chats, no key behind them
        _chunk("prompts8_27b_f16", "f16", 24, 4, 256, 64, 8, 2003, 2003, rows_min=77, ctx_min=77, gate=True, out="bf16"),
        # a long document in chunks through a window: what is visible is bounded, however far the document has come
        _chunk("doc_27b_f16_w4k", "f16", 24, 4, 256, 256, 1, 4096, 32768, window=4096, sinks=64, out="bf16"),
        # a short turn of four chats over compact caches, statistics kept for the weights, everything in f32
        _chunk("turns4_d128_q4_w2k", "q4_0", 32, 8, 128, 64, 4, 150, 16000, rows_min=17, ctx_min=900, window=2048, sinks=16, lse=True),
        # weights of one decode step of 32 sequences
        _mass("mass_step32_27b_q8", "q8_0", 24, 4, 256, 256, 32, 1, 8190, ctx_min=1000),
        # weights that the last tokens of a long prompt give, before it is cut down
        _mass("mass_tail_d128_f16", "f16", 32, 8, 128, 16, 1, 64, 30011, q="bf16"),
        # weights of whole prompts
        _mass("mass_prompts4_27b_f16", "f16", 24, 4, 256, 64, 4, 2003, 4099, rows_min=300, ctx_min=600),
        # one short session of the smallest model over its budget
        _evict("evict_one_d64", 4, 1, 64, 16, 1, 1100, 1024),
        # sixteen sessions of the 27B shape cut from up to twice their budget
        _evict("evict16_27b", 24, 4, 256, 256, 16, 8190, 4096, ctx_min=4200, sinks=4, recent=512),
        # a long prompt cut to a tenth
        _evict("evict_prompt_d128", 32, 8, 128, 64, 1, 100003, 10000, sinks=16, recent=1000),
    ]


HEADS = [(4, 1), (24, 4), (16, 2), (32, 8), (8, 8), (16, 4)]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        heads, kv_heads = rng.choice(HEADS)
        dim, page = rng.choice([64, 128, 256]), rng.choice([16, 64, 256])
        kind = rng.choice(["chunk", "chunk", "chunk", "mass", "mass", "evict"])
        if kind == "evict":
            ctx, seqs = _log_uniform(rng, 200, 100003), rng.choice([1, 1, 2, 4, 16])
            budget = max(150, int(ctx / rng.uniform(1.05, 10)))
            sinks, recent = rng.choice([0, 4, 16]), rng.choice([0, 64, budget // 8])
            c = _evict("", heads, kv_heads, dim, page, seqs, ctx, budget, ctx_min=max(1, ctx // rng.choice([1, 2, 4])), sinks=sinks, recent=recent)
        else:
            kv, q = rng.choice(["f16", "q8_0", "q4_0"]), rng.choice(["f32", "f32", "bf16"])
            seqs = rng.choice([1, 1, 2, 4, 8, 32])
            rows = rng.choice([1, 1, _log_uniform(rng, 2, 64), _log_uniform(rng, 64, 4096)])
            ctx = _log_uniform(rng, max(64, rows), 32768)
            window = rng.choice([0, 0, _log_uniform(rng, 16, 8192)])
            at = dict(rows_min=max(1, rows // rng.choice([1, 4, 16])), ctx_min=max(1, ctx // rng.choice([1, 4, 16])), window=window,
                      sinks=rng.choice([0, 4, 64]) if window else 0, q=q)
            if kind == "chunk":
                c = _chunk("", kv, heads, kv_heads, dim, page, seqs, rows, ctx, gate=rng.random() < 0.5, lse=rng.random() < 0.3,
                           out=rng.choice(["f32", "bf16"]), **at)
            else:
                c = _mass("", kv, heads, kv_heads, dim, page, seqs, rows, ctx, **at)
        del c["name"]
        n, pool = max(_lengths(c)), sum(_lengths(c)) * kv_heads * dim
        scores = 0 if kind == "evict" else seqs * max(_row_counts(c)) * heads * n
        if pool <= 1.3e8 and seqs * n * kv_heads * dim <= 5.5e8 and scores <= 3.3e9 and work(c)["flops"] <= 4.3e11:
            return c


def _spread(n, lo, hi, seed):
    """n whole numbers, evenly spread over the logarithm from lo to hi, in an order that is not sorted"""
    if n == 1:
        return [hi]
    at = random.Random(seed).sample(range(n), n)
    return [max(1, int(round(lo * (hi / lo) ** (a / (n - 1))))) for a in at]


def _row_counts(case):
    return _spread(case["seqs"], case["rows_min"], case["rows"], 1)


def _lengths(case):
    """the sequences' lengths, the new tokens included"""
    n = _spread(case["seqs"], case["ctx_min"], case["ctx"], 2)
    return n if case["kind"] == "evict" else [max(a, r) for a, r in zip(n, _row_counts(case))]


def _pairs(case):
    """visible (row, key) pairs, and keys that some row sees"""
    pairs = union = 0
    w, sinks = case["window"], case["sinks"]
    for n, r in zip(_lengths(case), _row_counts(case)):
        p = np.arange(n - r, n)
        seen = p + 1 if not w else np.minimum(p + 1, w + np.minimum(sinks, np.maximum(p - w + 1, 0)))
        pairs += int(seen.sum())
        low = max(0, n - r - w + 1) if w else 0
        union += n - low + min(sinks, low)
    return pairs, union


def work(case):
    hkv, d, hq = case["kv_heads"], case["dim"], case["heads"]
    hb = _head_bytes(case["kv"], d)
    if case["kind"] == "evict":
        kept = sum(max(0, min(n, case["budget"]) - case["sinks"]) if n > case["budget"] else 0 for n in _lengths(case))
        return {"bytes": 4 * hkv * sum(_lengths(case)) + 4 * hkv * case["seqs"] * case["budget"] + 4 * hkv * kept * hb + 8 * hkv * kept, "flops": 0}
    pairs, union = _pairs(case)
    t = sum(_row_counts(case))
    size = {"f32": 4, "bf16": 2}
    if case["kind"] == "mass":
        return {"bytes": t * hq * (d * size[case["q"]] + 4) + union * hkv * (hb + 8), "flops": 2 * hq * d * pairs}
    rows = t * hq * d * (size[case["q"]] + size[case["out"]] + (4 if case["gate"] else 0)) + (4 * t * hq if case["lse"] else 0)
    return {"bytes": rows + 2 * union * hkv * hb, "flops": 4 * hq * d * pairs}


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


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    hq, hkv, d, page, seqs, kv = (case[k] for k in ("heads", "kv_heads", "dim", "page", "seqs", "kv"))
    lens = _lengths(case)
    per = [-(-n // page) for n in lens]
    n_pages, max_pages = sum(per) + 2, max(per)
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.zeros(seqs, max_pages, dtype=torch.int32, device="cuda")
    at = 0
    for s, p in enumerate(per):
        table[s, :p] = order[at: at + p]
        at += p
    hb = _head_bytes(kv, d)
    k, v = (torch.empty(n_pages, page, hkv, hb, dtype=torch.uint8, device="cuda") for _ in range(2))
    step = max(1, (1 << 25) // (page * hkv * d))
    for a in range(0, n_pages, step):
        m = min(step, n_pages - a)
        k[a: a + m] = _encode(kv, _normed(randn(m, page, hkv, d)))
        v[a: a + m] = _encode(kv, randn(m, page, hkv, d))
    st = {"case": case, "k": k, "v": v, "table": table, "offsets": (torch.arange(seqs, device="cuda") * max_pages).int(), "max_n": max(lens)}
    if case["kind"] == "evict":
        ld = max(lens)
        st["mass"] = (2 * randn(seqs, hkv, ld)).exp()
        st["n"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["keep"] = torch.empty(seqs, hkv, case["budget"], dtype=torch.int32, device="cuda")
        st["mass_out"] = torch.zeros_like(st["mass"])
        return st
    rows = _row_counts(case)
    t = sum(rows)
    st["t"], st["max_rows"] = t, max(rows)
    st["row0"] = torch.tensor([0] + list(np.cumsum(rows)), dtype=torch.int32, device="cuda")
    st["pos0"] = torch.tensor([n - r for n, r in zip(lens, rows)], dtype=torch.int32, device="cuda")
    st["q"] = _normed(randn(t, hq, d)).to(TYPES[case["q"]])
    st["scale"] = d ** -0.5
    if case["kind"] == "mass":
        st["mass"] = torch.rand(seqs, hkv, max(lens), generator=g, device="cuda") * (2 * hq / hkv / max(lens))   # (as a step before this one left it)
        st["lse"] = torch.cat([x[1] for x in _rows64(st, values=False)]).float()
        return st
    st["gate"] = randn(t, hq * d) if case["gate"] else None
    st["out"] = torch.empty(t, hq, d, dtype=TYPES[case["out"]], device="cuda")
    st["lse"] = torch.empty(t, hq, device="cuda") if case["lse"] else None
    return st


# ---- the definition in 64 bits, sequence by sequence ----
def _rows64(st, values=True):
    """per sequence (out [rows, heads, D], lse [rows, heads], weights' sum per (kv head, position))"""
    case = st["case"]
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    grp, page, got = hq // hkv, case["page"], []
    row0, pos0 = st["row0"].tolist(), st["pos0"].tolist()
    for s in range(case["seqs"]):
        r, p0 = row0[s + 1] - row0[s], pos0[s]
        n = p0 + r
        where = st["table"][s, : -(-n // page)].long()
        heads = [_decode(case["kv"], x[where].flatten(0, 1)[:n], d, torch.float64) for x in ((st["k"], st["v"]) if values else (st["k"],))]
        q = st["q"][row0[s]: row0[s + 1]].double()
        out, lse = torch.zeros(r, hq, d, dtype=torch.float64, device="cuda"), torch.zeros(r, hq, dtype=torch.float64, device="cuda")
        total = torch.zeros(hkv, n, dtype=torch.float64, device="cuda")
        most = max(1, int(2e8 // (n * grp)))
        for a in range(0, r, most):
            b = min(r, a + most)
            p, j = (p0 + torch.arange(a, b, device="cuda"))[:, None], torch.arange(n, device="cuda")[None]
            seen = j <= p
            if case["window"]:
                seen &= (j > p - case["window"]) | (j < case["sinks"])
            for h in range(hkv):
                x = torch.matmul(q[a:b, h * grp: (h + 1) * grp].reshape(-1, d), heads[0][:, h].t().contiguous()).mul_(st["scale"]).view(b - a, grp, n)
                x.masked_fill_(~seen[:, None], -math.inf)
                z = torch.logsumexp(x, -1)
                lse[a:b, h * grp: (h + 1) * grp] = z
                if not values and "lse" not in st:
                    continue
                x.sub_(z[..., None] if values else st["lse"][row0[s] + a: row0[s] + b, h * grp: (h + 1) * grp].double()[..., None]).exp_()
                if values:
                    out[a:b, h * grp: (h + 1) * grp] = torch.matmul(x.view(-1, n), heads[1][:, h].contiguous()).view(b - a, grp, d)
                else:
                    total[h] += x.sum((0, 1))
        got.append((out, lse, total))
    return got


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(st)
    got = _rows64(st, values=case["kind"] == "chunk")
    if case["kind"] == "mass":
        total = st["mass"].double()
        for s, x in enumerate(got):
            total[s, :, : x[2].shape[1]] += x[2]
        return total
    out = torch.cat([x[0] for x in got])
    if case["gate"]:
        out = out / (1 + torch.exp(-st["gate"].double())).view_as(out)
    return (out, torch.cat([x[1] for x in got])) if case["lse"] else (out,)


def _exact_evict(st):
    case = st["case"]
    page, budget = case["page"], case["budget"]
    k, v = (x.view(torch.float16).double() for x in (st["k"], st["v"]))
    mass, table = st["mass"].double().cpu().numpy(), st["table"].cpu().numpy()
    keep, left = np.full(tuple(st["keep"].shape), -1, np.int32), np.zeros_like(mass)
    for s, n in enumerate(st["n"].tolist()):
        for h in range(case["kv_heads"]):
            m = mass[s, h, :n]
            if n <= budget:
                chosen = np.arange(n)
            else:
                mid = np.arange(case["sinks"], n - case["recent"])
                best = mid[np.lexsort((mid, -m[mid]))[: budget - case["sinks"] - case["recent"]]]
                chosen = np.sort(np.concatenate([np.arange(case["sinks"]), best, np.arange(n - case["recent"], n)]))
            keep[s, h, : len(chosen)] = chosen
            left[s, h, : len(chosen)] = m[chosen]
            src, dst = (torch.from_numpy(x).cuda() for x in (chosen, np.arange(len(chosen))))
            where = torch.from_numpy(table[s]).cuda().long()
            for x in (k, v):
                x[where[dst // page], dst % page, h] = x[where[src // page], src % page, h]
    return (torch.from_numpy(keep).cuda(), k, v, torch.from_numpy(left).cuda())


# ---- one pass ----
def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"chunk": _own_chunk, "mass": _own_mass, "evict": _own_evict}[kind](st)
    return {"chunk": _plain_chunk, "mass": _plain_mass, "evict": _plain_evict}[kind](st)


def _own_cache(p1a, st):
    case = st["case"]
    page, rows = case["page"], st["table"].shape[1]
    return p1a.KVCache(KV_TYPES[case["kv"]], rows * page, case["kv_heads"], case["dim"], st["k"].data_ptr(), st["v"].data_ptr(), pt=st["table"],
                       rtab=st["offsets"], psh=page.bit_length() - 1, pstride=st["k"].stride(0))


def _own_rows(p1a, st):
    case = st["case"]
    return p1a.Rows(st["t"], n_seq=case["seqs"], row0=st["row0"], pos0=st["pos0"], max_rows=st["max_rows"], max_n=st["max_n"], window=case["window"],
                    n_sink=case["sinks"])


def _own_chunk(st):
    p1a = importlib.import_module("p100e-engine_amd")
    p1a.attn_chunk(st["q"], _own_cache(p1a, st), st["out"], _own_rows(p1a, st), st["case"]["heads"], st["scale"], gate=st["gate"], lse=st["lse"])
    return (st["out"], st["lse"]) if st["lse"] is not None else (st["out"],)


def _own_mass(st):
    p1a = importlib.import_module("p100e-engine_amd")
    p1a.attn_mass(st["q"], _own_cache(p1a, st), st["lse"], st["mass"], _own_rows(p1a, st), st["case"]["heads"], st["scale"])
    return st["mass"]


def _own_evict(st):
    p1a = importlib.import_module("p100e-engine_amd")
    case = st["case"]
    p1a.evict_select(st["mass"], st["n"], st["keep"], n_sink=case["sinks"], n_recent=case["recent"])
    p1a.kv_compact(_own_cache(p1a, st), st["keep"], mass=st["mass"], mass_out=st["mass_out"])
    return st["keep"], st["k"].view(torch.float16), st["v"].view(torch.float16), st["mass_out"]


def _padded(st):
    """keys [seqs, kv heads, keys, D], values, queries [seqs, kv heads, rows * group, D] and what is seen [seqs, rows, keys], in 32 bits"""
    case = st["case"]
    hq, hkv, d, page, seqs = (case[k] for k in ("heads", "kv_heads", "dim", "page", "seqs"))
    n, r = st["max_n"], st["max_rows"]
    where = st["table"].long()
    k, v = (_decode(case["kv"], x[where].flatten(1, 2)[:, :n], d).transpose(1, 2) for x in (st["k"], st["v"]))
    row0, pos0 = st["row0"].long(), st["pos0"].long()
    count = row0[1:] - row0[:-1]
    i = torch.arange(r, device="cuda")
    live = i[None] < count[:, None]
    at = (row0[:-1, None] + i[None]).clamp_max(st["t"] - 1)
    q = st["q"].float()[at].view(seqs, r, hkv, hq // hkv, d).transpose(1, 2).flatten(2, 3)
    p, j = (pos0[:, None] + i[None])[..., None], torch.arange(n, device="cuda")
    seen = j <= p
    if case["window"]:
        seen = seen & ((j > p - case["window"]) | (j < case["sinks"]))
    return k, v, q, seen, live, at


def _scores(st, k, q, seen):
    """[seqs, kv heads, rows, group, keys], -inf where a row does not see the key"""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(st["scale"])
    x = x.unflatten(2, (st["max_rows"], -1))
    return x.masked_fill_(~seen[:, None, :, None], -math.inf)


def _plain_chunk(st):
    case = st["case"]
    k, v, q, seen, live, at = _padded(st)
    x = _scores(st, k, q, seen)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.flatten(2, 3), v.contiguous()).unflatten(2, (st["max_rows"], -1)) / total
    lse = (top + total.log()).squeeze(-1)
    out = out.transpose(1, 2).flatten(2, 3)[live]
    if case["gate"]:
        out = out / (1 + torch.exp(-st["gate"])).view_as(out)
    out = out.to(st["out"].dtype)
    return (out, lse.transpose(1, 2).flatten(2, 3)[live]) if case["lse"] else (out,)


def _plain_mass(st):
    k, _, q, seen, live, at = _padded(st)
    x = _scores(st, k, q, seen)
    lse = st["lse"][at].unflatten(-1, (st["case"]["kv_heads"], -1)).transpose(1, 2)
    x = x.sub_(lse[..., None]).exp_().mul_(live[:, None, :, None, None])
    st["mass"] += x.sum((2, 3))
    return st["mass"]


def _plain_evict(st):
    case = st["case"]
    seqs, hkv, budget, sinks, page = case["seqs"], case["kv_heads"], case["budget"], case["sinks"], case["page"]
    mass, n = st["mass"], st["n"].long()[:, None, None]
    ld = mass.shape[-1]
    j = torch.arange(ld, device="cuda")
    rank = mass.masked_fill((j < sinks) | ((j >= n - case["recent"]) & (j < n)), math.inf).masked_fill(j >= n, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    best = torch.where(best < n, best, ld).sort(-1).values
    if ld < budget:
        best = torch.cat([best, torch.full((seqs, hkv, budget - ld), ld, device="cuda")], -1)
    kept = best < n
    st["keep"].copy_(torch.where(kept, best, -1))
    src = torch.where(kept, best, 0)
    dst = torch.arange(budget, device="cuda").expand_as(src)
    s, h = torch.arange(seqs, device="cuda")[:, None, None].expand_as(src), torch.arange(hkv, device="cuda")[None, :, None].expand_as(src)
    where = st["table"].long()
    s, h, src, dst = s[kept], h[kept], src[kept], dst[kept]
    for x in (st["k"], st["v"]):
        x[where[s, dst // page], dst % page, h] = x[where[s, src // page], src % page, h]
    st["mass_out"].zero_()
    st["mass_out"][s, h, dst] = mass[s, h, src]
    return st["keep"], st["k"].view(torch.float16), st["v"].view(torch.float16), st["mass_out"]
