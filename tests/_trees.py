"""Trees of drafted tokens: random trees, and what the operators on them are to give, in 64 bits."""
import numpy as np
import torch


def tree(g, n, branch=3):
    """parents of n nodes, at most `branch` children each"""
    parent, kids = [-1] * min(n, 1), [0] * n
    for i in range(1, n):
        free = [j for j in range(max(0, i - 12), i) if kids[j] < branch]
        p = int(free[g.integers(len(free))])
        kids[p] += 1
        parent.append(p)
    return parent


def paths(parent):
    """[n][n] bool: node i sees node j; [n] depths"""
    n = len(parent)
    see, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i, p in enumerate(parent):
        if 0 <= p < i:
            see[i] = see[p]
            depth[i] = depth[p] + 1
        see[i, i] = True
    return see, depth


def words_of(see, words):
    """[n][m] bool -> [n][words] int32"""
    out = np.zeros((see.shape[0], words * 32), np.uint8)
    m = min(see.shape[1], words * 32)
    out[:, :m] = see[:, :m]
    return np.packbits(out, axis=1, bitorder="little").view(np.uint32).view(np.int32).reshape(see.shape[0], words)


def sees(see, pos0, n_ctx, window, n_sink):
    """[rows][positions]: positions 0 .. of the sequence that rows with in-tree masks see [rows][rows]"""
    n = see.shape[0]
    end = max(min(pos0 + n, n_ctx), 0)
    j = np.arange(end)[None]
    p = pos0 + np.maximum(see.sum(1) - 1, 0)[:, None]
    m = np.broadcast_to(j < pos0, (n, end)).copy()
    if window:
        m &= (j > p - window) | (j < n_sink)
    for b in range(n):
        if 0 <= pos0 + b < end:
            m[:, pos0 + b] |= see[:, b]
    slot = pos0 + np.arange(n)
    m[(slot < 0) | (slot >= n_ctx)] = False
    return m


def distribution(row, logits, temp):
    """float64 [V] weights of a row of the target (all 0: it has none)"""
    x = row.astype(np.float64)
    if not logits:
        return np.where(x > 0, x, 0.0)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    if not temp > 0:
        return (np.arange(len(x)) == x.argmax()).astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(temp)))
    w[np.isnan(w)] = 0
    return w / w.sum()


def verify(target, token, parent, u, u_next, draft=None, temp=1.0, logits=True, max_children=1 << 30, distinct=False):
    """one sequence: (accepted nodes, next token). target, draft float arrays [n][V]"""
    n, V = target.shape[0], target.shape[1]
    if n == 0:
        return [], -1
    kids = [[c for c in range(1, n) if parent[c] == r and parent[c] < c and 0 <= token[c] < V] for r in range(n)]
    at, path = 0, []
    while True:
        p = distribution(target[at], logits, temp)
        left, mass, gone, chosen = p.copy(), 1.0, 0.0, -1
        q = None if draft is None else np.where(draft[at] > 0, draft[at].astype(np.float64), 0.0)
        for c in kids[at][:max_children] if draft is not None else kids[at]:
            x = token[c]
            if q is None:
                if float(u[c]) * mass < left[x]:
                    chosen = c
                    break
                mass -= left[x]
                left[x] = 0
                continue
            if not 1 - gone > 0:
                continue
            if float(u[c]) * (q[x] / (1 - gone)) * mass < left[x]:
                chosen = c
                break
            left = np.maximum(left - mass / (1 - gone) * q, 0)
            mass = left.sum()
            if distinct:
                gone += q[x]
        if chosen < 0:
            break
        path.append(chosen)
        at = chosen
    if not left.sum() > 0:
        left = p
    total = np.cumsum(left)
    if not total[-1] > 0:
        return path, -1
    over = np.nonzero((total > float(u_next) * total[-1]) & (left > 0))[0]
    return path, int(over[0]) if len(over) else int(np.nonzero(left > 0)[0][-1])


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def bf16_values(x):
    """the values of a float array as bf16 holds them"""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).float().numpy()
