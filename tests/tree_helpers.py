"""Plain forms for the tests of trees of drafted tokens: what a tree's parents say, its attention and its verification in
64 bits on the CPU."""
import numpy as np
import torch

from decode_helpers import U, values


def random_parents(requests, nodes, seed=0, roots=False):
    """int32 [requests][nodes]: each node after some earlier one; roots: sometimes after the context itself."""
    rng = np.random.default_rng(seed)
    p = np.full((requests, nodes), -1, np.int32)
    for b in range(requests):
        for t in range(1, nodes):
            p[b, t] = rng.integers(-1 if roots else 0, t)
    return torch.from_numpy(p)


def chain(requests, nodes):
    return torch.arange(-1, nodes - 1, dtype=torch.int32).repeat(requests, 1)


def ways(parents):
    """For each node of one tree the nodes from its first ancestor to itself; None where it is no node."""
    out = []
    for t, p in enumerate(int(x) for x in parents):
        if p < -1 or p >= t or (p >= 0 and out[p] is None):
            out.append(None)
        else:
            out.append((out[p] if p >= 0 else []) + [t])
    return out


def tree_attention(cache, table, q, base, parents, q_heads, scale, max_len=None):
    """(out, bound) in 64 bits, as decode_helpers.attention with what each node sees: the same derivation."""
    K, V = values(cache, "k"), values(cache, "v")
    D, G, P, T = cache.dim, q_heads // cache.heads, cache.page_size, parents.shape[1]
    most = table.shape[1] * P if max_len is None else min(max_len, table.shape[1] * P)
    q = q.cpu().double().view(len(base), T, q_heads, D)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(base):
        for t, way in enumerate(ways(parents[b if parents.shape[0] > 1 else 0])):
            if n < 0 or way is None:
                continue
            pos = torch.tensor([p for p in list(range(min(n, most))) + [n + j for j in way] if p < most], dtype=torch.long)
            page = table[b].long()[pos // P]
            there = (page >= 0) & (page < cache.pages)
            page, off = page[there], (pos % P)[there]
            if not len(page):
                continue
            for h in range(q_heads):
                k, v, x = K[page, h // G, off], V[page, h // G, off], q[b, t, h]
                p = torch.softmax(scale * (k @ x), 0)
                out[b, t, h] = p @ v
                reach = abs(scale) * float((k.abs() @ x.abs()).max())
                bound[b, t, h] = U * (2 * (D + 8) * reach + (n + T) / 4 + 64) * (p @ v.abs())
    return out.view(len(base) * T, -1), bound.view(len(base) * T, -1)


def probabilities(x, temperature):
    """softmax(x / temperature) of one row in 64 bits; greedy: the first of the largest alone; None: nothing has any."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return None
    p = np.zeros(len(x))
    if not temperature > 0:
        p[int(x.argmax())] = 1
        return p
    if top == np.inf:
        p[x == np.inf] = 1
    else:
        p = np.exp((x - top) / np.float64(np.float32(temperature)))
    return p / p.sum()


def verification(x, tokens, parents, uniform, temperature=None, draft=None):
    """[(accepted, path, token, gap)] for each request, all arguments numpy arrays: gap is the smallest distance of a
    comparison from its border, in probability."""
    out = []
    B, T = tokens.shape
    for b in range(B):
        up = parents[b if len(parents) > 1 else 0]
        if up[0] != -1:
            out.append((-1, [-1] * T, -1, 1.0))
            continue
        temp = 1.0 if temperature is None else float(temperature[b])
        cur, path, gap = 0, [0], 1.0
        while True:
            p = probabilities(x[b * T + cur], temp)
            if p is None:
                break
            q = None if draft is None else draft[b * T + cur].astype(np.float64)
            left, Z, a, nxt = p.copy(), 1.0, 0.0, None
            for c in range(1, T):
                if up[c] != cur or c <= cur or not 0 <= tokens[b, c] < len(p):
                    continue
                tok, u = int(tokens[b, c]), float(uniform[b, c])
                lhs = u * Z * (1.0 if q is None else q[tok])
                if lhs < left[tok]:
                    nxt = c
                if left[tok] > 0 or lhs > 0:
                    gap = min(gap, abs(lhs - left[tok]) / (1 + a))
                if nxt is not None:
                    break
                if q is None:
                    Z -= left[tok]
                    left[tok] = 0
                else:
                    a += Z
                    left = np.maximum(p - a * q, 0)
                    Z = left.sum()
            if nxt is None:
                break
            cur = nxt
            path.append(nxt)
        token = -1
        if p is not None:
            if not left.sum() > 0:
                left = p
            run = left.cumsum()
            target = float(uniform[b, 0]) * run[-1]
            token = int(np.argmax(run > target))
            gap = min(gap, abs(run[token] - target) / (1 + a), abs(target - (run[token - 1] if token else -1)) / (1 + a))
        out.append((len(path) - 1, path + [-1] * (T - len(path)), token, gap))
    return out


# Weights are off by some 1e-14 of themselves (2^z by a polynomial, its argument by 2^-53 of up to 1000), sums of up to 2^18 of
# them by as much again: comparisons nearer than this may fall either way.
NEAR = 1e-12
