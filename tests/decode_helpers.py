"""Inputs and plain 64-bit forms for the tests of the paged cache, its attention and the penalised pick."""
import numpy as np
import torch

from kq import kv

U = 2.0 ** -24                     # half a step of fp32, relative


def page_table(lens, page, width=None, extra=0, seed=0):
    """Table [requests][width] of pages in a random order, -1 past a request's; and the pool's size."""
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    pages = sum(need) + extra
    order = np.random.default_rng(seed).permutation(max(pages, 1))
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table), max(pages, 1)


def make_cache(dtype, pages, heads, page, dim, dev, seed=0, order="heads", fill=None):
    """A cache of random values; order: "heads" [pages][heads][page][dim], "positions" [pages][page][heads][dim], or
    "apart": inside a larger tensor, so that no stride is the natural one."""
    g = torch.Generator().manual_seed(seed)
    dt = kv.DTYPES[dtype]
    shape = (pages, heads, page, dim)

    def put(x):
        if order == "positions":
            return x.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        if order == "apart":
            big = torch.zeros((pages, heads + 1, page + 1, *[n + 16 for n in x.shape[3:]]), dtype=x.dtype).to(dev)
            view = big[:, 1:, 1:, 16:] if x.dim() == 4 else big[:, 1:, 1:]
            view.copy_(x)
            return view
        return x.to(dev)

    if dtype == "i8":
        k, v = (torch.randint(-127, 128, shape, generator=g, dtype=dt) for _ in range(2))
        scales = [put((1 + torch.rand(shape[:3], generator=g)) / 64) for _ in range(2)]
    else:
        k, v = (torch.randn(shape, generator=g).to(dt) for _ in range(2))
        scales = [None, None]
    return kv.KVCache.over(put(k), put(v), *scales)


def values(cache, name):
    """The pool's values in 64 bits on the CPU, [pages][heads][page][dim]."""
    x = getattr(cache, name).cpu().double()
    if cache.k.dtype == torch.int8:
        x = x * getattr(cache, name + "_scale").cpu().double()[..., None]
    return x


def attention(cache, table, q, lens, T, q_heads, scale):
    """(out, bound) in 64 bits: the formula's rows [requests * T][q_heads * dim], and how far an fp32 evaluation may be.

    A score is a sum of dim products in fp32: off by at most (dim + 8) u sum|q k| scale, with u = 2^-24 (the products'
    splits, the scale and the exponent's argument in the 8).  exp turns a score's error into a relative one of its
    probability, and a softmax into at most twice the largest.  The sum over positions is a chain of
    at most len / 4 + 64 roundings of partial sums below sum p |v|."""
    K, V = values(cache, "k"), values(cache, "v")
    D, G, P = cache.dim, q_heads // cache.heads, cache.page_size
    q = q.cpu().double().view(len(lens), T, q_heads, D)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(lens):
        pos = torch.arange(max(n, 0))
        page = table[b].long()[pos // P]
        there = (page >= 0) & (page < cache.pages)
        page, off, pos = page[there], (pos % P)[there], pos[there]
        for h in range(q_heads):
            k, v = K[page, h // G, off], V[page, h // G, off]
            for t in range(T):
                see = pos < n - T + 1 + t
                if not see.any():
                    continue
                x = q[b, t, h]
                p = torch.softmax(scale * (k[see] @ x), 0)
                out[b, t, h] = p @ v[see]
                reach = abs(scale) * float((k[see].abs() @ x.abs()).max())
                bound[b, t, h] = U * (2 * (D + 8) * reach + n / 4 + 64) * (p @ v[see].abs())
    return out.view(len(lens) * T, -1), bound.view(len(lens) * T, -1)


def check_attention(got, ref, bound):
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() / bound.clamp(min=1e-300))[bound > 0]
    assert (got[bound == 0] == 0).all()
    assert worst.numel() == 0 or float(worst.max()) <= 1, float(worst.max())
