"""kq_kv_keep: the accepted nodes' entries moved together, entry for entry, and nothing else written."""
import numpy as np
import pytest
import torch

from decode_helpers import make_cache, page_table
from kq import kv

pytestmark = pytest.mark.gpu


def moved(full, table, base, path, page, pages):
    """What a pool [pages][heads][page]... holds afterwards (numpy)."""
    out = full.copy()
    for b, n in enumerate(base):
        cap = table.shape[1] * page
        last = -1
        for i, j in enumerate(path[b].tolist()):
            if j < i or j <= last or j >= path.shape[1]:
                break
            last = j
            if n < 0 or n + j >= cap or i == j:
                continue
            src, dst = int(table[b, (n + j) // page]), int(table[b, (n + i) // page])
            if 0 <= src < pages and 0 <= dst < pages:
                out[dst, :, (n + i) % page] = full[src, :, (n + j) % page]
    return out


def paths(requests, nodes, seed):
    """Rising paths of every length from the root, some through neighbouring nodes."""
    rng = np.random.default_rng(seed)
    p = np.full((requests, nodes), -1, np.int32)
    for b in range(requests):
        n = rng.integers(1, nodes + 1) if b else nodes
        p[b, :n] = np.sort(rng.permutation(nodes)[:n])
    return torch.from_numpy(p)


def check(dev, caches, table, base, path, page):
    att = kv.PagedAttention(caches, table.to(dev), caches[0].heads)
    names = [n for n in ("k", "v", "k_scale", "v_scale")]

    def hold(t):
        return None if t is None else (t.cpu().contiguous().view(torch.int16).numpy() if t.element_size() == 2 else t.cpu().numpy()).copy()

    before = [[hold(getattr(c, n)) for n in names] for c in caches]
    att.keep(path.to(dev), torch.tensor(base, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    for c, full in zip(caches, before):
        for n, x in zip(names, full):
            if x is not None:
                np.testing.assert_array_equal(hold(getattr(c, n)), moved(x, table, base, path, page, c.pages))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("D,heads,page,T", [(16, 1, 16, 1), (16, 1, 1, 5), (64, 2, 16, 8), (80, 3, 4, 33), (128, 8, 16, 64),
                                            (256, 4, 64, 24), (240, 40, 8, 64)])
@pytest.mark.parametrize("order", ["heads", "positions", "apart"])
def test_paths(dev, dtype, D, heads, page, T, order):
    print("keep", dtype, D, heads, page, T, order, flush=True)
    base = [0, 1, 15, 16, 40, 7]
    table, pages = page_table([n + T for n in base], page, extra=2)
    caches = [make_cache(dtype, pages, heads, page, D, dev, seed=i, order=order) for i in range(2)]
    check(dev, caches, table, base, paths(len(base), T, T), page)


@pytest.mark.parametrize("layers", [1, 31, 32, 33, 70])
def test_layers(dev, layers):
    """More layers than a launch takes, of types and orders of their own."""
    base, T = [3, 20], 12
    table, pages = page_table([n + T for n in base], 16, extra=1)
    caches = [make_cache(["f16", "bf16", "i8"][i % 3], pages, 2, 16, 64, dev, seed=i, order=["heads", "apart"][i % 2])
              for i in range(layers)]
    check(dev, caches, table, base, paths(2, T, layers), 16)


def test_paths_that_end(dev):
    """At the first entry that names no node: below its place, not above the one before, past the tree."""
    T = 8
    path = torch.tensor([[0, 2, 2, 5, 6, -1, -1, -1], [0, 3, 1, 4, -1, -1, -1, -1], [1, 2, 3, 4, 5, 6, 7, 8],
                         [0, 2, 2 ** 31 - 1, 3, -1, -1, -1, -1], [-1, 1, 2, 3, 4, 5, 6, 7], [0, -2 ** 31, 5, 6, -1, -1, -1, -1],
                         [0, 1, 2, 3, 4, 5, 6, 7], [7, -1, -1, -1, -1, -1, -1, -1]], dtype=torch.int32)
    base = [5] * 8
    table, pages = page_table([16] * 8, 4)
    check(dev, [make_cache("bf16", pages, 2, 4, 64, dev)], table, base, path, 4)


def test_holes_and_bounds(dev):
    """Entries from or into pages that are not there, slots past the table, requests that sit out: nothing is moved."""
    T, page = 12, 4
    path = torch.tensor([[0, 2, 4, 5, 7, 9, 11] + [-1] * 5] * 6, dtype=torch.int32)
    base = [2, 2, 20, -1, 2 ** 31 - 1, -(2 ** 31)]
    table, pages = page_table([24] * 6, page)
    table[0, 1], table[1, 2] = -1, pages
    check(dev, [make_cache("i8", pages, 2, page, 32, dev)], table, base, path, page)


def test_offsets_past_32_bits(dev):
    D, page, heads = 128, 16, 8
    pages = 2 ** 32 // (D * page * heads) + 40
    k, v = (torch.empty((pages, heads, page, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.ones((pages, heads, page), device=dev) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    k[-2:].random_(-100, 100)
    want = k[pages - 2, :, 3].clone()
    cache = kv.KVCache.over(k, v, ks, vs)
    kv.PagedAttention([cache], table, heads).keep(torch.tensor([[0, 9]], dtype=torch.int32, device=dev)[:, :2].repeat(1, 1),
                                                  torch.tensor([10], dtype=torch.int32, device=dev))
    assert not torch.equal(k[pages - 1, :, 11], want)          # node 9 of a tree of two is none
    path = torch.full((1, 10), -1, dtype=torch.int32, device=dev)
    path[0, 0], path[0, 1] = 0, 9
    kv.PagedAttention([cache], table, heads).keep(path, torch.tensor([10], dtype=torch.int32, device=dev))
    assert torch.equal(k[pages - 1, :, 11], want)


def test_stream_and_graph(dev):
    base, T = [3, 20], 12
    table, pages = page_table([n + T for n in base], 16, extra=1)
    caches = [make_cache("bf16", pages, 2, 16, 64, dev, seed=i) for i in range(3)]
    held = [(c.k.clone(), c.v.clone()) for c in caches]
    att = kv.PagedAttention(caches, table.to(dev), 2)
    path, bd = paths(2, T, 0).to(dev), torch.tensor(base, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.keep(path, bd)
    for i in range(4):
        path.copy_(paths(2, T, i))
        bd[0] = i
        for c, (k, v) in zip(caches, held):
            c.k.copy_(k), c.v.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for c, (k, v) in zip(caches, held):
            for x, y in ((c.k, k), (c.v, v)):
                want = moved(y.cpu().view(torch.int16).numpy(), table, bd.tolist(), path.cpu(), 16, pages)
                np.testing.assert_array_equal(x.cpu().view(torch.int16).numpy(), want)


def test_refusals_on_the_device(dev):
    table, pages = page_table([32, 32], 16)
    cache = make_cache("bf16", pages, 2, 16, 64, dev)
    att = kv.PagedAttention([cache], table.to(dev), 2)
    path, base = torch.zeros(2, 8, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    before = cache.k.clone()
    for a in ((path.long(), base), (path[:1], base), (path[0], base), (path, base.long()), (path, base[:1]), (path.cpu(), base),
              (path, base.cpu()), (None, base), (path, None), (path.t().contiguous().t(), base), (path.repeat(1, 9), base),
              (path[:, :0], base)):
        with pytest.raises(ValueError):
            att.keep(*a)
    torch.cuda.synchronize()
    assert torch.equal(cache.k, before)


@pytest.mark.parametrize("layers", [2, 33, 64])
def test_layers_that_share_a_cache(dev, layers):
    """Their entries move once, among a launch's layers and across launches."""
    base, T = [3, 20], 12
    table, pages = page_table([n + T for n in base], 16, extra=1)
    own = [make_cache("bf16", pages, 2, 16, 64, dev, seed=i) for i in range(max(layers - 2, 1))]
    check(dev, own + [own[0]] * (layers - len(own)), table, base, paths(2, T, 5), 16)
