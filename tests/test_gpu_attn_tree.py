"""kq_tree_plan and kq_attn_tree: trees of drafted tokens against the softmax formula in 64 bits (tolerance derived in
decode_helpers.attention), what no row sees, and how they meet the attention of a chain."""
import math

import pytest
import torch

from decode_helpers import check_attention, make_cache, page_table
from kq import kv, ops
from tree_helpers import chain, random_parents, tree_attention, ways

pytestmark = pytest.mark.gpu


def setup(dev, dtype, D, q_heads, heads, page, base, T, order="heads", seed=0, width=None):
    table, pages = page_table([max(n, 0) + T for n in base], page, extra=1, seed=seed, width=width)
    cache = make_cache(dtype, pages, heads, page, D, dev, seed=seed, order=order)
    g = torch.Generator().manual_seed(seed + 1)
    return cache, table, torch.randn((len(base) * T, q_heads * D), generator=g)


def i32(x, dev):
    return torch.as_tensor(x, dtype=torch.int32, device=dev)


def attend(dev, cache, table, q, base, parents, q_heads, scale=None, max_len=None, out=None):
    T = parents.shape[1]
    att = kv.PagedAttention([cache], table.to(dev), q_heads, nodes=T, max_len=max_len, scale=scale)
    tree = kv.Tree(len(base), T, dev).plan(parents.to(dev), i32(base, dev))
    return att.attend_tree(0, q.to(dev), tree, out)


def check(dev, dtype, D, q_heads, heads, page, base, T, order="heads", seed=0, scale=None, parents=None):
    print("tree", dtype, D, q_heads, heads, page, base, T, order, scale, flush=True)
    cache, table, q = setup(dev, dtype, D, q_heads, heads, page, base, T, order, seed)
    parents = random_parents(len(base), T, seed, roots=True) if parents is None else parents
    got = attend(dev, cache, table, q, base, parents, q_heads, scale)
    ref, bound = tree_attention(cache, table, q, base, parents, q_heads, D ** -0.5 if scale is None else scale)
    check_attention(got, ref, bound)
    # typical roundings add as their squares: far below the worst case of the bound
    if ref.norm() > 0:
        assert float((got.cpu().double() - ref).norm() / ref.norm()) <= 16 * math.sqrt(D) * 2.0 ** -24


@pytest.mark.parametrize("T", [1, 2, 7, 31, 32, 33, 64])
def test_plan(dev, T):
    parents = random_parents(4, T, seed=T, roots=True)
    if T > 4:
        parents[1, 2], parents[1, 4], parents[2, 3], parents[2, 0] = 2, -2, 63, 0
    base = [0, 17, 1 << 30, -1]
    tree = kv.Tree(4, T, dev).plan(parents.to(dev), i32(base, dev))
    seen = tree.seen.cpu()
    got = [t.cpu().view(4, T).tolist() for t in (tree.seq, tree.pos, tree.slot)]
    for b, n in enumerate(base):
        for t, way in enumerate(ways(parents[b])):
            word = sum(1 << j for j in way) if way else 0
            assert int(seen[b, t]) & (2 ** 64 - 1) == word
            there = way is not None and n >= 0
            assert [g[b][t] for g in got] == ([b, n + len(way) - 1, n + t] if there else [-1, -1, -1])
    one = kv.Tree(4, T, dev).plan(parents[:1].to(dev), i32(base, dev))       # one tree for all
    assert all(torch.equal(one.seen[b].cpu(), seen[0]) for b in range(4))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 128, 160, 192, 240, 256])
def test_head_sizes(dev, dtype, D):
    check(dev, dtype, D, 4, 2, 16, [1, 37, 300], 13, seed=D)
    check(dev, dtype, D, 8, 2, 16, [2, 290], 40, seed=D)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("T", [1, 3, 16, 64])
def test_lengths(dev, dtype, T):
    """None, one, and both sides of every tile's, split's and page's end, ahead of the tree and with it."""
    edges = [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 192, 255, 256, 257, 448, 511, 513, 1024 - T]
    check(dev, dtype, 64, 2, 1, 16, edges, T)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("q_heads,heads,T", [(1, 1, 64), (5, 5, 17), (7, 1, 9), (32, 8, 16), (16, 1, 5), (40, 1, 64), (64, 2, 2),
                                             (24, 4, 33)])
def test_head_layouts(dev, dtype, q_heads, heads, T):
    check(dev, dtype, 64, q_heads, heads, 16, [3, 290], T)


@pytest.mark.parametrize("page", [1, 2, 8, 64, 256, 1024])
def test_page_sizes(dev, page):
    for dtype in ("f16", "bf16", "i8"):
        check(dev, dtype, 64, 4, 2, page, [5, 100, 700], 20)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("order", ["positions", "apart"])
def test_orders(dev, dtype, order):
    check(dev, dtype, 128, 8, 2, 16, [40, 333], 20, order=order)
    check(dev, dtype, 80, 3, 3, 32, [40, 333], 5, order=order)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_long(dev, dtype):
    check(dev, dtype, 128, 4, 1, 16, [20011], 24)
    check(dev, dtype, 64, 2, 1, 128, [9000, 17, 30000], 5)


@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0])
def test_scales(dev, scale):
    for dtype in ("f16", "bf16", "i8"):
        check(dev, dtype, 64, 4, 2, 16, [1, 50, 700], 24, scale=scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_large_and_small_values(dev, dtype):
    """Queries and values far from 1, zero queries, and scores apart by more than the exponent's range."""
    D, H, base, T = 64, 4, [300, 41], 21
    parents = random_parents(2, T, 3)
    for qs, vs in ((1e4, 1.0), (1e-20, 1.0), (1.0, 2.0 ** 14), (1.0, 2.0 ** -14), (0.0, 1.0), (30.0, 1.0)):
        cache, table, q = setup(dev, dtype, D, H, 2, 16, base, T)
        (cache.v_scale if dtype == "i8" else cache.v).mul_(vs / (8 if dtype == "f16" and vs > 1 else 1))
        q = q * qs
        print("values", dtype, qs, vs, flush=True)
        got = attend(dev, cache, table, q, base, parents, H)
        check_attention(got, *tree_attention(cache, table, q, base, parents, H, D ** -0.5))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T", [6, 40])
def test_elements_far_apart(dev, dtype, T):
    """Queries whose elements lie 2^60 apart, each beside keys that have only its own dimension: every element keeps its
    24 bits.  f16: keys and values among the subnormals as well."""
    D, H, base = 64, 2, [70]
    cache, table, q = setup(dev, dtype, D, H, 1, 16, base, T)
    q = q * torch.exp2(torch.randint(-30, 31, q.shape, generator=torch.Generator().manual_seed(1)).float())
    cache.k.mul_((torch.arange(16, device=dev)[:, None] % 2 == 0) | (torch.arange(D, device=dev) == 5))
    cache.k[:, :, 1::2, 5] = cache.k[:, :, 1::2, 5] * 2.0 ** -12
    cache.v.mul_(2.0 ** -16)
    q[:, 5] = torch.where(q[:, 5].abs() > 1, 1 / q[:, 5], q[:, 5])
    parents = random_parents(1, T, 4)
    for s in (1.0, 1e-8):
        got = attend(dev, cache, table, q, base, parents, H, scale=s)
        check_attention(got, *tree_attention(cache, table, q, base, parents, H, s))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("T,H", [(5, 2), (20, 8), (64, 4)])
def test_what_no_row_sees_changes_no_bit(dev, dtype, T, H):
    """NaN and infinities past the tree, in slots of nodes that are none, in pages no table names, in table entries past
    the request's."""
    base = [5, 40, 250, 0, 30]
    cache, table, q = setup(dev, dtype, 128, H, 2, 16, base, T, width=40)
    parents = random_parents(len(base), T, 7)
    parents[2, T - 2:] = -5
    base[4] = -1                                     # sits out
    clean = attend(dev, cache, table, q, base, parents, H)
    assert (clean.view(len(base), T, -1)[4] == 0).all() and (clean.view(len(base), T, -1)[2, -2:] == 0).all()
    dirty = torch.ones(cache.k.shape[:3], dtype=torch.bool)
    for b, n in enumerate(base):
        for p in range(n + T if n >= 0 else 0):
            if not (b == 2 and p >= n + T - 2):
                dirty[table[b, p // 16], :, p % 16] = False
    if dtype == "i8":
        cache.k_scale[dirty.to(dev)] = float("nan")
        cache.v_scale[dirty.to(dev)] = float("inf")
        cache.k[dirty.to(dev)] = -128
    else:
        cache.k[dirty.to(dev)] = float("nan")
        cache.v[dirty.to(dev)] = float("inf")
    for b, n in enumerate(base):
        table[b, -(-(n + T) // 16) if n >= 0 else 0:] = 2 ** 31 - 1
    assert torch.equal(attend(dev, cache, table, q, base, parents, H), clean)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("T,H", [(4, 4), (30, 8)])
def test_holes(dev, dtype, T, H):
    """Pages given up are passed over, also those that hold nodes, also when they leave a row nothing."""
    base = [300, 64 - T, 30, 700]
    cache, table, q = setup(dev, dtype, 64, H, 2, 16, base, T)
    table[0, [0, 3, 18]] = torch.tensor([-1, cache.pages, -2 ** 31], dtype=torch.int32)
    table[1] = -1                                   # nothing left
    table[2, 1:] = -7                               # the end of the context, and most of the tree
    table[3, :40] = -1                              # the first 640 positions are gone
    parents = random_parents(4, T, 2, roots=True)
    got = attend(dev, cache, table, q, base, parents, H)
    check_attention(got, *tree_attention(cache, table, q, base, parents, H, 64 ** -0.5))
    assert (got.view(4, T, -1)[1] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 240])
@pytest.mark.parametrize("T,H", [(6, 2), (40, 8)])
@pytest.mark.parametrize("n", [3, 40, 254, 300])
def test_infinities_that_some_nodes_see(dev, dtype, D, T, H, n):
    """Drafts that bring infinities and NaN: nodes that do not see them keep every bit; those that do get them where they
    lie, and the formula's values elsewhere."""
    base = [n, 70]
    cache, table, q = setup(dev, dtype, D, H, 2, 16, base, T, seed=n)
    parents = random_parents(2, T, 1)
    parents[0, :6] = torch.tensor([-1, 0, 0, 1, 2, 2])
    clean = attend(dev, cache, table, q, base, parents, H).view(2, T, H, D)
    bound = tree_attention(cache, table, q, base, parents, H, D ** -0.5)[1].view(2, T, H, D).to(dev)

    def at(t):
        return table[0, (n + t) // 16], (n + t) % 16

    def check(got, want, marked):
        for t, way in enumerate(ways(parents[0])):
            if not marked & set(way):
                assert torch.equal(got[0, t], clean[0, t])
        assert torch.equal(got[1], clean[1])
        fine = torch.isfinite(want)
        torch.testing.assert_close(got[~fine], want[~fine], rtol=0, atol=0, equal_nan=True)
        assert ((got - want).abs()[fine] <= 2 * bound[fine]).all()

    for h, t, d, x in ((0, 1, 3, "inf"), (1, 2, D - 1, "nan"), (0, 4, 5, "-inf")):
        cache.v[at(t)[0], h, at(t)[1], d] = float(x)
    want = clean.clone()
    G = H // 2
    for t, way in enumerate(ways(parents[0])):
        if 1 in way:
            want[0, t, :G, 3] = float("inf")
        if 2 in way:
            want[0, t, G:, D - 1] = float("nan")
        if 4 in way:
            want[0, t, :G, 5] = float("-inf")
    check(attend(dev, cache, table, q, base, parents, H).view(2, T, H, D), want, {1, 2, 4})
    cache.k[at(2)[0], 1, at(2)[1], 0] = float("nan")                    # a NaN key: the row of whoever sees it
    for t, way in enumerate(ways(parents[0])):
        if 2 in way:
            want[0, t, G:] = float("nan")
    check(attend(dev, cache, table, q, base, parents, H).view(2, T, H, D), want, {1, 2, 4})


def test_an_infinity_in_the_context(dev):
    """An infinite value that all see, and an infinite key: queries on its side give it all weight, others none."""
    D, H, T, base = 64, 8, 20, [40]
    for dtype in ("f16", "bf16"):
        cache, table, q = setup(dev, dtype, D, H, 1, 16, base, T)
        parents = random_parents(1, T, 1)
        q = q.abs() + 0.1
        clean = attend(dev, cache, table, q, base, parents, H).view(T, H, D)
        cache.v[table[0, 1], 0, 3, 7] = float("-inf")
        got = attend(dev, cache, table, q, base, parents, H).view(T, H, D)
        bound = tree_attention(cache, table, q, base, parents, H, D ** -0.5)[1].view(T, H, D).to(dev)
        assert (got[..., 7] == float("-inf")).all()
        rest = torch.arange(D, device=dev) != 7
        assert ((got - clean).abs() <= 2 * bound)[..., rest].all()
        cache.v[table[0, 1], 0, 3, 7] = 1.0
        cache.k[table[0, 0], 0, 5] = cache.k[table[0, 0], 0, 5].abs().clamp(max=2)
        cache.k[table[0, 0], 0, 5, 9] = float("-inf")                   # a score of -inf: no weight
        got = attend(dev, cache, table, q, base, parents, H)
        assert torch.isfinite(got).all()
        far = attend(dev, _without(cache, table, 5), table, q, base, parents, H).view(T, H, D)
        assert ((got.view(T, H, D) - far).abs() <= 4 * bound)[..., rest].all()


def _without(cache, table, p):
    """The cache with position p of request 0 so far off that it has no weight."""
    k = cache.k.clone()
    k[table[0, p // 16], 0, p % 16] = 0
    k[table[0, p // 16], 0, p % 16, 9] = -30000
    return kv.KVCache.over(k, cache.v)


def test_bounds(dev):
    """Bases above max_len or the table's positions; nodes past either are not there; negative bases."""
    T, H = 6, 4
    cache, table, q = setup(dev, "bf16", 64, H, 2, 16, [58, 58, 58], T)
    parents = random_parents(3, T, 5)
    full = dict(cache=cache, table=table, q=q, parents=parents, q_heads=H)
    for base, most in (([58, 61, 64], None), ([58, 20, 3], 60), ([58, 70, 1 << 30], 59), ([100, 2 ** 31 - 1, -(2 ** 31)], None)):
        got = attend(dev, base=base, max_len=most, **full)
        check_attention(got, *tree_attention(base=base, scale=64 ** -0.5, max_len=most, **full))


@pytest.mark.parametrize("dtype,D", [("f16", 128), ("bf16", 128), ("i8", 80), ("bf16", 256)])
def test_a_chain_is_the_attention_of_its_tokens(dev, dtype, D):
    """A chain sees what kq_attn_paged's tokens see: both within the bound of the same formula."""
    T, H, lens = 5, 8, [700, 1300, 12, 256]
    cache, table, q = setup(dev, dtype, D, H, 2, 16, [n - T for n in lens], T)
    got = attend(dev, cache, table, q, [n - T for n in lens], chain(4, T), H)
    att = kv.PagedAttention([cache], table.to(dev), H, tokens=T)
    want = att.attend(0, q.to(dev), i32(lens, dev))
    _, bound = tree_attention(cache, table, q, [n - T for n in lens], chain(4, T), H, D ** -0.5)
    assert ((got - want).cpu().double().abs() <= 2 * bound).all()


@pytest.mark.parametrize("dtype,D,T,H", [("f16", 128, 7, 8), ("bf16", 128, 40, 8), ("i8", 80, 16, 4), ("bf16", 256, 24, 16)])
def test_a_row_does_not_depend_on_other_requests(dev, dtype, D, T, H):
    """The same bits beside requests of other lengths, trees and contents, with its pages elsewhere, call after call."""
    base = [700, 1300, 12, 256]
    cache, table, q = setup(dev, dtype, D, H, 2, 16, base, T)
    parents = random_parents(4, T, 1)
    rows = attend(dev, cache, table, q, base, parents, H, max_len=2000).view(4, T, -1)
    for b in range(4):
        others, p = [5, -1, 900, 40], random_parents(4, T, 9)
        others[b], p[b] = base[b], parents[b]
        again = attend(dev, cache, table, torch.where(torch.arange(4 * T)[:, None] // T == b, q, q.flip(0)), others, p, H, max_len=2000)
        assert torch.equal(again.view(4, T, -1)[b], rows[b])
    perm = torch.randperm(cache.pages)
    moved = kv.KVCache.over(*[x[perm.to(dev)] if x is not None else None
                              for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    back = torch.argsort(perm).int()
    there = torch.where(table >= 0, back[table.clamp(min=0).long()], -1).int()
    assert torch.equal(attend(dev, moved, there, q, base, parents, H, max_len=2000).view(4, T, -1), rows)


def test_strided_rows(dev):
    """Queries out of a fused projection's rows, outputs into wider rows, both from odd floats on."""
    for T, H in ((2, 4), (24, 8)):
        base, D = [77, 300], 64
        cache, table, q = setup(dev, "bf16", D, H, 2, 16, base, T)
        parents = random_parents(2, T, 1)
        wide = torch.zeros(2 * T, H * D + 133, device=dev)
        wide[:, 3:3 + H * D] = q.to(dev)
        out = torch.full((2 * T, H * D + 9), 7.0, device=dev)
        attend(dev, cache, table, wide[:, 3:3 + H * D], base, parents, H, out=out[:, 5:5 + H * D])
        assert torch.equal(out[:, 5:5 + H * D], attend(dev, cache, table, q, base, parents, H))
        assert (out[:, :5] == 7).all() and (out[:, 5 + H * D:] == 7).all()


def test_offsets_past_32_bits(dev):
    """A request in the last pages of a pool whose offsets pass 2^32."""
    D, page, heads = 128, 16, 8
    pages = 2 ** 32 // (D * page * heads) + 40
    k, v = (torch.empty((pages, heads, page, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.ones((pages, heads, page), device=dev) for _ in range(2))
    for T in (2, 33):
        small, table, q = setup(dev, "i8", D, 16, heads, page, [300], T)
        for big, x in ((k, small.k), (v, small.v), (ks, small.k_scale), (vs, small.v_scale)):
            big[-small.pages:] = x
        parents = random_parents(1, T, 1)
        got = attend(dev, kv.KVCache.over(k, v, ks, vs), table + (pages - small.pages), q, [300], parents, 16)
        assert torch.equal(got, attend(dev, small, table, q, [300], parents, 16))


@pytest.mark.parametrize("T", [6, 48])
def test_other_stream_and_graph(dev, T):
    """On a stream of its own, and captured with the plan: parents, bases, tables and queries are read when the graph runs."""
    base, H = [600, 40], 8
    cache, table, q = setup(dev, "bf16", 128, H, 2, 16, base, T)
    td, qd, pd, bd = table.to(dev), q.to(dev), random_parents(2, T, 1).to(dev), i32(base, dev)
    att, tree = kv.PagedAttention([cache], td, H, nodes=T), kv.Tree(2, T, dev)
    want = att.attend_tree(0, qd, tree.plan(pd, bd))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = att.attend_tree(0, qd, tree.plan(pd, bd))
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.attend_tree(0, qd, tree.plan(pd, bd), out)
    for i, n in enumerate((600, 17, 599, 1, 0, -1)):
        bd.fill_(min(n, 40))
        bd[0] = n
        pd.copy_(random_parents(2, T, i))
        qd.normal_()
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        seen = tree.seen.clone()
        assert torch.equal(out, att.attend_tree(0, qd, tree.plan(pd, bd)))
        assert torch.equal(seen, tree.seen)


def test_repeated_calls_leave_the_workspace_ready(dev):
    """Calls of trees of changing sizes and of chains on one workspace: each as on a new one."""
    H, D = 8, 64
    cache, table, _ = setup(dev, "bf16", D, H, 2, 16, [2000, 900, 40], 64)
    att = kv.PagedAttention([cache], table.to(dev), H, tokens=16, nodes=64)
    g = torch.Generator().manual_seed(3)
    for i in range(24):
        T = [1, 4, 64, 16][i % 4]
        base = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in (2000, 900, 40)]
        q = torch.randn((3 * T, H * D), generator=g)
        if i % 4 == 3:
            lens = i32([n + T for n in base], dev)
            got = att.attend(0, q.to(dev), lens, tokens=T)
            assert torch.equal(got, kv.PagedAttention([cache], table.to(dev), H, tokens=T).attend(0, q.to(dev), lens))
            continue
        parents = random_parents(3, T, i)
        got = att.attend_tree(0, q.to(dev), kv.Tree(3, T, dev).plan(parents.to(dev), i32(base, dev)))
        assert torch.equal(got, attend(dev, cache, table, q, base, parents, H)), (i, base)


def test_workspace_grows_with_its_sizes():
    base = ops.attn_tree_workspace_bytes(4, 8, 64, 4, 5000)
    for more in ((8, 8, 64, 4, 5000), (4, 16, 64, 4, 5000), (4, 8, 128, 4, 5000), (4, 8, 64, 64, 5000), (4, 8, 64, 4, 50000)):
        assert ops.attn_tree_workspace_bytes(*more) >= base


def test_refusals_on_the_device(dev):
    """Device tensors of another type, too small, of another layout or left out: refused before any launch."""
    H, D, T = 4, 64, 6
    cache, table, q = setup(dev, "bf16", D, H, 2, 16, [40, 40], T)
    att = kv.PagedAttention([cache], table.to(dev), H, nodes=T)
    tree, q = kv.Tree(2, T, dev), q.to(dev)
    parents, base = chain(2, T).to(dev), i32([40, 40], dev)
    for a in ((parents.long(), base), (parents[:, :-1], base), (parents[0], base), (parents.t().contiguous().t(), base),
              (parents, base.long()), (parents, base[:1]), (parents, base.cpu()), (None, base), (parents, None),
              (torch.cat([parents, parents])[:0], base)):
        with pytest.raises(ValueError):
            tree.plan(*a)
    tree.plan(parents, base)
    for a in ((q.half(), tree), (q[:-1], tree), (q[:, :-1], tree), (q.t().contiguous().t(), tree), (q.cpu(), tree),
              (q, kv.Tree(2, T, dev)), (q, tree, torch.empty_like(q)[:-1]), (q, tree, q.half())):
        with pytest.raises(ValueError):
            att.attend_tree(0, *a)
    assert att.attend_tree(0, q, tree).shape == q.shape
