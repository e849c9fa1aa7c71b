"""kq_attn_paged against the softmax formula in 64 bits (tolerance derived in decode_helpers.attention), its masks, and
its contract that a row's result depends on its query, its cache and its length alone."""
import math

import pytest
import torch

from decode_helpers import attention, check_attention, make_cache, page_table
from kq import kv, ops

pytestmark = pytest.mark.gpu


def setup(dev, dtype, D, q_heads, heads, page, lens, T, order="heads", seed=0, width=None):
    table, pages = page_table(lens, page, extra=1, seed=seed, width=width)
    cache = make_cache(dtype, pages, heads, page, D, dev, seed=seed, order=order)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((len(lens) * T, q_heads * D), generator=g)
    return cache, table, q


def attend(dev, cache, table, q, lens, T, q_heads, scale=None, max_len=None, out=None):
    att = kv.PagedAttention([cache], table.to(dev), q_heads, tokens=T, max_len=max_len, scale=scale)
    return att.attend(0, q.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), out)


def check(dev, dtype, D, q_heads, heads, page, lens, T=1, order="heads", seed=0, scale=None):
    print("attention", dtype, D, q_heads, heads, page, lens, T, order, scale, flush=True)
    cache, table, q = setup(dev, dtype, D, q_heads, heads, page, lens, T, order, seed)
    got = attend(dev, cache, table, q, lens, T, q_heads, scale)
    ref, bound = attention(cache, table, q, lens, T, q_heads, D ** -0.5 if scale is None else scale)
    check_attention(got, ref, bound)
    # typical roundings add as their squares: far below the worst case of the bound
    if ref.norm() > 0:
        assert float((got.cpu().double() - ref).norm() / ref.norm()) <= 16 * math.sqrt(D) * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 128, 160, 192, 240, 256])
def test_head_sizes(dev, dtype, D):
    check(dev, dtype, D, 4, 2, 16, [1, 37, 300, 770], seed=D)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_lengths(dev, dtype):
    """None, one, and both sides of every tile's, split's and page's end."""
    check(dev, dtype, 128, 4, 1, 16, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512,
                                      513, 1023, 1024, 1025])


@pytest.mark.parametrize("dtype", ["bf16", "i8"])
@pytest.mark.parametrize("q_heads,heads", [(1, 1), (5, 5), (7, 1), (32, 8), (16, 1), (17, 1), (40, 1), (64, 2)])
def test_head_layouts(dev, dtype, q_heads, heads):
    check(dev, dtype, 64, q_heads, heads, 16, [3, 290])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("T", [2, 3, 4, 5, 8, 16])
def test_tokens(dev, dtype, T):
    """Drafted tokens: each sees up to itself; a request shorter than the draft leaves its first rows empty."""
    check(dev, dtype, 128, 8, 2, 16, [T, 0, 1, T - 1, 100, 257, 513], T=T)
    check(dev, dtype, 256, 12, 2, 64, [T + 40, 300], T=T)


@pytest.mark.parametrize("page", [1, 2, 8, 64, 256, 1024])
def test_page_sizes(dev, page):
    check(dev, "bf16", 64, 4, 2, page, [5, 100, 700])
    check(dev, "i8", 64, 4, 2, page, [5, 100, 700])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("order", ["positions", "apart"])
def test_orders(dev, dtype, order):
    check(dev, dtype, 128, 8, 2, 16, [40, 333], order=order)
    check(dev, dtype, 80, 3, 3, 32, [40, 333], T=2, order=order)


def test_strided_rows(dev):
    """Queries out of a fused projection's rows, outputs into wider rows, both from odd floats on."""
    lens, T, H, D = [77, 300], 2, 4, 64
    cache, table, q = setup(dev, "bf16", D, H, 2, 16, lens, T)
    wide = torch.zeros(4, H * D + 133, device=dev)
    wide[:, 3:3 + H * D] = q.to(dev)
    out = torch.full((4, H * D + 9), 7.0, device=dev)
    attend(dev, cache, table, wide[:, 3:3 + H * D], lens, T, H, out=out[:, 5:5 + H * D])
    assert torch.equal(out[:, 5:5 + H * D], attend(dev, cache, table, q, lens, T, H))
    assert (out[:, :5] == 7).all() and (out[:, 5 + H * D:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "i8"])
def test_long(dev, dtype):
    check(dev, dtype, 128, 4, 1, 16, [20011])
    check(dev, dtype, 64, 2, 1, 128, [9000, 17, 40000], T=2)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-3, 3.0])
def test_scales(dev, scale):
    """No scale at all averages; a large one leaves one position."""
    check(dev, "bf16", 64, 4, 2, 16, [1, 50, 700], scale=scale)
    check(dev, "f16", 64, 4, 2, 16, [1, 50, 700], scale=scale)
    check(dev, "i8", 64, 4, 2, 16, [1, 50, 700], scale=scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_large_and_small_values(dev, dtype):
    """Queries and values far from 1, zero queries, and scores apart by more than the exponent's range."""
    D, H, lens = 64, 4, [300, 41]
    for qs, vs in ((1e4, 1.0), (1e-20, 1.0), (1.0, 2.0 ** 14), (1.0, 2.0 ** -14), (0.0, 1.0), (30.0, 1.0)):
        cache, table, q = setup(dev, dtype, D, H, 2, 16, lens, 1)
        (cache.v_scale if dtype == "i8" else cache.v).mul_(vs / (8 if dtype == "f16" and vs > 1 else 1))
        q = q * qs
        print("values", dtype, qs, vs, flush=True)
        got = attend(dev, cache, table, q, lens, 1, H)
        check_attention(got, *attention(cache, table, q, lens, 1, H, D ** -0.5))


def test_scales_far_apart_in_an_8_bit_cache(dev):
    """Positions whose value scales differ by 2^40, and rows of zeros (scale 0)."""
    D, H, lens = 64, 4, [500]
    cache, table, q = setup(dev, "i8", D, H, 2, 16, lens, 1)
    cache.v_scale.mul_(torch.exp2(torch.randint(-20, 21, cache.v_scale.shape, device=dev).float()))
    cache.k_scale[:, :, 3] = 0
    cache.v_scale[:, :, 5] = 0
    check_attention(attend(dev, cache, table, q, lens, 1, H), *attention(cache, table, q, lens, 1, H, D ** -0.5))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("T", [1, 3])
def test_nothing_past_the_length_is_used(dev, dtype, T):
    """NaN and infinities in the rest of a request's last page, in pages that no table names and in table entries past
    the request's pages change no bit."""
    lens = [5, 40, 257, 0]
    cache, table, q = setup(dev, dtype, 128, 8, 2, 16, lens, T, width=40)
    clean = attend(dev, cache, table, q, lens, T, 8)
    dirty = torch.ones(cache.k.shape[:3], dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            dirty[table[b, p // 16], :, p % 16] = False
    if dtype == "i8":
        cache.k_scale[dirty.to(dev)] = float("nan")
        cache.v_scale[dirty.to(dev)] = float("inf")
        cache.k[dirty.to(dev)] = -128
    else:
        cache.k[dirty.to(dev)] = float("nan")
        cache.v[dirty.to(dev)] = float("inf")
    for b, n in enumerate(lens):
        table[b, -(-n // 16):] = 2 ** 31 - 1
    assert torch.equal(attend(dev, cache, table, q, lens, T, 8), clean)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_holes(dev, dtype):
    """Pages given up (-1, or any number outside the pool) are passed over, also when they leave a row nothing."""
    lens, H, T = [300, 64, 30, 700], 4, 2
    cache, table, q = setup(dev, dtype, 64, H, 2, 16, lens, T)
    table[0, [0, 3, 18]] = torch.tensor([-1, cache.pages, -2 ** 31], dtype=torch.int32)
    table[1] = -1                                   # nothing left
    table[2, 1] = -7                                # the last page
    table[3, :40] = -1                              # a window: the first 640 positions are gone
    got = attend(dev, cache, table, q, lens, T, H)
    ref, bound = attention(cache, table, q, lens, T, H, 64 ** -0.5)
    check_attention(got, ref, bound)
    assert (got.view(4, T, -1)[1] == 0).all()


def test_infinite_and_nan_positions_that_are_seen(dev):
    """What a row sees counts: an infinite value gives an infinite output, a NaN key a NaN row; other rows keep theirs."""
    lens, H, D = [40, 40], 2, 64
    cache, table, q = setup(dev, "bf16", D, H, 2, 16, lens, 1)
    clean = attend(dev, cache, table, q, lens, 1, H)
    cache.v[table[0, 2], 0, 7, 5] = float("inf")     # position 39, the last
    cache.k[table[1, 0], 1, 3, 0] = float("nan")
    got = attend(dev, cache, table, q, lens, 1, H).view(2, H, D)
    want = clean.view(2, H, D).clone()
    want[0, 0, 5] = float("inf")
    want[1, 1] = float("nan")
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


def test_lengths_past_the_bounds(dev):
    """Lengths above max_len or above the table's positions count as those; negative ones as none."""
    cache, table, q = setup(dev, "bf16", 64, 4, 2, 16, [64, 64, 64], 1)
    full = attend(dev, cache, table, q, [64, 50, 0], 1, 4)
    assert torch.equal(attend(dev, cache, table, q, [1 << 30, 50, -5], 1, 4), full)
    assert torch.equal(attend(dev, cache, table, q, [1 << 30, 50, -(1 << 31)], 1, 4, max_len=1 << 29), full)
    short = attend(dev, cache, table, q, [33, 33, 0], 1, 4)
    assert torch.equal(attend(dev, cache, table, q, [64, 50, 0], 1, 4, max_len=33), short)


@pytest.mark.parametrize("dtype,D", [("f16", 128), ("bf16", 128), ("i8", 128), ("bf16", 256), ("i8", 80)])
def test_a_row_depends_on_nothing_else(dev, dtype, D):
    """The same bits alone, in a batch, as one token or among drafted ones, under another bound, with other pages."""
    H, T, lens = 8, 5, [700, 1300, 12, 256]
    cache, table, q = setup(dev, dtype, D, H, 2, 16, lens, T)
    rows = attend(dev, cache, table, q, lens, T, H).view(len(lens), T, -1)
    qs = q.view(len(lens), T, -1)
    for t in range(T):
        one = attend(dev, cache, table, qs[:, t].contiguous(), [n - T + 1 + t for n in lens], 1, H, max_len=5000)
        assert torch.equal(one, rows[:, t])
    for b, n in enumerate(lens):
        alone = attend(dev, cache, table[b:b + 1], qs[b], [n], T, H)
        assert torch.equal(alone, rows[b])
    perm = torch.randperm(cache.pages)
    moved = kv.KVCache.over(*[x[perm.to(dev)] if x is not None else None
                              for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)])
    back = torch.argsort(perm).int()
    there = torch.where(table >= 0, back[table.clamp(min=0).long()], -1).int()
    assert torch.equal(attend(dev, moved, there, q, lens, T, H).view(len(lens), T, -1), rows)


def test_offsets_past_32_bits(dev):
    """A request in the last pages of a pool whose offsets pass 2^32."""
    D, page, heads = 128, 16, 8
    pages = 2 ** 32 // (D * page * heads) + 40
    k, v = (torch.empty((pages, heads, page, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.ones((pages, heads, page), device=dev) for _ in range(2))
    small, table, q = setup(dev, "i8", D, 16, heads, page, [300], 1)
    for big, x in ((k, small.k), (v, small.v), (ks, small.k_scale), (vs, small.v_scale)):
        big[-small.pages:] = x
    got = attend(dev, kv.KVCache.over(k, v, ks, vs), table + (pages - small.pages), q, [300], 1, 16)
    assert torch.equal(got, attend(dev, small, table, q, [300], 1, 16))


def test_other_stream_and_graph(dev):
    """On a stream of its own, and captured: lengths, tables and queries are read when the graph runs."""
    lens, H, T = [600, 40], 8, 2
    cache, table, q = setup(dev, "bf16", 128, H, 2, 16, lens, T)
    td, qd = table.to(dev), q.to(dev)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    att = kv.PagedAttention([cache], td, H, tokens=T)
    want = att.attend(0, qd, ld)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = att.attend(0, qd, ld)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.attend(0, qd, ld, out)
    for n in (600, 17, 599, 1, 0):
        ld.fill_(min(n, 40))
        ld[0] = n
        qd.normal_()
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, att.attend(0, qd, ld))


def test_fewer_tokens_than_the_workspace_holds(dev):
    lens, H = [90, 300], 4
    cache, table, q = setup(dev, "bf16", 64, H, 2, 16, lens, 1)
    att = kv.PagedAttention([cache], table.to(dev), H, tokens=16)
    got = att.attend(0, q.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), tokens=1)
    assert torch.equal(got, attend(dev, cache, table, q, lens, 1, H))


def test_workspace_grows_with_its_sizes():
    base = ops.attn_paged_workspace_bytes(4, 8, 64, 1, 5000)
    for more in ((8, 8, 64, 1, 5000), (4, 16, 64, 1, 5000), (4, 8, 128, 1, 5000), (4, 8, 64, 2, 5000), (4, 8, 64, 1, 50000)):
        assert ops.attn_paged_workspace_bytes(*more) >= base


@pytest.mark.parametrize("dtype,D,T", [("bf16", 128, 1), ("f16", 256, 4), ("i8", 80, 3)])
def test_a_longer_bound_changes_no_bit(dev, dtype, D, T):
    """Tables for contexts of one chunk, of some and of very many: the joins that each leads to agree."""
    H, lens = 8, [130, 256, 0, 3]
    cache, table, q = setup(dev, dtype, D, H, 2, 16, lens, T)
    narrow = attend(dev, cache, table, q, lens, T, H)
    for width in (17, 100, 1200, 40000):
        wide = torch.full((len(lens), width), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        assert torch.equal(attend(dev, cache, wide, q, lens, T, H), narrow), width
    lens = [700, 5000, 255, 1025]
    cache, table, q = setup(dev, dtype, D, H, 2, 16, lens, T)
    here = attend(dev, cache, table, q, lens, T, H)
    for width in (3000, 10000, 40000):              # one, two and four chunks a workgroup
        wide = torch.full((len(lens), width), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        assert torch.equal(attend(dev, cache, wide, q, lens, T, H), here), width


def test_repeated_calls_leave_the_workspace_ready(dev):
    """Calls of changing tokens, lengths and bounds on one workspace: each as on a new one."""
    H, D = 8, 64
    cache, table, _ = setup(dev, "bf16", D, H, 2, 16, [2000, 900, 40], 1)
    att = kv.PagedAttention([cache], table.to(dev), H, tokens=16)
    g = torch.Generator().manual_seed(3)
    for i in range(30):
        T = [1, 4, 16][i % 3]
        lens = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in (2000, 900, 40)]
        q = torch.randn((3 * T, H * D), generator=g)
        got = att.attend(0, q.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), tokens=T)
        assert torch.equal(got, attend(dev, cache, table, q, lens, T, H)), (i, lens)


def test_refusals_on_the_device(dev):
    """Device tensors of another type, too small, of another layout or left out: refused before any launch."""
    H, D = 4, 64
    cache, table, q = setup(dev, "bf16", D, H, 2, 16, [40, 40], 1)
    att = kv.PagedAttention([cache], table.to(dev), H, rope=kv.rope_table(64, D, device=dev))
    q, lens = q.to(dev), torch.tensor([40, 40], dtype=torch.int32, device=dev)
    new = torch.randn(2, 2 * D, device=dev)
    seq, pos = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 1], [39, 39]))
    before = cache.k.clone()
    for a in ((q.half(), lens), (q[:1], lens), (q[:, :-1], lens), (q.t().contiguous().t(), lens), (q.view(-1), lens),
              (q, lens.long()), (q, lens[:1]), (q, None), (q.cpu(), lens), (None, lens, torch.empty_like(q))):
        with pytest.raises(ValueError):
            att.attend(0, *a)
    for a in ((q, new.half(), new, seq, pos), (q, new, new[:1], seq, pos), (q, new, new[:, :-1], seq, pos),
              (q, new, new, seq.long(), pos), (q, new, new, seq, pos[:1]), (q, new, new, None, pos), (q[:1], new, new, seq, pos),
              (q, new, new, torch.stack([seq, seq], 1)[:, 0], pos), (None, new, new, seq, pos, q)):
        with pytest.raises(ValueError):
            att.append(0, *a)
    torch.cuda.synchronize()
    assert torch.equal(cache.k, before)
    att.append(0, q, new, new, seq, pos)
    assert not torch.equal(cache.k, before)


@pytest.mark.parametrize("dtype,D,q_heads", [("bf16", 64, 4), ("f16", 128, 8), ("f16", 256, 4), ("bf16", 240, 6)])
@pytest.mark.parametrize("n", [3, 40, 258, 515])
def test_infinities_that_some_tokens_see(dev, dtype, D, q_heads, n):
    """Drafted tokens that bring infinities and NaN: each row is what it is alone, at its own length."""
    T, heads, lens = 5, 2, [n, 700]
    cache, table, q = setup(dev, dtype, D, q_heads, heads, 16, lens, T, seed=n)
    page, off = (table[0, (n - 1) // 16], (n - 1) % 16), (table[0, max(n - 3, 0) // 16], max(n - 3, 0) % 16)
    cache.v[page[0], 1, page[1], 7] = float("inf")
    cache.v[off[0], 0, off[1], D - 1] = float("nan")
    cache.k[off[0], 1, off[1], 0] = float("-inf")
    rows = attend(dev, cache, table, q, lens, T, q_heads).view(2, T, -1)
    qs = q.view(2, T, -1)
    for t in range(T):
        alone = attend(dev, cache, table, qs[:, t].contiguous(), [m - T + 1 + t for m in lens], 1, q_heads)
        torch.testing.assert_close(rows[:, t], alone, rtol=0, atol=0, equal_nan=True)
    assert torch.isfinite(rows[1]).all() and not torch.isfinite(rows[0, -1]).all()
    wide = torch.full((2, 60000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    torch.testing.assert_close(attend(dev, cache, wide, q, lens, T, q_heads).view(2, T, -1), rows, rtol=0, atol=0, equal_nan=True)
