"""Attention of trees where fp32's range and each number's own 24 bits count, against the formula in 64 bits."""
import math

import pytest
import torch

from decode_helpers import U, attention, check_attention, values
from test_gpu_attn_range import sinks
from test_gpu_attn_tree import attend, setup
from tree_helpers import chain, tree_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("gap", [12, 25, 40, 80])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 40), (256, 5)])
def test_weights_far_below_the_largest(dev, dtype, gap, D, T):
    lens = [T + n for n in (8, 65, 700, 4096)]
    print("tree sinks", dtype, gap, D, T, flush=True)
    cache, table, q = sinks(dev, dtype, D, gap, lens, T)
    got = attend(dev, cache, table, q, [n - T for n in lens], chain(4, T), 2, scale=1.0)
    check_attention(got, *attention(cache, table, q, lens, T, 2, 1.0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gap", [0, 20, 80, 120, 1000])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 40), (256, 4)])
def test_infinite_values_of_small_weight(dev, dtype, gap, D, T):
    """An infinity or NaN that a row sees counts however small its weight, in whichever part of the context it lies; the other
    columns keep their sums."""
    lens = [700, 40]
    print("tree infinite values", dtype, gap, D, T, flush=True)
    cache, table, q = sinks(dev, dtype, D, gap, lens, T)
    # one in a tile with a position that takes all the weight, one in a tile without
    hits = [(330, 10), (100, 20)]
    for p, d in hits:
        cache.v[table[0, p // 16], 0, p % 16:p % 16 + 2, d:d + 4] = 0
    ref, bound = attention(cache, table, q, lens, T, 2, 1.0)
    # exp(-120) is below fp32's least normal number 2^-126: such a weight may be lost, and with it 2^-126 |v| a position
    bound += 2.0 ** -126 * 700 * float(cache.v.abs().max())
    for p, d in hits:
        page, off = table[0, p // 16], p % 16
        cache.v[page, 0, off, d:d + 4] = torch.tensor([math.inf, -math.inf, math.nan, math.inf], device=dev).to(cache.v.dtype)
        cache.v[page, 0, off + 1, d + 3] = -math.inf
    got = attend(dev, cache, table, q, [n - T for n in lens], chain(2, T), 2, scale=1.0).view(2, T, 2, D)
    for p, d in hits:
        hit = got[0, :, :, d:d + 4].cpu()
        assert (hit[..., 0] == math.inf).all() and (hit[..., 1] == -math.inf).all() and hit[..., 2:].isnan().all()
        for x in (got, ref.view(2, T, 2, D), bound.view(2, T, 2, D)):
            x[0, :, :, d:d + 4] = 0
    check_attention(got.view(2 * T, -1), ref, bound)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 20), (240, 4)])
def test_infinite_keys_that_are_seen(dev, dtype, D, T):
    """A key of -inf in one channel: no weight where the query is positive there, however small, and a NaN row where it is
    negative.  Pages of one position, so that a hole is what has no weight."""
    base, H = [300, 41], 4
    print("tree infinite keys", dtype, D, T, flush=True)
    cache, table, q = setup(dev, dtype, D, H, 2, 1, base, T)
    q.view(-1, H, D)[:, :, 3] = torch.tensor([8.0, -8.0, 1e-6, 1e-14])
    cache.k[table[0, 100], :, 0, 3] = -math.inf
    got = attend(dev, cache, table, q, base, chain(2, T), H).view(2, T, H, D)
    table[0, 100] = -1
    want = attend(dev, cache, table, q, base, chain(2, T), H).view(2, T, H, D)
    assert torch.isfinite(want).all()
    want[0, :, 1] = math.nan
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


def own(cache, table, q, base, T, q_heads, scale):
    """(out, bound) as decode_helpers.attention, of chains, with each score's error from its own products alone: position i's
    score is off by at most e_i = (D + 8) u scale sum|q k_i|, so the row by sum p e |v| + (sum p e)(sum p |v|) to first
    order (a score that has no weight moves nothing), twice for the second, and the sum over positions as there.  A weight below
    fp32's least normal number 2^-126, beside the largest, may be lost."""
    K, V = values(cache, "k"), values(cache, "v")
    D, G, P = cache.dim, q_heads // cache.heads, cache.page_size
    q = q.cpu().double().view(len(base), T, q_heads, D)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(base):
        pos = torch.arange(n + T)
        page, off = table[b].long()[pos // P], pos % P
        for h in range(q_heads):
            for t in range(T):
                see = pos <= n + t
                k, v, x = K[page, h // G, off][see], V[page, h // G, off][see], q[b, t, h]
                p = torch.softmax(scale * (k @ x), 0)
                e = p * (U * (D + 8) * abs(scale) * (k.abs() @ x.abs()))
                out[b, t, h] = p @ v
                bound[b, t, h] = 2 * (e @ v.abs() + e.sum() * (p @ v.abs())) + U * ((n + T) / 4 + 64) * (p @ v.abs()) + 2.0 ** -126 * v.abs().sum(0)
    return out.view(len(base) * T, -1), bound.view(len(base) * T, -1)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("far", [10, 100, 3000, 60000, 1e7])
@pytest.mark.parametrize("D,T,H", [(64, 1, 2), (64, 40, 4), (128, 20, 2), (256, 3, 4)])
def test_scores_that_rise_from_far_below(dev, dtype, far, D, T, H):
    """A context that opens with scores far below 0, behind it ordinary ones: their weights are as exact as without it.  The largest
    score rises in the middle of a tile, at the start of one, in the tree itself, and in steps.  (A table of many more pages leaves
    each context in one part.)"""
    if dtype == "f16" and far > 60000:
        pytest.skip("past f16's range")
    base = [200, 333, 64, 96]
    first = [[(0, 70, 1.0)], [(0, 96, 1.0)], [(0, 64, 1.0)], [(0, 32, 1.0), (32, 64, 0.25)]]
    print("tree rise", dtype, far, D, T, H, flush=True)
    cache, table, q = setup(dev, dtype, D, H, 2, 16, base, T, width=16384)
    q.view(-1, H, D)[:, :, 0] = 1.0
    cache.k[..., 0] = 0
    for b, spans in enumerate(first):
        for a, z, part in spans:
            for p in range(a, z):
                at = (table[b, p // 16], slice(None), p % 16)
                if dtype == "i8":
                    cache.k[at] = 0
                    cache.k_scale[at] = far * part / 127
                cache.k[(*at, 0)] = -127 if dtype == "i8" else -far * part
    got = attend(dev, cache, table, q, base, chain(4, T), H, scale=1.0 / 8)
    check_attention(got, *own(cache, table, q, base, T, H, 1.0 / 8))


@pytest.mark.parametrize("dtype,D,H", [("f16", 128, 8), ("bf16", 64, 4), ("i8", 80, 2), ("bf16", 256, 16)])
def test_a_row_beside_other_sizes_of_call(dev, dtype, D, H):
    """How many requests, nodes and positions a call is made for changes the order of a row's sums alone: each time it is
    the formula's, and with the same sizes the same bits."""
    T, n, most = 8, 1000, 64
    cache, table, q = setup(dev, dtype, D, H, 2, 16, [n], most)
    want, bound = tree_attention(cache, table, q[:T], [n], chain(1, T), H, D ** -0.5)
    for seqs, nodes, max_len in ((1, T, 1016), (1, T, 60000), (2, T, 1016), (9, T, 5000), (70, T, 1064), (1, most, 1064), (1, most, 60000),
                                 (5, 40, 2000)):
        wide = torch.full((seqs, 60000 // 16 + 1), -1, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        rows = q[:nodes].repeat(seqs, 1)
        base = [n] + [n - 7 * b for b in range(1, seqs)]
        got = attend(dev, cache, wide, rows, base, chain(seqs, nodes), H, max_len=max_len)
        print("sizes", dtype, D, H, seqs, nodes, max_len, flush=True)
        check_attention(got[:T], want, bound)
        assert torch.equal(got[:T], attend(dev, cache, wide, rows, [n] + [5] * (seqs - 1), chain(seqs, nodes), H, max_len=max_len)[:T])
