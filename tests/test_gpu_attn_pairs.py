"""Attention where a workgroup takes two chunks, and two such pairs one after the other: the same bits as a request has alone, where
it is split otherwise."""
import math

import pytest
import torch

from decode_helpers import make_cache
from test_gpu_attn_paged import attend, check

pytestmark = pytest.mark.gpu

HEADS, PAGE, POOL, WIDTH = 8, 16, 64, 4096        # 65536 positions, 256 chunks; every table names the same pages
# the second pairs of workgroups start at position 32768 where 8 requests share the chip
LENS = [65536, 65535, 40000, 33025, 32769, 32768, 700, 0]
FORMS = [("f16", 128, 4, 1), ("bf16", 128, 4, 1), ("i8", 128, 4, 1), ("f16", 128, 4, 8), ("bf16", 128, 4, 8),
         ("i8", 128, 4, 8), ("f16", 64, 4, 5), ("bf16", 256, 4, 5), ("i8", 256, 2, 16), ("f16", 240, 4, 5),
         ("bf16", 16, 1, 1), ("i8", 80, 8, 3)]


def batch(dev, dtype, D, G, T, lens):
    cache = make_cache(dtype, POOL + len(lens), HEADS, PAGE, D, dev, seed=D + T)
    g = torch.Generator().manual_seed(T)
    table = torch.randint(0, POOL, (len(lens), WIDTH), generator=g, dtype=torch.int32)
    for b, n in enumerate(lens):                    # the last page of a request is its own
        if n:
            table[b, (n - 1) // PAGE] = POOL + b
    return cache, table, torch.randn((len(lens) * T, HEADS * G * D), generator=g)


@pytest.mark.parametrize("dtype,D,G,T", FORMS)
def test_several_pairs_a_workgroup(dev, dtype, D, G, T):
    print("pairs", dtype, D, G, T, flush=True)
    cache, table, q = batch(dev, dtype, D, G, T, LENS)
    rows = attend(dev, cache, table, q, LENS, T, HEADS * G).view(len(LENS), T, -1)
    assert torch.isfinite(rows).all() and (rows[-1] == 0).all()
    for b, n in enumerate(LENS):
        alone = attend(dev, cache, table[b:b + 1], q[b * T:(b + 1) * T], [n], T, HEADS * G)
        assert torch.equal(alone, rows[b]), n
        if T > 1 and n:
            first = attend(dev, cache, table[b:b + 1], q[b * T:b * T + 1], [n - T + 1], 1, HEADS * G)
            assert torch.equal(first, rows[b, :1]), n


@pytest.mark.parametrize("dtype,D,G,T", [f for f in FORMS if f[0] != "i8" and f[3] > 1])
def test_infinities_in_several_pairs(dev, dtype, D, G, T):
    """Infinities and NaN that only a draft's last tokens see, in the first pair and in the second of a workgroup, and in both
    chunks of a pair: each row is what it is alone, at its own length."""
    lens = [32768 + 3, 33025, 65536, 32768 + 256 + 2, 258, 700, 512 + 2, 40000]
    print("infinities in pairs", dtype, D, G, T, flush=True)
    cache, table, q = batch(dev, dtype, D, G, T, lens)
    for b, n in enumerate(lens):
        cache.v[POOL + b, 1, (n - 1) % PAGE, 7] = math.inf
        cache.v[POOL + b, 0, (n - 1) % PAGE, D - 1] = math.nan
        cache.k[POOL + b, 2, (n - 1) % PAGE, 0] = -math.inf
        if n % PAGE != 1:
            cache.v[POOL + b, 3, (n - 2) % PAGE, 3] = -math.inf
    rows = attend(dev, cache, table, q, lens, T, HEADS * G).view(len(lens), T, -1)
    assert torch.isfinite(rows[:, :T - 2]).all() and not torch.isfinite(rows[:, -1]).all()
    qs = q.view(len(lens), T, -1)
    for b, n in enumerate(lens):
        for t in range(T):
            one = attend(dev, cache, table[b:b + 1], qs[b, t:t + 1], [n - T + 1 + t], 1, HEADS * G)
            torch.testing.assert_close(one, rows[b, t:t + 1], rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("D,q_heads,heads,T", [(128, 8, 1, 4), (256, 8, 1, 5), (64, 40, 2, 1)])
def test_the_formula_with_more_rows_than_a_tile(dev, dtype, D, q_heads, heads, T):
    check(dev, dtype, D, q_heads, heads, 16, [4099, 513, 2], T=T)


def test_long_f16(dev):
    check(dev, "f16", 128, 4, 1, 16, [20011])
