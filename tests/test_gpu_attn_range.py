"""Attention where fp32's range and each number's own 24 bits count, against the formula in 64 bits within
decode_helpers.attention's bound."""
import math

import pytest
import torch

from decode_helpers import attention, check_attention, make_cache, page_table
from test_gpu_attn_paged import attend, setup

pytestmark = pytest.mark.gpu


def sinks(dev, dtype, D, gap, lens, T, every=64):
    """Every 64th position takes all the weight and has a value of 0; the others' scores lie `gap` below.  Two query heads on
    one key-value head; the score is the first value of the key."""
    table, pages = page_table(lens, 16)
    cache = make_cache(dtype, pages, 1, 16, D, dev)
    flat = torch.zeros(pages * 16, dtype=torch.bool)
    for b, n in enumerate(lens):
        p = torch.arange(5, n, every)
        flat[table[b].long()[p // 16] * 16 + p % 16] = True
    sink = flat.view(pages, 1, 16).to(dev)
    cache.k.zero_()
    if dtype == "i8":
        cache.k[..., 0] = 127 * sink
        cache.k_scale.fill_(gap / 127)
        cache.v.abs_()                                  # of one sign, so that errors of one sign do not cancel
    else:
        cache.k[..., 0] = gap * sink
        cache.v.add_(1)
    cache.v.masked_fill_(sink[..., None], 0)
    q = torch.zeros(len(lens) * T, 2 * D)
    q[:, [0, D]] = 1
    return cache, table, q


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("gap", [12, 18, 25, 30, 40, 60, 80])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 3), (256, 1)])
def test_weights_far_below_the_largest(dev, dtype, gap, D, T):
    lens = [40, 65, 700, 4096]
    print("sinks", dtype, gap, D, T, flush=True)
    cache, table, q = sinks(dev, dtype, D, gap, lens, T)
    got = attend(dev, cache, table, q, lens, T, 2, scale=1.0)
    check_attention(got, *attention(cache, table, q, lens, T, 2, 1.0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gap", [0, 20, 40, 80])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 4), (256, 1)])
def test_infinite_values_of_small_weight(dev, dtype, gap, D, T):
    """An infinity or NaN that a row sees counts however small its weight; the other columns keep their sums."""
    lens = [700, 40]
    print("infinite values", dtype, gap, D, T, flush=True)
    cache, table, q = sinks(dev, dtype, D, gap, lens, T)
    page, off = table[0, 300 // 16], 300 % 16
    cache.v[page, 0, off:off + 2, 10:14] = 0
    ref, bound = attention(cache, table, q, lens, T, 2, 1.0)
    cache.v[page, 0, off, 10:14] = torch.tensor([math.inf, -math.inf, math.nan, math.inf], device=dev).to(cache.v.dtype)
    cache.v[page, 0, off + 1, 13] = -math.inf
    got = attend(dev, cache, table, q, lens, T, 2, scale=1.0).view(2, T, 2, D)
    hit = got[0, :, :, 10:14].cpu()
    assert (hit[..., 0] == math.inf).all() and (hit[..., 1] == -math.inf).all() and hit[..., 2:].isnan().all()
    got[0, :, :, 10:14] = 0
    ref.view(2, T, 2, D)[0, :, :, 10:14] = 0
    bound.view(2, T, 2, D)[0, :, :, 10:14] = 0
    check_attention(got.view(2 * T, -1), ref, bound)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 4), (240, 1)])
def test_infinite_keys_that_are_seen(dev, dtype, D, T):
    """A key of -inf in one channel: no weight where the query is positive there, however small, and a NaN row where it is
    negative.  Pages of one position, so that a hole is what has no weight."""
    lens, H = [300, 41], 4
    print("infinite keys", dtype, D, T, flush=True)
    cache, table, q = setup(dev, dtype, D, H, 2, 1, lens, T)
    q.view(-1, H, D)[:, :, 3] = torch.tensor([8.0, -8.0, 1e-6, 1e-14])
    cache.k[table[0, 100], :, 0, 3] = -math.inf
    got = attend(dev, cache, table, q, lens, T, H).view(2, T, H, D)
    table[0, 100] = -1
    want = attend(dev, cache, table, q, lens, T, H).view(2, T, H, D)
    assert torch.isfinite(want).all()
    want[0, :, 1] = math.nan
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("ratio", [1e2, 1e3, 1e4, 1e6, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("D", [48, 128])
def test_a_query_channel_far_above_the_others(dev, dtype, ratio, D):
    """Where the keys are 0 in that channel, the others' products are the whole score."""
    lens, T, H = [41, 700], 2, 4
    print("channel", dtype, ratio, D, flush=True)
    cache, table, q = setup(dev, dtype, D, H, 2, 16, lens, T)
    q.view(-1, H, D)[..., 17] = ratio
    cache.k[..., 17] = 0
    check_attention(attend(dev, cache, table, q, lens, T, H), *attention(cache, table, q, lens, T, H, D ** -0.5))


def test_an_f16_row_beside_rows_of_other_ranges(dev):
    """Drafted tokens with and without elements that f16 parts do not hold: each row's bits are those it has alone."""
    D, H, T, lens = 128, 4, 4, [700, 41]
    cache, table, q = setup(dev, "f16", D, H, 2, 16, lens, T)
    qs = q.view(2, T, H, D)
    qs[:, 1, :, 17] = 1e15
    qs[:, 2, 1, 5:9] = 1e-20
    cache.k[..., 17] = 0
    rows = attend(dev, cache, table, q, lens, T, H).view(2, T, -1)
    for t in range(T):
        alone = attend(dev, cache, table, qs[:, t].reshape(2, -1).contiguous(), [n - T + 1 + t for n in lens], 1, H)
        assert torch.equal(alone, rows[:, t]), t
    check_attention(rows.view(2 * T, -1), *attention(cache, table, q, lens, T, H, D ** -0.5))


@pytest.mark.parametrize("keys,queries", [(-100, 100), (60, -60), (95, -95), (104, -95)])
def test_key_scales_far_from_1(dev, keys, queries):
    """An 8-bit cache's key scales at 2^keys under queries at 2^queries: ordinary scores."""
    D, H, lens = 64, 4, [41, 300]
    print("key scales", keys, queries, flush=True)
    cache, table, q = setup(dev, "i8", D, H, 2, 16, lens, 1)
    cache.k_scale.mul_(2.0 ** keys)
    q, scale = q * 2.0 ** queries, 2.0 ** -(keys + queries) * D ** -0.5
    check_attention(attend(dev, cache, table, q, lens, 1, H, scale), *attention(cache, table, q, lens, 1, H, scale))
