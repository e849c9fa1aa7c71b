"""kq_attn_tree_workspace: what holds the largest step holds every smaller one (host only: a call without a workspace says what it
needs before any launch)."""
import itertools
import random
import re

import pytest

from kq import _lib, ops
from test_paged_host import P, cache_struct
from test_tree_host import attend


def need(seqs, q_heads, heads, dim, T, max_len):
    cache = cache_struct(heads=heads, dim=dim, page_stride=heads * 16 * dim, head_stride=16 * dim, pos_stride=dim)
    assert attend(cache, seqs=seqs, T=T, max_len=max_len, q_heads=q_heads, ldq=q_heads * dim, ldo=q_heads * dim, ws=P,
                  ws_bytes=0) == _lib.KQ_ERR_ARG
    return int(re.search(r"(\d+) needed", _lib.kq().kq_last_error().decode()).group(1))


@pytest.mark.parametrize("q_heads,heads", [(32, 8), (16, 4), (8, 8), (7, 1), (40, 5)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_smaller_calls_fit(q_heads, heads, dim):
    rng = random.Random(q_heads * dim)
    lengths = [1, 31, 32, 33, 600, 1058, 2047, 2048, 2051, 2080, 5003, 16384, 16385, 50001, 65536, 131072]
    for S, T, M in [(1, 64, 2051), (4, 16, 2080), (5, 16, 2048), (32, 16, 8208), (64, 64, 131072), (300, 3, 40000), (2, 1, 1 << 20)]:
        most = ops.attn_tree_workspace_bytes(S, q_heads, dim, T, M)
        sizes = itertools.product({1, 2, 3, S // 2, S - 1, S}, {1, 2, 5, T // 2, T - 1, T}, [m for m in lengths if m <= M] + [M])
        for s, t, m in itertools.chain(sizes, ((rng.randint(1, S), rng.randint(1, T), rng.randint(1, M)) for _ in range(200))):
            if 0 < s <= S and 0 < t <= T:
                assert need(s, q_heads, heads, dim, t, m) <= most, (S, T, M, s, t, m)


@pytest.mark.parametrize("q_heads,dim,T", [(32, 128, 64), (32, 128, 16), (16, 256, 24), (8, 64, 2)])
def test_never_falls(q_heads, dim, T):
    """In any of requests, nodes and positions."""
    for sizes in ([(s, T, 2048) for s in range(1, 200)], [(4, t, 5000) for t in range(1, 65)],
                  [(s, T, m) for s in (1, 5) for m in range(1, 70000, 307)][:228]):
        held = [ops.attn_tree_workspace_bytes(s, q_heads, dim, t, m) for s, t, m in sizes]
        assert held == sorted(held)


def test_a_buffer_for_the_longest_context_takes_a_shorter_one():
    most = ops.attn_tree_workspace_bytes(4, 32, 128, 16, 2080)
    assert need(4, 32, 8, 128, 16, 1058) <= most and need(1, 32, 8, 128, 16, 2048) <= most
