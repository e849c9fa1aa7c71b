"""kq_kv_append against the same steps in numpy's fp32 (each product, sum and rounding alike: equal bits) and against
the formula in 64 bits."""
import numpy as np
import pytest
import torch

from decode_helpers import U, make_cache, page_table
from kq import kv, ops

pytestmark = pytest.mark.gpu
F32 = np.float32


def turned(x, pos, rope, rot, interleaved, dt):
    """x [N][heads][D] (numpy) with its first rot values rotated, every step in dt."""
    y = x.astype(dt)
    c, s = (r[:, None] for r in np.split(rope[pos].astype(dt), 2, 1))
    a = (slice(0, rot, 2) if interleaved else slice(0, rot // 2))
    b = (slice(1, rot, 2) if interleaved else slice(rot // 2, rot))
    u, v = y[..., a].copy(), y[..., b].copy()
    y[..., a] = u * c - v * s
    y[..., b] = v * c + u * s
    return y


def stored(x, dtype):
    """(elements, scales or None) of x [N][heads][D] fp32."""
    if dtype == "i8":
        scale = np.abs(x).max(-1) * (F32(1) / F32(127))
        return np.where(scale[..., None] > 0, np.rint(x / np.where(scale > 0, scale, 1)[..., None]), 0).astype(np.int8), scale
    t = torch.from_numpy(x).to(kv.DTYPES[dtype])
    return t.view(torch.int16).numpy(), None


def bits(t):
    t = t.cpu()
    return t.numpy() if t.dtype == torch.int8 else t.contiguous().view(torch.int16).numpy()


def run(dev, dtype, D, q_heads, heads, page, start, tokens, rot, interleaved, order="heads", shift=0, seed=0, with_q=True):
    """Append `tokens` tokens to each request standing at start[b]; checks everything that the call may write."""
    print("append", dtype, D, q_heads, heads, page, start, tokens, rot, interleaved, order, shift, flush=True)
    rng = np.random.default_rng(seed)
    lens = [s + tokens for s in start]
    table, pages = page_table(lens, page, extra=2, seed=seed)
    cache = make_cache(dtype, pages, heads, page, D, dev, seed=seed, order=order)
    N = len(start) * tokens
    seq = np.repeat(np.arange(len(start)), tokens).astype(np.int32)
    pos = (np.array(start)[:, None] + np.arange(tokens)).reshape(-1).astype(np.int32)
    shuffle = rng.permutation(N)
    seq, pos = seq[shuffle], pos[shuffle]
    width = (q_heads + 2 * heads) * D
    flat = rng.standard_normal(N * width + shift).astype(F32)
    x = flat[shift:].reshape(N, width)
    xd = torch.from_numpy(flat).to(dev)[shift:].view(N, width)
    q, k, v = xd.split([q_heads * D, heads * D, heads * D], 1)
    rope = kv.rope_table(int(max(lens)) + 3, rot, device="cpu") if rot else None
    before = {n: bits(getattr(cache, n)).copy() for n in "kv"}
    before.update({n: getattr(cache, n).cpu().numpy().copy() for n in ("k_scale", "v_scale")} if dtype == "i8" else {})
    q_out = torch.full((N, q_heads * D), 7.0, device=dev)
    ops.kv_append(cache, table.to(dev), q if with_q else None, k, v, torch.from_numpy(seq).to(dev),
                  torch.from_numpy(pos).to(dev), q_out if with_q else None, q_heads, None if rope is None else rope.to(dev),
                  interleaved)
    torch.cuda.synchronize()

    xq, xk, xv = (p.reshape(N, -1, D) for p in np.split(x, [q_heads * D, (q_heads + heads) * D], 1))
    rp = rope.numpy() if rot else None
    turn = (lambda t, dt: turned(t, pos, rp, rot, interleaved, dt)) if rot else (lambda t, dt: t.astype(dt))
    if with_q:
        got = q_out.cpu().numpy().reshape(N, q_heads, D)
        np.testing.assert_array_equal(got, turn(xq, F32))
        # two products and a sum, each off by half a step of at most |a| + |b|
        exact = turn(xq, np.float64)
        reach = np.abs(xq).max(-1, keepdims=True) * 2
        assert (np.abs(got - exact) <= 3 * U * reach).all()
    else:
        assert (q_out == 7.0).all()
    pg, off = table.numpy()[seq, pos // page], pos % page
    for name, new in (("k", turn(xk, F32)), ("v", xv)):
        want, scale = stored(np.ascontiguousarray(new), dtype)
        full = before[name]
        full[pg, :, off] = want
        np.testing.assert_array_equal(bits(getattr(cache, name)), full)       # and nothing else was written
        if dtype == "i8":
            full = before[name + "_scale"]
            full[pg, :, off] = scale
            np.testing.assert_array_equal(getattr(cache, name + "_scale").cpu().numpy(), full)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(16, 8), (64, 64), (80, 40), (96, 96), (128, 128), (176, 16), (256, 64)])
def test_head_sizes(dev, dtype, D, rot, interleaved):
    run(dev, dtype, D, 4, 2, 16, [0, 15, 31], 3, rot, interleaved, seed=D)


@pytest.mark.parametrize("dtype", ["bf16", "i8"])
@pytest.mark.parametrize("q_heads,heads,page,start,tokens", [
    (1, 1, 1, [0], 1), (32, 8, 16, [700], 1), (7, 1, 8, [5, 6, 7, 8, 9], 1), (10, 5, 256, [255], 2), (4, 4, 32, [0, 100], 70)])
def test_layouts(dev, dtype, q_heads, heads, page, start, tokens):
    run(dev, dtype, 128, q_heads, heads, page, start, tokens, 128, False, seed=q_heads)


@pytest.mark.parametrize("dtype", ["f16", "i8"])
@pytest.mark.parametrize("order", ["positions", "apart"])
@pytest.mark.parametrize("shift", [0, 1])
def test_orders_and_unaligned_rows(dev, dtype, order, shift):
    run(dev, dtype, 64, 4, 2, 16, [3, 40], 9, 32, False, order=order, shift=shift)
    run(dev, dtype, 64, 4, 2, 16, [3, 40], 9, 32, True, order=order, shift=shift)


def test_without_queries_and_without_rotation(dev):
    run(dev, "bf16", 128, 4, 2, 16, [3, 40], 5, 128, False, with_q=False)
    run(dev, "bf16", 128, 4, 2, 16, [3, 40], 5, 0, False)


def test_in_place_queries(dev):
    cache = make_cache("bf16", 4, 2, 16, 64, dev)
    att = kv.PagedAttention([cache], torch.arange(4, dtype=torch.int32, device=dev)[None], 4,
                            rope=kv.rope_table(64, 64, device=dev))
    q, k, v = (torch.randn(5, n * 64, device=dev) for n in (4, 2, 2))
    seq, pos = torch.zeros(5, dtype=torch.int32, device=dev), torch.arange(9, 14, dtype=torch.int32, device=dev)
    apart = att.append(0, q, k, v, seq, pos)
    assert apart.data_ptr() != q.data_ptr()
    assert att.append(0, q, k, v, seq, pos, q) is q
    assert torch.equal(q, apart)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_skipped_tokens_and_holes(dev, dtype):
    """Padding tokens (seq -1), requests, positions and pages that do not exist: nothing of the cache or of a skipped
    token's queries is written; a token over a hole has its queries rotated."""
    D, N = 64, 8
    cache = make_cache(dtype, 5, 2, 16, D, dev)
    table = torch.tensor([[0, -1, 5], [2 ** 31 - 1, 3, -2 ** 31]], dtype=torch.int32, device=dev)
    #         kept, hole, page 5 of 5, past table, seq -1, seq 2, pos -1, kept
    seq = torch.tensor([0, 0, 0, 0, -1, 2, 1, 1], dtype=torch.int32, device=dev)
    pos = torch.tensor([3, 16, 40, 48, 5, 5, -1, 30], dtype=torch.int32, device=dev)
    q, k, v = (torch.randn(N, n * D, device=dev) for n in (2, 2, 2))
    rope = kv.rope_table(48, D, device=dev)
    before = cache.k.clone(), cache.v.clone()
    out = torch.full_like(q, 7.0)
    ops.kv_append(cache, table, q, k, v, seq, pos, out, 2, rope)
    torch.cuda.synchronize()
    kept = torch.zeros(cache.k.shape[:3], dtype=torch.bool)
    kept[0, :, 3] = kept[3, :, 14] = True
    for now, was in zip((cache.k, cache.v), before):
        assert torch.equal(now.cpu()[~kept], was.cpu()[~kept])
        assert not torch.equal(now.cpu()[kept], was.cpu()[kept])
    written = (out != 7.0).any(1).cpu().tolist()
    assert written == [True, True, True, False, False, False, False, True]
    # a rope table shorter than the requests' positions: the tokens past it are skipped
    out.fill_(7.0)
    ops.kv_append(cache, table, q, k, v, seq, pos, out, 2, kv.rope_table(10, D, device=dev))
    assert (out != 7.0).any(1).cpu().tolist() == [True] + [False] * 7


def test_values_at_the_types_borders(dev):
    """f16 overflows to infinity and bf16 ties go to even as torch rounds them; an 8-bit row of zeros has scale 0; the
    largest value of a row is code 127 or -127; subnormal scales stay in range."""
    one = torch.zeros(1, dtype=torch.int32, device=dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    x = torch.zeros(1, 64)
    x[0, :8] = torch.tensor([65519.0, 65520.0, -1e6, 1 + 2 ** -9, 1 + 3 * 2 ** -9, 6e-8, -3e-8, 1e-41])
    for dtype in ("f16", "bf16"):
        cache = make_cache(dtype, 1, 1, 1, 64, dev)
        ops.kv_append(cache, table, None, x.to(dev), (-x).to(dev), one, one, None, 1)
        assert torch.equal(cache.k.cpu().view(-1), x[0].to(cache.k.dtype))
        assert torch.equal(cache.v.cpu().view(-1), (-x[0]).to(cache.v.dtype))
    cache = make_cache("i8", 1, 1, 1, 64, dev)
    ops.kv_append(cache, table, None, x.to(dev), torch.zeros(1, 64, device=dev), one, one, None, 1)
    assert cache.k.min() == -127 and (cache.v == 0).all() and float(cache.v_scale) == 0
    tiny = torch.full((1, 64), 1e-44)
    ops.kv_append(cache, table, None, tiny.to(dev), -tiny.to(dev), one, one, None, 1)
    assert cache.k.abs().max() <= 127 and cache.v.abs().max() <= 127


def test_offsets_past_32_bits(dev):
    """The last pages of a pool whose elements' offsets and bytes pass 2^32."""
    D, page, heads = 128, 16, 8
    pages = 2 ** 32 // (D * page * heads) + 3
    k, v = (torch.zeros((pages, heads, page, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((pages, heads, page), device=dev) for _ in range(2))
    cache = kv.KVCache.over(k, v, ks, vs)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=dev)
    pos = torch.tensor([7, 16, 47], dtype=torch.int32, device=dev)
    x = torch.randn(3, heads * D, device=dev)
    ops.kv_append(cache, table, None, x, -x, torch.zeros(3, dtype=torch.int32, device=dev), pos, None, heads)
    want, scale = stored(x.cpu().numpy().reshape(3, heads, D), "i8")
    for n, (p, off) in enumerate([(pages - 1, 7), (0, 0), (pages - 2, 15)]):
        np.testing.assert_array_equal(k[p, :, off].cpu().numpy(), want[n])
        np.testing.assert_array_equal(ks[p, :, off].cpu().numpy(), scale[n])
        np.testing.assert_array_equal(v[p, :, off].cpu().numpy(), -want[n])
    assert int(k[pages - 3].abs().sum()) == 0


def test_other_stream_and_graph(dev):
    """On a stream of its own, and captured: positions are read when the graph runs."""
    D = 64
    cache = make_cache("bf16", 4, 2, 16, D, dev)
    table = torch.arange(4, dtype=torch.int32, device=dev)[None]
    att = kv.PagedAttention([cache], table, 2, rope=kv.rope_table(64, D, device=dev))
    q, k, v = (torch.randn(1, 2 * D, device=dev) for _ in range(3))
    seq, pos = (torch.zeros(1, dtype=torch.int32, device=dev) for _ in range(2))
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        att.append(0, q, k, v, seq, pos, out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.append(0, q, k, v, seq, pos, out)
    for p in (5, 17, 40):
        pos.fill_(p)
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got, rotated = cache.k.clone(), out.clone()
        att.append(0, q, k, v, seq, pos, out)
        torch.cuda.synchronize()
        assert torch.equal(got, cache.k) and torch.equal(rotated, out)
        assert cache.k[p // 16, :, p % 16].abs().sum() > 0
