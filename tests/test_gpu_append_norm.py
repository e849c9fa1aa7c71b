"""kq_kv_append_norm: norms against the formula in 64 bits, tokens stored apart from their position, and nothing else written."""
import numpy as np
import pytest
import torch

from decode_helpers import U, make_cache, page_table, values
from kq import kv

pytestmark = pytest.mark.gpu


def exact_head(x, w, eps, pos, rope, rot, interleaved):
    """x [N][heads][D] (64 bits) normed by w (or not), then rotated by pos."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    y = x.clone()
    if rot:
        c, s = (r[:, None] for r in rope[pos].double().chunk(2, 1))
        a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
        b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    # a square, up to 12 sums of positive terms, a quotient, the eps, a root (which halves those) and a reciprocal: r is off by
    # at most (14 + 2) / 2 + 2 = 10 u; two products more, and the rotation's three steps on values of up to twice the largest
    bound = (12 + 2 + 3) * U * 2 * x.abs().amax(-1, keepdim=True) * torch.ones_like(y)
    return y, bound


def run(dev, dtype, D, q_heads, heads, page, base, T, rot, interleaved=False, order="heads", shift=0, q_norm=True, k_norm=True,
        eps=1e-6, with_q=True, with_slot=True, scale=1.0, seed=0):
    print("append_norm", dtype, D, q_heads, heads, page, base, T, rot, interleaved, order, shift, q_norm, k_norm, flush=True)
    g = torch.Generator().manual_seed(seed)
    table, pages = page_table([n + T for n in base], page, extra=2, seed=seed)
    cache = make_cache(dtype, pages, heads, page, D, dev, seed=seed, order=order)
    N = len(base) * T
    order_ = torch.randperm(N, generator=g)
    seq = torch.arange(len(base)).repeat_interleave(T).int()[order_]
    slot = (torch.tensor(base)[:, None] + torch.arange(T)).reshape(-1).int()[order_]
    pos = (torch.tensor(base)[:, None] + torch.randint(0, T, (len(base), T), generator=g)).reshape(-1).int()[order_]
    if not with_slot:
        pos = slot
    width = (q_heads + 2 * heads) * D
    flat = torch.randn(N * width + shift, generator=g) * scale
    x = flat[shift:].view(N, width)
    xd = flat.to(dev)[shift:].view(N, width)
    q, k, v = xd.split([q_heads * D, heads * D, heads * D], 1)
    wq, wk = (1 + 0.3 * torch.randn(1, D, generator=g) for _ in range(2))
    rope = kv.rope_table(max(base) + T + 3, rot, device="cpu") if rot else None
    att = kv.PagedAttention([cache], table.to(dev), q_heads, rope=None if rope is None else rope.to(dev), interleaved=interleaved,
                            q_norm=wq.to(dev) if q_norm else None, k_norm=wk.to(dev) if k_norm else None, eps=eps)
    before = {n: values(cache, n) for n in "kv"}
    out = torch.full((N, q_heads * D), 7.0, device=dev)
    att.append(0, q if with_q else None, k, v, seq.to(dev), pos.to(dev), out if with_q else None, slot=slot.to(dev) if with_slot else None)
    xq, xk, xv = (p.reshape(N, -1, D).double() for p in x.split([q_heads * D, heads * D, heads * D], 1))
    at = pos.long()
    if with_q:
        want, bound = exact_head(xq, wq.double() if q_norm else None, eps, at, rope, rot, interleaved)
        assert ((out.cpu().double().view(N, -1, D) - want).abs() <= bound).all()
    else:
        assert (out == 7.0).all()
    pg, off = table[seq.long(), slot.long() // page].long(), slot.long() % page
    for name, (want, bound) in (("k", exact_head(xk, wk.double() if k_norm else None, eps, at, rope, rot, interleaved)),
                                ("v", (xv, 0 * xv))):
        got = values(cache, name)
        if dtype == "i8":                              # half a code, and the codes' own rounding at the bound
            step = getattr(cache, name + "_scale").cpu().double()[pg, :, off][..., None]
            top = want.abs().amax(-1, keepdim=True)
            assert ((step - top / 127).abs() <= (bound.amax(-1, keepdim=True) + 2 * U * top) / 127).all()
            room = step / 2 + bound + 4 * U * top
        else:                                          # half a step of the cache's type; f16: or of its subnormals
            half = torch.finfo(kv.DTYPES[dtype]).eps / 2
            room = bound + half * (want.abs() + bound) + (2.0 ** -25 if dtype == "f16" else 0)
        assert ((got[pg, :, off] - want).abs() <= room).all()
        full = before[name]
        full[pg, :, off] = got[pg, :, off]
        assert torch.equal(got, full)                  # nothing else was written


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 192, 240, 256])
def test_head_sizes(dev, dtype, D):
    run(dev, dtype, D, 4, 2, 16, [0, 37, 300], 5, D if D % 8 == 0 else 16, seed=D)
    run(dev, dtype, D, 3, 1, 8, [1], 9, 8, interleaved=True, seed=D)


@pytest.mark.parametrize("rot,interleaved", [(0, False), (8, False), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("q_norm,k_norm", [(True, True), (True, False), (False, True), (False, False)])
def test_norms_and_rotations(dev, rot, interleaved, q_norm, k_norm):
    run(dev, "bf16", 128, 8, 2, 16, [3, 40], 7, rot, interleaved, q_norm=q_norm, k_norm=k_norm)


@pytest.mark.parametrize("order", ["positions", "apart"])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_orders_and_odd_floats(dev, order, shift):
    for dtype in ("f16", "bf16", "i8"):
        run(dev, dtype, 128, 8, 2, 16, [3, 40], 7, 64, order=order, shift=shift)


def test_sizes(dev):
    run(dev, "bf16", 128, 32, 8, 16, [11], 1, 128)
    run(dev, "f16", 256, 16, 4, 64, [11, 200, 3], 64, 64)
    run(dev, "bf16", 128, 32, 8, 16, [0, 5], 700, 128, with_slot=False)
    run(dev, "i8", 64, 64, 64, 1, [2], 33, 64)
    run(dev, "bf16", 64, 4, 2, 16, [2], 5, 64, with_q=False)


@pytest.mark.parametrize("scale,eps", [(1e-12, 1e-6), (1e-12, 0.0), (1e15, 1e-6), (1e-3, 0.5)])
def test_large_and_small_values(dev, scale, eps):
    run(dev, "bf16", 64, 4, 2, 16, [3, 40], 7, 64, scale=scale, eps=eps)


def test_a_head_of_zeros(dev):
    """eps keeps it 0; without, 0 times the reciprocal of 0 is what the formula gives."""
    table, pages = page_table([4], 16)
    cache = make_cache("bf16", pages, 1, 16, 64, dev)
    one = torch.ones(1, 64, device=dev)
    x, at = torch.zeros(1, 64, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    for eps in (1e-6, 0.0):
        att = kv.PagedAttention([cache], table.to(dev), 1, q_norm=one, k_norm=one, eps=eps)
        got = att.append(0, x, x, x, at, at)
        assert (got == 0).all() if eps else torch.isnan(got).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8"])
def test_slots_alone_are_the_append_of_another_position(dev, dtype):
    """Without norms the bits are kq_kv_append's, stored in the slots."""
    D, H, heads, T = 64, 4, 2, 9
    table, pages = page_table([60], 16)
    a, b = (make_cache(dtype, pages, heads, 16, D, dev) for _ in range(2))
    rope = kv.rope_table(64, D, device=dev)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(T, n * D, generator=g).to(dev) for n in (H, heads, heads))
    seq = torch.zeros(T, dtype=torch.int32, device=dev)
    pos, slot = torch.arange(10, 10 + T, device=dev).int(), torch.arange(40, 40 + T, device=dev).int()
    qa = kv.PagedAttention([a], table.to(dev), H, rope=rope).append(0, q, k, v, seq, pos)
    qb = kv.PagedAttention([b], table.to(dev), H, rope=rope).append(0, q, k, v, seq, pos, slot=slot)
    assert torch.equal(qa, qb)
    flat = [t.to(dev).long() for t in (table[0, (pos.cpu() // 16).long()], table[0, (slot.cpu() // 16).long()])]
    for n in ("k", "v") + (("k_scale", "v_scale") if dtype == "i8" else ()):
        assert torch.equal(getattr(a, n)[flat[0], :, (pos % 16).long()], getattr(b, n)[flat[1], :, (slot % 16).long()])


def test_tokens_that_are_skipped(dev):
    """Requests and slots outside the table, positions outside the rotation: nothing of them is read or written."""
    D, H = 64, 2
    table, pages = page_table([32, 32], 16)
    cache = make_cache("bf16", pages, 1, 16, D, dev)
    rope, one = kv.rope_table(20, D, device=dev), torch.ones(1, D, device=dev)
    att = kv.PagedAttention([cache], table.to(dev), H, rope=rope, q_norm=one, k_norm=one)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)              # noqa: E731
    seq, pos, slot = i32(0, -1, 2, 0, 0, 1, 1, 1), i32(3, 3, 3, -1, 20, 19, 3, 3), i32(3, 3, 3, 4, 5, 31, 32, -1)
    q, new = torch.randn(8, H * D, device=dev), torch.randn(8, D, device=dev)
    out, before = torch.full_like(q, 7.0), cache.k.clone()
    att.append(0, q, new, new, seq, pos, out, slot=slot)
    wrote = (out != 7.0).all(1).tolist()
    assert wrote == [True, False, False, False, False, True, False, False]
    assert (out[[1, 2, 3, 4, 6, 7]] == 7.0).all()
    changed = (cache.k != before).any(-1)[:, 0].nonzero().tolist()
    assert sorted(changed) == sorted([[int(table[0, 0]), 3], [int(table[1, 1]), 15]])
    # no rotation: any position will do, as the slot alone says where
    att = kv.PagedAttention([cache], table.to(dev), H, q_norm=one, k_norm=one)
    att.append(0, q, new, new, i32(*[0] * 8), i32(-5, 10 ** 9, 0, 0, 0, 0, 0, 0), out, slot=i32(*range(8)))
    assert (out != 7.0).all()


def test_layers_have_their_own_weights(dev):
    D, L = 64, 3
    table, pages = page_table([10], 16)
    caches = [make_cache("bf16", pages, 1, 16, D, dev) for _ in range(L)]
    w = torch.rand(L, D, device=dev) + 0.5
    att = kv.PagedAttention(caches, table.to(dev), 1, q_norm=w, k_norm=w, eps=0.0)
    x, at = torch.randn(1, D, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    got = torch.cat([att.append(i, x, x, x, at, at) for i in range(L)])
    want = x.double() / x.double().square().mean().sqrt() * w.double()
    assert ((got.double() - want).abs() <= 17 * U * want.abs()).all()
    assert torch.equal(att.append(-1, x, x, x, at, at)[0], got[L - 1])


def test_in_place_and_graph(dev):
    D, H, T = 128, 4, 6
    table, pages = page_table([40], 16)
    cache = make_cache("f16", pages, 2, 16, D, dev)
    w = torch.rand(1, D, device=dev) + 0.5
    att = kv.PagedAttention([cache], table.to(dev), H, rope=kv.rope_table(64, D, device=dev), q_norm=w, k_norm=w)
    q, k, v = (torch.randn(T, n * D, device=dev) for n in (H, 2, 2))
    seq, pos = torch.zeros(T, dtype=torch.int32, device=dev), torch.arange(T, device=dev).int()
    slot, out = pos.clone(), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.append(0, q, k, v, seq, pos, out, slot=slot)
    for i in range(4):
        q.normal_(), k.normal_()
        slot.copy_(torch.randperm(40, device=dev)[:T])
        cache.k.zero_()
        graph.replay()
        torch.cuda.synchronize()
        here = cache.k.clone()
        cache.k.zero_()
        want = q.clone()
        att.append(0, want, k, v, seq, pos, want, slot=slot)                   # in place
        assert torch.equal(out, want) and torch.equal(cache.k, here)


def test_refusals_on_the_device(dev):
    D, H = 64, 2
    table, pages = page_table([32], 16)
    cache = make_cache("bf16", pages, 1, 16, D, dev)
    one = torch.ones(1, D, device=dev)
    att = kv.PagedAttention([cache], table.to(dev), H, q_norm=one, k_norm=one)
    q, new, at = torch.randn(3, H * D, device=dev), torch.randn(3, D, device=dev), torch.arange(3, device=dev).int()
    for slot in (at.long(), at[:2], at.cpu(), torch.stack([at, at], 1)[:, 0], [0, 1, 2]):
        with pytest.raises(ValueError):
            att.append(0, q, new, new, at * 0, at, slot=slot)
    with pytest.raises(ValueError):
        att.append(0, q.half(), new, new, at * 0, at)
    with pytest.raises(ValueError, match="device"):
        kv.PagedAttention([cache], table.to(dev), H, q_norm=one.cpu())
