"""kq_logits_penalize against the same steps in numpy's fp32 (each rounding alike: equal bits) and the pick's rule."""
import numpy as np
import pytest
import torch

from kq import ops, sampling

pytestmark = pytest.mark.gpu
F32 = np.float32


def steps(x, hist=None, length=None, prompt=None, rep=None, freq=None, pres=None, ids=None, vals=None, allowed=None, dt=F32):
    y = x.astype(dt)
    V = y.shape[1]
    for b in range(len(y)):
        row = y[b]
        if hist is not None:
            n = min(max(int(length[b]), 0), hist.shape[1])
            h = hist[b, :n]
            late = h[max(int(prompt[b]) if prompt is not None else 0, 0):]
            h, late = (a[(a >= 0) & (a < V)] for a in (h, late))
            seen, count = np.unique(h), np.bincount(late, minlength=V)
            if rep is not None:
                row[seen] = np.where(row[seen] > 0, row[seen] / dt(rep[b]), row[seen] * dt(rep[b]))
            c = np.nonzero(count)[0]
            if freq is not None:
                row[c] -= dt(freq[b]) * count[c].astype(dt)
            if pres is not None:
                row[c] -= dt(pres[b])
        if ids is not None:
            last = {int(i): v for i, v in zip(ids[b], vals[b]) if 0 <= i < V}
            for i, v in last.items():
                row[i] += dt(v)
        if allowed is not None:
            words = allowed[b if len(allowed) > 1 else 0].view(np.uint32)
            bits = (words[np.arange(V) >> 5] >> (np.arange(V) & 31).astype(np.uint32)) & 1
            row[bits == 0] = -np.inf
    return y


def picks(y):
    out = []
    for row in y:
        r = np.where(np.isnan(row), -np.inf, row)
        i = int(np.argmax(r))
        out.append(i if r[i] > F32(-1e30) else -1)
    return out


NAMES = ("history", "length", "prompt", "repetition", "frequency", "presence", "bias_ids", "bias_values", "allowed")


def check(dev, x, *args, shift=0):
    """args in NAMES' order (numpy or None).  The logits from `shift` floats past an aligned place on."""
    B, V = x.shape
    print("logits", B, V, [n for n, a in zip(NAMES, args) if a is not None], shift, flush=True)
    flat = np.zeros(x.size + shift, F32)
    flat[shift:] = x.reshape(-1)
    xd = torch.from_numpy(flat).to(dev)[shift:].view(B, V)
    kw = {n: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev) for n, a in zip(NAMES, args)}
    p = sampling.Picker(B, dev)
    want = steps(x, *args)
    out = torch.full((B, V + 3), 7.0, device=dev)
    picked = p.pick(xd, out=out[:, :V], **kw)
    np.testing.assert_array_equal(out[:, :V].cpu().numpy(), want)
    assert (out[:, V:] == 7).all()
    assert picked.cpu().tolist() == picks(want)
    assert p.pick(xd, **kw).cpu().tolist() == picks(want)                     # without the logits; workspace used again
    aligned = torch.empty((B, V), device=dev)
    p.pick(xd, out=aligned, **kw)
    np.testing.assert_array_equal(aligned.cpu().numpy(), want)
    ops.logits_penalize(xd, *[kw[n] for n in NAMES], y=xd)                     # in place, without a pick
    np.testing.assert_array_equal(xd.cpu().numpy(), want)
    assert int(p.ws.to(torch.int32).abs().sum()) == 0


def inputs(B, V, L, nb, masked, seed=0):
    rng = np.random.default_rng(seed)
    x = (3 * rng.standard_normal((B, V))).astype(F32)
    hist = length = prompt = rep = freq = pres = ids = vals = allowed = None
    if L:
        hist = (V ** rng.random((B, L)) - 1).astype(np.int32)
        length = rng.integers(0, L + 1, B).astype(np.int32)
        length[0] = L
        prompt = (length * rng.random(B)).astype(np.int32)
        rep = (0.7 + rng.random(B)).astype(F32)
        freq, pres = (rng.random((2, B)) - 0.3).astype(F32)
    if nb:
        ids = rng.integers(-1, V, (B, nb)).astype(np.int32)
        vals = (5 * rng.standard_normal((B, nb))).astype(F32)
    if masked:
        allowed = rng.integers(-2 ** 31, 2 ** 31, (B, (V + 31) // 32)).astype(np.int32)
    return x, hist, length, prompt, rep, freq, pres, ids, vals, allowed


@pytest.mark.parametrize("B,V,L,nb", [(1, 1, 1, 1), (2, 31, 5, 3), (3, 4095, 40, 7), (1, 4096, 0, 0), (5, 4097, 300, 0),
                                      (2, 8195, 0, 20), (4, 32000, 1000, 300), (1, 151936, 5000, 50), (3, 248320, 100, 1)])
@pytest.mark.parametrize("masked", [False, True])
def test_sizes(dev, B, V, L, nb, masked):
    check(dev, *inputs(B, V, L, nb, masked, seed=V))


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_unaligned_rows(dev, shift):
    check(dev, *inputs(3, 5000, 50, 4, True), shift=shift)


@pytest.mark.parametrize("drop", [(0, 1, 2, 3, 4, 5), (2,), (3,), (4,), (5,), (6, 7), (8,), (3, 4, 5), tuple(range(9))])
def test_each_step_may_be_left_out(dev, drop):
    x, *args = inputs(3, 6000, 200, 10, True)
    check(dev, x, *[None if i in drop else a for i, a in enumerate(args)])


def test_many_rows(dev):
    check(dev, *inputs(300, 4200, 60, 4, True))


def test_histories(dev):
    """Lengths of none, below none and above what is held, prompts past the length, ids outside the vocabulary, one
    id over and over, and one that the slices of a row would each count."""
    B, V, L = 6, 9000, 400
    x, hist, length, prompt, rep, freq, pres, *_ = inputs(B, V, L, 0, False)
    hist[0], hist[1, ::2], hist[1, 1::2] = 4321, -1, V
    hist[2, :] = np.array([-2 ** 31, 2 ** 31 - 1, 0, V - 1] * 100)
    length[:] = [L, L, L, 0, -7, 10 ** 9]
    prompt[:] = [10, 0, 7, 0, 0, 10 ** 6]
    check(dev, x, hist, length, prompt, rep, freq, pres, None, None, None)


def test_an_ids_last_bias_counts(dev):
    x = np.zeros((2, 500), F32)
    ids = np.array([[3, 7, 3, -1, 7, 499, 3], [500, 2 ** 31 - 1, 0, 0, 0, 0, 0]], np.int32)
    vals = np.arange(1, 15, dtype=F32).reshape(2, 7)
    check(dev, x, None, None, None, None, None, None, ids, vals, None)


def test_values(dev):
    """Infinities, NaN, zeros of both signs, subnormals and the type's lowest value go through as fp32 steps them."""
    v = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-41, -1e-41, np.finfo(F32).min, np.finfo(F32).max, 1.0, -1.0], F32)
    x = np.tile(v, (3, 40))
    hist = np.tile(np.arange(0, 440, 3, dtype=np.int32), (3, 1))
    length = np.full(3, hist.shape[1], np.int32)
    rep, freq, pres = np.array([1.5, 0.5, 1.0], F32), np.array([0.1, -0.2, 0], F32), np.array([0.3, 0, 0], F32)
    ids = np.tile(np.arange(22, dtype=np.int32), (3, 1))
    vals = np.tile(np.array([1, -np.inf], F32), (3, 11))
    with np.errstate(all="ignore"):
        check(dev, x, hist, length, None, rep, freq, pres, ids, vals, None)


def test_rows_that_leave_nothing(dev):
    """A mask without a bit, logits of -inf, NaN or at most -1e30: -1.  Ties go to the lowest id, across slices too."""
    V = 10000
    x = np.random.default_rng(0).standard_normal((6, V)).astype(F32)
    x[1], x[2], x[3] = -np.inf, np.nan, -1e30
    x[4, [9999, 4096, 4095]] = 50.0
    x[5] = 0.0
    allowed = np.full((6, (V + 31) // 32), -1, np.int32)
    allowed[0] = 0
    allowed[0, -1] = ~((1 << (V % 32)) - 1)          # only bits past the vocabulary
    with np.errstate(all="ignore"):
        check(dev, x, None, None, None, None, None, None, None, None, allowed)
    p = sampling.Picker(6, dev).pick(torch.from_numpy(x).to(dev), allowed=torch.from_numpy(allowed).to(dev))
    assert p.cpu().tolist() == [-1, -1, -1, -1, 4095, 0]


def test_one_mask_for_all_rows(dev):
    x, *_, allowed = inputs(4, 3000, 0, 0, True)
    check(dev, x, *[None] * 8, allowed[:1])


def test_other_stream_and_graph(dev):
    B, V = 3, 20000
    x, hist, length, prompt, rep, freq, pres, ids, vals, allowed = (
        torch.from_numpy(a).to(dev) for a in inputs(B, V, 100, 5, True))
    args = dict(history=hist, length=length, prompt=prompt, repetition=rep, frequency=freq, presence=pres, bias_ids=ids,
                bias_values=vals, allowed=allowed)
    p = sampling.Picker(B, dev)
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = p.pick(x, out=out, **args).clone()
    side.synchronize()
    assert torch.equal(a, p.pick(x, out=out, **args))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.pick(x, out=out, **args)
    for _ in range(3):
        x.normal_()
        length.random_(0, 101)
        graph.replay()
        torch.cuda.synchronize()
        a, y = p.picked.clone(), out.clone()
        assert torch.equal(p.pick(x, out=out, **args), a) and torch.equal(out, y)


@pytest.mark.parametrize("B,V", [(200, 9001), (600, 5000), (300, 20003)])
def test_slices(dev, B, V):
    """Batches whose rows are cut into fewer, larger slices."""
    check(dev, *inputs(B, V, 70, 6, True, seed=B))


@pytest.mark.parametrize("L,nb", [(3000, 2047), (3000, 2048), (3000, 5000), (1 << 20, 10), ((1 << 20) - 1, 10)])
def test_long_lists(dev, L, nb):
    """Bias lists and histories on both sides of what one note per id holds."""
    check(dev, *inputs(2, 6000, L, nb, True, seed=nb))


def test_refusals_on_the_device(dev):
    """Device tensors of another type, too small, of another layout or left out: refused before any launch."""
    B, V = 2, 300
    x, *args = (torch.from_numpy(a).to(dev) for a in inputs(B, V, 20, 5, True))
    good = dict(zip(NAMES, args))
    p = sampling.Picker(B, dev)
    for name, bad in (("history", good["history"].long()), ("history", good["history"][:1]), ("length", None),
                      ("length", good["length"][:1]), ("prompt", good["prompt"].long()), ("repetition", good["repetition"].double()),
                      ("frequency", good["frequency"][:1]), ("bias_values", None), ("bias_values", good["bias_values"][:, :4]),
                      ("bias_ids", good["bias_ids"].t().contiguous().t()), ("allowed", good["allowed"][:, :9]),
                      ("out", torch.empty(B, V - 1, device=dev)), ("out", torch.empty(B, V)), ("out", torch.empty(V, B, device=dev).t())):
        with pytest.raises(ValueError):
            p.pick(x, **{**good, name: bad})
    for logits in (x.double(), x.t().contiguous().t(), x.cpu()):
        with pytest.raises(ValueError):
            p.pick(logits, **good)
    assert p.pick(x, **good).cpu().tolist() == picks(steps(x.cpu().numpy(), *[a.cpu().numpy() for a in args]))
