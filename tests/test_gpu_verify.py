"""kq_verify against its definition in 64 bits (tree_helpers.verification): choices are equal unless a comparison falls
nearer its border than the weights' last bits; and that tokens come with the target's own probabilities."""
import numpy as np
import pytest
import torch

from kq import sampling
from tree_helpers import NEAR, chain, random_parents, verification

pytestmark = pytest.mark.gpu


def inputs(B, T, V, seed=0, spread=2.5, draft=False, parents=None, likely=True):
    """Logits with a few likely ids, drafts among them (or drawn from the draft's rows), random numbers."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((B, T, V)) * spread).astype(np.float32)
    n = min(4, V)
    top = np.stack([rng.permutation(V)[:n] if V < 1000 else rng.choice(V, n, replace=False) for _ in range(B * T)]).reshape(B, T, n)
    if likely:
        lift = np.log(V) + spread ** 2 / 2 + np.array([0.5, -0.7, -1.5, -2.2])[:n]
        np.put_along_axis(x, top, np.broadcast_to(lift, (B, T, n)).astype(np.float32), 2)
    parents = random_parents(B, T, seed).numpy() if parents is None else parents
    up = np.clip(np.broadcast_to(parents, (B, T)), 0, T - 1)
    q = None
    if draft:
        y = x + 0.7 * rng.standard_normal(x.shape)
        e = np.exp(y - y.max(-1, keepdims=True))
        q = (e / e.sum(-1, keepdims=True)).astype(np.float32)
        tokens = np.zeros((B, T), np.int32)
        for b in range(B):
            for t in range(T):
                run = q[b, up[b, t]].astype(np.float64).cumsum()
                tokens[b, t] = np.argmax(run > rng.random() * run[-1])
        q = q.reshape(B * T, V)
    else:
        tokens = np.take_along_axis(top.reshape(B, -1), up * n + rng.integers(0, n, (B, T)), 1).astype(np.int32)
    return x.reshape(B * T, V), tokens, parents.astype(np.int32), rng.random((B, T), dtype=np.float32), q


def call(dev, x, tokens, parents, uniform, temperature=None, draft=None, ver=None):
    (B, T), V = tokens.shape, x.shape[1]
    ver = sampling.Verifier(B, T, V, dev) if ver is None else ver

    def put(a):
        return None if a is None else a if isinstance(a, torch.Tensor) else torch.from_numpy(a).to(dev)

    got = ver.verify(put(x), put(tokens), put(parents), put(uniform), put(temperature), put(draft))
    return [g.cpu().tolist() for g in got]


def check(dev, x, tokens, parents, uniform, temperature=None, draft=None, ver=None):
    print("verify", tokens.shape, x.shape[1], temperature is not None, draft is not None, flush=True)
    got = call(dev, x, tokens, parents, uniform, temperature, draft, ver)
    want = verification(x, tokens, parents, uniform, temperature, draft)
    near = 0
    for b, (accepted, path, token, gap) in enumerate(want):
        if gap <= NEAR:
            near += 1
            continue
        assert (got[0][b], got[1][b], got[2][b]) == (accepted, path, token), (b, gap)
    assert near <= 1 + len(want) // 50
    return got


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("V", [1, 2, 3, 5, 31, 1000, 1024, 2047, 2048, 2049, 8191, 8192, 8193, 20000, 50257])
def test_vocabularies(dev, V, draft):
    check(dev, *inputs(5, 6, V, seed=V, draft=draft)[:4], draft=inputs(5, 6, V, seed=V, draft=draft)[4])


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("B,T", [(1, 1), (1, 2), (1, 64), (3, 33), (64, 5), (300, 3)])
def test_batches_and_trees(dev, B, T, draft):
    x, tokens, parents, u, q = inputs(B, T, 700, seed=T, draft=draft)
    check(dev, x, tokens, parents, u, draft=q)
    x, tokens, parents, u, q = inputs(B, T, 700, seed=T + 1, draft=draft, parents=chain(B, T).numpy())
    check(dev, x, tokens, parents, u, draft=q)
    one = random_parents(1, T, 5).numpy()                       # one tree for all
    x, tokens, parents, u, q = inputs(B, T, 700, seed=T + 2, draft=draft, parents=one)
    check(dev, x, tokens, one, u, draft=q)


def test_large(dev):
    for draft in (False, True):
        x, tokens, parents, u, q = inputs(3, 7, 151936, seed=1, draft=draft)
        check(dev, x, tokens, parents, u, np.array([0.8, 1.0, 1.3], np.float32), q)
    x, tokens, parents, u, q = inputs(2, 64, 32000, seed=2)
    check(dev, x, tokens, parents, u)


@pytest.mark.parametrize("B,T,V,draft", [(40, 24, 60001, False), (17, 64, 50000, False), (170, 5, 100000, False),
                                         (20, 16, 140000, True)])
def test_more_rows_than_are_read_at_once(dev, B, T, V, draft):
    """Walks that go on where the rows read so far end, in chains, trees and stars; accepted to the last node by random numbers of 0."""
    for seed in range(2):
        parents = chain(B, T).numpy() if draft else random_parents(B, T, seed).numpy()
        parents[B // 2:] = np.maximum(np.arange(T) - 1, 0) - (np.arange(T) == 0)
        parents[0, 1:] = 0
        x, tokens, parents, u, q = inputs(B, T, V, seed=seed, draft=draft, parents=parents)
        u[1::3, 1:] = 0
        got = check(dev, x, tokens, parents, u, draft=q)
        assert max(got[0]) == T - 1


@pytest.mark.parametrize("draft", [False, True])
def test_temperatures(dev, draft):
    """Cold, hot, greedy (0, below, NaN); infinitely hot: every finite logit alike."""
    t = np.array([1e-3, 0.1, 0.5, 1.0, 3.0, 50.0, 0.0, -1.0, np.nan, 1e-30, 1e30], np.float32)
    x, tokens, parents, u, q = inputs(len(t), 6, 900, seed=3, draft=draft)
    check(dev, x, tokens, parents, u, t, q)


def test_ties_under_greedy(dev):
    """The first of equal largest logits alone: drafts of it are taken, of its equals not."""
    V = 9000
    x = np.zeros((4, V), np.float32)
    x[:, [77, 4000, 8999]] = 5.0
    tokens, parents = np.array([[0, 4000, 77, 8999]], np.int32), np.array([[-1, 0, 0, 2]], np.int32)
    u = np.full((1, 4), 0.999, np.float32)
    assert check(dev, x, tokens, parents, u, np.zeros(1, np.float32)) == [[1], [[0, 2, -1, -1]], [77]]


def test_logits_without_probability(dev):
    """-inf and NaN have none; a row of them ends the walk with no token; +inf takes all."""
    V, B, T = 3000, 6, 4
    x, tokens, parents, u, _ = inputs(B, T, V, seed=4)
    x = x.reshape(B, T, V)
    x[0, :, ::2] = -np.inf
    x[1, :, 5:] = np.nan
    x[2] = -np.inf
    x[3, 1:] = np.nan
    tokens[3, 1], parents[3, 1] = int(np.nanargmax(x[3, 0])), 0
    u[3, 1] = 0
    x[4, :, [9, 2000]] = np.inf
    x[5, :, :-1] = -np.inf
    got = check(dev, x.reshape(-1, V), tokens, parents, u)
    assert got[2][2] == -1 and got[0][2] == 0 and got[0][3] == 1 and got[2][3] == -1
    assert got[2][4] in (9, 2000) and got[2][5] == V - 1


def test_two_ids_left(dev):
    """A mask that leaves two ids, both drafted: one of them is always taken."""
    V, B = 5000, 64
    rng = np.random.default_rng(0)
    x = np.full((B, 3, V), -np.inf, np.float32)
    x[:, :, [40, 4100]] = rng.standard_normal((B, 3, 2))
    tokens = np.tile(np.array([[0, 4100, 40]], np.int32), (B, 1))
    parents, u = np.array([[-1, 0, 0]], np.int32), rng.random((B, 3), dtype=np.float32)
    u[:8, 1:] = 1 - 2.0 ** -24
    got = check(dev, x.reshape(-1, V), tokens, parents, u)
    assert got[0] == [1] * B


def test_drafts_that_are_none(dev):
    """Ids outside the vocabulary, parents that are none, the same id twice among siblings, requests that sit out."""
    V, B, T = 400, 6, 6
    x, tokens, parents, u, q = inputs(B, T, V, seed=5, draft=True)
    tokens[0], tokens[1, 1:3] = V, [-1, 2 ** 31 - 1]
    parents[2, 1:] = [5, -1, -2, 63, 9]
    parents[3] = [-1, 0, 0, 0, 0, 0]
    tokens[3] = tokens[3, 1]
    parents[4, 0], parents[5, 0] = 0, -2
    for draft in (None, q):
        got = check(dev, x, tokens, parents, u, draft=draft)
        assert got[0][0] == 0 and got[0][2] == 0 and got[0][4:] == [-1, -1] and got[2][4:] == [-1, -1]
        assert got[1][4] == [-1] * T


def test_random_numbers_at_the_ends(dev):
    """0 takes every draft that has a probability and the first id that has one; just below 1 the last."""
    V, T = 2500, 5
    x, tokens, parents, u, _ = inputs(2, T, V, seed=6, parents=chain(2, T).numpy())
    x[:, 0] = -np.inf
    x[:, -1] = -np.inf
    u[0], u[1] = 0, 1 - 2.0 ** -24
    got = call(dev, x, tokens, parents, u)
    assert got[0] == [T - 1, 0] and got[2] == [1, V - 2]


def test_nothing_left(dev):
    """A draft's probabilities that cover the target's everywhere: the token is then drawn from the target itself."""
    V = 600
    x, tokens, parents, u, _ = inputs(3, 2, V, seed=7, parents=chain(3, 2).numpy())
    q = np.full((6, V), 1.0, np.float32)
    u[:, 1] = 0.9999
    got = check(dev, x, tokens, parents, u, draft=q)
    assert got[0] == [0, 0, 0]


def test_the_target_itself_as_draft(dev):
    """Drafts drawn from the target's own probabilities: p and q differ by roundings alone, so all are taken."""
    V, T, B = 2000, 5, 40
    x, tokens, parents, u, _ = inputs(B, T, V, seed=8, parents=chain(B, T).numpy())
    e = np.exp(x.astype(np.float64) - x.max(-1, keepdims=True))
    q = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    u = np.minimum(u, np.float32(0.999))
    got = call(dev, x, tokens, parents, u, draft=q)
    assert got[0] == [T - 1] * B


@pytest.mark.parametrize("draft", [False, True])
def test_tokens_have_the_targets_probabilities(dev, draft):
    """First tokens of 60000 requests whose drafts are two siblings and a grandchild: each id as often as the target has
    it, within six standard deviations."""
    B, T, V = 15000, 4, 6
    rng = np.random.default_rng(9)
    logits = rng.standard_normal((T, V)).astype(np.float32)
    p = np.exp(logits[0].astype(np.float64))
    p /= p.sum()
    dq = rng.random((T, V)).astype(np.float32)
    dq /= dq.sum(-1, keepdims=True)
    parents = np.array([[-1, 0, 0, 1]], np.int32)
    x = np.tile(logits, (B, 1))
    q = np.tile(dq, (B, 1)) if draft else None
    ver, count = sampling.Verifier(B, T, V, dev), np.zeros(V)
    xd, qd = torch.from_numpy(x).to(dev), torch.from_numpy(q).to(dev) if draft else None
    for i in range(4):
        tokens = np.zeros((B, T), np.int32)
        for t in (1, 2, 3):
            tokens[:, t] = rng.choice(V, B, p=dq[parents[0, t]] / dq[parents[0, t]].sum()) if draft else rng.integers(0, V, B)
        u = rng.random((B, T), dtype=np.float32)
        accepted, path, token = call(dev, xd, tokens, parents, u, draft=qd, ver=ver)
        path, token, accepted = np.array(path), np.array(token), np.array(accepted)
        first = np.where(accepted > 0, tokens[np.arange(B), path[:, 1]], token)
        count += np.bincount(first, minlength=V)
    n = 4 * B
    assert (np.abs(count - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all(), (count / n, p)


def test_strided_rows_and_fewer_than_held(dev):
    """Logits, drafts and lists out of wider rows from odd places on; fewer requests, nodes and ids than the verifier holds."""
    B, T, V = 3, 5, 3001
    x, tokens, parents, u, q = inputs(B, T, V, seed=10, draft=True)

    def wide(a, pad, shift):
        big = torch.full((a.shape[0], a.shape[1] + pad), 7, dtype=torch.from_numpy(a).dtype, device=dev)
        big[:, shift:shift + a.shape[1]] = torch.from_numpy(a).to(dev)
        return big[:, shift:shift + a.shape[1]]

    ver = sampling.Verifier(5, 9, 4000, dev)
    for draft in (None, q):
        want = call(dev, x, tokens, parents, u, draft=draft)
        got = call(dev, wide(x, 10, 3), wide(tokens, 3, 1), wide(parents, 2, 2), wide(u, 5, 1), None,
                   None if draft is None else wide(draft, 7, 5), ver)
        assert got == want


def test_repeats_streams_and_graphs(dev):
    """The same bits call after call; on another stream; captured, with inputs read when the graph runs."""
    B, T, V = 4, 6, 9000
    ver = sampling.Verifier(B, T, V, dev)
    x, tokens, parents, u, q = (torch.from_numpy(a).to(dev) for a in inputs(B, T, V, seed=11, draft=True))
    for draft in (None, q):
        want = [g.clone() for g in ver.verify(x, tokens, parents, u, draft=draft)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [g.clone() for g in ver.verify(x, tokens, parents, u, draft=draft)]
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ver.verify(x, tokens, parents, u, draft=draft)
        for i in range(5):
            nx, nt, np_, nu, nq = inputs(B, T, V, seed=20 + i, draft=True)
            for a, b in ((x, nx), (tokens, nt), (parents, np_), (u, nu), (q, nq)):
                a.copy_(torch.from_numpy(b))
            graph.replay()
            torch.cuda.synchronize()
            got = [g.clone() for g in held]
            again = ver.verify(x, tokens, parents, u, draft=draft)
            assert all(torch.equal(a, b) for a, b in zip(got, again))
            check(dev, nx, nt, np_, nu, draft=None if draft is None else nq)


def test_refusals_on_the_device(dev):
    B, T, V = 2, 4, 500
    ver = sampling.Verifier(B, T, V, dev)
    x, tokens, parents, u, q = (torch.from_numpy(a).to(dev) for a in inputs(B, T, V, seed=12, draft=True))
    temp = torch.ones(B, device=dev)
    for a in ((x.half(), tokens, parents, u), (x[:-1], tokens, parents, u), (x.t().contiguous().t(), tokens, parents, u),
              (x.cpu(), tokens, parents, u), (x, tokens.long(), parents, u), (x, tokens.cpu(), parents, u),
              (x, tokens, parents.long(), u), (x, tokens, parents[:, :-1], u), (x, tokens, parents[0], u), (x, tokens, None, u),
              (x, tokens, parents, u.double()), (x, tokens, parents, u[:1]), (x, tokens, parents, None),
              (x, tokens, parents, u, temp.half()), (x, tokens, parents, u, temp[:1]), (x, tokens, parents, u, None, q.half()),
              (x, tokens, parents, u, None, q[:-1]), (x, tokens, parents, u, None, q[:, :-1])):
        with pytest.raises(ValueError):
            ver.verify(*a)
