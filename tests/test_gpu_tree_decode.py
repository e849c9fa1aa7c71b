"""A step by trees of drafted tokens as the example runs it: plan, append with norms of the heads, attention, verification and
the accepted entries kept, over all layers and many steps.  In fp32 numerics the products' rows depend on that row alone, so a
greedy continuation by trees is the one token by token wherever the two largest logits lie further apart than the
two attentions' rounding, and the caches then hold the same entries up to it."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "oxcoder-9b_amd", "examples"))


def prompts(n):
    """Texts that repeat themselves, so that something can be drafted."""
    g = torch.Generator().manual_seed(11)
    out = []
    for m, again in ((12, 3), (1, 1), (7, 4), (20, 2))[:n]:
        out.append(torch.randint(0, 1024, (m,), generator=g).tolist() * again)
    return out


def decoder(dev, requests, cache, nodes, mode="f32", norms=True):
    from decode_batch import Decoder
    return Decoder(2, 512, 8, 2, 64, 1024, 1024, requests, 192, cache, mode=mode, device=dev, nodes=nodes, head_norms=norms)


def test_drafts():
    from decode_batch import draft_tree
    assert draft_tree([5], 3) == ([5, -1, -1], [-1, -2, -2])
    assert draft_tree([1, 2, 3, 1, 2, 4, 1], 6) == ([1, 2, 4, 1, 3, 1], [-1, 0, 1, 2, 1, 4])
    assert draft_tree([1, 2, 3, 1, 2, 4, 1], 3) == ([1, 2, 4], [-1, 0, 1])
    assert draft_tree([7, 7, 7], 8) == ([7, 7, 7, -1, -1, -1, -1, -1], [-1, 0, 1, -2, -2, -2, -2, -2])
    ids, parents = draft_tree([3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3], 64, depth=4)
    assert len(ids) == 64 and all(p < t for t, p in enumerate(parents))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,nodes,norms", [("f16", 16, True), ("bf16", 16, False), ("i8", 9, True), ("f16", 64, True), ("bf16", 1, True)])
def test_greedy_as_token_by_token(dev, cache, nodes, norms):
    ids, steps = prompts(4), 40
    plain, tree = decoder(dev, 4, cache, nodes, norms=norms), decoder(dev, 4, cache, nodes, norms=norms)
    want = plain.generate(ids, steps, penalty=1.0)
    got, passes = tree.generate_tree(ids, steps)
    print("tree decode", cache, nodes, passes, "passes", flush=True)
    assert got == want
    assert passes <= steps                                     # a request's every pass gives a token at least
    # the entries of the tokens that both have fed, all but the last one: the attentions' rounding moves an element to its neighbour
    # in the cache's type at times, 2^-8 of bf16 or one code of 127, and to no more than two of those
    for a, b in zip(plain.caches, tree.caches):
        for r, p in enumerate(ids):
            for n in range(len(p) + steps - 1):
                page, off = r * (192 // 16) + n // 16, n % 16
                for x, y in ((a.k, b.k), (a.v, b.v)):
                    x, y = x[page, :, off].float(), y[page, :, off].float()
                    assert torch.allclose(x, y, rtol=0, atol=2.0 ** -6 * float(x.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_right_drafts_among_wrong_ones(dev, cache):
    """Trees that hold the next tokens on a way of every other node, wrong ones between them: the way is taken whole and its
    entries, which lie apart, are moved together, so that the next step's way is taken too."""
    ids, steps, nodes = prompts(4), 40, 15
    want = decoder(dev, 4, cache, nodes).generate(ids, steps, penalty=1.0)
    dec = decoder(dev, 4, cache, nodes)
    dec._feed(ids)
    done = 0
    while done + 8 <= steps:
        # node 0, then at 2 j - 1 a wrong token and at 2 j the right one, both after node 2 j - 2
        tokens = [[(ids[b] + want[b])[len(ids[b]) - 1 + done]] for b in range(4)]
        for b in range(4):
            for t in want[b][done:done + 7]:
                tokens[b] += [(t + 1) % 1024, t]
        up = [-1] + [2 * (j // 2) for j in range(14)]
        parents = torch.tensor([up] * 4, dtype=torch.int32, device=dev)
        base = torch.tensor([len(p) - 1 + done for p in ids], dtype=torch.int32, device=dev)
        logits = dec.forward_tree(tokens, parents, base)
        uniform = torch.rand((4, nodes), device=dev)
        accepted, path, token = dec.verifier.verify(logits, torch.tensor(tokens, dtype=torch.int32, device=dev), parents, uniform,
                                                    temperature=torch.zeros(4, device=dev))
        dec.att.keep(path, base)
        assert accepted.tolist() == [7] * 4 and path.tolist() == [list(range(0, 15, 2)) + [-1] * 7] * 4
        assert token.tolist() == [w[done + 7] for w in want]
        done += 8


@pytest.mark.gpu
def test_drawn(dev):
    """The same random numbers give the same text again; each id is one of the vocabulary."""
    ids = prompts(4)
    a, passes = decoder(dev, 4, "bf16", 16).generate_tree(ids, 24, temperature=0.7, seed=3)
    assert (a, passes) == decoder(dev, 4, "bf16", 16).generate_tree(ids, 24, temperature=0.7, seed=3)
    assert a != decoder(dev, 4, "bf16", 16).generate_tree(ids, 24, temperature=0.7, seed=4)[0]
    assert all(len(row) == 24 and all(0 <= t < 1024 for t in row) for row in a)


@pytest.mark.gpu
def test_quantized_activations(dev):
    """The engine's default numerics: the products of 64 rows go through the GEMM."""
    ids = prompts(4)
    out, _ = decoder(dev, 4, "f16", 16, "q8k").generate_tree(ids, 16)
    assert out == decoder(dev, 4, "f16", 16, "q8k").generate_tree(ids, 16)[0]
    assert all(len(row) == 16 and all(0 <= t < 1024 for t in row) for row in out)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_a_captured_step(dev, cache):
    """Plan, append, attention, verification and the kept entries of two layers as one graph: each replay, with other trees, bases and
    random numbers in its tensors and eager work between, leaves the bits of the eager calls."""
    from kq import kv, sampling
    from tree_helpers import random_parents
    B, T, H, KV, D, V, W = 3, 24, 4, 2, 64, 5000, 12
    table = torch.randperm(B * W, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(B, W).to(dev)
    g = torch.Generator().manual_seed(2)
    norm = (1 + 0.1 * torch.randn((2, D), generator=g)).to(dev)

    class Side:
        def __init__(self):
            self.caches = [kv.KVCache(B * W, 16, KV, D, cache, dev) for _ in range(2)]
            self.att = kv.PagedAttention(self.caches, table, H, rope=kv.rope_table(W * 16, D, device=dev), q_norm=norm, k_norm=norm,
                                         nodes=T)
            self.tree, self.ver = kv.Tree(B, T, dev), sampling.Verifier(B, T, V, dev)
            self.out = [torch.zeros((B * T, H * D), device=dev) for _ in range(2)]
            self.turned = torch.zeros((B * T, H * D), device=dev)

        def step(self, x):
            self.tree.plan(x["parents"], x["base"])
            for i in range(2):
                self.att.append(i, x["q"], x["k"], x["v"], self.tree.seq, self.tree.pos, self.turned, slot=self.tree.slot)
                self.att.attend_tree(i, self.turned, self.tree, self.out[i])
            accepted, path, token = self.ver.verify(x["logits"], x["tokens"], x["parents"], x["uniform"])
            self.att.keep(path, x["base"])
            return accepted, path, token

        def held(self):
            return [t for c in self.caches for t in (c.k, c.v)] + self.out

    def given(i):
        g = torch.Generator().manual_seed(10 + i)
        logits = torch.randn((B * T, V), generator=g)
        tokens = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32)
        logits.view(B, T, V).scatter_add_(2, tokens.long()[:, None].expand(B, T, T).contiguous(), torch.full((B, T, T), 9.0))
        base = torch.tensor([[5, 70, 0], [9, -1, 17], [31, 80, 2], [0, 100, 160]][i], dtype=torch.int32)
        return dict(logits=logits, tokens=tokens, parents=random_parents(B, T, i), base=base, uniform=torch.rand((B, T), generator=g),
                    q=torch.randn((B * T, H * D), generator=g), k=torch.randn((B * T, KV * D), generator=g),
                    v=torch.randn((B * T, KV * D), generator=g))

    eager, replayed = Side(), Side()
    x = {n: t.to(dev) for n, t in given(0).items()}
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        replayed.step(x)                                       # (every kernel is loaded)
    s.synchronize()
    eager.step(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = replayed.step(x)
    some = 0
    for i in (1, 2, 3, 1):
        for n, t in given(i).items():
            x[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        mine = [t.clone() for t in got]
        want = eager.step(x)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mine, want))
        assert all(torch.equal(a, b) for a, b in zip(replayed.held(), eager.held()))
        some += int(mine[0].clamp(min=0).sum())
    assert some > 0
