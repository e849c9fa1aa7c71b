"""Several requests decoded together: the products of kq.gpu4 with the paged cache, its attention and the penalised pick.

    python oxcoder-9b_amd/examples/decode_batch.py [--requests 8] [--steps 64] [--layers 4] [--cache bf16] [--nodes 16]

builds layers of the benchmark's 9B-class shape with synthetic weights (there is no checkpoint here), feeds every
request a prompt of its own length 16 tokens at a time, decodes greedily under a repetition penalty, and prints the
time of a step.  With --nodes it decodes once more, now several tokens a step: each request's earlier text drafts a tree of
continuations, one pass over all its nodes gives the logits after each, and what they accept is kept.  ``Decoder`` is
what a serving program keeps: the pages belong to it, requests may come and go with their rows of the table.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from kq import gpu4, kv, sampling  # noqa: E402
from kq import quantize as kqq  # noqa: E402
from kq.formats import Q4_K  # noqa: E402


class Decoder:
    """A llama-like stack over quantized weights for ``requests`` requests of up to ``positions`` positions each."""

    def __init__(self, layers, dim, q_heads, kv_heads, head_dim, ffn, vocab, requests, positions, cache="bf16", page=16,
                 mode="q8k", seed=0, device="cuda", nodes=0, head_norms=False):
        self.layers, self.dim, self.vocab, self.requests, self.nodes = layers, dim, vocab, requests, nodes
        self.kv_dim, self.device = kv_heads * head_dim, torch.device(device)
        w = gpu4.Weights(device)
        shapes = {"q": (q_heads * head_dim, dim), "k": (self.kv_dim, dim), "v": (self.kv_dim, dim),
                  "o": (dim, q_heads * head_dim), "gate": (ffn, dim), "up": (ffn, dim), "down": (dim, ffn)}
        for i in range(layers):
            for j, (name, (R, C)) in enumerate(shapes.items()):
                w.add("%d.%s" % (i, name), kqq.synthetic_matrix(R, C, Q4_K, seed=seed + 100 * i + j), R, C, Q4_K)
        for j, name in enumerate(("token_embd.weight", "output")):
            w.add(name, kqq.synthetic_matrix(vocab, dim, Q4_K, seed=seed + 90 + j), vocab, dim, Q4_K)
        rows = max(16, nodes) * max(requests, 1)
        self.eng = gpu4.Engine(w, mode=mode, chunk=rows)
        self.norm = torch.ones(dim, device=device)
        # a pool with a page for every position of every request; a serving program hands pages out as contexts grow
        width = -(-positions // page)
        table = torch.arange(requests * width, dtype=torch.int32, device=device).view(requests, width)
        self.caches = [kv.KVCache(requests * width, page, kv_heads, head_dim, cache, device) for _ in range(layers)]
        g = torch.Generator().manual_seed(seed)
        q_norm, k_norm = ((1 + 0.2 * torch.randn((layers, head_dim), generator=g)).to(device) if head_norms else None for _ in range(2))
        self.att = kv.PagedAttention(self.caches, table, q_heads, tokens=16, rope=kv.rope_table(positions, head_dim, device=device),
                                     q_norm=q_norm, k_norm=k_norm, nodes=nodes)
        self.picker = sampling.Picker(requests, device)
        if nodes:
            self.tree = kv.Tree(requests, nodes, device)
            self.verifier = sampling.Verifier(requests, nodes, vocab, device)
        self.h, self.xn, self.res = (torch.empty((rows, dim), device=device) for _ in range(3))
        self.q, self.a = (torch.empty((rows, q_heads * head_dim), device=device) for _ in range(2))
        self.k, self.v = (torch.empty((rows, self.kv_dim), device=device) for _ in range(2))
        self.gate, self.up, self.act = (torch.empty((rows, ffn), device=device) for _ in range(3))
        self.logits = torch.empty((requests * max(nodes, 1), vocab), device=device)

    def _rows(self, names, x, outs):
        """The named matrices on the rows of x."""
        self.eng.feed_rows(names, x, outs)

    def _stack(self, ids, attend):
        """The layers on one row for each of ids (below 0: anything), attend(i, q, k, v, out) being layer i's cache; the normed rows."""
        N = len(ids)
        h, xn, res = self.h[:N], self.xn[:N], self.res[:N]
        for n, tok in enumerate(ids):
            self.eng.embed(max(tok, 0), h[n])
        q, k, v, a = self.q[:N], self.k[:N], self.v[:N], self.a[:N]
        gate, up, act = self.gate[:N], self.up[:N], self.act[:N]
        add = None
        for i in range(self.layers):
            self.eng.rmsfold_q8k(h, self.norm, residual=add, xn=xn)
            self._rows(["%d.q" % i, "%d.k" % i, "%d.v" % i], xn, [q, k, v])
            attend(i, q, k, v, a)
            self._rows(["%d.o" % i], a, [res])
            self.eng.rmsfold_q8k(h, self.norm, residual=res, xn=xn)
            self._rows(["%d.gate" % i, "%d.up" % i], xn, [gate, up])
            self.eng.swiglu_q8k(gate, up, y=act)
            self._rows(["%d.down" % i], act, [res])
            add = res
        self.eng.rmsfold_q8k(h, self.norm, residual=add, xn=xn)
        return xn

    def forward(self, tokens, pos):
        """tokens: a list of T ids (1..16) for each request, pos int32 [requests]: where the first of them stands.
        A request without tokens is given ids and a position of -1: it reads nothing, writes nothing and
        its logits mean nothing.  Returns the logits [requests][vocab] after each request's last token."""
        B, T = len(tokens), len(tokens[0])
        dev = self.device
        at = pos[:, None] + torch.arange(T, dtype=torch.int32, device=dev)
        at = torch.where(pos[:, None] < 0, -1, at).reshape(-1).to(torch.int32)
        seq = torch.arange(B, dtype=torch.int32, device=dev).repeat_interleave(T)
        lens = torch.where(pos < 0, 0, pos + T).to(torch.int32)

        def attend(i, q, k, v, a):
            self.att.append(i, q, k, v, seq, at, q)
            self.att.attend(i, q, lens, a, tokens=T)

        xn = self._stack([t for row in tokens for t in row], attend)
        self._rows(["output"], xn[T - 1::T].contiguous(), [self.logits[:B]])
        return self.logits[:B]

    def forward_tree(self, tokens, parents, base):
        """tokens: a list of the constructor's ``nodes`` ids for each request, parents int32 [requests][nodes] and base int32
        [requests] as kv.Tree.plan takes them.  Returns the logits [requests * nodes][vocab], a row after each node."""
        tree = self.tree.plan(parents, base)

        def attend(i, q, k, v, a):
            self.att.append(i, q, k, v, tree.seq, tree.pos, q, slot=tree.slot)
            self.att.attend_tree(i, q, tree, a)

        self._rows(["output"], self._stack([t for row in tokens for t in row], attend), [self.logits])
        return self.logits

    def _feed(self, prompts):
        """All but each prompt's last token, 16 at a time while every request has as many, then one by one."""
        B, done = len(prompts), [0] * len(prompts)
        while any(done[b] < len(prompts[b]) - 1 for b in range(B)):
            left = [len(prompts[b]) - 1 - done[b] for b in range(B)]
            T = 16 if min(n for n in left if n) >= 16 else 1
            rows = [prompts[b][done[b]:done[b] + T] if left[b] else [-1] * T for b in range(B)]
            self.forward(rows, torch.tensor([done[b] if left[b] else -1 for b in range(B)], dtype=torch.int32, device=self.device))
            done = [done[b] + (T if left[b] else 0) for b in range(B)]

    def generate(self, prompts, steps, penalty=1.1):
        """Greedy continuations of the prompts (lists of ids), ``steps`` tokens each."""
        B, dev = len(prompts), self.device
        history = torch.zeros((B, max(map(len, prompts)) + steps), dtype=torch.int32, device=dev)
        for b, p in enumerate(prompts):
            history[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        length = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
        repetition = torch.full((B,), float(penalty), device=dev)
        self._feed(prompts)
        out, last = [[] for _ in range(B)], [p[-1] for p in prompts]
        for _ in range(steps):
            logits = self.forward([[t] for t in last], length - 1)
            picked = self.picker.pick(logits, history=history, length=length, repetition=repetition)
            history.scatter_(1, length[:, None].long(), picked[:, None])
            length += 1
            last = picked.tolist()
            for b in range(B):
                out[b].append(last[b])
        return out

    def generate_tree(self, prompts, steps, temperature=0.0, seed=0):
        """Continuations of the prompts, ``steps`` tokens each, drawn at a temperature (0: greedy), by trees of ``nodes`` drafted
        tokens: what came after a request's last token earlier in its text.  The prompts and ``steps`` + ``nodes`` further
        tokens fit the cache.  Returns (continuations, passes over the layers)."""
        B, T, dev = len(prompts), self.nodes, self.device
        g = torch.Generator(device=dev).manual_seed(seed)
        heat = torch.full((B,), float(temperature), device=dev)
        self._feed(prompts)
        text, passes = [list(p) for p in prompts], 0
        while any(len(text[b]) < len(prompts[b]) + steps for b in range(B)):
            on = [len(text[b]) < len(prompts[b]) + steps for b in range(B)]
            drafts = [draft_tree(text[b], T) if on[b] else ([-1] * T, [-2] * T) for b in range(B)]
            tokens, parents = ([d[i] for d in drafts] for i in range(2))
            ids, parents = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (tokens, parents))
            base = torch.tensor([len(text[b]) - 1 if on[b] else -1 for b in range(B)], dtype=torch.int32, device=dev)
            logits = self.forward_tree(tokens, parents, base)
            uniform = torch.rand((B, T), generator=g, device=dev)
            accepted, path, token = self.verifier.verify(logits, ids, parents, uniform, temperature=heat)
            self.att.keep(path, base)
            for b, (n, way, t) in enumerate(zip(accepted.tolist(), path.tolist(), token.tolist())):
                if on[b]:
                    text[b] += [tokens[b][i] for i in way[1:n + 1]] + [t]
            passes += 1
        return [text[b][len(prompts[b]):len(prompts[b]) + steps] for b in range(B)], passes


def draft_tree(text, nodes, depth=8):
    """(ids, parents) of a tree below text's last token: what followed it earlier, the latest first, up to ``depth`` ids each
    time; the nodes that are left over are none."""
    ids, parents, child = [text[-1]], [-1], {}
    for i in range(len(text) - 2, -1, -1):
        if text[i] != text[-1]:
            continue
        at = 0
        for t in text[i + 1:i + 1 + depth]:
            if (at, t) not in child:
                if len(ids) == nodes:
                    return ids, parents
                child[at, t] = len(ids)
                ids.append(t)
                parents.append(at)
            at = child[at, t]
    left = nodes - len(ids)
    return ids + [-1] * left, parents + [-2] * left


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--cache", default="bf16", choices=sorted(kv.DTYPES))
    p.add_argument("--nodes", type=int, default=0, help="decode by trees of so many tokens as well")
    a = p.parse_args()
    dec = Decoder(a.layers, 4096, 32, 8, 128, 12288, 4096, a.requests, 1024, a.cache, nodes=a.nodes)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 4096, (17 + 13 * b,), generator=g).tolist() for b in range(a.requests)]
    dec.generate(prompts, 2)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    out = dec.generate(prompts, a.steps)
    torch.cuda.synchronize()
    fed = max(map(len, prompts)) - 1
    print("%d requests, %d layers: %d tokens each after prompts of up to %d in %.1f ms" % (
        a.requests, a.layers, a.steps, fed + 1, 1e3 * (time.perf_counter() - t0)))
    print("first request:", out[0][:16])
    if a.nodes:
        dec.generate_tree(prompts, 2)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        out, passes = dec.generate_tree(prompts, a.steps)
        torch.cuda.synchronize()
        print("trees of %d: %d tokens each in %d passes, %.1f ms" % (a.nodes, a.steps, passes, 1e3 * (time.perf_counter() - t0)))


if __name__ == "__main__":
    main()
