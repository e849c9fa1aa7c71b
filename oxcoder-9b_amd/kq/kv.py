"""A paged key-value cache for several requests, and attention over it.

The reference's engine keeps one contiguous cache for its one request (scripts/kindi_q4/kindi/engine.py:255-280);
here requests share a pool of pages.  ``KVCache`` is one layer's pool, ``PagedAttention`` what a decoding
program calls between its q/k/v and output projections: ``append`` rotates the new tokens' queries and
keys and stores keys and values (kq_kv_append), ``attend`` runs their attention (kq_attn_paged).

    cache = [KVCache(pages, 16, 8, 128, "bf16") for _ in range(layers)]
    att = PagedAttention(cache, table, 32, tokens=1, rope=rope_table(4096, 128))
    att.append(layer, q, k, v, seq, pos, q)          # q is rotated in place
    att.attend(layer, q, lens, out)

A step that verifies drafts feeds a tree of tokens per request, whose node j lies in slot base + j of the cache:

    tree = Tree(requests, nodes)                      # one for all layers and steps
    att = PagedAttention(cache, table, 32, nodes=nodes, rope=rope_table(4096, 128))
    tree.plan(parents, base)                          # once a step
    att.append(layer, q, k, v, tree.seq, tree.pos, q, slot=tree.slot)
    att.attend_tree(layer, q, tree, out)
    att.keep(path, base)                              # the accepted nodes (sampling.Verifier), in all layers at once

``table`` is int32 [requests][pages of one]: the page of each run of ``page_size`` positions; the program
that owns the pool fills it, and may change it between calls (the kernels read it when they run).  An entry
outside the pool is a hole: nothing is stored there, and attention passes over it.
"""
import ctypes as C

import torch

from . import _lib, ops

_TYPES = {torch.float16: _lib.KQ_KV_F16, torch.bfloat16: _lib.KQ_KV_BF16, torch.int8: _lib.KQ_KV_I8}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}


def rope_table(positions, rot, base=10000.0, device="cuda"):
    """[positions][rot] floats for PagedAttention: rot/2 cosines of a position's angles p * base^(-2i/rot), then
    rot/2 sines, from angles in 64 bits."""
    inv = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], -1).float()


class KVCache:
    """One layer's pool: k and v [pages][heads][page_size][dim], for "i8" with fp32 scales [pages][heads]
    [page_size] (a value is code * scale)."""

    def __init__(self, pages, page_size, heads, dim, dtype="bf16", device="cuda"):
        if dtype not in DTYPES:
            raise ValueError("dtype must be one of %s" % sorted(DTYPES))
        shape, dt = (pages, heads, page_size, dim), DTYPES[dtype]
        k, v = (torch.zeros(shape, dtype=dt, device=device) for _ in range(2))
        ks, vs = ((torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)) if dt == torch.int8
                  else (None, None))
        self._bind(k, v, ks, vs)

    @classmethod
    def over(cls, k, v, k_scale=None, v_scale=None):
        """A cache in tensors that exist: k and v [pages][heads][page_size][dim] of any strides with contiguous heads
        (pages held position by position: pass k.transpose(1, 2)), alike for k and v."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _TYPES:
            raise ValueError("k and v must be [pages][heads][page_size][dim] of one type: float16, bfloat16 or int8")
        if k.stride() != v.stride():
            raise ValueError("k and v must have the same strides")
        pages, heads, size, dim = k.shape
        unit = 16 // k.element_size()
        # the stride of a dimension of one element is never used: any valid one does
        st = [s if n > 1 else -(-dim // unit) * unit for n, s in zip(k.shape, k.stride())][:3]
        sc = [0, 0, 0]
        if k.dtype == torch.int8:
            if k_scale is None or v_scale is None or k_scale.shape != k.shape[:3] or v_scale.shape != k.shape[:3]:
                raise ValueError("an int8 cache needs k_scale and v_scale [pages][heads][page_size]")
            if k_scale.stride() != v_scale.stride():
                raise ValueError("k_scale and v_scale must have the same strides")
            if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
                raise ValueError("scales must be float32")
            sc = [s if n > 1 else 1 for n, s in zip(k_scale.shape, k_scale.stride())]
        elif k_scale is not None or v_scale is not None:
            raise ValueError("only an int8 cache has scales")
        if dim > 1 and k.stride(3) != 1:
            raise ValueError("k and v must have unit stride along dim")
        held = [t for t in (k, v, k_scale, v_scale) if t is not None]
        if any(t.device != k.device for t in held):
            raise ValueError("k, v and their scales must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page_size, self.dim = pages, heads, size, dim
        self.device = k.device
        ptr = [t.data_ptr() if t is not None else None for t in (k, v, k_scale, v_scale)]
        self._kv = _lib.KV(*ptr, _TYPES[k.dtype], heads, dim, pages, size, *st, *sc)
        self.ref = C.addressof(self._kv)      # the const kq_kv* of the C ABI; lives as long as this object


class Tree:
    """What the calls of every layer take of a step's trees: ``plan`` fills, from the parents of each request's nodes, seq, pos
    and slot (int32 [requests * nodes], PagedAttention.append's) and seen (int64 [requests][nodes]: bit j of node t's
    word says that it sees node j, its ancestors and itself; 0: no node)."""

    def __init__(self, requests, nodes, device="cuda"):
        if not 1 <= requests <= 65535 or not 1 <= nodes <= _lib.KQ_MAX_TREE:
            raise ValueError("1..65535 requests of 1..%d nodes" % _lib.KQ_MAX_TREE)
        self.requests, self.nodes = requests, nodes
        self.seen = torch.zeros((requests, nodes), dtype=torch.int64, device=device)
        self.seq, self.pos, self.slot = (torch.full((requests * nodes,), -1, dtype=torch.int32, device=device) for _ in range(3))
        self.device, self.base = self.seen.device, None
        # what every call passes on, as addresses: the tensors stay as long as the tree
        self._held = tuple(t.data_ptr() for t in (self.seen, self.seq, self.pos, self.slot))
        self._calls = _lib.calls() if self.device.type == "cuda" else None

    def plan(self, parents, base):
        """parents: int32 [requests][nodes], or [1][nodes] for all requests: the node that node t follows, below t, or -1 where
        it follows the context; another value: no node, nor those that follow it.  base: int32 [requests], the
        positions ahead of the tree; below 0: the request sits out.  Node t lies in slot base + t and
        stands at position base + its ancestors' number.  base is read by attend_tree too: it stays as it is until
        the step's last call."""
        if not isinstance(base, torch.Tensor) or base.device != self.device:
            raise ValueError("base must be a device tensor, on the tree's device")
        rc = self._calls and self._calls.tree_plan(*self._held, ops._stream(self.device), parents, base, self.requests, self.nodes)
        if rc is None:                       # a tensor is not as it should be
            ops.tree_plan(parents, base, self.seen, self.seq, self.pos, self.slot, self.requests, self.nodes)
        elif rc:
            _lib.check(rc)
        self.base = base
        return self


class PagedAttention:
    """The attention of a decoding program over its layers' caches, with the one workspace it needs.

    caches: a KVCache per layer, all of one shape (types may differ); table: int32 [requests][width]; tokens: the most
    new tokens per request that attend will see (1..16); max_len: the most positions a request will hold
    (default: what its row of the table covers); rope: rope_table's, or None (nothing is rotated), whose width is
    the number of values that turn (append skips tokens at positions past its rows); interleaved: pairs (2i, 2i + 1)
    instead of (i, i + rot/2); scale: default dim ** -0.5.
    q_norm, k_norm: float32 [layers][dim], weights of a norm of each head of q (of k) that append applies ahead of the
    rotation, x / sqrt(mean(x^2) + eps) * w; nodes: the most nodes of a tree that attend_tree will see (0: none, up to 64).
    attend_tree shares a request's positions out by max_len, not by their number: it is fastest where that is near the longest
    request's (16 requests of 5000 positions: 173 us with 5027, 535 with 131072).
    These are for the object's life: another table or rotation takes another object, what is in them may change.
    Calls on one PagedAttention share its workspace and so must be ordered: one stream, or synchronised."""

    def __init__(self, caches, table, q_heads, tokens=1, max_len=None, rope=None, interleaved=False, scale=None,
                 q_norm=None, k_norm=None, eps=1e-6, nodes=0):
        if not caches:
            raise ValueError("one cache per layer")
        c = caches[0]
        if any((x.k.shape, x.device) != (c.k.shape, c.device) for x in caches):
            raise ValueError("the layers' caches must have the same pages, heads, page size, dim and device")
        if table.dim() != 2 or table.dtype != torch.int32 or table.device != c.device:
            raise ValueError("table must be int32 [requests][pages] on the caches' device")
        if not 1 <= tokens <= _lib.KQ_MAX_BATCH:
            raise ValueError("tokens must be 1..%d" % _lib.KQ_MAX_BATCH)
        if q_heads < 1 or q_heads % c.heads:
            raise ValueError("q_heads must be a multiple of the cache's %d heads" % c.heads)
        if not 0 <= nodes <= _lib.KQ_MAX_TREE:
            raise ValueError("nodes must be 0..%d" % _lib.KQ_MAX_TREE)
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None and (w.shape != (len(caches), c.dim) or w.dtype != torch.float32 or not w.is_contiguous()
                                  or w.device != c.device):
                raise ValueError("%s must be float32 [%d layers][%d], contiguous, on the caches' device"
                                 % (name, len(caches), c.dim))
        if not (eps >= 0 and eps < float("inf")):
            raise ValueError("eps must be finite, at least 0")
        self.caches, self.table, self.q_heads, self.tokens = tuple(caches), table, q_heads, tokens
        self.rope, self._interleaved = rope, 1 if interleaved else 0
        self.scale = c.dim ** -0.5 if scale is None else float(scale)
        self.max_len = table.shape[1] * c.page_size if max_len is None else int(max_len)
        n = ops.attn_paged_workspace_bytes(table.shape[0], q_heads, c.dim, tokens, self.max_len)
        self.nodes, self.q_norm, self.k_norm, self.eps = nodes, q_norm, k_norm, float(eps)
        if n and nodes:
            n = max(n, ops.attn_tree_workspace_bytes(table.shape[0], q_heads, c.dim, nodes, self.max_len))
        if not n:
            raise ValueError("%d requests of %d positions, %d heads of %d: not supported"
                             % (table.shape[0], self.max_len, q_heads, c.dim))
        buf = torch.empty(n + 256, dtype=torch.uint8, device=c.device)
        self.ws = buf[-buf.data_ptr() % 256:][:n]
        # what every call passes on, as addresses: the tensors stay as long as the plan
        self._plan, self._keep = None, (table, rope, q_norm, k_norm, buf)
        self._refs = (C.c_void_p * len(self.caches))(*[x.ref for x in self.caches])
        self._norms = [tuple(None if w is None else w.data_ptr() + 4 * c.dim * i for w in (q_norm, k_norm))
                       for i in range(len(self.caches))] if q_norm is not None or k_norm is not None else None
        if c.device.type == "cuda":
            self._calls = _lib.calls()
            self._plan = self._calls.plan(ops._table(table), ops._rope(rope), q_heads, c.heads, c.dim, self.max_len,
                                          self._interleaved, self.scale, self.eps, (self.ws.data_ptr(), n))

    def append(self, layer, q, k, v, seq, pos, q_out=None, slot=None):
        """Norm (where the constructor has weights) and rotate q [N][q_heads * dim] into q_out (q itself: in place; None: a new tensor) and k
        [N][heads * dim], store k and v for token n of request seq[n] at position pos[n] (both int32 [N]).
        q None: keys and values only.  slot (int32 [N]): where the tokens are stored, in the place of pos, which then
        only rotates.  Returns q_out."""
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        c = self.caches[layer]
        if self._norms is None and slot is None:
            rc = self._plan and self._calls.append(self._plan, c.ref, ops._stream(c.device), q, k, v, seq, pos, q_out)
        else:
            norms = self._norms[layer] if self._norms else (None, None)
            rc = self._plan and self._calls.append_norm(self._plan, c.ref, ops._stream(c.device), q, k, v, seq, pos, q_out, slot,
                                                        *norms)
        if rc is None:                       # a tensor is not as it should be
            qn, kn = (w if w is None else w[layer] for w in (self.q_norm, self.k_norm))
            ops.kv_append(c, self.table, q, k, v, seq, pos, q_out, self.q_heads, self.rope, self._interleaved, slot, qn, kn,
                          self.eps)
        elif rc:
            _lib.check(rc)
        return q_out

    def attend(self, layer, q, lens, out=None, tokens=None):
        """Attention of the last ``tokens`` (default: the constructor's) tokens of each request; q and out
        [requests * tokens][q_heads * dim], lens int32 [requests] counting the new tokens.  Returns out."""
        T = self.tokens if tokens is None else tokens
        if not 1 <= T <= self.tokens:
            raise ValueError("tokens must be 1..%d" % self.tokens)
        c = self.caches[layer]
        if out is None:
            out = torch.empty((q.shape[0], self.q_heads * c.dim), dtype=torch.float32, device=q.device)
        rc = self._plan and self._calls.attend(self._plan, c.ref, ops._stream(c.device), q, lens, out, T)
        if rc is None:                       # a tensor is not as it should be
            ops.attn_paged(c, self.table, q, lens, out, self.q_heads, T, self.scale, self.max_len, self.ws)
        elif rc:
            _lib.check(rc)
        return out

    def attend_tree(self, layer, q, tree, out=None):
        """Attention of every request's tree as ``tree`` (a Tree of this object's requests, planned) says: node t sees the
        positions ahead of the tree, its ancestors and itself.  q and out [requests * nodes][q_heads * dim]; a node that is
        none, or of a request that sits out, gets 0.  Returns out."""
        T = tree.nodes
        if tree.requests != self.table.shape[0] or T > self.nodes:
            raise ValueError("a tree of %d requests and %d nodes, made for %d requests and up to %d nodes"
                             % (tree.requests, T, self.table.shape[0], self.nodes))
        c = self.caches[layer]
        if tree.device != c.device or tree.base is None:
            raise ValueError("the tree must be planned, on the caches' device")
        if out is None:
            out = torch.empty((q.shape[0], self.q_heads * c.dim), dtype=torch.float32, device=q.device)
        rc = self._plan and self._calls.attend_tree(self._plan, c.ref, ops._stream(c.device), q, tree.base, tree._held[0], out, T)
        if rc is None:                       # a tensor is not as it should be
            ops.attn_tree(c, self.table, q, tree.base, tree.seen, out, self.q_heads, T, self.scale, self.max_len, self.ws)
        elif rc:
            _lib.check(rc)
        return out

    def keep(self, path, base):
        """Move the entries of each request's accepted nodes together in every layer's cache: from position base[b] +
        path[b][i] to base[b] + i, for i up to the first entry that names no node (below i, not above the one
        before, or at least the row's width; -1 ends it).  path: int32 [requests][nodes], as wide as the trees and not cut to
        the longest path, since its width says how many nodes there are; base: int32 [requests]."""
        c = self.caches[0]
        rc = self._plan and self._calls.keep(self._plan, C.addressof(self._refs), len(self.caches), ops._stream(c.device), path, base)
        if rc is None:                       # a tensor is not as it should be
            ops.kv_keep(self.caches, self.table, path, base)
        elif rc:
            _lib.check(rc)
