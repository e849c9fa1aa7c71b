"""A paged key-value cache for several requests, and attention over it.

The reference's engine keeps one contiguous cache for its one request (scripts/kindi_q4/kindi/engine.py:255-280);
here requests share a pool of pages.  ``KVCache`` is one layer's pool, ``PagedAttention`` what a decoding
program calls between its q/k/v and output projections: ``append`` rotates the new tokens' queries and
keys and stores keys and values (kq_kv_append), ``attend`` runs their attention (kq_attn_paged).

    cache = [KVCache(pages, 16, 8, 128, "bf16") for _ in range(layers)]
    att = PagedAttention(cache, table, 32, tokens=1, rope=rope_table(4096, 128))
    att.append(layer, q, k, v, seq, pos, q)          # q is rotated in place
    att.attend(layer, q, lens, out)

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


class PagedAttention:
    """The attention of a decoding program over its layers' caches, with the one workspace it needs.

    caches: a KVCache per layer, all of one shape (types may differ); table: int32 [requests][width]; tokens: the most
    new tokens per request that attend will see (1..16); max_len: the most positions a request will hold
    (default: what its row of the table covers); rope: rope_table's, or None (nothing is rotated), whose width is
    the number of values that turn (append skips tokens at positions past its rows); interleaved: pairs (2i, 2i + 1)
    instead of (i, i + rot/2); scale: default dim ** -0.5.
    These are for the object's life: another table or rotation takes another object, what is in them may change.
    Calls on one PagedAttention share its workspace and so must be ordered: one stream, or synchronised."""

    def __init__(self, caches, table, q_heads, tokens=1, max_len=None, rope=None, interleaved=False, scale=None):
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
        self.caches, self.table, self.q_heads, self.tokens = tuple(caches), table, q_heads, tokens
        self.rope, self._interleaved = rope, 1 if interleaved else 0
        self.scale = c.dim ** -0.5 if scale is None else float(scale)
        self.max_len = table.shape[1] * c.page_size if max_len is None else int(max_len)
        n = ops.attn_paged_workspace_bytes(table.shape[0], q_heads, c.dim, tokens, self.max_len)
        if not n:
            raise ValueError("%d requests of %d positions, %d heads of %d: not supported"
                             % (table.shape[0], self.max_len, q_heads, c.dim))
        buf = torch.empty(n + 256, dtype=torch.uint8, device=c.device)
        self.ws = buf[-buf.data_ptr() % 256:][:n]
        # what every call passes on, as addresses: the tensors stay as long as the plan
        self._plan, self._keep = None, (table, rope, buf)
        if c.device.type == "cuda":
            self._calls = _lib.calls()
            self._plan = self._calls.plan(ops._table(table), ops._rope(rope), q_heads, c.heads, c.dim, self.max_len,
                                          self._interleaved, self.scale, (self.ws.data_ptr(), n))

    def append(self, layer, q, k, v, seq, pos, q_out=None):
        """Rotate q [N][q_heads * dim] into q_out (q itself: in place; None: a new tensor) and k
        [N][heads * dim], store k and v for token n of request seq[n] at position pos[n] (both int32 [N]).
        q None: keys and values only.  Returns q_out."""
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        c = self.caches[layer]
        rc = self._plan and self._calls.append(self._plan, c.ref, ops._stream(c.device), q, k, v, seq, pos, q_out)
        if rc is None:                       # a tensor is not as it should be
            ops.kv_append(c, self.table, q, k, v, seq, pos, q_out, self.q_heads, self.rope, self._interleaved)
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
