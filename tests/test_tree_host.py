"""Refusals of the operators on trees of drafted tokens: argument errors are returned before any launch (host only; the
pointers are never read), and the Python layer refuses tensors that do not fit."""
import ctypes as ct

import pytest
import torch

from kq import _lib, kv, ops, sampling
from test_paged_host import CACHE, P, cache_struct, refused


def plan(parents=P, ldp=8, base=P, seqs=2, T=8, seen=P, seq=P, pos=P, slot=P):
    return _lib.kq().kq_tree_plan(parents, ldp, base, seqs, T, seen, seq, pos, slot, None)


def append(kvs, table=P, ldt=8, seqs=2, width=8, N=3, seq=P, pos=P, slot=P, q=P, ldq=256, q_heads=4, q_out=P, ldqo=256, k=P,
           ldk=128, v=P, ldv=128, rope=P, rope_rows=100, rot=64, interleaved=0, q_norm=P, k_norm=P, eps=1e-6):
    return _lib.kq().kq_kv_append_norm(ct.addressof(kvs) if kvs is not None else None, table, ldt, seqs, width, N, seq, pos,
                                       slot, q, ldq, q_heads, q_out, ldqo, k, ldk, v, ldv, rope, rope_rows, rot, interleaved,
                                       q_norm, k_norm, eps, None)


def attend(kvs, table=P, ldt=8, seqs=2, width=8, base=P, seen=P, max_len=100, T=5, q=P, ldq=256, q_heads=4, scale=1.0, out=P,
           ldo=256, ws=P, ws_bytes=1 << 40):
    return _lib.kq().kq_attn_tree(ct.addressof(kvs) if kvs is not None else None, table, ldt, seqs, width, base, seen,
                                  max_len, T, q, ldq, q_heads, scale, out, ldo, ws, ws_bytes, None)


def keep(*kvs, table=P, ldt=8, seqs=2, width=8, base=P, path=P, ldp=8, T=8, layers=None):
    refs = (ct.c_void_p * max(len(kvs), 1))(*[ct.addressof(x) if x is not None else None for x in kvs])
    return _lib.kq().kq_kv_keep(ct.addressof(refs) if kvs else None, len(kvs) if layers is None else layers, table, ldt, seqs,
                                width, base, path, ldp, T, None)


def verify(x=P, ldx=1000, B=2, T=5, V=1000, tokens=P, ldt=5, parents=P, ldp=5, uniform=P, ldu=5, temperature=P, draft=P,
           ldd=1000, accepted=P, path=P, token=P, ws=P, ws_bytes=1 << 40):
    return _lib.kq().kq_verify(x, ldx, B, T, V, tokens, ldt, parents, ldp, uniform, ldu, temperature, draft, ldd, accepted,
                               path, token, ws, ws_bytes, None)


@pytest.mark.parametrize("change,msg", CACHE)
def test_cache_rules(change, msg):
    refused(append(cache_struct(**change)), msg)
    refused(attend(cache_struct(**change)), msg)
    refused(keep(cache_struct(), cache_struct(**change)), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(seqs=0), "seqs=0"), (dict(seqs=65536), "seqs=65536"), (dict(T=0), "T=0"), (dict(T=65), "T=65"),
    (dict(parents=None), "parents is NULL"), (dict(ldp=7), "ldp=7"), (dict(ldp=-1), "ldp=-1"), (dict(base=None), "base is NULL"),
    (dict(seen=None), "seen is NULL"), (dict(seen=P + 4), "seen must be 8-byte"), (dict(seq=None), "seq is NULL"),
    (dict(pos=P + 1), "pos must be 4-byte"), (dict(slot=None), "slot is NULL"),
])
def test_plan_argument_errors(change, msg):
    refused(plan(**change), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(N=-1), "N=-1"), (dict(q=None), "q and q_out"), (dict(seq=None), "seq is NULL"), (dict(pos=None), "pos is NULL"),
    (dict(slot=P + 2), "slot must be 4-byte"), (dict(q_norm=P + 1), "q_norm must be"), (dict(k_norm=P + 2), "k_norm must be"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(rot=72), "rot=72"),
    (dict(ldk=127), "127 of k"), (dict(q_heads=3), "q_heads=3"), (dict(table=None), "table is NULL"), (dict(ldt=7), "ldt=7"),
    (dict(N=1 << 28), "too many"),
])
def test_append_argument_errors(change, msg):
    refused(append(cache_struct(), **change), msg)


def test_append_of_no_token_is_nothing():
    assert append(cache_struct(), N=0, k=None, v=None, q=None, q_out=None, seq=None, pos=None, slot=None) == 0


@pytest.mark.parametrize("change,msg", [
    (dict(base=None), "base is NULL"), (dict(seen=None), "seen is NULL"), (dict(seen=P + 4), "seen must be 8-byte"),
    (dict(T=0), "T=0"), (dict(T=65), "T=65"), (dict(max_len=0), "max_len=0"), (dict(q=None), "q is NULL"),
    (dict(out=None), "out is NULL"), (dict(ldo=100), "100 of out"), (dict(scale=float("nan")), "scale"), (dict(ws=None), "ws is NULL"),
    (dict(ws=P + 16), "ws must be 256-byte"), (dict(ws_bytes=0), "workspace of 0 bytes"), (dict(seqs=0), "seqs=0"),
    (dict(q_heads=3), "q_heads=3"), (dict(ldq=255), "255 of q"), (dict(width=1 << 27, ldt=1 << 27), "2^30 positions"),
])
def test_attention_argument_errors(change, msg):
    refused(attend(cache_struct(), **change), msg)


@pytest.mark.parametrize("args", [(0, 4, 64, 1, 10), (1, 0, 64, 1, 10), (1, 4, 60, 1, 10), (1, 4, 64, 0, 10),
                                  (1, 4, 64, 65, 10), (1, 4, 64, 1, 0)])
def test_attention_workspace_of_bad_sizes_is_zero(args):
    assert ops.attn_tree_workspace_bytes(*args) == 0


def test_keep_argument_errors():
    c = cache_struct()
    refused(keep(), "no layer")
    refused(keep(c, layers=0), "no layer")
    refused(keep(c, None), "kv is NULL")
    for change in (dict(heads=4), dict(dim=48), dict(pages=5), dict(page_size=32)):
        refused(keep(c, cache_struct(**change)), "the same heads")
    refused(keep(c, cache_struct(), cache_struct(v=P + 4096)), "layers 0 and 2 share one of k and v")
    for change, msg in ((dict(table=None), "table is NULL"), (dict(base=None), "base is NULL"), (dict(path=None), "path is NULL"),
                        (dict(ldp=7), "7 of path"), (dict(T=0), "T=0"), (dict(T=65, ldp=65), "T=65"), (dict(seqs=0), "seqs=0")):
        refused(keep(c, c, **change), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(B=0), "seqs=0"), (dict(T=0), "T=0"), (dict(T=65), "T=65"), (dict(B=20000), "65535 rows"), (dict(V=0), "V=0"),
    (dict(x=None), "x is NULL"), (dict(ldx=999), "999 of x"), (dict(tokens=None), "tokens is NULL"), (dict(ldt=4), "4 of tokens"),
    (dict(parents=None), "parents is NULL"), (dict(ldp=4), "ldp=4"), (dict(uniform=None), "uniform is NULL"),
    (dict(ldu=4), "4 of uniform"), (dict(temperature=P + 1), "temperature must be"), (dict(ldd=10), "10 of draft"),
    (dict(draft=P + 2), "draft must be"), (dict(accepted=None), "accepted is NULL"), (dict(path=None), "path is NULL"),
    (dict(token=None), "token is NULL"), (dict(ws=None), "ws is NULL"), (dict(ws=P + 8), "ws must be"),
    (dict(ws_bytes=0), "workspace of 0 bytes"),
])
def test_verify_argument_errors(change, msg):
    refused(verify(**change), msg)


@pytest.mark.parametrize("args", [(0, 5, 100), (1, 0, 100), (1, 65, 100), (1, 5, 0), (20000, 5, 100), (1, 1, (1 << 30) + 1)])
def test_verify_workspace_of_bad_sizes_is_zero(args):
    assert ops.verify_workspace_bytes(*args) == 0
    with pytest.raises(ValueError):
        sampling.Verifier(*args, device="cpu")


def test_python_refusals():
    cache = kv.KVCache(4, 16, 2, 64, "bf16", "cpu")
    table = torch.zeros(1, 4, dtype=torch.int32)
    w = torch.ones(1, 64)
    for bad in (dict(nodes=65), dict(nodes=-1), dict(q_norm=w[0]), dict(k_norm=w.half()), dict(q_norm=torch.ones(2, 64)),
                dict(k_norm=torch.ones(64, 1).t()[:, ::1].expand(1, 64)[:, :32]), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            kv.PagedAttention([cache], table, 4, **bad)
    for bad in ((0, 4), (1, 0), (1, 65), (65536, 1)):
        with pytest.raises(ValueError):
            kv.Tree(*bad, device="cpu")
    att, tree = kv.PagedAttention([cache], table, 4, nodes=8), kv.Tree(1, 8, "cpu")
    q, new, one = torch.zeros(8, 256), torch.zeros(8, 128), torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError, match="planned"):
        att.attend_tree(0, q, tree)
    with pytest.raises(ValueError, match="device tensor"):
        tree.plan(torch.zeros(1, 8, dtype=torch.int32), one[:1])
    for bad in (kv.Tree(2, 8, "cpu"), kv.Tree(1, 9, "cpu")):
        with pytest.raises(ValueError, match="made for"):
            att.attend_tree(0, q, bad)
    with pytest.raises(ValueError, match="device tensor"):
        att.append(0, q, new, new, one, one, slot=one)
    with pytest.raises(ValueError, match="device tensor"):
        att.keep(torch.zeros(1, 8, dtype=torch.int32), one[:1])
    ver, toks = sampling.Verifier(1, 4, 100, "cpu"), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ver.verify(torch.zeros(4, 100), toks, toks, torch.zeros(1, 4))
    for x, t in ((torch.zeros(8, 100), torch.zeros(2, 4)), (torch.zeros(5, 100), torch.zeros(1, 5)), (torch.zeros(4, 101), toks)):
        with pytest.raises(ValueError, match="holds"):
            ver.verify(x, t.int(), toks, torch.zeros(1, 4))
    with pytest.raises(ValueError, match="must be"):
        ver.verify(torch.zeros(4, 100), toks[0], toks, torch.zeros(1, 4))
