"""Refusals of the paged cache, its attention and the penalised pick: every argument error is returned before any
launch (host only; the pointers are never read), and the Python layer refuses tensors that do not fit."""
import ctypes as ct

import pytest
import torch

from kq import _lib, kv, ops, sampling

P = 4096                                        # an aligned address that nothing reads


def cache_struct(**change):
    f = dict(k=P, v=P, k_scale=None, v_scale=None, type=30, heads=2, dim=64, pages=4, page_size=16,
             page_stride=2 * 16 * 64, head_stride=16 * 64, pos_stride=64, scale_page_stride=32, scale_head_stride=16,
             scale_pos_stride=1)
    f.update(change)
    return _lib.KV(**f)


def refused(rc, msg):
    assert rc == _lib.KQ_ERR_ARG
    assert msg in _lib.kq().kq_last_error().decode()


CACHE = [
    (dict(type=12), "cache type 12"), (dict(heads=0), "heads=0"), (dict(dim=24), "dim=24"), (dict(dim=272), "dim=272"),
    (dict(dim=0), "dim=0"), (dict(page_size=12), "page_size=12"), (dict(page_size=0), "page_size=0"),
    (dict(page_size=1 << 21), "page_size"), (dict(pages=0), "pages=0"), (dict(k=None), "k of the cache is NULL"),
    (dict(v=P + 8), "16-byte aligned"), (dict(pos_stride=48), "stride 48"), (dict(pos_stride=68), "stride 68"),
    (dict(head_stride=-1024), "stride -1024"), (dict(page_stride=1 << 60), "stride"),
    (dict(type=24), "k_scale of the cache is NULL"), (dict(type=24, k_scale=P), "v_scale of the cache is NULL"),
    (dict(type=24, k_scale=P, v_scale=P, pos_stride=72, dim=64), "stride 72"),
    (dict(type=24, k_scale=P, v_scale=P, scale_pos_stride=0), "scale stride 0"),
]


def append(kvs, table=P, ldt=8, seqs=2, width=8, N=3, seq=P, pos=P, q=P, ldq=256, q_heads=4, q_out=P, ldqo=256, k=P,
           ldk=128, v=P, ldv=128, rope=P, rope_rows=100, rot=64, interleaved=0):
    return _lib.kq().kq_kv_append(ct.addressof(kvs) if kvs is not None else None, table, ldt, seqs, width, N, seq, pos, q,
                                  ldq, q_heads, q_out, ldqo, k, ldk, v, ldv, rope, rope_rows, rot, interleaved, None)


def attend(kvs, table=P, ldt=8, seqs=2, width=8, lens=P, max_len=100, T=1, q=P, ldq=256, q_heads=4, scale=1.0, out=P,
           ldo=256, ws=P, ws_bytes=1 << 40):
    return _lib.kq().kq_attn_paged(ct.addressof(kvs) if kvs is not None else None, table, ldt, seqs, width, lens, max_len,
                                   T, q, ldq, q_heads, scale, out, ldo, ws, ws_bytes, None)


def penalize(x=P, ldx=1000, B=2, V=1000, hist=P, ldh=50, max_hist=50, hist_len=P, prompt=P, rep=P, freq=P, pres=P, bid=P,
             bval=P, ldb=4, nb=4, allowed=P, ldm=32, y=P, ldy=1000, ws=P, ws_bytes=1 << 30, picked=P):
    return _lib.kq().kq_logits_penalize(x, ldx, B, V, hist, ldh, max_hist, hist_len, prompt, rep, freq, pres, bid, bval,
                                        ldb, nb, allowed, ldm, y, ldy, ws, ws_bytes, picked, None)


@pytest.mark.parametrize("change,msg", CACHE)
def test_cache_rules(change, msg):
    refused(append(cache_struct(**change)), msg)
    refused(attend(cache_struct(**change)), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(table=None), "table is NULL"), (dict(table=P + 2), "table must be 4-byte"), (dict(seqs=0), "seqs=0"),
    (dict(seqs=65536), "seqs=65536"), (dict(width=0), "width=0"), (dict(width=1 << 27, ldt=1 << 27), "2^30 positions"),
    (dict(ldt=7), "ldt=7"), (dict(q_heads=3), "q_heads=3"), (dict(q_heads=0), "q_heads=0"), (dict(ldq=255), "255 of q"),
    (dict(q=P + 1), "q must be 4-byte"),
])
def test_shared_argument_errors(change, msg):
    refused(append(cache_struct(), **change), msg)
    refused(attend(cache_struct(), **change), msg)


@pytest.mark.parametrize("change,msg", [
    (dict(N=-1), "N=-1"), (dict(q=None), "q and q_out"), (dict(q_out=None), "q and q_out"), (dict(seq=None), "seq is NULL"),
    (dict(pos=None), "pos is NULL"), (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(ldk=127), "127 of k"),
    (dict(ldv=0), "0 of v"), (dict(ldqo=128), "128 of q_out"), (dict(rot=4), "rot=4"), (dict(rot=72), "rot=72"),
    (dict(rot=12), "rot=12"), (dict(rope_rows=0), "rope_rows=0"), (dict(rope=P + 2), "rope must be 4-byte"),
    (dict(N=1 << 28), "too many"),
])
def test_append_argument_errors(change, msg):
    refused(append(cache_struct(), **change), msg)


def test_append_of_no_token_is_nothing():
    assert append(cache_struct(), N=0, k=None, v=None, q=None, q_out=None, seq=None, pos=None) == 0


@pytest.mark.parametrize("change,msg", [
    (dict(lens=None), "lens is NULL"), (dict(T=0), "T=0"), (dict(T=17), "T=17"), (dict(max_len=0), "max_len=0"),
    (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"), (dict(ldo=100), "100 of out"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(ws=None), "ws is NULL"),
    (dict(ws=P + 16), "ws must be 256-byte"), (dict(ws_bytes=0), "workspace of 0 bytes"),
])
def test_attention_argument_errors(change, msg):
    refused(attend(cache_struct(), **change), msg)


@pytest.mark.parametrize("args", [(0, 4, 64, 1, 10), (1, 0, 64, 1, 10), (1, 4, 60, 1, 10), (1, 4, 272, 1, 10),
                                  (1, 4, 64, 0, 10), (1, 4, 64, 17, 10), (1, 4, 64, 1, 0)])
def test_attention_workspace_of_bad_sizes_is_zero(args):
    assert ops.attn_paged_workspace_bytes(*args) == 0


@pytest.mark.parametrize("change,msg", [
    (dict(B=0), "B=0"), (dict(B=65536), "B=65536"), (dict(V=0), "V=0"), (dict(x=None), "x is NULL"), (dict(ldx=999), "999 of x"),
    (dict(max_hist=-1), "max_hist=-1"), (dict(ldh=49), "49 of hist"), (dict(hist_len=None), "hist_len is NULL"),
    (dict(nb=-1), "nb=-1"), (dict(ldb=3), "3 of bias_id"), (dict(bval=None), "bias_val is NULL"), (dict(ldm=31), "ldm=31"),
    (dict(ldm=-1), "ldm=-1"), (dict(rep=P + 1), "per-row"), (dict(y=None, picked=None), "neither"), (dict(ldy=0), "0 of y"),
    (dict(ws=None), "ws is NULL"), (dict(ws_bytes=10), "workspace of 10 bytes"), (dict(picked=P + 2), "picked must be"),
])
def test_logits_argument_errors(change, msg):
    refused(penalize(**change), msg)


def test_logits_workspace_of_bad_sizes_is_zero():
    assert ops.logits_workspace_bytes(0) == ops.logits_workspace_bytes(65536) == 0
    with pytest.raises(ValueError):
        sampling.Picker(0, "cpu")


def test_python_refusals():
    """Tensors that are not on the device, of another type or too small, and caches that do not fit together."""
    with pytest.raises(ValueError, match="dtype"):
        kv.KVCache(4, 16, 2, 64, "f32", "cpu")
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one type"):
        kv.KVCache.over(k, k.half())
    with pytest.raises(ValueError, match="same strides"):
        kv.KVCache.over(k, torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16).transpose(1, 2))
    with pytest.raises(ValueError, match="only an int8"):
        kv.KVCache.over(k, k, torch.zeros(4, 2, 16), torch.zeros(4, 2, 16))
    with pytest.raises(ValueError, match="k_scale"):
        kv.KVCache.over(k.to(torch.int8), k.to(torch.int8))
    with pytest.raises(ValueError, match="unit stride"):
        kv.KVCache.over(*[torch.zeros(4, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3)] * 2)
    cache = kv.KVCache(4, 16, 2, 64, "bf16", "cpu")
    table = torch.zeros(1, 4, dtype=torch.int32)
    for bad in (dict(q_heads=3), dict(tokens=17), dict(max_len=0), dict(table=table.long()), dict(table=table[0]),
                dict(caches=[])):
        with pytest.raises(ValueError):
            kv.PagedAttention(**{**dict(caches=[cache], table=table, q_heads=4), **bad})
    att = kv.PagedAttention([cache], table, 4)
    q, new = torch.zeros(1, 256), torch.zeros(1, 128)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        att.append(0, q, new, new, one, one)
    with pytest.raises(ValueError, match="device tensor"):
        att.attend(0, q, one)
    with pytest.raises(ValueError, match="tokens"):
        att.attend(0, q, one, tokens=2)
    with pytest.raises(ValueError, match="device tensor"):
        sampling.Picker(2, "cpu").pick(torch.zeros(2, 100))
    with pytest.raises(ValueError, match="rows"):
        sampling.Picker(1, "cpu").pick(torch.zeros(2, 100))


def test_a_one_element_dimension_has_any_stride():
    """torch gives a dimension of one element whatever stride; the cache's rules hold for the ones that are used."""
    k = torch.zeros(3, 1, 1, 32, dtype=torch.float16)
    c = kv.KVCache.over(k.as_strided((3, 1, 1, 32), (32, 5, 7, 1)), k.as_strided((3, 1, 1, 32), (32, 5, 7, 1)))
    assert append(c._kv, width=8, q_heads=4, ldk=32, ldv=32, ldq=128, ldqo=128, rot=32, N=0) == 0
