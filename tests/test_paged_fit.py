"""What the paged cache's objects take and refuse (host only)."""
import pytest
import torch

from kq import kv

TABLE = torch.zeros(1, 4, dtype=torch.int32)


@pytest.mark.parametrize("other", [(4, 32, 2, 64), (4, 8, 2, 64), (5, 16, 2, 64), (4, 16, 4, 64), (4, 16, 2, 128)])
def test_layers_of_another_shape(other):
    """One table and one bound serve all layers: pages of another size would hold other positions than they say."""
    caches = [kv.KVCache(4, 16, 2, 64, "bf16", "cpu"), kv.KVCache(*other, "bf16", "cpu")]
    for pair in (caches, caches[::-1]):
        with pytest.raises(ValueError, match="same"):
            kv.PagedAttention(pair, TABLE, 8)


def test_layers_of_one_shape_in_any_order_of_memory_and_type():
    k, v = (torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    kv.PagedAttention([kv.KVCache.over(k, v), *(kv.KVCache(4, 16, 2, 64, t, "cpu") for t in ("bf16", "f16", "i8"))], TABLE, 4)


def test_append_of_no_token_into_rows_that_are_there():
    """An empty tensor's address is NULL: no token with an output of more rows than that is still nothing to do."""
    from test_paged_host import P, append, cache_struct
    for q, out in ((None, P), (P, None)):
        assert append(cache_struct(), N=0, k=None, v=None, q=q, q_out=out, seq=None, pos=None) == 0


@pytest.fixture
def bf16_by_default():
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_dtype(torch.float32)


def test_scales_are_fp32_whatever_the_default_type(bf16_by_default):
    cache = kv.KVCache(4, 16, 2, 64, "i8", "cpu")
    assert cache.k_scale.dtype == cache.v_scale.dtype == torch.float32


@pytest.mark.gpu
def test_outputs_are_fp32_whatever_the_default_type(dev, bf16_by_default):
    cache = kv.KVCache(4, 16, 2, 64, "bf16", dev)
    att = kv.PagedAttention([cache], TABLE.to(dev), 4)
    q, lens = torch.zeros(1, 256, dtype=torch.float32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    assert att.attend(0, q, lens).dtype == torch.float32
