"""The example's token loop: products, paged cache, attention and pick together.  In fp32 numerics every operator's row
depends on that row's request alone, so a request's logits are the same bits however it is fed and whoever is beside it."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "oxcoder-9b_amd", "examples"))

pytestmark = pytest.mark.gpu


def decoder(dev, requests, cache, mode="f32"):
    from decode_batch import Decoder
    return Decoder(2, 512, 8, 2, 64, 1024, 1024, requests, 128, cache, mode=mode, device=dev)


def prompts(n):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 1024, (m,), generator=g).tolist() for m in (40, 1, 23, 33)[:n]]


@pytest.mark.parametrize("cache", ["f16", "bf16", "i8"])
def test_fed_in_chunks_or_one_by_one(dev, cache):
    ids = prompts(1)[0]
    pos = lambda n: torch.tensor([n], dtype=torch.int32, device=dev)          # noqa: E731
    a, b = decoder(dev, 1, cache), decoder(dev, 1, cache)
    for i, t in enumerate(ids):
        one = a.forward([[t]], pos(i)).clone()
    for i in range(0, len(ids), 8):
        many = b.forward([ids[i:i + 8]], pos(i)).clone()
    assert torch.equal(one, many)
    for x, y in zip(a.caches, b.caches):
        assert torch.equal(x.k, y.k) and torch.equal(x.v, y.v)
    assert torch.isfinite(one).all() and float(one.std()) > 0


@pytest.mark.parametrize("cache", ["bf16", "i8"])
def test_alone_or_beside_others(dev, cache):
    ids = prompts(4)
    together = decoder(dev, 4, cache).generate(ids, 12)
    for b in range(4):
        assert decoder(dev, 1, cache).generate(ids[b:b + 1], 12)[0] == together[b]
    # the penalty counts: with none, another continuation; with a huge one, no id twice
    distinct = decoder(dev, 4, cache).generate(ids, 12, penalty=1e6)
    for b in range(4):
        assert len(set(distinct[b])) == 12 and not set(distinct[b]) & set(ids[b])


def test_quantized_activations(dev):
    """The engine's default numerics: the same loop runs, and gives one continuation each time."""
    ids = prompts(4)
    out = decoder(dev, 4, "bf16", "q8k").generate(ids, 8)
    assert out == decoder(dev, 4, "bf16", "q8k").generate(ids, 8)
    assert all(0 <= t < 1024 for row in out for t in row)
