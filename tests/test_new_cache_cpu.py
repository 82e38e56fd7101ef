"""The cache that a model makes for itself, without its weights."""
from types import SimpleNamespace

import pytest
import torch

from sharq_b200.decoder import DecoderConfig, SharqDecoder


def new_cache(head_dim, *args, theta=1e4, **kw):
    model = SimpleNamespace(cfg=DecoderConfig(head_dim=head_dim, rope_theta=theta), embed=torch.zeros(1), layers=[SimpleNamespace(local_kv=2)] * 3)
    return SharqDecoder.new_cache(model, *args, **kw)


@pytest.mark.parametrize("head_dim", [16, 32, 80, 96, 192, 256])
def test_heads_that_attention_does_not_take_are_refused(head_dim):
    """Before a prompt is stored, not at the first decode step."""
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        new_cache(head_dim, 2, 40)


@pytest.mark.parametrize("head_dim", [64, 128])
def test_sizes(head_dim):
    cache = new_cache(head_dim, 4, 100, page_size=16)
    assert cache.k.shape == cache.v.shape == (3, 4 * 7, 2, 16, head_dim) and cache.cos.shape == (100, head_dim)
