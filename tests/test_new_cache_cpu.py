"""The cache that a model makes for itself, without its weights."""
from types import SimpleNamespace

import numpy as np
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


@pytest.mark.parametrize("head_dim,theta", [(128, 5e5), (128, 1e6), (64, 1e4)])
def test_angles_of_far_positions(head_dim, theta):
    """The tables are the cosines and sines of the definition, rounded once to bf16 (half a step: 2^-8), to the last position of a long cache."""
    n = 131072
    cache = new_cache(head_dim, 1, n, theta=theta, page_size=64, pages=1)
    at = np.unique(np.concatenate((np.arange(64), np.arange(1, n, 977), np.arange(n - 64, n))))
    turns = np.outer(at, theta ** (-np.arange(0, head_dim, 2) / head_dim))
    for got, want in ((cache.cos, np.cos(turns)), (cache.sin, np.sin(turns))):
        assert got.dtype == torch.bfloat16 and torch.equal(got[:, :head_dim // 2], got[:, head_dim // 2:])
        off = np.abs(got[at, :head_dim // 2].double().numpy() - want)
        # the float64 angle itself is off by some 2^-53 of the position, twice
        assert (off <= 2.0 ** -8 * np.abs(want) + n * 2.0 ** -51).all()
