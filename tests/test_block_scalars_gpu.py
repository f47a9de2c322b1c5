"""Scalars that are not finite in the 32 bits that the kernels compute in are refused."""
import math

import pytest
import torch

import onebitsparsemul_b200 as ob

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 1e39, -1e300])
def test_scalars_beyond_32_bits(value):
    x, w = torch.ones(2, 64, dtype=torch.float16, device=DEV), torch.ones(64, dtype=torch.float16, device=DEV)
    k, pos, freq = x.view(2, 1, 64), torch.arange(2, device=DEV), ob.rotary_frequencies(64)[0]
    cache = ob.KVCache8.empty(1, 1, 64)
    batch = ob.CacheBatch(*(torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 2], [2], [[0]])))
    for call in (lambda: ob.residual_norm(x, w, residual=x, residual_scale=value), lambda: ob.residual_norm(x, w, eps=value),
                 lambda: ob.rotary_tokens(k, pos, freq, magnitude=value), lambda: ob.cache_append(k, k, cache, batch, inv_freq=freq, magnitude=value),
                 lambda: ob.cache_append(k, k, cache, batch, q=k, inv_freq=freq, magnitude=value), lambda: ob.cache_attend(k, cache, batch, scale=value)):
        with pytest.raises(ValueError):
            call()
    assert not cache.k_pages.view(torch.uint8).any()
    ob.rotary_tokens(k, pos, freq, magnitude=3e38), ob.cache_attend(k, cache, batch, scale=-1e38)
